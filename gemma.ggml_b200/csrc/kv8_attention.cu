// kv8_attention.cu — grouped-query soft-max attention of a batch of sequences over the 8-bit paged cache (kv8.cuh).
//
// A CTA per (token, head): its warps have the visible keys in turn, a lane eight numbers of a row, running maximum and sum in registers, and the warps'
// parts are joined in shared memory.  A row of a sequence without tokens, or behind the last sequence, stays as it was.
#include <algorithm>

#include "dense.cuh"
#include "kv8.cuh"

namespace {

constexpr int kWarps = 8;

struct attn_args {
    const float *q;
    const uint8_t *cache;
    const int32_t *tables;
    int64_t table_ld;
    int B;
    int64_t T;
    int n_seq;
    const int32_t *starts, *pos0;
    int H, G, D, Dv;
    int64_t window, keep;
    float cap;
    const float *sink, *gate;
    int64_t ldg, record;
    void *out;
};

template <int CODE, typename E> __global__ void __launch_bounds__(32 * kWarps) kv8_plain_kernel(const __grid_constant__ attn_args a) {
    __shared__ float s_o[kWarps][kKv8MaxHead], s_m[kWarps], s_l[kWarps];
    using code = kv8_code<CODE>;
    step_wait();
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, g = h / (a.H / a.G), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (t >= a.starts[a.n_seq]) return;
    const int s = last_not_behind(a.n_seq, t, [&](int i) { return (int64_t)a.starts[i]; });
    const int64_t i = (int64_t)a.pos0[s] + (t - a.starts[s]);
    const int64_t lo = a.window > 0 ? max((int64_t)0, i - a.window + 1) : 0, n_keep = min(a.keep, lo), total = n_keep + i - lo + 1;
    float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int u = 0; u < 8; u++) {
        q[u] = lane + 32 * u < a.D ? a.q[(t * a.H + h) * a.D + lane + 32 * u] : 0.f;
        o[u] = 0.f;
    }
    for (int64_t n = warp; n < total; n += kWarps) {
        const int64_t j = n < n_keep ? n : lo + (n - n_keep);
        const int row = (int)(j % a.B);
        const uint8_t *rec = a.cache + ((int64_t)a.tables[s * a.table_ld + j / a.B] * a.G + g) * a.record;
        const float *sc = reinterpret_cast<const float *>(rec + (int64_t)a.B * (a.D + a.Dv)) + row / kKv8Group;
        const uint8_t *k = rec + (int64_t)row * a.D, *v = rec + (int64_t)a.B * a.D + (int64_t)row * a.Dv;
        float x = 0.f;
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (lane + 32 * u < a.D) x = fmaf(code::decode(k[lane + 32 * u]), q[u], x);
        x = warp_sum_f32(x) * sc[0];
        if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
        const float mx = fmaxf(m, x), corr = expf(m - mx), w = expf(x - mx), wv = w * sc[a.B / kKv8Group];
        l = fmaf(l, corr, w);
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (lane + 32 * u < a.Dv) o[u] = fmaf(o[u], corr, wv * code::decode(v[lane + 32 * u]));
        m = mx;
    }
#pragma unroll
    for (int u = 0; u < 8; u++) s_o[warp][lane + 32 * u] = o[u];
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
    __syncthreads();
    float M = a.sink ? a.sink[h] : -INFINITY, L = 0.f;
    for (int w = 0; w < kWarps; w++) M = fmaxf(M, s_m[w]);
    if (a.sink) L = expf(a.sink[h] - M);
    for (int w = 0; w < kWarps; w++) L = fmaf(s_l[w], s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - M), L);
    for (int c = threadIdx.x; c < a.Dv; c += 32 * kWarps) {
        float y = 0.f;
        for (int w = 0; w < kWarps; w++) y = fmaf(s_o[w][c], s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - M), y);
        y /= L;
        if (a.gate) y *= 1.f / (1.f + expf(-a.gate[t * a.ldg + (int64_t)h * a.Dv + c]));
        reinterpret_cast<E *>(a.out)[(t * a.H + h) * a.Dv + c] = from_f32<E>(y);
    }
}

} // namespace

extern "C" {

size_t ggb_kv8_attn_scratch_bytes(int Dv) { return (size_t)512 * 2 * 32 * (Dv + 2) * 4; }

int ggb_op_kv8_attn(int dt, int code, const float *q, const void *cache, const int32_t *tables, int64_t table_ld, int block_size, int64_t T, int64_t max_new,
                    int n_seq, const int32_t *starts, const int32_t *pos0, int H, int G, int D, int Dv, int64_t window, int64_t keep_first, float softcap,
                    const float *sink, const float *gate, int64_t ldg, void *out, void *scratch, size_t scratch_bytes) {
    GGB_REQUIRE_INIT();
    GGB_CHECK_ARG(dt == GGB_TYPE_BF16 || dt == GGB_TYPE_F32, "kv8_attn: dtype %d is neither bf16 nor f32", dt);
    GGB_CHECK_ARG(code == GGB_KV8_INT8 || code == GGB_KV8_E4M3, "kv8_attn: code %d is neither int8 nor e4m3", code);
    GGB_CHECK_ARG(kv8_sizes_fit(code, H, G, D, Dv, block_size),
                  "kv8_attn: %d heads over %d of %d / %d numbers in pages of %d: heads are whole groups, sizes multiples of 16 up to %d, pages multiples of 16", H, G, D, Dv,
                  block_size, kKv8MaxHead);
    GGB_CHECK_ARG(q && cache && tables && starts && pos0 && out, "kv8_attn: a pointer is null");
    GGB_CHECK_ARG(T > 0 && n_seq > 0 && T <= (1 << 24) && n_seq <= (1 << 20) && max_new > 0 && max_new <= T && table_ld > 0 && H <= 65535,
                  "kv8_attn: %lld tokens of %d sequences, at most %lld each", (long long)T, n_seq, (long long)max_new);
    GGB_CHECK_ARG(softcap >= 0.f && keep_first >= 0 && (!gate || ldg >= (int64_t)H * Dv), "kv8_attn: a soft cap or kept positions below zero, or a gate row too short");
    GGB_CHECK_ARG((uintptr_t)cache % 16 == 0, "kv8_attn: the cache must begin on a 16-byte boundary");
    GGB_CHECK_ARG(!scratch || ((uintptr_t)scratch % 16 == 0 && scratch_bytes >= ggb_kv8_attn_scratch_bytes(Dv)), "kv8_attn: %zu bytes of scratch, %zu needed on a 16-byte boundary",
                  scratch_bytes, ggb_kv8_attn_scratch_bytes(Dv));
    const attn_args a{q, (const uint8_t *)cache, tables, table_ld, block_size, T, n_seq, starts, pos0, H, G, D, Dv, window, window > 0 ? keep_first : 0, softcap, sink, gate, ldg,
                      kv8_record(D, Dv, block_size), out};
    const dim3 grid((unsigned)T, (unsigned)H), block(32 * kWarps);
#define PLAIN(CODE, E) GGB_CUDA(ggb_launch_step(kv8_plain_kernel<CODE, E>, grid, block, 0, a))
    if (dt == GGB_TYPE_BF16) {
        if (code == GGB_KV8_INT8) PLAIN(GGB_KV8_INT8, __nv_bfloat16);
        else PLAIN(GGB_KV8_E4M3, __nv_bfloat16);
    } else {
        if (code == GGB_KV8_INT8) PLAIN(GGB_KV8_INT8, float);
        else PLAIN(GGB_KV8_E4M3, float);
    }
#undef PLAIN
    GGB_LAUNCH_CHECK();
    return GGB_OK;
}

} // extern "C"
