// kv8_store.cu — new keys and values of a batch of sequences into the 8-bit paged cache (kv8.cuh), queries and keys turned by their positions on
// the way.
//
// A group of 16 positions has one scale per head, for keys and for values.  Tokens that begin a group find their scale from themselves: the
// largest magnitude over the largest code.  Tokens that join one keep its scale where they fit; where they do not, the scale grows to what they need, or to
// twice what it was if that is more, and the codes that stand there are rounded once more.  A scale that grows at least doubles, so a code that was rounded again
// and again is off by less than 1/2 + 1/4 + ... = 1 step of the last scale.
//
// One launch: a CTA owns one (group, key head) that new tokens reach, a thread 16 numbers of a row; the CTAs behind those turn a token's queries each.  Multiply
// and add round apart (as everywhere in this library), so codes are the same bits as those of the formulas in 32-bit arithmetic.
//
// What bounds it: single tokens the launch (in replays of a captured graph, one 2.6 us, 64 of different sequences 5.6 us; call by call the host takes longer); portions the bytes of the projections and of the turned queries (4,096
// tokens, 32 heads over 8 of 128: 42.9 us, 4.6 TB/s, 70 % of what a copy moves; 55 us when a query's loads waited for its sequence, cosines and one another).
#include <algorithm>

#include "kv8.cuh"

namespace {

struct store_args {
    const float *q, *k, *v;
    int64_t ld, T;
    int n_seq;
    const int32_t *starts, *pos0;
    int H, G, D, Dv, rot, halves;
    const float *cs;
    float scale;
    const int32_t *tables;
    int64_t table_ld;
    int B;
    uint8_t *cache;
    float *q_out;
    int64_t record;
    unsigned kv_ctas;
    int vec; // rows, and those of cos_sin, begin on 16-byte boundaries
};

// number d of a head's row x at a position whose [cos, sin] are cs; rot of them are turned: pairs (2m, 2m + 1) or, halves, (m, m + rot / 2)
__device__ __forceinline__ float turned(const float *x, int d, int rot, int halves, const float *cs) {
    const float a = x[d];
    if (d >= rot) return a;
    const int h = rot / 2, m = halves ? (d < h ? d : d - h) : d / 2;
    const bool first = halves ? d < h : !(d & 1);
    const float b = x[halves ? (first ? d + h : d - h) : d ^ 1], c = cs[2 * m], s = cs[2 * m + 1];
    return first ? a * c - b * s : a * c + b * s;
}
// N consecutive ones from d on (N a multiple of 4), in 16-byte pieces: all turned or none, and with halves all in one of them
template <int N> __device__ __forceinline__ void turned_piece(const float *x, int d, int rot, int halves, const float *cs, float (&y)[N]) {
    const float4 *x4 = reinterpret_cast<const float4 *>(x + d);
#pragma unroll
    for (int u = 0; u < N / 4; u++) {
        const float4 t = x4[u];
        y[4 * u] = t.x, y[4 * u + 1] = t.y, y[4 * u + 2] = t.z, y[4 * u + 3] = t.w;
    }
    if (d >= rot) return;
    if (halves) {
        const int h = rot / 2;
        const bool first = d < h;
        const float4 *o4 = reinterpret_cast<const float4 *>(x + (first ? d + h : d - h)), *c4 = reinterpret_cast<const float4 *>(cs + 2 * (first ? d : d - h));
#pragma unroll
        for (int u = 0; u < N / 4; u++) {
            const float4 o = o4[u], c0 = c4[2 * u], c1 = c4[2 * u + 1];
            const float other[4] = {o.x, o.y, o.z, o.w}, c[4] = {c0.x, c0.z, c1.x, c1.z}, s[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float a = y[4 * u + e];
                y[4 * u + e] = first ? a * c[e] - other[e] * s[e] : a * c[e] + other[e] * s[e];
            }
        }
    } else {
        const float4 *c4 = reinterpret_cast<const float4 *>(cs + d);
#pragma unroll
        for (int u = 0; u < N / 4; u++) {
            const float4 c = c4[u];
            const float a0 = y[4 * u], b0 = y[4 * u + 1], a1 = y[4 * u + 2], b1 = y[4 * u + 3];
            y[4 * u] = a0 * c.x - b0 * c.y, y[4 * u + 1] = b0 * c.x + a0 * c.y;
            y[4 * u + 2] = a1 * c.z - b1 * c.w, y[4 * u + 3] = b1 * c.z + a1 * c.w;
        }
    }
}

__device__ __forceinline__ bool piece_fits(int vec, int n, int d, int rot, int halves) { return vec && (d >= rot || (rot % n == 0 && (!halves || (rot / 2) % n == 0))); }

template <int CODE> __global__ void __launch_bounds__(512, 2) kv8_store_kernel(const __grid_constant__ store_args a) {
    __shared__ unsigned s_max[2];
    using code = kv8_code<CODE>;
    step_wait();
    const int tid = threadIdx.x;
    if (blockIdx.x >= a.kv_ctas) { // ---- the queries of a token
        // A thread has the same four numbers of every n-th head, so that it loads their cosines and sines once; the heads' numbers are asked for four at a time, the
        // first ones before the token's sequence is looked for
        const int64_t t = blockIdx.x - a.kv_ctas;
        const int quads = a.D / 4, n = blockDim.x / quads, h0 = tid / quads, d = 4 * (tid - h0 * quads);
        const float *row = a.q + t * a.ld + d;
        float *out = a.q_out + t * a.H * a.D + d;
        const int half = a.rot / 2;
        const bool turns = d < a.rot, piece = piece_fits(a.vec, 4, d, a.rot, a.halves), first = a.halves ? d < half : true;
        const int other = turns && a.halves ? (first ? half : -half) : 0;
        constexpr int U = 4;
        float4 x[U], o[U];
        auto ask = [&](int h) {
            if (!piece || h0 >= n) return;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (h + u * n < a.H) {
                    x[u] = *reinterpret_cast<const float4 *>(row + (h + u * n) * a.D);
                    if (other) o[u] = *reinterpret_cast<const float4 *>(row + (h + u * n) * a.D + other);
                }
        };
        ask(h0);
        if (t >= a.starts[a.n_seq]) return;
        const int s = last_not_behind(a.n_seq, t, [&](int i) { return (int64_t)a.starts[i]; });
        const int64_t pos = (int64_t)a.pos0[s] + (t - a.starts[s]);
        const float *cs = a.cs + pos * a.rot;
        if (h0 >= n) return;
        if (!piece) { // odd strides, or a turn that ends inside
            for (int h = h0; h < a.H; h += n)
#pragma unroll
                for (int u = 0; u < 4; u++) out[h * a.D + u] = turned(row - d + h * a.D, d + u, a.rot, a.halves, cs) * a.scale;
            return;
        }
        float4 c0, c1;
        if (turns) {
            const float4 *c4 = reinterpret_cast<const float4 *>(cs + (a.halves ? 2 * (first ? d : d - half) : d));
            c0 = c4[0];
            if (a.halves) c1 = c4[1];
        }
        for (int h = h0; h < a.H; h += U * n) {
            if (h != h0) ask(h);
#pragma unroll
            for (int u = 0; u < U; u++) {
                float4 y = x[u];
                if (turns) {
                    if (!a.halves) {
                        y = make_float4(x[u].x * c0.x - x[u].y * c0.y, x[u].y * c0.x + x[u].x * c0.y, x[u].z * c0.z - x[u].w * c0.w, x[u].w * c0.z + x[u].z * c0.w);
                    } else if (first) {
                        y = make_float4(x[u].x * c0.x - o[u].x * c0.y, x[u].y * c0.z - o[u].y * c0.w, x[u].z * c1.x - o[u].z * c1.y, x[u].w * c1.z - o[u].w * c1.w);
                    } else {
                        y = make_float4(x[u].x * c0.x + o[u].x * c0.y, x[u].y * c0.z + o[u].y * c0.w, x[u].z * c1.x + o[u].z * c1.y, x[u].w * c1.z + o[u].w * c1.w);
                    }
                }
                if (h + u * n < a.H) *reinterpret_cast<float4 *>(out + (h + u * n) * a.D) = make_float4(y.x * a.scale, y.y * a.scale, y.z * a.scale, y.w * a.scale);
            }
        }
        return;
    }
    // ---- a group and head.  Sequence s has the places from starts[s] / 16 + 2 s on: as many as its tokens can reach groups, at most
    const int64_t unit = blockIdx.x / a.G;
    const int g = blockIdx.x - (int)unit * a.G;
    const int s = last_not_behind(a.n_seq, unit, [&](int i) { return (int64_t)(a.starts[i] / kKv8Group) + 2 * i; });
    const int64_t t0 = a.starts[s], n = a.starts[s + 1] - t0, p0 = a.pos0[s];
    const int64_t grp = p0 / kKv8Group + (unit - (t0 / kKv8Group + 2 * s)), first = grp * kKv8Group; // first position of the group
    if (n <= 0 || first >= p0 + n) return;
    const int held = (int)max((int64_t)0, p0 - first), end = (int)min((int64_t)kKv8Group, p0 + n - first); // rows [held, end) are new
    uint8_t *rec = a.cache + ((int64_t)a.tables[s * a.table_ld + first / a.B] * a.G + g) * a.record;
    const int row0 = (int)(first % a.B);
    float *scales = reinterpret_cast<float *>(rec + (int64_t)a.B * (a.D + a.Dv)) + row0 / kKv8Group;

    const bool is_v = tid >= a.D; // D threads a key piece each, Dv a value's
    const int piece = is_v ? tid - a.D : tid, width = is_v ? a.Dv : a.D, ppr = width / 16;
    const int r = piece / ppr, d = 16 * (piece - r * ppr);
    const bool mine = tid < a.D + a.Dv, fresh = mine && r >= held && r < end;
    float y[16];
    unsigned top = 0;
    if (fresh) {
        const int64_t t = t0 + (first + r - p0);
        const float *x = is_v ? a.v + t * a.ld + g * a.Dv : a.k + t * a.ld + g * a.D, *cs = a.cs + (first + r) * a.rot;
        const int rot = is_v ? 0 : a.rot;
        if (piece_fits(a.vec, 16, d, rot, a.halves)) {
            turned_piece<16>(x, d, rot, a.halves, cs, y);
        } else {
#pragma unroll
            for (int u = 0; u < 16; u++) y[u] = turned(x, d + u, rot, a.halves, cs);
        }
#pragma unroll
        for (int u = 0; u < 16; u++) { // what is no number is kept as zero; infinities as the largest code, they say nothing about the scale
            if (y[u] != y[u]) y[u] = 0.f;
            const unsigned m = __float_as_uint(fabsf(y[u]));
            if (m < 0x7f800000u) top = max(top, m);
        }
    }
    const float old = held && mine ? scales[is_v ? a.B / kKv8Group : 0] : 0.f;
    if (tid < 2) s_max[tid] = 0;
    __syncthreads();
    const unsigned mk = __reduce_max_sync(0xffffffffu, is_v ? 0u : top), mv = __reduce_max_sync(0xffffffffu, is_v ? top : 0u);
    if ((tid & 31) == 0) {
        if (mk) atomicMax(&s_max[0], mk);
        if (mv) atomicMax(&s_max[1], mv);
    }
    __syncthreads();
    if (!mine) return;
    const float amax = __uint_as_float(s_max[is_v]);
    const float least = amax > 0.f ? fmaxf(amax * code::inv_top, 7.8886090522101181e-31f) : 0.f; // 2^-100: its reciprocal is an fp32 number
    const float scale = least > old ? fmaxf(least, 2.f * old) : old;
    uint8_t *at = rec + (is_v ? (int64_t)a.B * a.D : 0) + (int64_t)(row0 + r) * width + d;
    if (fresh) {
        const float inv = 1.0f / (scale > 0.f ? scale : 1.f);
        union {
            uint8_t c[16];
            uint4 v;
        } o;
#pragma unroll
        for (int u = 0; u < 16; u++) o.c[u] = code::encode(y[u] * inv);
        *reinterpret_cast<uint4 *>(at) = o.v;
    } else if (r < held && scale > old) {
        const float ratio = old / scale;
        union {
            uint8_t c[16];
            uint4 v;
        } o;
        o.v = *reinterpret_cast<const uint4 *>(at);
#pragma unroll
        for (int u = 0; u < 16; u++) o.c[u] = code::encode(code::decode(o.c[u]) * ratio);
        *reinterpret_cast<uint4 *>(at) = o.v;
    }
    if (piece == 0) scales[is_v ? a.B / kKv8Group : 0] = scale;
}

} // namespace

extern "C" {

int64_t ggb_kv8_page_bytes(int G, int D, int Dv, int block_size) {
    return kv8_sizes_fit(GGB_KV8_INT8, G, G, D, Dv, block_size) ? G * kv8_record(D, Dv, block_size) : 0;
}

int ggb_op_kv8_store(int code, const float *q, const float *k, const float *v, int64_t ld, int64_t T, int n_seq, const int32_t *starts, const int32_t *pos0, int H,
                     int G, int D, int Dv, int rot_dims, int rot_halves, const float *cos_sin, float scale, const int32_t *tables, int64_t table_ld, int block_size,
                     void *cache, float *q_out) {
    GGB_REQUIRE_INIT();
    GGB_CHECK_ARG(code == GGB_KV8_INT8 || code == GGB_KV8_E4M3, "kv8_store: code %d is neither int8 nor e4m3", code);
    GGB_CHECK_ARG(kv8_sizes_fit(code, H, G, D, Dv, block_size),
                  "kv8_store: %d heads over %d of %d / %d numbers in pages of %d: heads are whole groups, sizes multiples of 16 up to %d, pages multiples of 16", H, G, D, Dv,
                  block_size, kKv8MaxHead);
    GGB_CHECK_ARG(q && k && v && starts && pos0 && tables && cache && q_out, "kv8_store: a pointer is null");
    GGB_CHECK_ARG(T > 0 && n_seq > 0 && T <= (1 << 24) && n_seq <= (1 << 20) && table_ld > 0 && ld >= std::max(std::max((int64_t)H * D, (int64_t)G * D), (int64_t)G * Dv),
                  "kv8_store: %lld tokens of %d sequences, rows of %lld numbers", (long long)T, n_seq, (long long)ld);
    GGB_CHECK_ARG(rot_dims >= 0 && rot_dims <= D && rot_dims % 2 == 0 && (rot_halves == 0 || rot_halves == 1) && (!rot_dims || cos_sin),
                  "kv8_store: %d of %d numbers cannot turn", rot_dims, D);
    GGB_CHECK_ARG((uintptr_t)cache % 16 == 0 && (uintptr_t)q_out % 4 == 0, "kv8_store: the cache must begin on a 16-byte boundary");
    const int64_t units = T / kKv8Group + 2 * (int64_t)n_seq;
    GGB_CHECK_ARG(units * G + T < (1ll << 31), "kv8_store: too many tokens and heads for a launch");
    const bool vec = ld % 4 == 0 && rot_dims % 4 == 0 && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (rot_dims ? (uintptr_t)cos_sin : 0)) % 16 == 0);
    const store_args a{q, k, v, ld, T, n_seq, starts, pos0, H, G, D, Dv, rot_dims, rot_halves, cos_sin, scale, tables, table_ld, block_size, (uint8_t *)cache, q_out,
                       kv8_record(D, Dv, block_size), (unsigned)(units * G), vec};
    const dim3 grid((unsigned)(units * G + T)), block((unsigned)((D + Dv + 31) / 32 * 32));
    if (code == GGB_KV8_INT8) {
        GGB_CUDA(ggb_launch_step(kv8_store_kernel<GGB_KV8_INT8>, grid, block, 0, a));
    } else {
        GGB_CUDA(ggb_launch_step(kv8_store_kernel<GGB_KV8_E4M3>, grid, block, 0, a));
    }
    GGB_LAUNCH_CHECK();
    return GGB_OK;
}

} // extern "C"
