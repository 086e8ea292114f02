// kv8_attention.cu — grouped-query soft-max attention of a batch of sequences over the 8-bit paged cache (kv8.cuh).
//
// Steps of a token or some drafted ones of every sequence, few rows of queries a key head:
//
// What has to be read are the codes, a byte a number, and a warp turns each into fp16 (exactly: 8 bits fit) once for all query heads of the key head.  Both products are
// mma.m16n8k16 with the keys, or the value coordinates, as the 16 rows and eight rows of queries as the columns, so no row of an MMA is empty for the usual four to
// eight query heads of a key head:
//
//   scores   S^T [16 keys][8 rows] = K Q^T, a lane's piece of a key is 16 consecutive codes straight from the cache: the order of a sum's terms is free, and queries
//            lie in shared memory in the same one
//   weights  in the registers that the scores are in: 2^(s - m); a kept maximum is followed only when a score exceeds it by 8 (a vote, no shuffles otherwise)
//   output   O^T [16 coordinates][8 rows] += V^T P^T, weights turned by movmatrix, values by byte permutes of the rows of two neighbouring keys
//
// PARTS: fp16 numbers that stand for an fp32 query or weight.  2 keep 22 bits of each (results in fp32); 1 keeps 11 (results in bf16, which keep 8).  A row of queries is
// multiplied by a power of two that brings its largest number to [2^10, 2^11), so nothing of weight gets too small for fp16; weights times their group's value scale are
// relative to a kept scale (`vref`) for the same reason.
//
// Work: items (sequence, R rows, key head), cut into tiles of 128 positions, a warp 16 of them; all tiles of a call in one row, dealt evenly to the CTAs, so
// ragged batches and single long sequences fill the chip alike.  A CTA that has only a piece of an item leaves it in the workspace (the first or the last
// of what it was dealt: two places), and kv8_join_kernel, a row a CTA, adds an item's pieces up in order.
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"

namespace {

using namespace kv8;

constexpr int kStepWarps = 8, kStepThreads = 32 * kStepWarps, kStepTile = 16 * kStepWarps; // keys of a tile
constexpr int kMaxRows = 32, kMaxCtas = 512;

inline size_t part_bytes(int Dv) { return (size_t)kMaxCtas * (2 * kMaxRows * (size_t)(Dv + 2) * 4 + sizeof(int4)); }

// the rows of an item and the tiles that they see: [0, n_keep) in kt tiles, then [lo, i1] in tiles from position kStepTile * w0 on
struct item {
    int s, rg, row0, rows; // rows [row0, row0 + rows) of the sequence: its tokens x the query heads of a key head
    int p0, i0, i1;        // positions of its first token, of the item's first and last
    int lo, n_keep, kt, w0, n;
    int64_t t0;            // its first token
};
template <int R> __device__ __forceinline__ item item_of(const attn_args &a, int s, int rg) {
    item x;
    const int hpg = a.H / a.G;
    x.s = s, x.rg = rg, x.t0 = a.starts[s], x.p0 = a.pos0[s], x.row0 = rg * R;
    const int64_t all = (a.starts[s + 1] - x.t0) * hpg;
    x.rows = (int)min((int64_t)R, all - x.row0);
    x.n = 0;
    if (x.rows <= 0) return x;
    x.i0 = x.p0 + x.row0 / hpg, x.i1 = x.p0 + (x.row0 + x.rows - 1) / hpg;
    x.lo = a.window > 0 ? (int)max((int64_t)0, x.i0 - a.window + 1) : 0;
    x.n_keep = (int)min(a.keep, (int64_t)x.lo);
    x.kt = (x.n_keep + kStepTile - 1) / kStepTile, x.w0 = x.lo / kStepTile;
    x.n = x.kt + x.i1 / kStepTile - x.w0 + 1;
    return x;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// P: numbers of a key and of a value, at most: 64, 128 or 256
template <int P, int NT, int PARTS> struct step_sizes {
    static constexpr int R = 8 * NT, KS = P / 16; // MMA steps along a key; blocks of 16 value coordinates
    static constexpr size_t q_bytes = (size_t)PARTS * NT * KS * 256, red_bytes = (size_t)kStepWarps * R * P * 4;
    static constexpr size_t smem = q_bytes + red_bytes + (size_t)kStepWarps * R * 8 + R * 4 + 64;
    static constexpr int min_ctas = (P <= 128 && NT == 1) || (P == 64 && NT == 2) ? 2 : 1;
};
// where the pair of coordinates 2 i, 2 i + 1 of the 16 (P = 64: 8) numbers of lane group g lies in its row of the reduction, in pairs: rows of a warp's stores in different banks
template <int P> __device__ __forceinline__ int red_at(int g, int i, int c) {
    constexpr int W = P == 64 ? 4 : 8; // pairs of a lane group (P = 256: of either half)
    return W * g + (i ^ ((((g >> 1) & 1) | (c << 1)) & (W - 1)));
}

template <int CODE, int P, int NT, int PARTS>
__global__ void __launch_bounds__(kStepThreads, step_sizes<P, NT, PARTS>::min_ctas) kv8_step_kernel(const __grid_constant__ attn_args a) {
    using Z = step_sizes<P, NT, PARTS>;
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    constexpr int R = Z::R, KS = Z::KS, NB = P / 64, VW = P == 64 ? 2 : 4, VC = P == 256 ? 2 : 1; // words of a lane's piece of a value row, pieces
    extern __shared__ __align__(16) uint8_t ks_smem[];
    __shared__ int64_t s_scan[kStepWarps], s_at[2];
    __shared__ int s_entry;
    step_wait();
    uint2 *sq = reinterpret_cast<uint2 *>(ks_smem);
    float2 *red = reinterpret_cast<float2 *>(ks_smem + Z::q_bytes);
    float *sm = reinterpret_cast<float *>(ks_smem + Z::q_bytes + Z::red_bytes), *sl = sm + kStepWarps * R, *srow = sl + kStepWarps * R, *svref = srow + R;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, c4 = lane & 3, hpg = a.H / a.G;

    // ---- what this CTA has been dealt: units [u, u_end) of the tiles of all items, and where the first lies
    int64_t u, u_end, U = 0;
    int entry, head, tile;
    item it;
    const int entries = a.n_seq * a.groups;
    if (a.part) {
        const int each = (entries + kStepThreads - 1) / kStepThreads, e0 = min(entries, tid * each), e1 = min(entries, e0 + each);
        int64_t mine = 0;
        for (int e = e0; e < e1; e++) mine += (int64_t)item_of<R>(a, e / a.groups, e % a.groups).n * a.G;
        int64_t run = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, run, off);
            if (lane >= off) run += x;
        }
        if (lane == 31) s_scan[warp] = run;
        __syncthreads();
        int64_t base = 0;
#pragma unroll
        for (int w = 0; w < kStepWarps; w++) {
            if (w < warp) base += s_scan[w];
            U += s_scan[w];
        }
        const int64_t N = min((int64_t)gridDim.x, U), b = blockIdx.x;
        if (tid == 0) a.desc[b] = make_int4(-1, 0, 0, 0);
        if (b >= N) return;
        u = U * b / N, u_end = U * (b + 1) / N;
        base += run - mine;
        if (u >= base && u < base + mine) {
            int e = e0;
            for (;; e++) {
                const int64_t n = (int64_t)item_of<R>(a, e / a.groups, e % a.groups).n * a.G;
                if (u < base + n) break;
                base += n;
            }
            s_entry = e, s_at[0] = u - base;
        }
        __syncthreads();
        entry = s_entry;
        it = item_of<R>(a, entry / a.groups, entry % a.groups);
        head = (int)(s_at[0] / it.n), tile = (int)(s_at[0] - (int64_t)head * it.n);
    } else {
        entry = blockIdx.x / a.G, head = blockIdx.x - entry * a.G, tile = 0;
        it = item_of<R>(a, entry / a.groups, entry % a.groups);
        u = 0, u_end = it.n;
    }

    while (u < u_end) {
        // ---- a piece of an item: tiles [tile, tile + n)
        const int n = (int)min((int64_t)(it.n - tile), u_end - u);
        // queries: rows as fp16 parts, in the order of a lane's pieces
        for (int r = warp; r < R; r += kStepWarps) {
            float4 x[(P + 127) / 128];
            float m = 0.f;
            const int row = it.row0 + r, tq = row / hpg, h = head * hpg + (row - tq * hpg);
            const float *src = a.q + ((it.t0 + tq) * a.H + h) * a.D;
#pragma unroll
            for (int k = 0; k < (P + 127) / 128; k++) {
                const int d = 4 * lane + 128 * k;
                x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < it.rows && d < a.D) {
                    if (a.vec_q) x[k] = *reinterpret_cast<const float4 *>(src + d);
                    else x[k] = make_float4(src[d], src[d + 1], src[d + 2], src[d + 3]);
                }
                m = fmaxf(m, fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
            }
            m = warp_max_f32(m);
            const float f = to_half_range(m);
            if (lane == 0) srow[r] = (a.cap > 0.f ? 1.f : kLog2e) / f;
            const float nan = m == INFINITY ? NAN : 0.f; // an infinite number spoils its row
#pragma unroll
            for (int k = 0; k < (P + 127) / 128; k++) {
                const int d = 4 * lane + 128 * k;
                if (d >= P) break;
                const float y[4] = {x[k].x * f + nan, x[k].y * f + nan, x[k].z * f + nan, x[k].w * f + nan};
                uint2 p = make_uint2(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]));
                const int step = 4 * (d / 64) + (d % 16) / 4, to = (r % 8) * 4 + (d % 64) / 16;
                sq[((r / 8) * KS + step) * 32 + to] = p;
                if (PARTS == 2) {
                    const float2 b0 = half2_floats(p.x), b1 = half2_floats(p.y);
                    p = make_uint2(half2_bits(y[0] - b0.x, y[1] - b0.y), half2_bits(y[2] - b1.x, y[3] - b1.y));
                    sq[((NT + r / 8) * KS + step) * 32 + to] = p;
                }
            }
        }
        __syncthreads();
        float rowf[NT][2], m[NT][2], l[NT][2], o[KS][NT][4], vref = 0.f;
        int pos[NT][2];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = 8 * t + 2 * c4 + e;
                rowf[t][e] = srow[r], m[t][e] = -INFINITY, l[t][e] = 0.f;
                pos[t][e] = r < it.rows ? it.p0 + (it.row0 + r) / hpg : -1; // sees nothing
            }
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][t][e] = 0.f;

        // the 16 positions of this warp in a tile: first one, or -1 where none of them is seen by any row
        auto group_of = [&](int k) {
            const int t = tile + k, first = (t < it.kt ? t : it.w0 + t - it.kt) * kStepTile + 16 * warp;
            const int lo = t < it.kt ? 0 : it.lo, hi = t < it.kt ? it.n_keep - 1 : it.i1;
            return k < n && first + 15 >= lo && first <= hi ? first : -1;
        };
        auto page_of = [&](int first) { return first < 0 ? 0 : a.tables[(int64_t)it.s * a.table_ld + first / a.B]; };
        uint4 kx[2][NB];
        uint32_t vx[4][VC][VW];
        float ksc = 0.f, vsc = 0.f;
        auto record_of = [&](int page) { return a.cache + ((int64_t)page * a.G + head) * a.record; };
        auto load_k = [&](int first, int page) {
            if (first < 0) return;
            const int row = first % a.B, last = min(15, it.i1 - first); // rows behind the last position: the last one again
            const uint8_t *rec = record_of(page);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint8_t *k = rec + (int64_t)(row + min(g8 + 8 * e, last)) * a.D + 16 * c4;
#pragma unroll
                for (int b = 0; b < NB; b++) kx[e][b] = 64 * b + 16 * c4 < a.D ? ld_stream_u4(k + 64 * b) : make_uint4(0, 0, 0, 0);
            }
            const float *sc = reinterpret_cast<const float *>(rec + (int64_t)a.B * (a.D + a.Dv)) + row / kKv8Group;
            ksc = sc[0], vsc = sc[a.B / kKv8Group];
        };
        auto load_v = [&](int first, int page) {
            if (first < 0) return;
            const int row = first % a.B, last = min(15, it.i1 - first);
            const uint8_t *v0 = record_of(page) + (int64_t)a.B * a.D;
#pragma unroll
            for (int e = 0; e < 4; e++) { // keys 2 c4, 2 c4 + 1, 2 c4 + 8, 2 c4 + 9
                const uint8_t *v = v0 + (int64_t)(row + min(2 * c4 + (e & 1) + 8 * (e >> 1), last)) * a.Dv + 4 * VW * g8;
#pragma unroll
                for (int c = 0; c < VC; c++) {
                    if (VW == 4) {
                        const uint4 x = 128 * c + 16 * g8 < a.Dv ? ld_stream_u4(v + 128 * c) : make_uint4(0, 0, 0, 0);
                        vx[e][c][0] = x.x, vx[e][c][1] = x.y, vx[e][c][VW - 2] = x.z, vx[e][c][VW - 1] = x.w;
                    } else {
                        uint2 x = make_uint2(0, 0);
                        if (8 * g8 < a.Dv) x = *reinterpret_cast<const uint2 *>(v);
                        vx[e][c][0] = x.x, vx[e][c][1] = x.y;
                    }
                }
            }
        };
        int first = group_of(0), page = page_of(first);
        load_k(first, page);
        load_v(first, page);
        int next = group_of(1), next_page = page_of(next);
        for (int k = 0; k < n; k++) {
            const int after = group_of(k + 2), after_page = page_of(after);
            if (first >= 0) {
                float z[NT][4];
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) z[t][e] = 0.f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const uint32_t w0[4] = {kx[0][b].x, kx[0][b].y, kx[0][b].z, kx[0][b].w}, w1[4] = {kx[1][b].x, kx[1][b].y, kx[1][b].z, kx[1][b].w};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        uint32_t a0, a1, a2, a3;
                        halves_of<CODE>(w0[w], a0, a2);
                        halves_of<CODE>(w1[w], a1, a3);
#pragma unroll
                        for (int part = PARTS - 1; part >= 0; part--)
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                const uint2 y = sq[((part * NT + t) * KS + 4 * b + w) * 32 + lane];
                                mma16816(z[t], a0, a1, a2, a3, y.x, y.y);
                            }
                    }
                }
                const float kscale = ksc, vscale = vsc;
                load_k(next, next_page);
                // ---- weights
                const bool window_tile = tile + k >= it.kt;
                const bool whole = first + 15 <= it.i0 && (window_tile ? first >= it.lo && (a.window <= 0 || first > it.i1 - a.window) : first + 15 < it.n_keep);
                bool grow = false;
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float s = z[t][e] * (rowf[t][e & 1] * kscale);
                        if (a.cap > 0.f) s = a.cap * kLog2e * tanhf(s / a.cap);
                        if (!whole) {
                            const int j = first + g8 + 8 * (e >> 1), i = pos[t][e & 1];
                            const bool in_tile = window_tile ? j >= it.lo : j < it.n_keep;
                            if (!(in_tile && j <= i && (a.window <= 0 || i - j < a.window || j < a.keep))) s = -INFINITY;
                        }
                        z[t][e] = s;
                        grow |= s > m[t][e & 1] + 8.f;
                    }
                }
                if (__any_sync(0xffffffffu, grow || vscale > 64.f * vref)) {
                    const float vnew = vscale > 64.f * vref ? vscale : vref, vf = vnew > 0.f ? vref / vnew : 0.f;
                    vref = vnew;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float x = fmaxf(z[t][e], z[t][e + 2]);
#pragma unroll
                            for (int off = 4; off <= 16; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                            x = fmaxf(x, m[t][e]);
                            const float f = m[t][e] == -INFINITY ? 0.f : exp2f(m[t][e] - x);
                            m[t][e] = x;
                            l[t][e] *= f;
#pragma unroll
                            for (int i = 0; i < KS; i++) o[i][t][e] *= f * vf, o[i][t][e + 2] *= f * vf;
                        }
                }
                const float vrel = vref > 0.f ? vscale / vref : 0.f;
                uint32_t pb[PARTS][NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = ex2_approx(z[t][e] - (m[t][e & 1] == -INFINITY ? 0.f : m[t][e & 1]));
                        l[t][e & 1] += w[e];
                        w[e] *= vrel;
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const uint32_t hi = half2_bits(w[2 * y], w[2 * y + 1]);
                        pb[0][t][y] = turn8x8(hi);
                        if (PARTS == 2) {
                            const float2 back = half2_floats(hi);
                            pb[PARTS - 1][t][y] = turn8x8(half2_bits(w[2 * y] - back.x, w[2 * y + 1] - back.y));
                        }
                    }
                }
                // ---- output: coordinates 2 i, 2 i + 1 of a lane's piece are rows g8 and g8 + 8 of block i
#pragma unroll
                for (int c = 0; c < VC; c++)
#pragma unroll
                    for (int w = 0; w < VW; w++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const uint32_t sel = y ? 0x7362 : 0x5140;
                            uint32_t a0, a1, a2, a3;
                            halves_of<CODE>(__byte_perm(vx[0][c][w], vx[1][c][w], sel), a0, a1);
                            halves_of<CODE>(__byte_perm(vx[2][c][w], vx[3][c][w], sel), a2, a3);
#pragma unroll
                            for (int part = PARTS - 1; part >= 0; part--)
#pragma unroll
                                for (int t = 0; t < NT; t++) mma16816(o[c * 8 + 2 * w + y][t], a0, a1, a2, a3, pb[part][t][0], pb[part][t][1]);
                        }
            } else {
                load_k(next, next_page);
            }
            load_v(next, next_page);
            first = next, page = next_page, next = after, next_page = after_page;
        }

        // ---- the warps' sums meet
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = 8 * t + 2 * c4 + e;
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], off);
                if (g8 == 0) sm[warp * R + r] = m[t][e], sl[warp * R + r] = l[t][e];
                float2 *row = red + (warp * R + r) * (P / 2);
#pragma unroll
                for (int i = 0; i < KS; i++) row[64 * (i / 8) + red_at<P>(g8, i % 8, c4)] = make_float2(o[i][t][e], o[i][t][e + 2]);
            }
        if (lane == 0) svref[warp] = vref;
        __syncthreads();
        const bool whole_item = n == it.n;
        float *part = a.part ? a.part + ((int64_t)blockIdx.x * 2 + (tile == 0)) * R * (a.Dv + 2) : nullptr;
        constexpr int TPR = kStepThreads / R; // threads a row
        const int r = tid / TPR;
        if (r < it.rows) {
            float M = -INFINITY, L = 0.f, f[kStepWarps];
#pragma unroll
            for (int w = 0; w < kStepWarps; w++) M = fmaxf(M, sm[w * R + r]);
#pragma unroll
            for (int w = 0; w < kStepWarps; w++) {
                f[w] = sm[w * R + r] == -INFINITY ? 0.f : exp2f(sm[w * R + r] - M);
                L = fmaf(sl[w * R + r], f[w], L);
                f[w] *= svref[w];
            }
            const int row = it.row0 + r, tq = row / hpg, h = head * hpg + (row - tq * hpg);
            const int64_t t = it.t0 + tq;
            const row_end end(a, h, M, L);
            for (int pr = tid - r * TPR; pr < a.Dv / 2; pr += TPR) {
                constexpr int W = P == 64 ? 4 : 8;
                const int at = 64 * (pr / 64) + red_at<P>((pr % 64) / W, pr % W, (r % 8) / 2);
                float2 y = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kStepWarps; w++) {
                    const float2 x = red[(w * R + r) * (P / 2) + at];
                    y.x = fmaf(x.x, f[w], y.x), y.y = fmaf(x.y, f[w], y.y);
                }
                if (whole_item) {
                    const int64_t to = (int64_t)h * a.Dv + 2 * pr;
                    E *out = reinterpret_cast<E *>(a.out) + t * a.H * a.Dv + to;
                    out[0] = from_f32<E>(gated(a, y.x * end.f, t, to)), out[1] = from_f32<E>(gated(a, y.y * end.f, t, to + 1));
                } else {
                    *reinterpret_cast<float2 *>(part + (int64_t)r * (a.Dv + 2) + 2 * pr) = y;
                }
            }
            if (!whole_item && tid == r * TPR) part[(int64_t)r * (a.Dv + 2) + a.Dv] = M, part[(int64_t)r * (a.Dv + 2) + a.Dv + 1] = L;
        }
        if (!whole_item && tile == 0 && tid == 0) { // it ends with the CTA that has its last tile
            const int64_t N = min((int64_t)gridDim.x, U), last = u - tile + it.n - 1;
            a.desc[blockIdx.x] = make_int4(it.s, it.rg, head, (int)(((last + 1) * N - 1) / U));
        }
        u += n;
        if (u >= u_end) break;
        __syncthreads(); // what is read above is written by the next piece
        tile = 0;
        if (++head == a.G) {
            head = 0;
            do {
                entry++;
                it = item_of<R>(a, entry / a.groups, entry % a.groups);
            } while (it.n == 0);
        }
    }
}

// an item's pieces: a row a CTA.  Threads of a column (four numbers) have the pieces in turn and are added up in order
template <int R, typename E> __global__ void __launch_bounds__(256) kv8_join_kernel(const __grid_constant__ attn_args a) {
    __shared__ float4 s_y[256];
    __shared__ float s_f[kMaxCtas], s_red[8], s_l[8];
    step_wait();
    const int b0 = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int4 d = a.desc[b0];
    if (d.x < 0) return;
    const int hpg = a.H / a.G, row = d.y * R + r, tq = row / hpg, h = d.z * hpg + (row - tq * hpg), pieces = d.w - b0 + 1;
    const int64_t t = a.starts[d.x] + tq;
    if (t >= a.starts[d.x + 1]) return;
    const int64_t pitch = a.Dv + 2;
    auto piece = [&](int k) { return a.part + (((int64_t)(b0 + k) * 2 + (k == 0)) * R + r) * pitch; };
    float M = -INFINITY;
    for (int k = tid; k < pieces; k += 256) M = fmaxf(M, s_f[k] = piece(k)[a.Dv]);
    M = warp_max_f32(M);
    if (lane == 0) s_red[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) M = fmaxf(M, s_red[w]);
    float L = 0.f;
    for (int k = tid; k < pieces; k += 256) {
        const float f = s_f[k] == -INFINITY ? 0.f : exp2f(s_f[k] - M);
        L = fmaf(piece(k)[a.Dv + 1], f, L);
        s_f[k] = f;
    }
    L = warp_sum_f32(L);
    if (lane == 0) s_l[warp] = L;
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int w = 0; w < 8; w++) L += s_l[w];
    const int quads = a.Dv / 4, ways = 256 / quads, way = tid / quads, c = 4 * (tid - way * quads);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (way < ways)
#pragma unroll 4
        for (int k = way; k < pieces; k += ways) {
            const float2 *x = reinterpret_cast<const float2 *>(piece(k) + c);
            const float2 p = x[0], q = x[1];
            const float f = s_f[k];
            y.x = fmaf(p.x, f, y.x), y.y = fmaf(p.y, f, y.y), y.z = fmaf(q.x, f, y.z), y.w = fmaf(q.y, f, y.w);
        }
    s_y[tid] = y;
    __syncthreads();
    if (way != 0) return;
    for (int w = 1; w < ways; w++) {
        const float4 x = s_y[w * quads + tid];
        y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
    }
    const row_end end(a, h, M, L);
    const int64_t to = (int64_t)h * a.Dv + c;
    E *out = reinterpret_cast<E *>(a.out) + t * a.H * a.Dv + to;
    out[0] = from_f32<E>(gated(a, y.x * end.f, t, to)), out[1] = from_f32<E>(gated(a, y.y * end.f, t, to + 1));
    out[2] = from_f32<E>(gated(a, y.z * end.f, t, to + 2)), out[3] = from_f32<E>(gated(a, y.w * end.f, t, to + 3));
}

template <int CODE, int P, int NT, int PARTS> int step_launch(attn_args a, int64_t max_new) {
    using Z = step_sizes<P, NT, PARTS>;
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    const int64_t groups = (max_new * (a.H / a.G) + Z::R - 1) / Z::R;
    GGB_CHECK_ARG(max_new * (a.H / a.G) < (1ll << 30) && a.n_seq * groups * a.G < (1ll << 31), "kv8_attn: too many sequences, tokens and heads for a launch");
    a.groups = (int)groups;
    auto k = kv8_step_kernel<CODE, P, NT, PARTS>;
    const int rc = ggb_allow_smem(k, Z::smem);
    if (rc) return rc;
    const unsigned ctas = a.part ? (unsigned)std::min(kMaxCtas, ggb_sm_count() * Z::min_ctas) : (unsigned)(a.n_seq * a.groups * a.G);
    GGB_CUDA(ggb_launch_step(k, dim3(ctas), dim3(kStepThreads), Z::smem, a));
    GGB_LAUNCH_CHECK();
    if (a.part) {
        GGB_CUDA(ggb_launch_step(kv8_join_kernel<Z::R, E>, dim3(ctas, Z::R), dim3(256), 0, a));
        GGB_LAUNCH_CHECK();
    }
    return GGB_OK;
}
// rows of an item: as many as a sequence and key head has, up to 32 (16 with the largest heads, whose sums fill the registers)
template <int CODE, int PARTS> int step_rows(const attn_args &a, int64_t max_new) {
    const int64_t rows = max_new * (a.H / a.G);
    const int size = std::max(a.D, a.Dv);
    if (size <= 64) return rows <= 8 ? step_launch<CODE, 64, 1, PARTS>(a, max_new) : rows <= 16 ? step_launch<CODE, 64, 2, PARTS>(a, max_new) : step_launch<CODE, 64, 4, PARTS>(a, max_new);
    if (size <= 128) return rows <= 8 ? step_launch<CODE, 128, 1, PARTS>(a, max_new) : rows <= 16 ? step_launch<CODE, 128, 2, PARTS>(a, max_new) : step_launch<CODE, 128, 4, PARTS>(a, max_new);
    return rows <= 8 ? step_launch<CODE, 256, 1, PARTS>(a, max_new) : step_launch<CODE, 256, 2, PARTS>(a, max_new);
}

} // namespace

extern "C" {

size_t ggb_kv8_attn_scratch_bytes(int Dv) { return part_bytes(Dv); }

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
    GGB_CHECK_ARG(T > 0 && n_seq > 0 && T <= (1 << 24) && n_seq <= (1 << 20) && max_new > 0 && max_new <= T && table_ld > 0,
                  "kv8_attn: %lld tokens of %d sequences, at most %lld each", (long long)T, n_seq, (long long)max_new);
    GGB_CHECK_ARG(softcap >= 0.f && keep_first >= 0 && (!gate || ldg >= (int64_t)H * Dv), "kv8_attn: a soft cap or kept positions below zero, or a gate row too short");
    GGB_CHECK_ARG((uintptr_t)cache % 16 == 0, "kv8_attn: the cache must begin on a 16-byte boundary");
    GGB_CHECK_ARG(!scratch || ((uintptr_t)scratch % 16 == 0 && scratch_bytes >= part_bytes(Dv)), "kv8_attn: %zu bytes of scratch, %zu needed on a 16-byte boundary",
                  scratch_bytes, part_bytes(Dv));
    float *part = (float *)scratch;
    const attn_args a{q, (const uint8_t *)cache, tables, table_ld, block_size, n_seq, starts, pos0, H, G, D, Dv, window, window > 0 ? keep_first : 0, softcap, sink, gate, ldg,
                           kv8_record(D, Dv, block_size), out, 0, part, part ? (int4 *)(part + (size_t)kMaxCtas * 2 * kMaxRows * (Dv + 2)) : nullptr,
                           (uintptr_t)q % 16 == 0};
    if (dt == GGB_TYPE_BF16) return code == GGB_KV8_INT8 ? step_rows<GGB_KV8_INT8, 1>(a, max_new) : step_rows<GGB_KV8_E4M3, 1>(a, max_new);
    return code == GGB_KV8_INT8 ? step_rows<GGB_KV8_INT8, 2>(a, max_new) : step_rows<GGB_KV8_E4M3, 2>(a, max_new);
}

} // extern "C"
