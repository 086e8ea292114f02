// kv8_tile.cuh — attention of many rows of queries over the 8-bit paged cache on tcgen05: portions of prompts.
//
// A CTA takes 128 rows of queries (tokens x the query heads of one key head) through tiles of 64 positions:
//
//   codes    four warps, 16 positions each: asked for three tiles ahead (cp.async, a lane for what it reads itself), turned into fp16 (exactly) and laid out as the
//            tensor cores want them
//   scores   S [128][64] = (q_l + q_h) K^T: queries as PARTS fp16 numbers, rows by a power of two in the upper part of the range (as in the steps' kernel)
//   weights  two threads a row, 32 positions each: S from tensor memory times the group's key scale and the row's factor, soft cap, mask, 2^(s - m), times the group's value
//            scale over a kept one, as PARTS fp16 numbers back to tensor memory, over the scores
//   output   O [128][Dv] += (p_l + p_h) V, weights from tensor memory, the values as they lie (MN-major B)
//
// Two groups of eight warps take the tiles alternately, each with scores, maxima, sums and output of its own, so that the tensor cores work for the one while the other
// computes weights.  A maximum, and the value scale that weights are relative to, are kept until they are exceeded far enough (2^8 and 64 times), so the
// output is hardly ever rescaled; both are a row's or a CTA's, no thread asks another but its row's other half.
//
// Work is dealt as in the steps' kernel: items (sequence, 128 rows, key head) of tiles in one row, an even share to every CTA, pieces of items joined behind.
#pragma once

#include "kv8.cuh"
#include "tile_attention.cuh"

namespace kv8 {

constexpr int kTileRows = 128, kTileKeys = 64, kTileBegin = 6; // (an item costs about six tiles to begin and to end)
constexpr int kTileCtas = 128;                                 // that share items: their pieces fill the workspace
constexpr int kSoftWarps = 16, kCodeWarps = 4, kTileThreads = 32 * (kSoftWarps + kCodeWarps + 4), kTileMma = kSoftWarps + kCodeWarps;
// registers: six groups of four warps are launched with 80 a thread, of which the weights' take 96 and the others 64 and 32 (4 x 96 + 64 + 32 = 6 x 80)
constexpr int kSoftRegs = 96, kCodeRegs = 64, kMmaRegs = 32;
constexpr int kAhead = 3; // tiles of codes asked for
enum { T_K_FULL = 0, T_K_FREE = 16, T_V_FULL = 32, T_V_FREE = 48, T_S_FULL = 64, T_P_FULL = 80, T_DONE = 96, T_Q_FULL = 104, T_SLOT = 128, T_DEAD = 132 };

template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct tile_sizes {
    uint32_t q, k, v, raw, raw_stage, stats, scales, bars, smem; // byte offsets behind the 1024-byte boundary, and bytes in all
    __host__ __device__ tile_sizes(int parts, int D, int Dv) {
        const uint32_t D64 = (D + 63) / 64, V64 = (Dv + 63) / 64;
        q = 0, k = parts * D64 * kTileRows * 128, v = k + 2 * D64 * kTileKeys * 128, raw = v + 2 * V64 * kTileKeys * 128;
        raw_stage = 1024 * (D64 + V64); // a warp's: two rows of 64 codes a lane and block
        stats = raw + kCodeWarps * kAhead * raw_stage;
        scales = stats + 13 * kTileRows * 4, bars = scales + 8 * 4 * 8, smem = 1024 + bars + 256;
    }
};
inline bool tile_fits(int D, int Dv, int H, int G) { return D <= 128 && Dv <= 128 && H / G <= kTileRows; }

struct tile_mma {
    uint32_t bars, q, q_part, k, k_stage, v, v_stage, tmem;
    int ksteps, Dv;
    volatile int *dead;
};
__device__ __forceinline__ constexpr uint32_t idesc_f16(int M, int N, bool b_mn) { return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
// the MMAs of a piece's n tiles: ph, uses of the two stages so far, `pieces` pieces so far.  KS: D / 16, or 0 for a number known at run time only
template <int PARTS, int KS> __device__ __forceinline__ void tile_products(const tile_mma &m, int n, int ph0, int ph1, int pieces) {
    const uint32_t id_s = idesc_f16(kTileRows, kTileKeys, false), id_o = idesc_f16(kTileRows, m.Dv, true);
    const uint32_t q_lo = umma_desc_lo(m.q, 16), k_lo = umma_desc_lo(m.k, 16), v_lo = umma_desc_lo(m.v, kTileKeys * 128);
    auto scores = [&](int t) {
        const uint32_t s = t & 1, par = ((s ? ph1 : ph0) + (t >> 1)) & 1, d = m.tmem + s * 64, kl = k_lo + ((s * m.k_stage) >> 4);
        mbar_wait_bounded(m.bars + T_K_FULL + 8 * s, par, m.dead);
        tc_fence_after();
#pragma unroll
        for (int part = PARTS - 1; part >= 0; part--) { // the small part first
            const uint32_t ql = q_lo + part * (m.q_part >> 4);
            if (KS > 0) {
#pragma unroll
                for (int b = 0; b < KS / 4; b++) umma_ss_k4(d, ql + b * (kTileRows * 8), kl + b * (kTileKeys * 8), id_s, part < PARTS - 1 || b > 0);
            } else {
                for (int k = 0; k < m.ksteps; k++)
                    umma_ss(d, ql + (k >> 2) * (kTileRows * 8) + 2 * (k & 3), kl + (k >> 2) * (kTileKeys * 8) + 2 * (k & 3), id_s, part < PARTS - 1 || k > 0);
            }
        }
        umma_arrive(m.bars + T_S_FULL + 8 * s);
        umma_arrive(m.bars + T_K_FREE + 8 * s);
    };
    mbar_wait_bounded(m.bars + T_Q_FULL, pieces & 1, m.dead);
    scores(0);
    if (n > 1) scores(1);
    for (int t = 0; t < n; t++) {
        const uint32_t s = t & 1, par = ((s ? ph1 : ph0) + (t >> 1)) & 1;
        mbar_wait_bounded(m.bars + T_P_FULL + 8 * s, par, m.dead);
        mbar_wait_bounded(m.bars + T_V_FULL + 8 * s, par, m.dead);
        tc_fence_after();
        const uint32_t o = m.tmem + 128 + s * m.Dv, p = m.tmem + s * 64, vl = v_lo + ((s * m.v_stage) >> 4);
#pragma unroll
        for (int part = PARTS - 1; part >= 0; part--) umma_ts_k4(o, p + part * 32, vl, 128, id_o, part < PARTS - 1 ? 1u : t >= 2);
        umma_arrive(m.bars + T_V_FREE + 8 * s);
        if (t + 2 < n) scores(t + 2);
    }
    umma_arrive(m.bars + T_DONE);
}

// without a workspace an item is one CTA's: the one that its first unit is dealt to
__device__ __forceinline__ void tile_piece_from(const attn_args &a, piece &x, unsigned at, unsigned end) {
    if (a.part) {
        piece_from<kTileRows, kTileKeys, kTileBegin>(a, x, at, end);
        return;
    }
    while (x.u < at) {
        x.u += x.it.n + kTileBegin, x.n = 0;
        if (x.u >= end) return;
        if (++x.head == a.G) {
            x.head = 0;
            do {
                x.entry++;
                x.it = item_of<kTileRows, kTileKeys>(a, x.entry / a.groups, x.entry % a.groups);
            } while (x.it.n == 0);
        }
    }
    x.tile = 0, x.n = x.it.n;
}

template <int CODE, int PARTS>
__global__ void __launch_bounds__(kTileThreads, 1) kv8_tile_kernel(const __grid_constant__ attn_args a) {
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    extern __shared__ uint8_t kt_raw[];
    __shared__ piece s_piece[2];
    __shared__ unsigned s_scan[kTileThreads / 32], s_end, s_all;
    const uint32_t raw0 = smem_u32(kt_raw), base = (raw0 + 1023u) & ~1023u;
    uint8_t *gbase = kt_raw + (base - raw0);
    const tile_sizes z(PARTS, a.D, a.Dv);
    const uint32_t bars = base + z.bars;
    volatile int *dead = reinterpret_cast<volatile int *>(gbase + z.bars + T_DEAD);
    float *st = reinterpret_cast<float *>(gbase + z.stats);
    float2 *scales = reinterpret_cast<float2 *>(gbase + z.scales); // [8 tiles][4 groups]: keys', values'
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hpg = a.H / a.G;
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(bars + T_K_FULL + 8 * s, kCodeWarps);
            mbar_init(bars + T_K_FREE + 8 * s, 1);
            mbar_init(bars + T_V_FULL + 8 * s, kCodeWarps);
            mbar_init(bars + T_V_FREE + 8 * s, 1);
            mbar_init(bars + T_S_FULL + 8 * s, 1);
            mbar_init(bars + T_P_FULL + 8 * s, kSoftWarps / 2);
        }
        mbar_init(bars + T_DONE, 1);
        mbar_init(bars + T_Q_FULL, kSoftWarps);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTileMma) tmem_alloc512(bars + T_SLOT);
    early_wait();

    // ---- what this CTA has been dealt
    {
        const int entries = a.n_seq * a.groups, each = (entries + kTileThreads - 1) / kTileThreads, e0 = min(entries, tid * each), e1 = min(entries, e0 + each);
        unsigned mine = 0, U = 0, front = 0;
        piece x;
        for (x.entry = e0; x.entry < e1; x.entry++) {
            x.it = item_of<kTileRows, kTileKeys>(a, x.entry / a.groups, x.entry % a.groups);
            if (x.it.n) mine += (x.it.n + kTileBegin) * a.G;
        }
        unsigned run = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, run, off);
            if (lane >= off) run += y;
        }
        if (lane == 31) s_scan[warp] = run;
        if (tid == 0) {
            s_piece[0].n = 0;
            if (a.part) a.desc[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        step_next();
        for (int w = 0; w < kTileThreads / 32; w++) {
            if (w < warp) front += s_scan[w];
            U += s_scan[w];
        }
        const deal d(U, gridDim.x);
        const unsigned u = d.first(blockIdx.x), end = d.first(blockIdx.x + 1);
        front += run - mine;
        if (u < end && u >= front && u < front + mine) {
            for (x.entry = e0;; x.entry++) {
                x.it = item_of<kTileRows, kTileKeys>(a, x.entry / a.groups, x.entry % a.groups);
                const unsigned n = x.it.n ? (x.it.n + kTileBegin) * a.G : 0;
                if (u < front + n) break;
                front += n;
            }
            x.head = (int)((u - front) / (unsigned)(x.it.n + kTileBegin)), x.u = front + x.head * (x.it.n + kTileBegin);
            tile_piece_from(a, x, u, end);
            s_piece[0] = x, s_end = end, s_all = U;
        }
        __syncthreads();
    }
    const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<uint32_t *>(gbase + z.bars + T_SLOT), 0);
    const int D64 = (a.D + 63) / 64, V64 = (a.Dv + 63) / 64;
    const uint32_t q_part = D64 * kTileRows * 128, k_stage = D64 * kTileKeys * 128, v_stage = V64 * kTileKeys * 128;

    // the roles, each through all pieces; ph0, ph1: uses of the two stages so far
    auto next_piece = [&] { // all threads: what a piece was is no longer needed
        tc_fence_before();
        warp_meet();
        bar_sync(0, kTileThreads);
        tc_fence_after();
    };
    int ph0 = 0, ph1 = 0;
    if (warp >= kSoftWarps && warp < kTileMma) {
        // ---- codes: a warp has 16 positions of every tile, a lane rows (lane >> 2) and 8 on, 16 codes of every 64
        fewer_registers<kCodeRegs>();
        const int cw = warp - kSoftWarps, r0 = lane >> 2, c = 16 * (lane & 3);
        const uint32_t ring = base + z.raw + cw * kAhead * z.raw_stage + 16 * lane, scale_at = base + z.scales + 8 * cw + 4 * lane; // (lanes 0 and 1: keys', values')
        const int r = 16 * cw + r0, pc = 2 * (lane & 3); // rows r and r + 8 of a tile: the same place within 8 rows
        const uint32_t at0 = r * 128 + ((pc ^ (r & 7)) << 4), at1 = r * 128 + (((pc + 1) ^ (r & 7)) << 4);
        const int per_pages = kTileKeys / a.B, per_rows = kTileKeys - per_pages * a.B;
        int stage = 0;
        for (int slot = 0; s_piece[slot].n > 0; slot ^= 1) {
            const item &it = s_piece[slot].it;
            const int n = s_piece[slot].n, tile = s_piece[slot].tile, head = s_piece[slot].head;
            const int kt = it.kt, w0 = it.w0 - kt, n_keep = it.n_keep, lo = it.lo, i1 = it.i1;
            const int32_t *table = a.tables + it.s * a.table_ld;
            auto first_of = [&](int k) { return (tile + k < kt ? tile + k : w0 + tile + k) * kTileKeys + 16 * cw; };
            auto seen = [&](int k, int first) { return tile + k < kt ? first < n_keep : first + 15 >= lo && first <= i1; };
            // the group that is asked for next: its page, or -1, and row.  From a tile to the next the place in the table and the row move by what a tile is in pages and rows
            int page = -1, at_page = 0, at_row = 0;
            auto look = [&](int k) {
                const int first = first_of(k);
                if (k == 0 || tile + k == kt) {
                    at_page = first / a.B, at_row = first - at_page * a.B;
                } else {
                    at_page += per_pages, at_row += per_rows;
                    if (at_row >= a.B) at_row -= a.B, at_page++;
                }
                page = -1;
                if (k < n && seen(k, first)) page = table[at_page];
            };
            auto ask = [&](int k, int to_stage) {
                const uint32_t to_scale = scale_at + ((ph0 + ph1 + k) & 7) * 32;
                if (page >= 0) {
                    const int row = at_row;
                    const uint8_t *rec = a.cache + ((int64_t)page * a.G + head) * a.record, *kp = rec + (row + r0) * a.D + c, *vp = rec + a.B * a.D + (row + r0) * a.Dv + c;
                    const uint32_t to = ring + to_stage * z.raw_stage;
#pragma unroll
                    for (int b = 0; b < 2; b++)
                        if (64 * b + c < a.D) {
                            cp_async16(to + b * 1024, kp + 64 * b);
                            cp_async16(to + b * 1024 + 512, kp + 8 * a.D + 64 * b);
                        }
#pragma unroll
                    for (int b = 0; b < 2; b++)
                        if (64 * b + c < a.Dv) {
                            cp_async16(to + (D64 + b) * 1024, vp + 64 * b);
                            cp_async16(to + (D64 + b) * 1024 + 512, vp + 8 * a.Dv + 64 * b);
                        }
                    if (lane < 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to_scale), "l"(rec + a.B * (a.D + a.Dv) + (row + lane * a.B) / 4) : "memory");
                } else if (k < n && lane < 2) {
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(to_scale), "r"(0) : "memory");
                }
                cp_async_commit();
                look(k + 1);
            };
            // a lane's codes of keys, or of values, to their places
            auto lay_out = [&](uint32_t from, uint32_t to, int blocks, int width, bool zero0, bool zero1) {
#pragma unroll
                for (int b = 0; b < 2; b++)
                    if (b < blocks) {
                        uint4 w[2];
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[e].x), "=r"(w[e].y), "=r"(w[e].z), "=r"(w[e].w) : "r"(from + b * 1024 + e * 512) : "memory");
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            uint32_t h[8];
                            halves_of<CODE>(w[e].x, h[0], h[1]);
                            halves_of<CODE>(w[e].y, h[2], h[3]);
                            halves_of<CODE>(w[e].z, h[4], h[5]);
                            halves_of<CODE>(w[e].w, h[6], h[7]);
                            if (64 * b + c >= width || (e ? zero1 : zero0))
#pragma unroll
                                for (int u = 0; u < 8; u++) h[u] = 0;
                            const uint32_t row = to + b * (kTileKeys * 128) + e * 1024;
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + at0), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + at1), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                        }
                    }
                fence_async_smem();
                __syncwarp();
            };
            look(0);
            for (int k = 0, s = stage; k < kAhead - 1; k++) {
                ask(k, s);
                if (++s == kAhead) s = 0;
            }
            for (int k = 0; k < n; k++) {
                const int s = k & 1, uses = (s ? ph1 : ph0) + (k >> 1), first = first_of(k);
                ask(k + kAhead - 1, stage == 0 ? kAhead - 1 : stage - 1);
                cp_async_wait<kAhead - 1>();
                const uint32_t from = ring + stage * z.raw_stage;
                if (uses > 0 && !mbar_wait_warp(bars + T_K_FREE + 8 * s, (uses - 1) & 1, dead)) break;
                lay_out(from, base + z.k + s * k_stage, D64, a.D, false, false);
                if (lane == 0) mbar_arrive(bars + T_K_FULL + 8 * s);
                if (uses > 0 && !mbar_wait_warp(bars + T_V_FREE + 8 * s, (uses - 1) & 1, dead)) break;
                // behind the last position, and where nothing was asked for, there may be codes that are no numbers, which a weight of zero would not undo
                const bool none = !seen(k, first);
                lay_out(from + D64 * 1024, base + z.v + s * v_stage, V64, a.Dv, none || first + r0 > i1, none || first + r0 + 8 > i1);
                if (lane == 0) mbar_arrive(bars + T_V_FULL + 8 * s);
                if (++stage == kAhead) stage = 0;
            }
            cp_async_wait<0>();
            ph0 += (n + 1) / 2, ph1 += n / 2;
            next_piece();
        }
    } else if (warp >= kTileMma) {
        // ---- products, by the first of these warps
        fewer_registers<kMmaRegs>();
        int pieces = 0;
        for (int slot = 0; s_piece[slot].n > 0; slot ^= 1, pieces++) {
            const int n = s_piece[slot].n;
            if (warp == kTileMma) {
                const tile_mma m{bars, base + z.q, q_part, base + z.k, k_stage, base + z.v, v_stage, tmem, a.D / 16, a.Dv, dead};
                if (a.D == 128) tile_products<PARTS, 8>(m, n, ph0, ph1, pieces);
                else if (a.D == 64) tile_products<PARTS, 4>(m, n, ph0, ph1, pieces);
                else tile_products<PARTS, 0>(m, n, ph0, ph1, pieces);
            }
            ph0 += (n + 1) / 2, ph1 += n / 2;
            next_piece();
        }
    } else {
        more_registers<kSoftRegs>();
        int pieces = 0;
        for (int slot = 0; s_piece[slot].n > 0; slot ^= 1, pieces++) {
            const piece &x = s_piece[slot];
            const item &it = x.it;
            const int n = x.n, tile = x.tile;
            auto first_of = [&](int t) { return (t < it.kt ? t : it.w0 + t - it.kt) * kTileKeys; };
            // ---- queries: a warp's 8 rows
            float *srow = st + 12 * kTileRows;
#pragma unroll 1
            for (int u0 = 0; u0 < 8; u0 += 4) {
                float4 v[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int r = 8 * warp + u0 + u, row = it.row0 + r, tq = row / hpg, h = x.head * hpg + (row - tq * hpg);
                    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < it.rows && 4 * lane < a.D) {
                        const float *src = a.q + ((it.t0 + tq) * a.H + h) * a.D + 4 * lane;
                        if (a.vec_q) v[u] = *reinterpret_cast<const float4 *>(src);
                        else v[u] = make_float4(src[0], src[1], src[2], src[3]);
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int r = 8 * warp + u0 + u;
                    const float big = fmaxf(fmaxf(fabsf(v[u].x), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w))), most = warp_max_f32(big);
                    const bool odd = __any_sync(0xffffffffu, big == INFINITY || v[u].x != v[u].x || v[u].y != v[u].y || v[u].z != v[u].z || v[u].w != v[u].w);
                    const float f = odd ? 0.f : power_for(most, 10);
                    if (lane == 0) srow[r] = odd ? NAN : kLog2e / f; // what is not finite spoils its own row
                    if (4 * lane >= 64 * D64) continue;
                    const float y[4] = {odd ? 0.f : v[u].x * f, odd ? 0.f : v[u].y * f, odd ? 0.f : v[u].z * f, odd ? 0.f : v[u].w * f};
                    uint2 p = make_uint2(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]));
                    const uint32_t at = base + z.q + (lane >> 4) * (kTileRows * 128) + r * 128 + ((((lane >> 1) & 7) ^ (r & 7)) << 4) + (lane & 1) * 8;
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(p.x), "r"(p.y) : "memory");
                    if (PARTS == 2) {
                        const float2 b0 = half2_floats(p.x), b1 = half2_floats(p.y);
                        p = make_uint2(half2_bits(y[0] - b0.x, y[1] - b0.y), half2_bits(y[2] - b1.x, y[3] - b1.y));
                        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + q_part), "r"(p.x), "r"(p.y) : "memory");
                    }
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + T_Q_FULL);
            bar_sync(3, 32 * kSoftWarps); // the rows' factors
            if (tid == 32 * kSoftWarps - 1) { // while the first scores are under way: the piece behind this one
                piece y = x;
                const unsigned at = y.u + kTileBegin + y.tile + y.n;
                y.n = 0;
                if (at < s_end) tile_piece_from(a, y, at, s_end);
                s_piece[slot ^ 1] = y;
            }
            __syncwarp();
            // ---- weights: group grp takes the tiles k = grp, grp + 2, ...; a thread owns 32 positions of one row, two threads the row
            const int grp = warp >> 3, half = (warp >> 2) & 1, r = 32 * (warp & 3) + lane;
            const int i = r < it.rows ? it.p0 + (it.row0 + r) / hpg : -1, lo = a.window > 0 ? (int)max((int64_t)0, i - a.window + 1) : 0;
            const int lo_last = a.window > 0 ? (int)max((int64_t)0, it.i1 - a.window + 1) : 0;
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = tmem + lanes + grp * 64, to = tmem + lanes + 128 + grp * a.Dv;
            const float rowf = srow[r], cap = a.cap * kLog2e, inv_cap = a.cap > 0.f ? kLn2 / a.cap : 0.f;
            float m = kNone, l = 0.f, vref = 0.f, vinv = 0.f;
            bool lost = false;
            for (int k = grp; k < n; k += 2) {
                const int t = tile + k, j0 = first_of(t);
                const bool kept = t < it.kt, whole = kept ? j0 + kTileKeys <= it.n_keep : j0 >= max(it.lo, lo_last) && j0 + kTileKeys - 1 <= it.i0;
                if (!mbar_wait_warp(bars + T_S_FULL + 8 * grp, ((grp ? ph1 : ph0) + (k >> 1)) & 1, dead)) lost = true;
                tc_fence_after();
                const float2 *sc = scales + ((ph0 + ph1 + k) & 7) * 4;
                const float most_v = fmaxf(fmaxf(sc[0].y, sc[1].y), fmaxf(sc[2].y, sc[3].y));
                float y[2][16], mx = kNone;
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    tmem_load16(ts + 32 * half + 16 * g, reinterpret_cast<uint32_t *>(y[g]));
                    const float f = rowf * sc[2 * half + g].x;
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const float2 p = unpack2(mul2(pack2(y[g][2 * c], y[g][2 * c + 1]), pack2(f, f)));
                        y[g][2 * c] = p.x, y[g][2 * c + 1] = p.y;
                    }
                    if (a.cap > 0.f) tile_attn::soft_cap16(y[g], cap, inv_cap);
                    if (!whole) { // positions [from, upto) of the tile, and of those below `from` the kept ones
                        const int c0 = j0 + 32 * half + 16 * g, upto = (kept ? it.n_keep : i + 1) - c0, from = (kept ? 0 : lo) - c0, keep = (int)min(a.keep, (int64_t)lo) - c0, low = it.lo - c0;
#pragma unroll
                        for (int c = 0; c < 16; c++) y[g][c] = c < upto && (kept || (c >= low && (c >= from || c < keep))) && i >= 0 ? y[g][c] : -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < 16; c++) mx = fmaxf(mx, y[g][c]);
                }
                float *swap = st + (2 * grp + 4 * ((k >> 1) & 1)) * kTileRows + r; // two tables: the next tile writes the other one
                swap[half * kTileRows] = mx;
                bar_sync(1 + grp, 256); // both halves' scores are in registers, too, before either's weights go over them
                mx = fmaxf(mx, swap[(half ^ 1) * kTileRows]);
                float f = 1.f;
                if (mx > m + 8.f) {
                    f = exp2f(m - mx);
                    m = mx, l *= f;
                }
                const bool more = most_v > 64.f * vref;
                if (more) {
                    f *= vref / most_v;
                    vref = most_v, vinv = 1.f / most_v;
                }
                if (k >= 2 && __any_sync(0xffffffffu, f != 1.f)) { // (its MMAs precede this tile's scores)
#pragma unroll 1
                    for (int c = 16 * half; c < a.Dv; c += 32) {
                        uint32_t o[16];
                        tmem_load16(to + c, o);
#pragma unroll
                        for (int u = 0; u < 16; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
                        tmem_store16(to + c, o);
                    }
                }
                f32x2 sum[2] = {0, 0};
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const float rel = sc[2 * half + g].y * vinv;
                    uint32_t hi[8], lo2[8];
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const float2 t2 = unpack2(add2(pack2(y[g][2 * c], y[g][2 * c + 1]), pack2(-m, -m)));
                        f32x2 w = pack2(ex2_approx(t2.x), ex2_approx(t2.y));
                        sum[c & 1] = add2(sum[c & 1], w);
                        w = mul2(w, pack2(rel, rel));
                        const float2 wv = unpack2(w);
                        hi[c] = half2_bits(wv.x, wv.y);
                        if (PARTS == 2) {
                            const float2 back = half2_floats(hi[c]);
                            lo2[c] = half2_bits(wv.x - back.x, wv.y - back.y);
                        }
                    }
                    tmem_store8(ts + 8 * (2 * half + g), hi);
                    if (PARTS == 2) tmem_store8(ts + 32 + 8 * (2 * half + g), lo2);
                }
                const float2 s2 = unpack2(add2(sum[0], sum[1]));
                l += s2.x + s2.y;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bars + T_P_FULL + 8 * grp);
                if (lost) break;
            }
            // ---- both groups' sums meet
            mbar_wait_warp(bars + T_DONE, pieces & 1, dead);
            tc_fence_after();
            bar_sync(3, 32 * kSoftWarps); // the tables are no longer read
            st[(2 * grp + half) * kTileRows + r] = l;
            if (half == 0) st[(4 + 2 * grp) * kTileRows + r] = m, st[(5 + 2 * grp) * kTileRows + r] = vref;
            bar_sync(3, 32 * kSoftWarps);
            const float m0 = st[4 * kTileRows + r], m1 = st[6 * kTileRows + r], M = fmaxf(m0, m1), g0 = exp2f(m0 - M), g1 = n > 1 ? exp2f(m1 - M) : 0.f;
            const float L = fmaf(st[r] + st[kTileRows + r], g0, n > 1 ? (st[2 * kTileRows + r] + st[3 * kTileRows + r]) * g1 : 0.f);
            const float f0 = g0 * st[5 * kTileRows + r], f1 = g1 * st[7 * kTileRows + r];
            const bool whole_item = n == it.n;
            const int row = it.row0 + r, tq = row / hpg, h = x.head * hpg + (row - tq * hpg), quarter = 2 * grp + half;
            const int64_t t = it.t0 + tq;
            float *part = whole_item ? nullptr : a.part + (((int64_t)blockIdx.x * 2 + (tile == 0)) * kTileRows + r) * (a.Dv + 2);
            const row_end end(a, r < it.rows ? h : 0, M, L);
            for (int cb = quarter; cb < a.Dv / 16; cb += 4) {
                uint32_t o0[16], o1[16];
                tmem_load16(tmem + lanes + 128 + 16 * cb, o0);
                if (n > 1) tmem_load16(tmem + lanes + 128 + a.Dv + 16 * cb, o1);
                if (r < it.rows) {
                    const int64_t at = (int64_t)h * a.Dv + 16 * cb;
                    E *out = reinterpret_cast<E *>(a.out) + t * a.H * a.Dv + at;
#pragma unroll
                    for (int u = 0; u < 16; u += 4) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            v[e] = __uint_as_float(o0[u + e]) * f0;
                            if (n > 1) v[e] = fmaf(__uint_as_float(o1[u + e]), f1, v[e]);
                        }
                        if (whole_item) {
#pragma unroll
                            for (int e = 0; e < 4; e++) v[e] = gated(a, v[e] * end.f, t, at + u + e);
                            if (a.vec_out) store_vec<4, E>(out + u, v);
                            else
#pragma unroll
                                for (int e = 0; e < 4; e++) out[u + e] = from_f32<E>(v[e]);
                        } else {
                            *reinterpret_cast<float2 *>(part + 16 * cb + u) = make_float2(v[0], v[1]);
                            *reinterpret_cast<float2 *>(part + 16 * cb + u + 2) = make_float2(v[2], v[3]);
                        }
                    }
                }
            }
            if (!whole_item && quarter == 0 && r < it.rows) *reinterpret_cast<float2 *>(part + a.Dv) = make_float2(M, L);
            if (!whole_item && tile + n < it.n && tid == 0) {
                const deal d(s_all, gridDim.x);
                a.desc[2 * blockIdx.x] = make_int4(it.s, it.rows, x.head, it.row0);
                a.desc[2 * blockIdx.x + 1] = make_int4((int)d.owner(x.u + kTileBegin), (int)d.owner(x.u + kTileBegin + it.n - 1), (int)it.t0, 0);
            }
            ph0 += (n + 1) / 2, ph1 += n / 2;
            next_piece();
        }
    }
    warp_meet();
    __syncthreads();
    if (warp == kTileMma) {
        settle(dead);
        tc_fence_after();
        tmem_free512(tmem);
        if (lane == 0 && *dead) *a.wait_error = 1;
    }
}

// *joins: CTAs whose pieces are to be joined.  Few items are cut, an even share for kTileCtas; of many, whole ones make shares that are even enough, for every SM
template <int CODE, int PARTS> int tile_launch(attn_args a, int64_t T, int64_t max_new, unsigned *joins) {
    const int hpg = a.H / a.G;
    const int64_t groups = (max_new * hpg + kTileRows - 1) / kTileRows, items = (T * hpg + kTileRows - 1) / kTileRows * a.G;
    GGB_CHECK_ARG(a.n_seq * groups * a.G * ((a.table_ld * a.B + a.keep) / kTileKeys + kTileBegin + 2) < (1ll << 31), "kv8_attn: too many sequences, tokens, heads and positions for a launch");
    a.groups = (int)groups;
    if (items >= 8 * ggb_sm_count()) a.part = nullptr;
    const size_t smem = std::max((size_t)tile_sizes(PARTS, a.D, a.Dv).smem, kOneCtaSmem);
    auto kfn = kv8_tile_kernel<CODE, PARTS>;
    const int rc = ggb_allow_smem(kfn, smem);
    if (rc) return rc;
    static const int registers = [kfn] { // what the split takes has to be there, or it would be waited for without end
        cudaFuncAttributes at{};
        return cudaFuncGetAttributes(&at, kfn) == cudaSuccess ? at.numRegs : 0;
    }();
    GGB_CHECK_ARG(registers * (kTileThreads / 128) >= 4 * kSoftRegs + kCodeRegs + kMmaRegs, "kv8_attn: built with %d registers a thread", registers);
    const unsigned ctas = (unsigned)(a.part ? std::min(kTileCtas, ggb_sm_count()) : ggb_sm_count());
    GGB_CUDA(ggb_launch_early(kfn, ggb_cluster{1, 1, 1}, dim3(ctas), dim3(kTileThreads), smem, a));
    GGB_LAUNCH_CHECK();
    *joins = a.part ? ctas : 0;
    return GGB_OK;
}

} // namespace kv8
