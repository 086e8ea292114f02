// kv8_tile.cuh — attention of many rows of queries over the 8-bit paged cache on tcgen05: portions of prompts.
//
// A CTA takes 128 rows of queries (tokens x the query heads of one key head) through tiles of 64 positions:
//
//   codes    copied by TMA (one warp asks) three tiles ahead; four warps for keys and four for values, 16 positions each, turn them into fp16 (exactly) and lay them out as the
//            tensor cores want them
//   scores   S [128][64] = (q_l + q_h) K^T: queries as two fp16 numbers, rows by a power of two in the upper part of the range (as in the steps' kernel)
//   weights  a thread a row: S from tensor memory times the group's key scale and the row's factor, soft cap, mask, 2^(s - m), times the group's value
//            scale, as PARTS fp16 numbers in the upper part of the range back to tensor memory, over the scores
//   output   O [128][Dv] += (p_l + p_h) V, weights from tensor memory, the values as they lie (MN-major B)
//
// Two groups of four warps take the tiles alternately, each with scores, maxima, sums and output of its own, so that the tensor cores work for the one while the other
// computes weights.  A maximum, and the largest product of a weight and a scale that the row has met, are kept until they are exceeded by 2^8, so the
// output is hardly ever rescaled; both are a row's, and no thread asks another.
//
// Work is dealt as in the steps' kernel: items (sequence, 128 rows, key head) of tiles in one row, an even share to every CTA, pieces of items joined behind; where there are
// many items, whole ones.
//
// What bounds it: nothing is full.  With one part of the queries a tile took a group about 2 us and both together 1: weights some 1,600 cycles a tile and group, products (queries and
// keys from shared memory, which the code warps write at the same time) some 1,300 where 650 would do; the second part adds a third of a microsecond a tile, from shared memory or
// from tensor memory.  Beside that an item begins in 6 us (what was dealt, queries, the first codes) and ends in 4 to 8 (sums, gate, pieces).  1,024 tokens behind 1,024, window 1,024,
// 16 heads over 4 of 128, bf16, gate: 41.7 us (207 TFLOP/s; one part 38); 4,096 tokens from position 0: 254 us (270 TFLOP/s; one part 200), 8,192: 788 us (349 TFLOP/s).
#pragma once

#include "kv8.cuh"
#include "tile_attention.cuh"

namespace kv8 {

constexpr int kTileRows = 128, kTileKeys = 64, kTileBegin = 6; // (an item costs about six tiles to begin and to end)
constexpr int kTileCtas = 128;                                 // that share items: their pieces fill the workspace
constexpr int kSoftWarps = 8, kCodeWarps = 8, kTileThreads = 32 * (kSoftWarps + kCodeWarps + 4), kTileMma = kSoftWarps + kCodeWarps, kTileAsk = kTileMma + 1;
// registers: five groups of four warps are launched with 96 a thread, of which the weights' take 152 and the others 64 and 48 (2 x 152 + 2 x 64 + 48 = 5 x 96)
constexpr int kSoftRegs = 152, kCodeRegs = 64, kMmaRegs = 48;
constexpr int kAhead = 3; // tiles of codes asked for
// tensor cores cut their sums short, always towards zero: with fp32 results what a chain of so many tiles has summed up is added, rounded to the nearest, to the rest in memory
constexpr int kChain = 16;
enum { T_K_FULL = 0, T_K_FREE = 16, T_V_FULL = 32, T_V_FREE = 48, T_S_FULL = 64, T_P_FULL = 80, T_DONE = 96, T_Q_FULL = 104, T_S_FREE = 112, T_SLOT = 128, T_DEAD = 132, T_RAW = 136, T_RAW_FREE = 168 };
// tensor memory: two groups' scores, their weights, their output
constexpr uint32_t kScoreCol = 0, kWeightCol = 128, kOutCol = 256;

__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// mbar_wait_warp whose tries may each last a microsecond: many warps of this kernel wait at any time, and trying costs those that work their turns
__device__ __forceinline__ bool wait_long(uint32_t bar, uint32_t parity, volatile int *dead) {
    for (int i = 0; i < kWaitTries; i++) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
        if (__any_sync(0xffffffffu, *dead)) return false;
    }
    *dead = 1;
    return false;
}
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct tile_sizes {
    uint32_t q, k, v, raw, raw_stage, stats, scales, tables, bars, smem; // byte offsets behind the 1024-byte boundary, and bytes in all
    __host__ __device__ tile_sizes(int D, int Dv) {
        const uint32_t D64 = (D + 63) / 64, V64 = (Dv + 63) / 64;
        q = 0, k = kQueryParts * D64 * kTileRows * 128, v = k + 2 * D64 * kTileKeys * 128, raw = v + 2 * V64 * kTileKeys * 128;
        raw_stage = 4096 * (D64 + V64); // a tile's four groups of keys, then of values, as they are copied
        stats = raw + kAhead * raw_stage;
        scales = stats + 7 * kTileRows * 4, tables = scales + 16 * 4 * 8, bars = tables + 256, smem = 1024 + bars + 256;
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
        const uint32_t s = t & 1, par = ((s ? ph1 : ph0) + (t >> 1)) & 1, d = m.tmem + kScoreCol + s * 64, kl = k_lo + ((s * m.k_stage) >> 4);
        mbar_wait_bounded(m.bars + T_K_FULL + 8 * s, par, m.dead);
        tc_fence_after();
#pragma unroll
        for (int part = kQueryParts - 1; part >= 0; part--) { // the small part first
            const uint32_t ql = q_lo + part * (m.q_part >> 4);
            if (KS > 0) {
#pragma unroll
                for (int b = 0; b < KS / 4; b++) umma_ss_k4(d, ql + b * (kTileRows * 8), kl + b * (kTileKeys * 8), id_s, part < kQueryParts - 1 || b > 0);
            } else {
                for (int k = 0; k < m.ksteps; k++)
                    umma_ss(d, ql + (k >> 2) * (kTileRows * 8) + 2 * (k & 3), kl + (k >> 2) * (kTileKeys * 8) + 2 * (k & 3), id_s, part < kQueryParts - 1 || k > 0);
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
        if (t + 2 < n) { // this tile's scores are in registers: the next ones, ahead of its weights
            mbar_wait_bounded(m.bars + T_S_FREE + 8 * s, par, m.dead);
            scores(t + 2);
        }
        mbar_wait_bounded(m.bars + T_P_FULL + 8 * s, par, m.dead);
        mbar_wait_bounded(m.bars + T_V_FULL + 8 * s, par, m.dead);
        tc_fence_after();
        const uint32_t o = m.tmem + kOutCol + s * m.Dv, p = m.tmem + kWeightCol + s * 64, vl = v_lo + ((s * m.v_stage) >> 4);
#pragma unroll
        for (int part = PARTS - 1; part >= 0; part--) umma_ts_k4(o, p + part * 32, vl, 128, id_o, part < PARTS - 1 ? 1u : (PARTS == 1 ? t : t % kChain) >= 2);
        umma_arrive(m.bars + T_V_FREE + 8 * s);
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
            do next_entry<kTileRows, kTileKeys>(a, x);
            while (x.it.n == 0);
        }
    }
    x.tile = 0, x.n = x.it.n;
}

template <int CODE, int PARTS>
__global__ void __launch_bounds__(kTileThreads, 1) kv8_tile_kernel(const __grid_constant__ attn_args a, const __grid_constant__ line_maps maps) {
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    extern __shared__ uint8_t kt_raw[];
    __shared__ piece s_piece[2];
    __shared__ unsigned s_scan[kTileThreads / 32], s_end, s_all;
    const uint32_t raw0 = smem_u32(kt_raw), base = (raw0 + 1023u) & ~1023u;
    uint8_t *gbase = kt_raw + (base - raw0);
    const tile_sizes z(a.D, a.Dv);
    const uint32_t bars = base + z.bars;
    volatile int *dead = reinterpret_cast<volatile int *>(gbase + z.bars + T_DEAD);
    float *st = reinterpret_cast<float *>(gbase + z.stats);
    float2 *scales = reinterpret_cast<float2 *>(gbase + z.scales); // [16 tiles][4 groups]: keys', values'
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, hpg = a.H / a.G;
    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(bars + T_K_FULL + 8 * s, kCodeWarps / 2);
            mbar_init(bars + T_K_FREE + 8 * s, 1);
            mbar_init(bars + T_V_FULL + 8 * s, kCodeWarps / 2);
            mbar_init(bars + T_V_FREE + 8 * s, 1);
            mbar_init(bars + T_S_FULL + 8 * s, 1);
            mbar_init(bars + T_P_FULL + 8 * s, kSoftWarps / 2);
            mbar_init(bars + T_S_FREE + 8 * s, kSoftWarps / 2);
        }
        for (int s = 0; s < kAhead; s++) mbar_init(bars + T_RAW + 8 * s, 1), mbar_init(bars + T_RAW_FREE + 8 * s, kCodeWarps);
        mbar_init(bars + T_DONE, 1);
        mbar_init(bars + T_Q_FULL, kSoftWarps);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTileMma) tmem_alloc512(bars + T_SLOT);
    early_wait();

    // ---- what this CTA has been dealt
    {
        const int each = (a.entries + kTileThreads - 1) / kTileThreads, e0 = min(a.entries, tid * each), e1 = min(a.entries, e0 + each);
        unsigned mine = 0, U = 0, front = 0;
        piece x;
        if (e0 < e1)
            for (to_entry<kTileRows, kTileKeys>(a, x, e0);; next_entry<kTileRows, kTileKeys>(a, x)) {
                if (x.it.n) mine += (x.it.n + kTileBegin) * a.G;
                if (x.entry + 1 == e1) break;
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
            for (each > 1 ? to_entry<kTileRows, kTileKeys>(a, x, e0) : void();; next_entry<kTileRows, kTileKeys>(a, x)) {
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
        // ---- codes: a warp has the keys, or the values, of a group of every tile; a lane rows (lane >> 2) and 8 on, 16 codes of every 64
        fewer_registers<kCodeRegs>();
        const int cw = warp - kSoftWarps, grp = cw & 3, r0 = lane >> 2, c = 16 * (lane & 3), pc = 2 * (lane & 3);
        const bool is_k = cw < 4;
        const int blocks = is_k ? D64 : V64, width = is_k ? a.D : a.Dv;
        const uint32_t raw = base + z.raw + (is_k ? grp * 1024 * D64 : 4096 * D64 + grp * 1024 * V64), raw_bars = bars + T_RAW, raw_free = bars + T_RAW_FREE;
        const uint32_t full = bars + (is_k ? T_K_FULL : T_V_FULL), empty = bars + (is_k ? T_K_FREE : T_V_FREE), tile_bytes = is_k ? k_stage : v_stage;
        const uint32_t tiles = base + (is_k ? z.k : z.v) + (16 * grp + r0) * 128, at0 = (pc ^ r0) << 4, at1 = ((pc + 1) ^ r0) << 4; // (row r0 + 8: the same place within 8 rows)
        uint32_t from_at[2][2], keep_at[2]; // a lane's codes in a group; behind the end of a row: its first ones, which become zeros
#pragma unroll
        for (int b = 0; b < 2; b++) {
            keep_at[b] = 64 * b + c < width ? ~0u : 0u;
#pragma unroll
            for (int e = 0; e < 2; e++) from_at[b][e] = in_box((r0 + 8 * e) * width + (64 * b + c < width ? 64 * b + c : 0));
        }
        int stage = 0;
        uint32_t raw_parity = 0;
        for (int slot = 0; s_piece[slot].n > 0; slot ^= 1) {
            const item &it = s_piece[slot].it;
            const int n = s_piece[slot].n, tile = s_piece[slot].tile, kt = it.kt, w0 = it.w0 - kt, n_keep = it.n_keep, lo = it.lo, i1 = it.i1;
            for (int k = 0; k < n; k++) {
                const int s = k & 1, uses = (s ? ph1 : ph0) + (k >> 1);
                if (!wait_long(raw_bars + 8 * stage, raw_parity, dead)) break;
                if (uses > 0 && !wait_long(empty + 8 * s, (uses - 1) & 1, dead)) break;
                const uint32_t from = raw + stage * z.raw_stage, to = tiles + s * tile_bytes;
                // values behind the last position, and where nothing was asked for: there may be codes that are no numbers, which a weight of zero would not undo
                const int first = (tile + k < kt ? tile + k : w0 + tile + k) * kTileKeys + 16 * grp;
                const bool none = !is_k && !(tile + k < kt ? first < n_keep : first + 15 >= lo && first <= i1), ragged = none || (!is_k && first + 15 > i1) || (width & 63) != 0;
                uint4 w[2][2];
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (b < blocks) w[b][e] = lds_u4(from + from_at[b][e]);
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (b < blocks) {
                            uint32_t h[8];
                            halves_of<CODE>(w[b][e].x, h[0], h[1]);
                            halves_of<CODE>(w[b][e].y, h[2], h[3]);
                            halves_of<CODE>(w[b][e].z, h[4], h[5]);
                            halves_of<CODE>(w[b][e].w, h[6], h[7]);
                            if (ragged) {
                                const uint32_t keep = none || (!is_k && first + 8 * e + r0 > i1) ? 0u : keep_at[b];
#pragma unroll
                                for (int u = 0; u < 8; u++) h[u] &= keep;
                            }
                            const uint32_t row = to + b * (kTileKeys * 128) + e * 1024;
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + at0), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + at1), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                        }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(raw_free + 8 * stage);
                    mbar_arrive(full + 8 * s);
                }
                if (++stage == kAhead) stage = 0, raw_parity ^= 1;
            }
            ph0 += (n + 1) / 2, ph1 += n / 2;
            next_piece();
        }
    } else if (warp >= kTileMma) {
        // ---- products by the first of these warps, requests by the second
        fewer_registers<kMmaRegs>();
        int pieces = 0, stage = 0, asked = 0;
        uint32_t free_parity = 1; // (of the use before)
        int *lines = reinterpret_cast<int *>(gbase + z.tables); // [8 tiles][4 groups][keys', values'] (-1: no row sees any of the group)
        for (int slot = 0; s_piece[slot].n > 0; slot ^= 1, pieces++) {
            const int n = s_piece[slot].n;
            if (warp == kTileMma) {
                const tile_mma m{bars, base + z.q, q_part, base + z.k, k_stage, base + z.v, v_stage, tmem, a.D / 16, a.Dv, dead};
                if (a.D == 128) tile_products<PARTS, 8>(m, n, ph0, ph1, pieces);
                else if (a.D == 64) tile_products<PARTS, 4>(m, n, ph0, ph1, pieces);
                else tile_products<PARTS, 0>(m, n, ph0, ph1, pieces);
            } else if (warp == kTileAsk) {
                const item &it = s_piece[slot].it;
                const int tile = s_piece[slot].tile, head = s_piece[slot].head;
                for (int k = 0; k < n; k++) {
                    if ((k & 7) == 0) { // eight tiles at a time, a lane a group, are looked up
                        const int t = tile + k + (lane >> 2), first = (t < it.kt ? t : it.w0 + t - it.kt) * kTileKeys + 16 * (lane & 3);
                        int2 line = make_int2(-1, -1);
                        float2 scale = make_float2(0.f, 0.f);
                        if (k + (lane >> 2) < n && (t < it.kt ? first < it.n_keep : first + 15 >= it.lo && first <= it.i1)) {
                            const int pg = first / a.B, grp = (first - pg * a.B) / kKv8Group;
                            const int64_t rec = (int64_t)a.tables[it.s * a.table_ld + pg] * a.G + head;
                            const float *sc = reinterpret_cast<const float *>(a.cache + rec * a.record + a.B * (a.D + a.Dv)) + grp;
                            line.x = (int)(rec * (a.record / 128)) + grp * (a.D / 8);
                            line.y = (int)(rec * (a.record / 128)) + a.B / kKv8Group * (a.D / 8) + grp * (a.Dv / 8);
                            scale = make_float2(sc[0], sc[a.B / kKv8Group]);
                        }
                        *reinterpret_cast<int2 *>(lines + 2 * lane) = line;
                        scales[(4 * (ph0 + ph1 + k) + lane) & 63] = scale;
                        __syncwarp();
                    }
                    if (asked >= kAhead && !wait_long(bars + T_RAW_FREE + 8 * stage, free_parity, dead)) break;
                    if (lane == 0) {
                        const uint32_t to = base + z.raw + stage * z.raw_stage, bar = bars + T_RAW + 8 * stage;
                        const int4 *l4 = reinterpret_cast<const int4 *>(lines + 8 * (k & 7));
                        const int4 la = l4[0], lb = l4[1];
                        const int kl[4] = {la.x, la.z, lb.x, lb.z}, vl[4] = {la.y, la.w, lb.y, lb.w};
                        int groups = 0;
#pragma unroll
                        for (int g = 0; g < 4; g++) groups += kl[g] >= 0;
                        mbar_expect_tx(bar, 16 * (a.D + a.Dv) * groups); // (a tile that no row sees anything of is none)
#pragma unroll
                        for (int g = 0; g < 4; g++)
                            if (kl[g] >= 0) {
                                tma_load_2d(to + g * 1024 * D64, &maps.k, 0, kl[g], bar);
                                tma_load_2d(to + 4096 * D64 + g * 1024 * V64, &maps.v, 0, vl[g], bar);
                            }
                    }
                    __syncwarp();
                    asked++;
                    if (++stage == kAhead) stage = 0, free_parity ^= 1;
                }
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
            // ---- queries: a warp's 16 rows, eight at a time, four lanes a row
            float *srow = st + 6 * kTileRows;
#pragma unroll 1
            for (int r = 16 * warp + (lane >> 2), e = 0; e < 2; e++, r += 8) {
                const int row = it.row0 + r, tq = row / hpg, h = x.head * hpg + (row - tq * hpg), part = lane & 3;
                const float *src = a.q + ((it.t0 + tq) * a.H + h) * a.D + 4 * part;
                float4 v[8];
                float big = 0.f;
                bool odd = false;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < it.rows && 16 * u + 4 * part < a.D) {
                        if (a.vec_q) v[u] = *reinterpret_cast<const float4 *>(src + 16 * u);
                        else v[u] = make_float4(src[16 * u], src[16 * u + 1], src[16 * u + 2], src[16 * u + 3]);
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const float most = fmaxf(fmaxf(fabsf(v[u].x), fabsf(v[u].y)), fmaxf(fabsf(v[u].z), fabsf(v[u].w)));
                    big = fmaxf(big, most);
                    odd |= v[u].x != v[u].x || v[u].y != v[u].y || v[u].z != v[u].z || v[u].w != v[u].w;
                }
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                odd = ((__ballot_sync(0xffffffffu, odd) >> (lane & 28)) & 15) != 0;
                odd |= big == INFINITY;
                const float f = odd ? 0.f : power_for(big, 10);
                if (part == 0) srow[r] = odd ? NAN : kLog2e / f; // what is not finite spoils its own row
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    if (16 * u >= 64 * D64) break;
                    const float y[4] = {odd ? 0.f : v[u].x * f, odd ? 0.f : v[u].y * f, odd ? 0.f : v[u].z * f, odd ? 0.f : v[u].w * f};
                    uint2 p = make_uint2(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]));
                    const uint32_t at = base + z.q + (u >> 2) * (kTileRows * 128) + r * 128 + (((2 * (u & 3) + (part >> 1)) ^ (r & 7)) << 4) + (part & 1) * 8;
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(p.x), "r"(p.y) : "memory");
                    const float2 b0 = half2_floats(p.x), b1 = half2_floats(p.y);
                    p = make_uint2(half2_bits(y[0] - b0.x, y[1] - b0.y), half2_bits(y[2] - b1.x, y[3] - b1.y));
                    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + q_part), "r"(p.x), "r"(p.y) : "memory");
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + T_Q_FULL);
            warp_meet();
            bar_sync(3, 32 * kSoftWarps); // the rows' factors
            if (tid == 32 * kSoftWarps - 1) { // while the first scores are under way: the piece behind this one
                piece y = x;
                const unsigned at = y.u + kTileBegin + y.tile + y.n;
                y.n = 0;
                if (at < s_end) tile_piece_from(a, y, at, s_end);
                s_piece[slot ^ 1] = y;
            }
            __syncwarp();
            // ---- weights: group grp takes the tiles k = grp, grp + 2, ...; a thread has a row
            const int grp = warp >> 2, r = 32 * (warp & 3) + lane;
            const int i = r < it.rows ? it.p0 + (it.row0 + r) / hpg : -1, lo = a.window > 0 ? (int)max((int64_t)0, i - a.window + 1) : 0;
            const int lo_last = a.window > 0 ? (int)max((int64_t)0, it.i1 - a.window + 1) : 0, whole_from = max(it.lo, lo_last), ph = grp ? ph1 : ph0;
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = tmem + lanes + kScoreCol + grp * 64, tw = tmem + lanes + kWeightCol + grp * 64, to = tmem + lanes + kOutCol + grp * a.Dv;
            const float rowf = srow[r], cap = a.cap * kLog2e, inv_cap = a.cap > 0.f ? kLn2 / a.cap : 0.f;
            float m = kNone, l = 0.f, d = 0.f; // weights are relative to 2^m, their products with values' scales to 2^(m - d)
            bool lost = false;
            const bool whole_item = n == it.n;
            const int row = it.row0 + r, tq = row / hpg, h = x.head * hpg + (row - tq * hpg);
            const int64_t t_row = it.t0 + tq;
            const int64_t part_row = ((int64_t)blockIdx.x * 2 + (tile == 0)) * kTileRows + r;
            float *part = whole_item ? nullptr : a.part + part_row * a.Dv;
            float M = kNone, L = 0.f; // of the chains so far
            int k = grp;
            for (int upto = PARTS == 1 ? n : min(n, kChain);; upto = min(n, upto + kChain)) {
                for (; k < upto; k += 2) {
                    const int t = tile + k, j0 = first_of(t);
                    const bool kept = t < it.kt, whole = kept ? j0 + kTileKeys <= it.n_keep : j0 >= whole_from && j0 + kTileKeys - 1 <= it.i0;
                    if (!wait_long(bars + T_S_FULL + 8 * grp, (ph + (k >> 1)) & 1, dead)) lost = true;
                    tc_fence_after();
                    const float4 *sc4 = reinterpret_cast<const float4 *>(scales + ((ph0 + ph1 + k) & 15) * 4);
                    const float4 sa = sc4[0], sb = sc4[1];
                    const float ks[4] = {sa.x, sa.z, sb.x, sb.z}, vs[4] = {sa.y, sa.w, sb.y, sb.w};
                    float y[4][16], f[4], top[4];
                    tmem_load32(ts, reinterpret_cast<uint32_t *>(y[0]));
                    tmem_load32(ts + 32, reinterpret_cast<uint32_t *>(y[2]));
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + T_S_FREE + 8 * grp);
                    // a score is its product times f; where something is in between, it is taken into the scores and f is one
#pragma unroll
                    for (int g = 0; g < 4; g++) f[g] = rowf * ks[g];
                    if (a.cap > 0.f || !whole) {
#pragma unroll
                        for (int g = 0; g < 4; g++) {
#pragma unroll
                            for (int c = 0; c < 16; c++) y[g][c] *= f[g];
                            f[g] = 1.f;
                            if (a.cap > 0.f) tile_attn::soft_cap16(y[g], cap, inv_cap);
                        }
                        if (!whole) { // positions [from, upto) of the tile, and of those below `from` the kept ones
                            const int upto = i < 0 ? 0 : (kept ? it.n_keep : i + 1) - j0, from = (kept ? 0 : lo) - j0, keep = kept ? 0 : (int)min(a.keep, (int64_t)lo) - j0, low = kept ? 0 : it.lo - j0;
#pragma unroll
                            for (int g = 0; g < 4; g++)
#pragma unroll
                                for (int c = 0; c < 16; c++) {
                                    const int j = 16 * g + c;
                                    if (!(j < upto && j >= low && (j >= from || j < keep))) y[g][c] = -INFINITY;
                                }
                        }
                    }
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        float big[2] = {y[g][0], y[g][1]};
#pragma unroll
                        for (int c = 2; c < 16; c++) big[c & 1] = fmaxf(big[c & 1], y[g][c]);
                        top[g] = fmaxf(big[0], big[1]) * f[g];
                    }
                    const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m2 = mx > m + 8.f ? ceilf(mx) : m;
                    float pm = -INFINITY, over = 1.f; // the largest product of a weight and a scale, in powers of two: only what the row sees counts
#pragma unroll
                    for (int g = 0; g < 4; g++) pm = fmaxf(pm, (top[g] - m2) + (float)scale_exponent(vs[g]));
                    const float d2 = d + (m2 - m);
                    if (m2 != m || pm + d2 > (float)kMostWeight) {
                        l *= exp2f(m - m2), m = m2;
                        d = fminf(d2, (float)kNewWeight - ceilf(pm));
                        over = exp2f(d - d2);
                    }
                    // (from here on the weights that this tile's go over have been read, and the output that they went into is there: tile k - 2's products)
                    // Rows that grew have parted the lanes; the wait's vote joins them, as loads and stores of tensor memory ask for
                    if (k >= 2) {
                        if (!wait_long(bars + T_V_FREE + 8 * grp, (ph + (k >> 1) - 1) & 1, dead)) lost = true;
                    } else {
                        warp_meet();
                    }
                    tc_fence_after();
                    if ((PARTS == 1 ? k : k % kChain) >= 2 && __any_sync(0xffffffffu, over != 1.f)) {
#pragma unroll 1
                        for (int c = 0; c < a.Dv; c += 16) {
                            uint32_t o[16];
                            tmem_load16(to + c, o);
#pragma unroll
                            for (int u = 0; u < 16; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * over);
                            tmem_store16(to + c, o);
                        }
                    }
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        f32x2 sum[2] = {0, 0};
                        const float rel = PARTS == 1 ? 0.f : scale_times(vs[g], (int)d);
                        // one part: the scale goes with the exponent, and out of the sum again (2^-60: below every 16-bit number, and the weight of the sum still there)
                        const float power = PARTS == 1 ? fmaxf(lg2_approx(vs[g]) + d, -60.f) : 0.f, shift = power - m;
                        uint32_t hi[8], lo2[8];
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            const float2 t2 = unpack2(fma2(pack2(y[g][2 * c], y[g][2 * c + 1]), pack2(f[g], f[g]), pack2(shift, shift)));
                            f32x2 w = pack2(ex2_approx(t2.x), ex2_approx(t2.y));
                            sum[c & 1] = add2(sum[c & 1], w);
                            if (PARTS == 2) w = mul2(w, pack2(rel, rel));
                            const float2 wv = unpack2(w);
                            hi[c] = half2_bits(wv.x, wv.y);
                            if (PARTS == 2) {
                                const float2 back = half2_floats(hi[c]);
                                lo2[c] = half2_bits(wv.x - back.x, wv.y - back.y);
                            }
                        }
                        tmem_store8(tw + 8 * g, hi);
                        if (PARTS == 2) tmem_store8(tw + 32 + 8 * g, lo2);
                        const float2 s2 = unpack2(add2(sum[0], sum[1]));
                        l = PARTS == 1 ? fmaf(s2.x + s2.y, ex2_approx(-power), l) : l + (s2.x + s2.y);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + T_P_FULL + 8 * grp);
                    if (lost) break;
                }
                // ---- both groups' sums meet, and those of the chains before: these lie where the result goes
                const bool last = PARTS == 1 || upto == n, more = PARTS == 2 && upto > kChain;
                if (last) wait_long(bars + T_DONE, pieces & 1, dead);
                else wait_long(bars + T_V_FREE + 8 * grp, (ph + ((k - 2) >> 1)) & 1, dead);
                tc_fence_after();
                bar_sync(3, 32 * kSoftWarps); // the tables are no longer read
                st[3 * grp * kTileRows + r] = l, st[(3 * grp + 1) * kTileRows + r] = m, st[(3 * grp + 2) * kTileRows + r] = d;
                bar_sync(3, 32 * kSoftWarps);
                const float before = M, m0 = st[kTileRows + r], m1 = n > 1 ? st[4 * kTileRows + r] : kNone;
                M = fmaxf(fmaxf(m0, m1), before);
                const float g0 = exp2f(m0 - M), g1 = n > 1 ? exp2f(m1 - M) : 0.f, gb = more ? exp2f(before - M) : 0.f;
                L = fmaf(st[r], g0, n > 1 ? st[3 * kTileRows + r] * g1 : 0.f) + (more ? L * gb : 0.f);
                const float f0 = exp2f((m0 - M) - st[2 * kTileRows + r]), f1 = n > 1 ? exp2f((m1 - M) - st[5 * kTileRows + r]) : 0.f;
                const row_end end(a, r < it.rows ? h : 0, M, L);
#pragma unroll 1
                for (int cb = grp; cb < a.Dv / 16; cb += 2) {
                    const int64_t at = (int64_t)h * a.Dv + 16 * cb;
                    float4 gt[4];
                    const float *gate = a.gate + t_row * a.ldg + at;
                    if (last && whole_item && a.gate && r < it.rows)
#pragma unroll
                        for (int u = 0; u < 4; u++) gt[u] = a.vec_gate ? *reinterpret_cast<const float4 *>(gate + 4 * u) : make_float4(gate[4 * u], gate[4 * u + 1], gate[4 * u + 2], gate[4 * u + 3]);
                    uint32_t o0[16], o1[16];
                    warp_meet(); // lanes whose rows end ahead of the others go on alone, here and in the round before
                    tmem_load16(tmem + lanes + kOutCol + 16 * cb, o0);
                    if (n > 1) tmem_load16(tmem + lanes + kOutCol + a.Dv + 16 * cb, o1);
                    if (r >= it.rows) continue;
                    E *out = reinterpret_cast<E *>(a.out) + t_row * a.H * a.Dv + at;
                    float v[16];
#pragma unroll
                    for (int u = 0; u < 16; u++) {
                        v[u] = __uint_as_float(o0[u]) * f0;
                        if (n > 1) v[u] = fmaf(__uint_as_float(o1[u]), f1, v[u]);
                    }
                    if (more) {
                        const float *b = whole_item ? reinterpret_cast<const float *>(out) : part + 16 * cb;
                        if (!whole_item || a.vec_out) {
#pragma unroll
                            for (int u = 0; u < 16; u += 4) {
                                const float4 b4 = *reinterpret_cast<const float4 *>(b + u);
                                v[u] = fmaf(b4.x, gb, v[u]), v[u + 1] = fmaf(b4.y, gb, v[u + 1]), v[u + 2] = fmaf(b4.z, gb, v[u + 2]), v[u + 3] = fmaf(b4.w, gb, v[u + 3]);
                            }
                        } else {
#pragma unroll
                            for (int u = 0; u < 16; u++) v[u] = fmaf(b[u], gb, v[u]);
                        }
                    }
                    if (!whole_item) {
#pragma unroll
                        for (int u = 0; u < 16; u += 4) *reinterpret_cast<float4 *>(part + 16 * cb + u) = make_float4(v[u], v[u + 1], v[u + 2], v[u + 3]);
                        continue;
                    }
                    if (last) {
#pragma unroll
                        for (int u = 0; u < 16; u++) v[u] *= end.f;
                        if (a.gate) {
#pragma unroll
                            for (int u = 0; u < 4; u++) {
                                const float2 p = unpack2(tile_attn::sigmoid_fast2(pack2(gt[u].x, gt[u].y))), s = unpack2(tile_attn::sigmoid_fast2(pack2(gt[u].z, gt[u].w)));
                                v[4 * u] *= p.x, v[4 * u + 1] *= p.y, v[4 * u + 2] *= s.x, v[4 * u + 3] *= s.y;
                            }
                        }
                    }
                    if (!a.vec_out) {
#pragma unroll
                        for (int u = 0; u < 16; u++) out[u] = from_f32<E>(v[u]);
                    } else if (PARTS == 1) {
#pragma unroll
                        for (int u = 0; u < 16; u += 8)
                            *reinterpret_cast<uint4 *>(out + u) = make_uint4(pack_bf16x2(v[u], v[u + 1]), pack_bf16x2(v[u + 2], v[u + 3]), pack_bf16x2(v[u + 4], v[u + 5]), pack_bf16x2(v[u + 6], v[u + 7]));
                    } else {
#pragma unroll
                        for (int u = 0; u < 16; u += 4) *reinterpret_cast<float4 *>(out + u) = make_float4(v[u], v[u + 1], v[u + 2], v[u + 3]);
                    }
                }
                if (last) break;
                l = 0.f, m = kNone, d = 0.f;
                tc_fence_before(); // the next chain begins when the other group has read this one's too
                warp_meet();
                bar_sync(3, 32 * kSoftWarps);
                tc_fence_after();
            }
            if (!whole_item && grp == 0 && r < it.rows) a.part_ml[part_row] = make_float2(M, L);
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
    const int64_t places = list_items(a, T, max_new, kTileRows), items = (T * hpg + kTileRows - 1) / kTileRows * a.G;
    GGB_CHECK_ARG(places * a.G * ((a.positions + a.keep) / kTileKeys + kTileBegin + 2) < (1ll << 31), "kv8_attn: too many sequences, tokens, heads and positions for a launch");
    a.entries = (int)places;
    // (bf16 results, 16 heads over 4 of 128, 4,096 tokens, 3.5 items an SM: with a window of 1,024 whole 133 us, cut 168; without one, from position 0 on, whole ones are uneven there, 254 and 236, and
    // no longer with 10,240 tokens, 1,150 and 1,174.  In fp32, where what a chain leaves goes to memory and back, 2,560 tokens 177 and 153, 4,096 tokens 365 and 333, 16,384 4,087 and 4,279)
    if (items >= (PARTS == 1 ? 3 : 8) * ggb_sm_count()) a.part = nullptr;
    const size_t smem = std::max((size_t)tile_sizes(a.D, a.Dv).smem, kOneCtaSmem);
    auto kfn = kv8_tile_kernel<CODE, PARTS>;
    const int rc = ggb_allow_smem(kfn, smem);
    if (rc) return rc;
    cudaFuncAttributes built{}; // what the split takes has to be there, or it would be waited for without end
    GGB_CUDA(cudaFuncGetAttributes(&built, kfn));
    const int registers = built.numRegs;
    GGB_CHECK_ARG(registers * (kTileThreads / 128) >= kSoftWarps / 4 * kSoftRegs + kCodeWarps / 4 * kCodeRegs + kMmaRegs, "kv8_attn: built with %d registers a thread", registers);
    const unsigned ctas = (unsigned)(a.part ? std::min(kTileCtas, ggb_sm_count()) : ggb_sm_count());
    line_maps maps;
    const int rc2 = make_line_maps(a, maps);
    if (rc2) return rc2;
    GGB_CUDA(ggb_launch_early(kfn, ggb_cluster{1, 1, 1}, dim3(ctas), dim3(kTileThreads), smem, a, maps));
    GGB_LAUNCH_CHECK();
    *joins = a.part ? ctas : 0;
    return GGB_OK;
}

} // namespace kv8
