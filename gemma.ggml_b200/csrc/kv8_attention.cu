// kv8_attention.cu — grouped-query soft-max attention of a batch of sequences over the 8-bit paged cache (kv8.cuh).
//
// Steps of a token or some drafted ones of every sequence, few rows of queries a key head (portions of prompts: kv8_tile.cuh):
//
// What has to be read are the codes, a byte a number, and a warp turns each into what its MMAs take once for all query heads of the key head.  Keys, or value coordinates, are
// the 16 rows of an MMA and eight rows of queries its columns, so no row is empty for the usual four to eight query heads of a key head:
//
//   codes    copied by TMA, a group of 16 positions at a time, a stage or more ahead for every warp on its own
//   scores   S^T [16 keys][8 rows] = K Q^T.  int8 codes: m16n8k32 on integers, a row of queries as three (bf16 results) or four digits to the base 128 whose products are put
//            together exactly; e4m3: m16n8k16 on fp16 numbers.  A lane's piece of a key is 16 consecutive codes: the order of a sum's terms is free, and queries lie in
//            shared memory in the same one
//   weights  in the registers that the scores are in: 2^(s - m); a kept maximum is followed only when a score exceeds it by 8 (a vote, no shuffles otherwise)
//   output   O^T [16 coordinates][8 rows] += V^T P^T by m16n8k16 on fp16 numbers, weights turned by movmatrix, values by byte permutes of the rows of two neighbouring keys
//
// PARTS: fp16 numbers that stand for an fp32 weight.  2 keep 22 bits of it (results in fp32); 1 keeps 11 (results in bf16,
// which keep 8).  Queries are two (or digits) for either: what is cut off them a score multiplies, by 40 where two scores of 40 are weighed against one another, and 11 bits then
// left results 2 % off.  A row of queries is multiplied by a power of two that brings its largest number to [2^10, 2^11), so nothing of weight gets too small for fp16; so are a row's
// weights times their groups' value scales (kv8.cuh).
//
// Work: items (sequence, R rows, key head), cut into tiles of as many positions as the CTA's warps take at once; all tiles of a call in one row, dealt evenly to the CTAs, so
// ragged batches and single long sequences fill the chip alike.  A CTA that has only a piece of an item leaves it in the workspace (the first or the last
// of what it was dealt: two places), and kv8_join_kernel adds an item's pieces up in order.
//
// What bounds it: from some ten megabytes of codes on the bytes (32 sequences of 8,000 positions, 32 heads over 8 of 128: 63.3 us, 78 % of what a copy moves; of 32,000
// 203 us, 97 %).  Below that what a launch has to do one after the other: look up what was dealt (1.3 us), queries and the first codes (2.5), the warps' sums (1.1), the join (3.5).
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "kv8_tile.cuh"

namespace {

using namespace kv8;

constexpr int kMaxRows = 32, kMaxCtas = 512;
constexpr int kBegin = 2; // units that an item costs to begin: the queries, the warps' sums

inline size_t part_bytes(int Dv) { return (size_t)kMaxCtas * (2 * kMaxRows * (size_t)(Dv + 2) * 4 + 2 * sizeof(int4)); }

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same on sums that begin with it
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma16832_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// P: numbers of a key and of a value, at most: 64, 128 or 256
template <int CODE, int P, int NT, int PARTS> struct step_sizes {
    static constexpr int R = 8 * NT, KS = P / 16; // blocks of 16 value coordinates
    // groups of 16 keys that a warp takes at once: two where the sums leave registers for them, which also gives the warp independent work (32 sequences of 8,000 positions, 128
    // numbers: 63.6 us, one 66.8; with two more drafted tokens each 97 and 108); with heads of 256, whose sums fill the registers, one (16 over 2: 42.7 us, two 46.1).  Two CTAs of six warps
    // an SM, or one of eight
    static constexpr int min_ctas = P * NT <= 128 ? 2 : 1, W = min_ctas == 2 ? 6 : 8, U = P < 256 && P * NT <= 256 ? 2 : 1, threads = 32 * W, tile = 16 * W * U;
    // queries: int8 digits for steps of 32 numbers, or fp16 parts for steps of 16
    static constexpr bool digits = CODE == GGB_KV8_INT8;
    static constexpr int Q = digits ? PARTS + 2 : kQueryParts, QS = digits ? P / 32 : P / 16;
    static constexpr int half = 16 * P, stage = 2 * half; // a group's keys, then their values; S of them on their way or in use
    // the warps' sums of a piece meet beside the stages, on which the next piece's codes are arriving (16 rows of 256: no room, over them)
    static constexpr bool beside = P == 64 || (P == 128 && NT > 1) || (P == 256 && NT == 1);
    static constexpr int S = P == 256 ? (NT == 1 ? 2 : 3) : P == 128 ? (NT == 1 ? 4 : NT == 2 ? 4 : 2) : NT == 4 ? 7 : 4;
    static constexpr size_t q_bytes = (size_t)Q * NT * QS * 256, ring_bytes = (size_t)W * S * stage, red_bytes = (size_t)W * R * P * 4;
    static_assert((beside || red_bytes <= ring_bytes) && stage % 1024 == 0, "shared memory");
    static constexpr size_t smem = 1024 + q_bytes + ring_bytes + (beside ? red_bytes : 0) + (size_t)W * (R * 12 + 768) + R * 8 + 64;
    static_assert((smem + 2048) * min_ctas <= 227 * 1024, "shared memory of an SM");
};
// where the pair of coordinates 2 i, 2 i + 1 of the 16 (P = 64: 8) numbers of lane group g lies in its row of the reduction, in pairs: rows of a warp's stores in different banks
template <int P> __device__ __forceinline__ int red_at(int g, int i, int c) {
    constexpr int W = P == 64 ? 4 : 8; // pairs of a lane group (P = 256: of either half)
    return W * g + (i ^ ((((g >> 1) & 1) | (c << 1)) & (W - 1)));
}

// a row of queries to shared memory, by a warp: fp16 parts or int8 digits in the order of the lanes' pieces of a key, and what turns a product into a score (NaN where a query
// is not finite: the row's own matter)
template <int CODE, int P, int NT, int PARTS> __device__ __forceinline__ void stage_row(const attn_args &a, const float *src, bool real, int r, uint2 *sq, float *srow) {
    using Z = step_sizes<CODE, P, NT, PARTS>;
    const int lane = threadIdx.x & 31;
    float4 x[(P + 127) / 128];
    float m = 0.f;
    bool odd = false;
#pragma unroll
    for (int k = 0; k < (P + 127) / 128; k++) {
        const int d = 4 * lane + 128 * k;
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (real && d < a.D) {
            if (a.vec_q) x[k] = *reinterpret_cast<const float4 *>(src + d);
            else x[k] = make_float4(src[d], src[d + 1], src[d + 2], src[d + 3]);
        }
        const float t = fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
        m = fmaxf(m, t);
        odd |= t == INFINITY || x[k].x != x[k].x || x[k].y != x[k].y || x[k].z != x[k].z || x[k].w != x[k].w;
    }
    m = warp_max_f32(m);
    odd = __any_sync(0xffffffffu, odd);
    const float f = power_for(odd ? 0.f : m, Z::digits ? 7 * Z::Q - 2 : 10); // digits: the largest number below 2^(7 Q - 1), its first digit up to 64
    if (lane == 0) srow[r] = odd ? NAN : (a.cap > 0.f ? 1.f : kLog2e) / f;
#pragma unroll
    for (int k = 0; k < (P + 127) / 128; k++) {
        const int d = 4 * lane + 128 * k;
        if (d >= P) break;
        const float y[4] = {x[k].x * f, x[k].y * f, x[k].z * f, x[k].w * f};
        const int t = r / 8, to = (r % 8) * 4 + (d % 64) / 16;
        if (Z::digits) {
            int n[4];
            uint32_t *words = reinterpret_cast<uint32_t *>(sq + (t * Z::QS + 2 * (d / 64) + (d % 16) / 8) * 32 + to) + ((d >> 2) & 1);
#pragma unroll
            for (int e = 0; e < 4; e++) n[e] = odd ? 0 : __float2int_rn(y[e]);
#pragma unroll
            for (int part = 0; part < Z::Q; part++) { // the last digit first
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int digit = part == Z::Q - 1 ? n[e] : ((n[e] + 64) & 127) - 64;
                    word |= (uint32_t)(digit & 255) << (8 * e);
                    n[e] = (n[e] - digit) >> 7;
                }
                words[part * NT * Z::QS * 64] = word;
            }
        } else {
            uint2 p = make_uint2(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]));
            const int step = 4 * (d / 64) + (d % 16) / 4;
            sq[(t * Z::QS + step) * 32 + to] = p;
            const float2 b0 = half2_floats(p.x), b1 = half2_floats(p.y);
            p = make_uint2(half2_bits(y[0] - b0.x, y[1] - b0.y), half2_bits(y[2] - b1.x, y[3] - b1.y));
            sq[((NT + t) * Z::QS + step) * 32 + to] = p;
        }
    }
}

template <int CODE, int P, int NT, int PARTS>
__global__ void __launch_bounds__(step_sizes<CODE, P, NT, PARTS>::threads, step_sizes<CODE, P, NT, PARTS>::min_ctas) kv8_step_kernel(const __grid_constant__ attn_args a, const __grid_constant__ line_maps maps) {
    using Z = step_sizes<CODE, P, NT, PARTS>;
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    constexpr int R = Z::R, KS = Z::KS, NB = P / 64, VW = P == 64 ? 2 : 4, VC = P == 256 ? 2 : 1; // words of a lane's piece of a value row, pieces
    extern __shared__ __align__(16) uint8_t ks_smem[];
    __shared__ unsigned s_scan[Z::W], s_end, s_all;
    __shared__ int s_dead;
    __shared__ piece s_piece[3]; // one whose sums are being taken, the next one (asked for meanwhile), the one behind that
    __shared__ __align__(8) uint64_t s_bars[Z::W * Z::S];
    step_wait();
    volatile int *dead = &s_dead;
    const uint32_t raw = smem_u32(ks_smem), ring0 = (raw + 1023u) & ~1023u;
    uint8_t *base_at = ks_smem + (ring0 - raw);
    uint2 *sq = reinterpret_cast<uint2 *>(base_at + Z::ring_bytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, c4 = lane & 3;
    int2 *lines = reinterpret_cast<int2 *>(base_at + Z::ring_bytes + Z::q_bytes) + warp * 96; // [32]: lines of the tiles' keys and values
    float2 *scales = reinterpret_cast<float2 *>(lines + 32);                                  // [64]
    float *sm = reinterpret_cast<float *>(base_at + Z::ring_bytes + Z::q_bytes + Z::W * 768), *sl = sm + Z::W * R, *sd = sl + Z::W * R, *srow = sd + Z::W * R;
    int *spos = reinterpret_cast<int *>(srow + R);
    float2 *red = reinterpret_cast<float2 *>(base_at + (Z::beside ? Z::ring_bytes + Z::q_bytes + Z::W * (768 + R * 12) + R * 8 + 64 : 0));
    const uint32_t ring = ring0 + warp * Z::S * Z::stage, bars = smem_u32(s_bars) + 8 * warp * Z::S;
    if (lane == 0)
        for (int k = 0; k < Z::S; k++) mbar_init(bars + 8 * k, 1);
    if (tid == 0) s_dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

    // ---- what this CTA has been dealt
    if (a.part) {
        const int each = (a.entries + Z::threads - 1) / Z::threads, e0 = min(a.entries, tid * each), e1 = min(a.entries, e0 + each);
        unsigned mine = 0, U = 0, base = 0;
        piece x;
        if (e0 < e1)
            for (to_entry<R, Z::tile>(a, x, e0);; next_entry<R, Z::tile>(a, x)) {
                if (x.it.n) mine += (x.it.n + kBegin) * a.G;
                if (x.entry + 1 == e1) break;
            }
        unsigned run = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, run, off);
            if (lane >= off) run += y;
        }
        if (lane == 31) s_scan[warp] = run;
        if (tid == 0) a.desc[2 * blockIdx.x] = make_int4(-1, 0, 0, 0), s_piece[0].n = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < Z::W; w++) {
            if (w < warp) base += s_scan[w];
            U += s_scan[w];
        }
        const deal d(U, gridDim.x);
        const unsigned u = d.first(blockIdx.x), end = d.first(blockIdx.x + 1);
        base += run - mine;
        if (u < end && u >= base && u < base + mine) {
            if (each > 1)
                for (to_entry<R, Z::tile>(a, x, e0);; next_entry<R, Z::tile>(a, x)) {
                    const unsigned n = x.it.n ? (x.it.n + kBegin) * a.G : 0;
                    if (u < base + n) break;
                    base += n;
                }
            x.head = (int)((u - base) / (unsigned)(x.it.n + kBegin)), x.u = base + x.head * (x.it.n + kBegin);
            piece_from<R, Z::tile, kBegin>(a, x, u, end);
            s_piece[0] = x, s_end = end, s_all = U;
        }
    } else if (tid == 0) {
        piece x;
        to_entry<R, Z::tile>(a, x, blockIdx.x / a.G);
        x.head = blockIdx.x - x.entry * a.G, x.tile = 0, x.u = 0;
        x.n = x.it.n;
        s_piece[0] = x, s_end = 0, s_all = 0;
    }
    __syncthreads();
    const int hpg = a.H / a.G;
    auto write_following = [&](int from, int to) { // one thread
        piece x = s_piece[from];
        const unsigned at = x.u + kBegin + x.tile + x.n;
        const bool more = x.n > 0 && at < s_end;
        x.n = 0;
        if (more) piece_from<R, Z::tile, kBegin>(a, x, at, s_end);
        s_piece[to] = x;
    };
    auto stage_queries = [&](const piece &x) {
        for (int r = warp; r < R; r += Z::W) {
            const int row = x.it.row0 + r, tq = row / hpg, h = x.head * hpg + (row - tq * hpg);
            stage_row<CODE, P, NT, PARTS>(a, a.q + ((x.it.t0 + tq) * a.H + h) * a.D, r < x.it.rows, r, sq, srow);
            if (lane == 0) spos[r] = r < x.it.rows ? x.it.p0 + tq : -1; // sees nothing
        }
    };
    auto fetch_queries = [&](const piece &x) { // to the cache, ahead of that
        for (int r = warp; r < x.it.rows; r += Z::W) {
            const int row = x.it.row0 + r, tq = row / hpg, h = x.head * hpg + (row - tq * hpg);
            if (4 * lane < a.D) asm volatile("prefetch.global.L1 [%0];" ::"l"(a.q + ((x.it.t0 + tq) * a.H + h) * a.D + 4 * lane));
        }
    };
    // where a lane's pieces lie in a stage (behind the end of a row: the row's first piece, which meets zeros of the queries or leaves by no coordinate)
    uint32_t k_at[2][NB], v_at[4][VC];
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int b = 0; b < NB; b++) {
            k_at[e][b] = in_box((g8 + 8 * e) * a.D + (64 * b + 16 * c4 < a.D ? 64 * b + 16 * c4 : 0));
            asm volatile("" : "+r"(k_at[e][b])); // computed once
        }
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
        for (int c = 0; c < VC; c++) {
            v_at[e][c] = Z::half + in_box((2 * c4 + (e & 1) + 8 * (e >> 1)) * a.Dv + (128 * c + 4 * VW * g8 < a.Dv ? 128 * c + 4 * VW * g8 : 0));
            asm volatile("" : "+r"(v_at[e][c]));
        }
    // stages are asked for and used in turn: `asked` and `used` groups so far; of the piece that is asked for, groups [ask_k, ask_n) are left
    int asked = 0, used = 0, ask_stage = 0, stage = 0, ask_slot = 0, ask_k = 0, ask_n = Z::U * s_piece[0].n;
    uint32_t parity = 0;
    // the first of this warp's positions in a tile
    auto first_of = [&](const item &it, int t) { return (t < it.kt ? t : it.w0 + t - it.kt) * Z::tile + 16 * Z::U * warp; };
    // Asks for whatever stages are free, for the piece in `slot` and the next one.  32 groups at a time, a lane each, are looked up: the lines of a group's keys (-1: no row
    // sees any of it) and values; the scales of both (-1, too) are on their way to registers until keep_scale()
    float2 scale = make_float2(0.f, 0.f);
    int scale_at = -1;
    auto keep_scale = [&] {
        if (scale_at >= 0) scales[scale_at] = scale;
        scale_at = -1;
        __syncwarp();
    };
    auto ask = [&](int slot, bool next) {
        while (asked - used < Z::S) {
            if (ask_k == ask_n) {
                const int then = slot == 2 ? 0 : slot + 1;
                if (!next || ask_slot != slot || s_piece[then].n == 0) break;
                ask_slot = then, ask_k = 0, ask_n = Z::U * s_piece[then].n;
            }
            if (*dead) break; // a wait has run out: no more requests
            if ((ask_k & 31) == 0) {
                keep_scale();
                scale = make_float2(-1.f, 0.f), scale_at = (asked + lane) & 63;
                const piece &x = s_piece[ask_slot];
                const int t = x.tile + (ask_k + lane) / Z::U, first = first_of(x.it, t) + 16 * ((ask_k + lane) % Z::U);
                int2 line = make_int2(-1, 0);
                if (ask_k + lane < ask_n && (t < x.it.kt ? first < x.it.n_keep : first + 15 >= x.it.lo && first <= x.it.i1)) {
                    const int pg = first / a.B, grp = (first - pg * a.B) / kKv8Group;
                    const int64_t rec = (int64_t)a.tables[x.it.s * a.table_ld + pg] * a.G + x.head;
                    const float *sc = reinterpret_cast<const float *>(a.cache + rec * a.record + a.B * (a.D + a.Dv)) + grp;
                    line.x = (int)(rec * (a.record / 128)) + grp * (a.D / 8);
                    line.y = (int)(rec * (a.record / 128)) + a.B / kKv8Group * (a.D / 8) + grp * (a.Dv / 8);
                    scale = make_float2(sc[0], sc[a.B / kKv8Group]);
                }
                lines[lane] = line;
                __syncwarp();
            }
            do {
                if (lane == 0) {
                    const int2 line = lines[ask_k & 31];
                    const uint32_t to = ring + ask_stage * Z::stage, bar = bars + 8 * ask_stage;
                    if (line.x >= 0) request(maps, to, to + Z::half, line.x, line.y, 16 * (a.D + a.Dv), bar);
                    else mbar_arrive(bar);
                }
                asked++, ask_k++;
                if (++ask_stage == Z::S) ask_stage = 0;
            } while (asked - used < Z::S && ask_k < ask_n && (ask_k & 31) != 0);
        }
    };
    if (s_piece[0].n > 0) {
        fetch_queries(s_piece[0]);
        ask(0, false); // (the piece behind it is not known yet)
        stage_queries(s_piece[0]);
    }
    if (tid == Z::threads - 1) write_following(0, 1);
    __syncthreads();
    for (int slot = 0; s_piece[slot].n > 0; slot = slot == 2 ? 0 : slot + 1) {
        // ---- a piece of an item: its tiles [tile, tile + n)
        const item &s_it = s_piece[slot].it;
        const int tile = s_piece[slot].tile, n = s_piece[slot].n;
        if (ask_slot != slot) ask_slot = slot, ask_k = 0, ask_n = Z::U * n; // (nothing of it has been asked for)
        // tiles [whole0, whole0 + wholes) of the window: every row sees all of this warp's positions
        constexpr int last_of = 16 * Z::U - 1;
        const int up = s_it.i0 - last_of - 16 * Z::U * warp, down = max(s_it.lo, a.window > 0 ? (int)max((int64_t)0, s_it.i1 - a.window + 1) : 0) - 16 * Z::U * warp;
        const int whole0 = s_it.kt + max(0, (down + Z::tile - 1) / Z::tile - s_it.w0), wholes = up < 0 ? 0 : max(0, s_it.kt + up / Z::tile - s_it.w0 - whole0 + 1);

        float rowf[NT][2], m[NT][2], l[NT][2], o[KS][NT][4];
        int lift[NT][2]; // products of weights and scales are taken times 2^lift
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) rowf[t][e] = srow[8 * t + 2 * c4 + e], m[t][e] = kNone, l[t][e] = 0.f, lift[t][e] = 0;
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[i][t][e] = 0.f;

        for (int k = 0;; k++) {
            ask(slot, Z::beside);
            if (k == n) break;
            if (scale_at >= 0) keep_scale();
            bool here = true;
            uint32_t from[Z::U];
            float2 sc[Z::U];
#pragma unroll
            for (int u = 0; u < Z::U; u++) {
                here = here && mbar_wait_warp(bars + 8 * stage, parity, dead);
                from[u] = ring + stage * Z::stage, sc[u] = scales[(used + u) & 63];
                if (++stage == Z::S) stage = 0, parity ^= 1;
            }
            if (!here) break;
            // ---- scores
            float z[Z::U][NT][4];
#pragma unroll
            for (int u = 0; u < Z::U; u++) {
                uint4 kw[2][NB];
#pragma unroll
                for (int b = 0; b < NB; b++) kw[0][b] = lds_u4(from[u] + k_at[0][b]), kw[1][b] = lds_u4(from[u] + k_at[1][b]);
                if (Z::digits) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        int zi[Z::Q][4];
#pragma unroll
                        for (int b = 0; b < NB; b++)
#pragma unroll
                            for (int part = 0; part < Z::Q; part++) {
                                const uint2 y = sq[((part * NT + t) * Z::QS + 2 * b) * 32 + lane], x = sq[((part * NT + t) * Z::QS + 2 * b + 1) * 32 + lane];
                                if (b == 0) mma16832_first(zi[part], kw[0][b].x, kw[1][b].x, kw[0][b].y, kw[1][b].y, y.x, y.y);
                                else mma16832(zi[part], kw[0][b].x, kw[1][b].x, kw[0][b].y, kw[1][b].y, y.x, y.y);
                                mma16832(zi[part], kw[0][b].z, kw[1][b].z, kw[0][b].w, kw[1][b].w, x.x, x.y);
                            }
#pragma unroll
                        for (int e = 0; e < 4; e++) // whole numbers below 2^29 each
                            z[u][t][e] = Z::Q == 3 ? fmaf((float)(zi[2][e] * 128 + zi[1][e]), 128.f, (float)zi[0][e])
                                                   : fmaf((float)(zi[Z::Q - 1][e] * 128 + zi[Z::Q - 2][e]), 16384.f, (float)(zi[1][e] * 128 + zi[0][e]));
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint32_t w0[4] = {kw[0][b].x, kw[0][b].y, kw[0][b].z, kw[0][b].w}, w1[4] = {kw[1][b].x, kw[1][b].y, kw[1][b].z, kw[1][b].w};
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            uint32_t a0, a1, a2, a3;
                            halves_of<CODE>(w0[w], a0, a2);
                            halves_of<CODE>(w1[w], a1, a3);
#pragma unroll
                            for (int part = Z::Q - 1; part >= 0; part--)
#pragma unroll
                                for (int t = 0; t < NT; t++) {
                                    const uint2 y = sq[((part * NT + t) * Z::QS + 4 * b + w) * 32 + lane];
                                    if (b + w == 0 && part == Z::Q - 1) mma16816_first(z[u][t], a0, a1, a2, a3, y.x, y.y);
                                    else mma16816(z[u][t], a0, a1, a2, a3, y.x, y.y);
                                }
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) z[u][t][e] *= rowf[t][e & 1] * sc[u].x;
            }
            if (a.cap > 0.f) {
#pragma unroll
                for (int u = 0; u < Z::U; u++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) z[u][t][e] = a.cap * kLog2e * tanhf(z[u][t][e] / a.cap);
            }
            if ((unsigned)(tile + k - whole0) >= (unsigned)wholes) {
                const int now = tile + k, i1 = s_it.i1, lo = now < s_it.kt ? 0 : s_it.lo, hi = now < s_it.kt ? s_it.n_keep - 1 : i1;
#pragma unroll
                for (int u = 0; u < Z::U; u++) {
                    const int first = first_of(s_it, now) + 16 * u;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int j = first + g8 + 8 * (e >> 1), i = spos[8 * t + 2 * c4 + (e & 1)];
                            if (!(j >= lo && j <= hi && j <= i && (a.window <= 0 || i - j < a.window || j < a.keep))) z[u][t][e] = -INFINITY;
                        }
                    // behind the last position, and where nothing was asked for, there may be e4m3 codes that are no numbers, whose weight of zero would spoil a sum
                    if (CODE == GGB_KV8_E4M3 && (first + 15 > i1 || sc[u].x < 0.f)) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (first + 2 * c4 + (e & 1) + 8 * (e >> 1) > i1 || sc[u].x < 0.f)
#pragma unroll
                                for (int c = 0; c < VC; c++) {
                                    asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(from[u] + v_at[e][c]), "r"(0u) : "memory");
                                    if (VW == 4) asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(from[u] + v_at[e][c] + 8), "r"(0u) : "memory");
                                }
                        fence_async_smem();
                        __syncwarp();
                    }
                }
            }
            // ---- weights
            bool grow = false;
            int lv[Z::U];
#pragma unroll
            for (int u = 0; u < Z::U; u++) {
                lv[u] = scale_exponent(sc[u].y);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float most = m[t][e] + (float)min(8, kMostWeight - lv[u] - lift[t][e]);
                        grow |= z[u][t][e] > most || z[u][t][e + 2] > most;
                    }
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = kNone, p = -INFINITY;
#pragma unroll
                        for (int u = 0; u < Z::U; u++) x = fmaxf(x, fmaxf(z[u][t][e], z[u][t][e + 2]));
#pragma unroll
                        for (int off = 4; off <= 16; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                        x = fmaxf(ceilf(x), m[t][e]);
#pragma unroll
                        for (int u = 0; u < Z::U; u++) p = fmaxf(p, (fmaxf(z[u][t][e], z[u][t][e + 2]) - x) + (float)lv[u]);
#pragma unroll
                        for (int off = 4; off <= 16; off <<= 1) p = fmaxf(p, __shfl_xor_sync(0xffffffffu, p, off));
                        const float d2 = (float)lift[t][e] + (x - m[t][e]), d = fminf(d2, (float)kNewWeight - ceilf(p)), f = exp2f(d - d2);
                        l[t][e] *= exp2f(m[t][e] - x);
                        m[t][e] = x, lift[t][e] = (int)d;
#pragma unroll
                        for (int i = 0; i < KS; i++) o[i][t][e] *= f, o[i][t][e + 2] *= f;
                    }
            }
            uint32_t pb[Z::U][PARTS][NT][2];
#pragma unroll
            for (int u = 0; u < Z::U; u++) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float vrel[2] = {scale_times(sc[u].y, lift[t][0]), scale_times(sc[u].y, lift[t][1])};
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = ex2_approx(z[u][t][e] - m[t][e & 1]);
                        l[t][e & 1] += w[e];
                        w[e] *= vrel[e & 1];
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const uint32_t hi = half2_bits(w[2 * y], w[2 * y + 1]);
                        pb[u][0][t][y] = turn8x8(hi);
                        if (PARTS == 2) {
                            const float2 back = half2_floats(hi);
                            pb[u][PARTS - 1][t][y] = turn8x8(half2_bits(w[2 * y] - back.x, w[2 * y + 1] - back.y));
                        }
                    }
                }
            }
            // ---- output: coordinates 2 i, 2 i + 1 of a lane's piece are rows g8 and g8 + 8 of block i
#pragma unroll
            for (int u = 0; u < Z::U; u++)
#pragma unroll
                for (int c = 0; c < VC; c++) {
                    uint32_t vx[4][VW];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (VW == 4) {
                            const uint4 x = lds_u4(from[u] + v_at[e][c]);
                            vx[e][0] = x.x, vx[e][1] = x.y, vx[e][VW - 2] = x.z, vx[e][VW - 1] = x.w;
                        } else {
                            const uint2 x = lds_u2(from[u] + v_at[e][c]);
                            vx[e][0] = x.x, vx[e][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < VW; w++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const uint32_t sel = y ? 0x7362 : 0x5140;
                            uint32_t a0, a1, a2, a3;
                            halves_of<CODE>(__byte_perm(vx[0][w], vx[1][w], sel), a0, a1);
                            halves_of<CODE>(__byte_perm(vx[2][w], vx[3][w], sel), a2, a3);
#pragma unroll
                            for (int t = 0; t < NT; t++) {
                                if (PARTS == 1) {
                                    mma16816(o[c * 8 + 2 * w + y][t], a0, a1, a2, a3, pb[u][0][t][0], pb[u][0][t][1]);
                                } else { // tensor cores cut their sums short, always towards zero: not the long one, which is rounded to the nearest
                                    float z4[4];
                                    mma16816_first(z4, a0, a1, a2, a3, pb[u][PARTS - 1][t][0], pb[u][PARTS - 1][t][1]);
                                    mma16816(z4, a0, a1, a2, a3, pb[u][0][t][0], pb[u][0][t][1]);
#pragma unroll
                                    for (int e = 0; e < 4; e++) o[c * 8 + 2 * w + y][t][e] += z4[e];
                                }
                            }
                        }
                }
            used += Z::U;
            __syncwarp();
        }

        // ---- the warps' sums meet
        if (!Z::beside) __syncthreads(); // (every group that was asked for has been used)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = 8 * t + 2 * c4 + e;
#pragma unroll
                for (int off = 4; off <= 16; off <<= 1) l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], off);
                if (g8 == 0) sm[warp * R + r] = m[t][e], sl[warp * R + r] = l[t][e], sd[warp * R + r] = (float)lift[t][e];
                float2 *row = red + (warp * R + r) * (P / 2);
#pragma unroll
                for (int i = 0; i < KS; i++) row[64 * (i / 8) + red_at<P>(g8, i % 8, c4)] = make_float2(o[i][t][e], o[i][t][e + 2]);
            }
        __syncthreads();
        const bool whole_item = n == s_it.n;
        const int64_t part_row = ((int64_t)blockIdx.x * 2 + (tile == 0)) * R;
        constexpr int TPR = Z::threads / R; // threads a row
        const int r = tid / TPR;
        if (r < s_it.rows) {
            float M = -INFINITY, L = 0.f, f[Z::W];
#pragma unroll
            for (int w = 0; w < Z::W; w++) M = fmaxf(M, sm[w * R + r]);
#pragma unroll
            for (int w = 0; w < Z::W; w++) {
                f[w] = exp2f(sm[w * R + r] - M);
                L = fmaf(sl[w * R + r], f[w], L);
                f[w] = exp2f((sm[w * R + r] - M) - sd[w * R + r]);
            }
            const int row = s_it.row0 + r, tq = row / hpg, h = s_piece[slot].head * hpg + (row - tq * hpg);
            const int64_t t = s_it.t0 + tq;
            const row_end end(a, h, M, L);
            for (int pr = tid - r * TPR; pr < a.Dv / 2; pr += TPR) {
                constexpr int W = P == 64 ? 4 : 8;
                const int at = 64 * (pr / 64) + red_at<P>((pr % 64) / W, pr % W, (r % 8) / 2);
                float2 y = make_float2(0.f, 0.f);
#pragma unroll
                for (int w = 0; w < Z::W; w++) {
                    const float2 x = red[(w * R + r) * (P / 2) + at];
                    y.x = fmaf(x.x, f[w], y.x), y.y = fmaf(x.y, f[w], y.y);
                }
                if (whole_item) {
                    const int64_t to = (int64_t)h * a.Dv + 2 * pr;
                    E *out = reinterpret_cast<E *>(a.out) + t * a.H * a.Dv + to;
                    out[0] = from_f32<E>(gated(a, y.x * end.f, t, to)), out[1] = from_f32<E>(gated(a, y.y * end.f, t, to + 1));
                } else {
                    *reinterpret_cast<float2 *>(a.part + (part_row + r) * a.Dv + 2 * pr) = y;
                }
            }
            if (!whole_item && tid == r * TPR) a.part_ml[part_row + r] = make_float2(M, L);
        }
        if (!whole_item && tile + n < s_it.n && tid == 0) { // joined by the CTAs that have it but for the last, whose own last piece may be another one's
            const piece &x = s_piece[slot];
            const deal d(s_all, gridDim.x);
            a.desc[2 * blockIdx.x] = make_int4(x.it.s, x.it.rows, x.head, x.it.row0);
            a.desc[2 * blockIdx.x + 1] = make_int4((int)d.owner(x.u + kBegin), (int)d.owner(x.u + kBegin + x.it.n - 1), (int)x.it.t0, 0);
        }
        const int then = slot == 2 ? 0 : slot + 1, last = then == 2 ? 0 : then + 1;
        if (s_piece[then].n > 0) stage_queries(s_piece[then]);
        if (tid == Z::threads - 1) write_following(then, last);
        if (!Z::beside) fence_async_smem(); // sums are written over by copies
        __syncthreads();                    // and by sums
    }
    if (warp == 0) {
        settle(dead);
        if (lane == 0 && *dead) *a.wait_error = 1;
    }
}

// an item's pieces, by the CTAs of the same numbers as those that hold them, all but the last: a share of the item's numbers each (many rows: gridDim.y shares).  Threads of a column of four numbers have
// the pieces in turn, four of them asked for ahead of the rows' maxima and sums, and are added up in order
template <int R, typename E> __global__ void __launch_bounds__(256) kv8_join_kernel(const __grid_constant__ attn_args a) {
    __shared__ float4 s_y[256];
    __shared__ float s_f[3 * kMaxCtas], s_g[3 * kMaxCtas], s_m[R], s_l[R];
    step_wait();
    const int4 d = a.desc[2 * blockIdx.x], e = a.desc[2 * blockIdx.x + 1];
    if (d.x < 0) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hpg = a.H / a.G, b0 = e.x, pieces = e.y - b0 + 1, share = (blockIdx.x - b0) * gridDim.y + blockIdx.y, shares = (pieces - 1) * gridDim.y;
    const int quads = a.Dv / 4, rows = d.y, q0 = rows * quads * share / shares, q1 = rows * quads * (share + 1) / shares, r0 = q0 / quads;
    if (q0 == q1) return;
    const int nq = min(256, q1 - q0), ways = 256 / nq, way = tid / nq;
    auto piece = [&](int k, int r) { return ((int64_t)(b0 + k) * 2 + (k == 0)) * R + r; };
    float4 ahead[4];
    auto load = [&](int k, int r, int c) { return *reinterpret_cast<const float4 *>(a.part + piece(k, r) * a.Dv + c); };
    int q = q0 + tid - way * nq;
#pragma unroll
    for (int u = 0; u < 4; u++)
        if (way < ways && way + u * ways < pieces) ahead[u] = load(way + u * ways, q / quads, 4 * (q % quads));
    for (int r = r0 + warp; r <= (q1 - 1) / quads; r += 8) {
        float *f = s_f + (r - r0) * pieces, *g = s_g + (r - r0) * pieces, M = kNone, L = 0.f;
#pragma unroll 8
        for (int k = lane; k < pieces; k += 32) {
            const float2 ml = a.part_ml[piece(k, r)];
            M = fmaxf(M, f[k] = ml.x);
            g[k] = ml.y;
        }
        M = warp_max_f32(M);
        for (int k = lane; k < pieces; k += 32) L = fmaf(g[k], f[k] = exp2f(f[k] - M), L);
        L = warp_sum_f32(L);
        if (lane == 0) s_m[r - r0] = M, s_l[r - r0] = L;
    }
    __syncthreads();
    for (; q < q1 && (way == 0 || ways > 1); q += nq) {
        const int r = q / quads, c = 4 * (q - r * quads);
        const float *f = s_f + (r - r0) * pieces;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (way < ways) {
            auto add = [&](const float4 &x, float g) { y.x = fmaf(x.x, g, y.x), y.y = fmaf(x.y, g, y.y), y.z = fmaf(x.z, g, y.z), y.w = fmaf(x.w, g, y.w); };
            int k = way;
            if (q < q0 + nq) {
#pragma unroll
                for (int u = 0; u < 4; u++, k += ways)
                    if (k < pieces) add(ahead[u], f[k]);
            }
#pragma unroll 4
            for (; k < pieces; k += ways) add(load(k, r, c), f[k]);
        }
        if (ways > 1) { // (then there is one q a thread)
            auto add_way = [&](int w) {
                const float4 x = s_y[w * nq + (q - q0)];
                y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
            };
            s_y[tid] = y;
            __syncthreads();
            if (way < 8)
                for (int w = way + 8; w < ways; w += 8) add_way(w);
            __syncthreads();
            s_y[tid] = y;
            __syncthreads();
            if (way != 0) return;
            for (int w = 1; w < min(8, ways); w++) add_way(w);
        }
        const int row = d.w + r, tq = row / hpg, h = d.z * hpg + (row - tq * hpg);
        const int64_t t = e.z + tq, to = (int64_t)h * a.Dv + c;
        const row_end end(a, h, s_m[r - r0], s_l[r - r0]);
        E *out = reinterpret_cast<E *>(a.out) + t * a.H * a.Dv + to;
        out[0] = from_f32<E>(gated(a, y.x * end.f, t, to)), out[1] = from_f32<E>(gated(a, y.y * end.f, t, to + 1));
        out[2] = from_f32<E>(gated(a, y.z * end.f, t, to + 2)), out[3] = from_f32<E>(gated(a, y.w * end.f, t, to + 3));
    }
}

template <int CODE, int P, int NT, int PARTS> int step_launch(attn_args a, int64_t T, int64_t max_new) {
    using Z = step_sizes<CODE, P, NT, PARTS>;
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    const int64_t places = list_items(a, T, max_new, Z::R);
    GGB_CHECK_ARG(max_new * (a.H / a.G) < (1ll << 30) && places * a.G < (1ll << 31), "kv8_attn: too many sequences, tokens and heads for a launch");
    GGB_CHECK_ARG(places * a.G * ((a.positions + a.keep) / Z::tile + 4) < (1ll << 31), "kv8_attn: too many positions for a launch"); // the units of a deal, at most
    a.entries = (int)places;
    auto k = kv8_step_kernel<CODE, P, NT, PARTS>;
    int rc = ggb_allow_smem(k, Z::smem);
    if (rc) return rc;
    const unsigned ctas = a.part ? (unsigned)std::min(kMaxCtas, ggb_sm_count() * Z::min_ctas) : (unsigned)(a.entries * a.G);
    line_maps maps;
    rc = make_line_maps(a, maps);
    if (rc) return rc;
    GGB_CUDA(ggb_launch_step(k, dim3(ctas), dim3(Z::threads), Z::smem, a, maps));
    GGB_LAUNCH_CHECK();
    if (a.part) {
        GGB_CUDA(ggb_launch_step(kv8_join_kernel<Z::R, E>, dim3(ctas), dim3(256), 0, a));
        GGB_LAUNCH_CHECK();
    }
    return GGB_OK;
}
// rows of an item: as many as a sequence and key head has, up to 32 (16 with the largest heads, whose sums fill the registers)
template <int CODE, int PARTS> int step_rows(const attn_args &a, int64_t T, int64_t max_new) {
    const int64_t rows = max_new * (a.H / a.G);
    const int size = std::max(a.D, a.Dv);
    if (size <= 64) return rows <= 8 ? step_launch<CODE, 64, 1, PARTS>(a, T, max_new) : rows <= 16 ? step_launch<CODE, 64, 2, PARTS>(a, T, max_new) : step_launch<CODE, 64, 4, PARTS>(a, T, max_new);
    if (size <= 128) return rows <= 8 ? step_launch<CODE, 128, 1, PARTS>(a, T, max_new) : rows <= 16 ? step_launch<CODE, 128, 2, PARTS>(a, T, max_new) : step_launch<CODE, 128, 4, PARTS>(a, T, max_new);
    return rows <= 8 ? step_launch<CODE, 256, 1, PARTS>(a, T, max_new) : step_launch<CODE, 256, 2, PARTS>(a, T, max_new);
}

// sequences of many rows by the tiles' kernel, the others by the steps', which begin and end sooner.  One sequence at 2,000 positions (bf16, 16 heads over 4 of 128), steps against tiles: 64 rows
// 16.9 and 21.4 us, 96 rows 18.9 and 22.5, 128 rows 18.8 and 23.7, 256 rows 26.7 and 24.4.  16 sequences of up to 256 rows: 87 by steps, 82 by both kernels, one behind the other, as a batch with shorter
// sequences beside takes them; up to 132 rows 59 and 81.  (Were all rows of such a batch the tiles' kernel's: 41 us with 128 rows, where steps take 57, and 37 with 64, where they take 40.)
constexpr int64_t kFew = 128;
template <int CODE, int PARTS> int attend(attn_args a, int64_t T, int64_t max_new) {
    using E = typename std::conditional<PARTS == 1, __nv_bfloat16, float>::type;
    const int64_t hpg = a.H / a.G;
    const bool tiles = max_new * hpg > kFew && tile_fits(a.D, a.Dv, a.H, a.G), steps = !tiles || (a.n_seq > 1 && hpg <= kFew);
    if (steps) {
        a.rows_above = 0, a.rows_up_to = tiles ? kFew : INT64_MAX;
        const int rc = step_rows<CODE, PARTS>(a, T, tiles ? kFew / hpg : max_new);
        if (rc) return rc;
    }
    if (tiles) {
        a.rows_above = steps ? kFew : 0, a.rows_up_to = INT64_MAX;
        unsigned joins;
        const int rc = tile_launch<CODE, PARTS>(a, T, max_new, &joins);
        if (rc) return rc;
        if (joins) {
            GGB_CUDA(ggb_launch_step(kv8_join_kernel<kTileRows, E>, dim3(joins, 8), dim3(256), 0, a));
            GGB_LAUNCH_CHECK();
        }
    }
    return GGB_OK;
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
    const int64_t positions = std::min<int64_t>(table_ld, (1ll << 31) / block_size) * block_size; // (they are 32-bit numbers)
    float *part = (float *)scratch;
    const attn_args a{q, (const uint8_t *)cache, tables, table_ld, block_size, n_seq, starts, pos0, H, G, D, Dv, window, window > 0 ? std::min<int64_t>(keep_first, positions) : 0, softcap, sink, gate, ldg,
                      kv8_record(D, Dv, block_size), out, 0, 0, 0, 0, part, (float2 *)(part ? part + (size_t)kMaxCtas * 2 * kMaxRows * Dv : nullptr),
                      (int4 *)(part ? part + (size_t)kMaxCtas * 2 * kMaxRows * (Dv + 2) : nullptr), (uintptr_t)q % 16 == 0,
                      (uintptr_t)out % 16 == 0, (uintptr_t)gate % 16 == 0 && ldg % 4 == 0, positions, ggb_wait_error_flag()};
    if (dt == GGB_TYPE_BF16) return code == GGB_KV8_INT8 ? attend<GGB_KV8_INT8, 1>(a, T, max_new) : attend<GGB_KV8_E4M3, 1>(a, T, max_new);
    return code == GGB_KV8_INT8 ? attend<GGB_KV8_INT8, 2>(a, T, max_new) : attend<GGB_KV8_E4M3, 2>(a, T, max_new);
}

} // extern "C"
