// draft_verify.cu — which tokens of a smaller model's draft stand against the target model's probabilities, and the token behind them, by given
// random numbers (speculative sampling).
//
// Sequence s has rows starts[s] .. starts[s + 1] - 1 of target logits: row j follows j drafted tokens, so all but the last judge the drafted token of
// their row.  With p = soft-max(target / temperature), q = soft-max(draft / temperature) (without draft logits: 1 at the drafted token), the token d of
// a row stands where u q(d) < p(d).  Behind the tokens that stand up to the first that does not, one is drawn: from max(p - q, 0) over its sum where a draft
// has fallen, from p behind a whole draft; it is the first v at which the running sum exceeds the sequence's last u times the whole sum.  So the tokens have the
// target's distribution, whatever the draft's.  Temperature 0: a token stands where it is the target's first maximum, which is also what is drawn.
//
//   stats   a CTA a piece of a row: its maximum, the first place of it, and sum of exp(l / temperature - maximum); a sequence's last draft row is not read
//   pick    a CTA a piece of the row that is drawn from: joins the rows' pieces, decides what stands, sums its piece of the weights; the CTA that is done last finds
//           the token: the piece by the pieces' sums in order, the part of it by its warps', then the place in that
//
// Exponentials in fp32 and sums of four of them; beyond that, sums, and the probabilities that judge a draft, in 64 bits.  An exponential is off by 4 steps of 2^-24 of itself
// (the unit) and by three more (difference, constant, product) times its argument, which is below 20 where a weight counts: p and q are off by less than 4e-6 of
// themselves.  So a draft is judged otherwise than in 64 bits throughout only where u q and p are within twice that of one another.  A weight p - q is a 32-bit difference of 32-bit products,
// nothing where p and q are the same numbers; running sums of them are off by up to 8e-6, and the whole is, so the token that is drawn is one whose part of the
// running sum lies within 1.6e-5, over the sum of what is left, of u.  (Of a draft that is nearly the target 1e-5 may be left: then that says little, once in 1e5 rows.)  Sums are added in an
// order that the sizes alone set.
//
// What bounds it: for large batches (16 sequences of up to five drafts, 256,000 numbers: 39.9 us, some 25 of them in the first kernel, where the bytes of the logits, read once, take
// 16.3) neither bytes nor instructions alone (DRAM 57 % and issue 57 % of their peaks, 15 instructions a number): a CTA has one block of numbers, so nothing is on its way while it
// finds the block's maximum and adds up; and what the second kernel does one thing after the other.  For one sequence (11.3 us) and the greedy form (24
// sequences, 49,999 numbers: 7.9 us, the bytes 3.3) the two launches and that chain.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int kMaxPieces = 64, kThreads = 256, kWarps = kThreads / 32;

struct piece_stats {
    float m;    // maximum
    int32_t at; // first place of it
    double s;   // sum of exp((l - m) / temperature): not above 0 when the row has no distribution
};

struct verify_args {
    const float *target, *draft;
    int64_t ld_t, ld_d, V, R, piece;
    int n_seq, pieces;
    const int32_t *starts, *drafted;
    const float *u;
    float inv; // log2(e) / temperature
    double inv64; // 1 / temperature
    int32_t *tokens, *accepted;
    piece_stats *stats; // [R][2][pieces]: target, draft
    double *sums;       // [n_seq][pieces][warps]
    unsigned *done;     // [n_seq]
    int vec_t, vec_d;
};

__device__ __forceinline__ int sequence_of(const int32_t *starts, int n_seq, int64_t row) { // whole warps
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seq;
    while (n > 1) {
        const int step = (n + 31) / 32, k = lane * step;
        const int last = max(0, __popc(__ballot_sync(0xffffffffu, k < n && starts[lo + k] <= row)) - 1) * step;
        lo += last;
        n = min(step, n - last);
    }
    return lo;
}

// the larger of two maxima, the first place where they are equal; what is no number wins (its sum says so)
__device__ __forceinline__ bool ahead(float m, int at, float m2, int at2) { return m > m2 || (m == m2 && at < at2); }

constexpr int kPasses = 8, kBlock = 4 * kThreads * kPasses; // 16-byte pieces in flight a thread; numbers in those of a CTA
// numbers i .. i + 3 of n
__device__ __forceinline__ float4 load4(const float *x, int i, int n, bool vec) {
    if (vec && i + 4 <= n) return *reinterpret_cast<const float4 *>(x + i);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = i + e < n ? x[i + e] : -INFINITY;
    return make_float4(y[0], y[1], y[2], y[3]);
}
// exp((x - m) / temperature) as a power of two, c = log2(e) / temperature: the unit's 2^-22 and the argument's roundings of 2^-24 of itself.  It takes none of
// expf's steps for large arguments; below 2^-126 it is zero.
__device__ __forceinline__ float power(float x, float m, float c) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((x - m) * c));
    return y;
}

// Each block of numbers waits in registers until the CTA's threads have their common maximum, so that a number costs one exponential and sums are scaled once a block
template <bool GREEDY> __global__ void __launch_bounds__(kThreads, 5) verify_stats_kernel(const __grid_constant__ verify_args a) {
    __shared__ float s_m[2][kWarps];
    __shared__ int s_at[kWarps];
    __shared__ double s_s[kWarps];
    step_wait();
    const int64_t r = blockIdx.y;
    const int side = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (r >= a.starts[a.n_seq]) return;
    const int seq = sequence_of(a.starts, a.n_seq, r);
    if (blockIdx.x == 0 && side == 0 && tid == 0 && r == a.starts[seq]) a.done[seq] = 0;
    if (side == 1 && r == a.starts[seq + 1] - 1) return; // nothing is judged by it
    const float *row = side ? a.draft + r * a.ld_d : a.target + r * a.ld_t;
    const bool vec = side ? a.vec_d : a.vec_t;
    const int64_t v0 = blockIdx.x * a.piece, v1 = min(a.V, v0 + a.piece); // pieces are multiples of 32
    float m = -INFINITY;
    int at = 0x7fffffff;
    double s = 0.0;
    bool odd = false;
    int turn = 0;
    for (int64_t b = v0; b < v1; b += kBlock, turn ^= 1) {
        float4 x[kPasses];
        const int n = (int)min((int64_t)kBlock, v1 - b);
#pragma unroll
        for (int p = 0; p < kPasses; p++)
            x[p] = 4 * kThreads * p < n ? load4(row + b, 4 * kThreads * p + 4 * tid, n, vec) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        float best = m;
#pragma unroll
        for (int p = 0; p < kPasses; p++) {
            if (GREEDY) {
                const float y[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    odd |= y[e] != y[e];
                    if (y[e] > best) best = y[e], at = (int)(b + 4 * kThreads * p) + 4 * tid + e;
                }
            } else {
                best = fmaxf(best, fmaxf(fmaxf(x[p].x, x[p].y), fmaxf(x[p].z, x[p].w)));
            }
        }
        if (!GREEDY) {
            best = warp_max_f32(best);
            if (lane == 0) s_m[turn][warp] = best; // (two of them in turn: the next block's are written before the last warp has read these)
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; w++) best = fmaxf(best, s_m[turn][w]);
            if (best > m) s *= (double)power(m, best, a.inv); // m = -inf: 0
            const float top = best == -INFINITY ? 0.f : best; // (numbers of -inf are nothing then too)
#pragma unroll
            for (int p = 0; p < kPasses; p++)
                if (4 * kThreads * p < n) // inf and NaN leave NaN
                    s += (double)((power(x[p].x, top, a.inv) + power(x[p].y, top, a.inv)) + (power(x[p].z, top, a.inv) + power(x[p].w, top, a.inv)));
        }
        m = best;
    }
    if (GREEDY) {
        odd = __any_sync(0xffffffffu, odd);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
            const int at2 = __shfl_xor_sync(0xffffffffu, at, off);
            if (ahead(m2, at2, m, at)) m = m2, at = at2;
        }
        if (lane == 0) s_m[0][warp] = m, s_at[warp] = at;
        s = odd ? NAN : 0.0;
    } else {
        s = warp_sum_f64(s);
    }
    if (lane == 0) s_s[warp] = s;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarps; w++) {
            s += s_s[w];
            if (GREEDY && ahead(s_m[0][w], s_at[w], m, at)) m = s_m[0][w], at = s_at[w];
        }
        a.stats[(r * 2 + side) * a.pieces + blockIdx.x] = piece_stats{m, at, s};
    }
}

struct row_stats {
    float m;
    int at;
    double s;
};
// a row's pieces, joined by a warp: every lane the answer
template <bool GREEDY> __device__ __forceinline__ row_stats joined(const piece_stats *p, int pieces, double inv) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    int at = 0x7fffffff;
    double s = 0.0;
#pragma unroll 1
    for (int c = lane; c < pieces; c += 32) {
        const piece_stats x = p[c];
        if (x.m == m || GREEDY) s += x.s;
        else if (x.m > m) s = x.s + (s > 0.0 ? s * exp(((double)m - (double)x.m) * inv) : s);
        else s += x.s * exp(((double)x.m - (double)m) * inv); // of a piece of no numbers: NaN times 0
        if (ahead(x.m, x.at, m, at)) m = x.m, at = x.at;
    }
    float best = m;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, best, off);
        const int at2 = __shfl_xor_sync(0xffffffffu, at, off);
        if (ahead(m2, at2, best, at)) best = m2, at = at2;
    }
    if (!GREEDY && m != best) s = s * exp(((double)m - (double)best) * inv);
    return {best, at, warp_sum_f64(s)};
}

// the row that the token behind the draft is drawn from
struct drawn_row {
    const float *p, *q; // q: logits to take away from it, or null
    float mp, mq;
    float sp, sq;    // 1 / sum, where there is a q (p alone needs no division: the sums are in proportion)
    int64_t without; // a token that falls out, or -1
};
__device__ __forceinline__ float weight(const drawn_row &d, float inv, float lp, float lq, int64_t v) {
    float w = power(lp, d.mp, inv) * d.sp;
    if (d.q) w = __fsub_rn(w, __fmul_rn(power(lq, d.mq, inv), d.sq));
    return v == d.without || !(w > 0.f) ? 0.f : w;
}
__device__ __forceinline__ float weights(const drawn_row &d, float inv, float4 lp, float4 lq, int64_t v) { // of four numbers
    return (weight(d, inv, lp.x, lq.x, v) + weight(d, inv, lp.y, lq.y, v + 1)) + (weight(d, inv, lp.z, lq.z, v + 2) + weight(d, inv, lp.w, lq.w, v + 3));
}
__device__ __forceinline__ float pick4(float4 x, int e) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; }

struct place {
    int at;               // the first of the sums at which their running sum exceeds `to`; should none (rounding), the last with anything in it, or -1
    double before, whole; // running sum ahead of it, sum of all
};
// a warp, every lane the answer: lane l has sums E l .. E l + E - 1
template <int E> __device__ __forceinline__ place place_of(const double (&sum)[E], double from, double to) {
    const int lane = threadIdx.x & 31;
    double mine = sum[0];
#pragma unroll
    for (int e = 1; e < E; e++) mine += sum[e];
    double upto = mine; // with the lanes below
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += x;
    }
    place p{-1, 0.0, from + __shfl_sync(0xffffffffu, upto, 31)};
    const unsigned over = __ballot_sync(0xffffffffu, from + upto > to && mine > 0.0), any = __ballot_sync(0xffffffffu, mine > 0.0);
    if (!any) return p;
    const int who = over ? __ffs((int)over) - 1 : 31 - __clz((int)any);
    double run = from + (upto - mine);
    bool open = true;
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (open && sum[e] > 0.0) p.at = E * lane + e, p.before = run;
        run += sum[e];
        if (sum[e] > 0.0 && run > to) open = false;
    }
    p.at = __shfl_sync(0xffffffffu, p.at, who), p.before = __shfl_sync(0xffffffffu, p.before, who);
    return p;
}

template <bool GREEDY> __global__ void __launch_bounds__(kThreads) verify_pick_kernel(const __grid_constant__ verify_args a) {
    __shared__ int s_first, s_extra;
    __shared__ bool s_last;
    __shared__ double s_sum[2][kWarps];
    __shared__ row_stats s_p, s_q;
    step_wait();
    const int seq = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t r0 = a.starts[seq];
    const int rows = (int)(a.starts[seq + 1] - r0), drafts = rows - 1;
    if (rows <= 0) {
        if (blockIdx.x == 0 && tid == 0) a.accepted[seq] = 0;
        return;
    }
    if (tid == 0) s_first = drafts;
    __syncthreads();
    // a warp a row, until one does not stand: the first of them is the row to draw from, else the last row
    row_stats t{0.f, 0, 0.0}, s{0.f, 0, 0.0};
    int fallen = -1;
    for (int j = warp; j <= drafts && fallen < 0; j += kWarps) {
        const int64_t r = r0 + j;
        t = joined<GREEDY>(a.stats + r * 2 * a.pieces, a.pieces, a.inv64);
        bool stands = false;
        if (j < drafts) {
            const int64_t d = a.drafted[r];
            if (GREEDY) {
                stands = t.s == 0.0 && t.m > -INFINITY && d == t.at;
            } else {
                double q = 1.0;
                if (a.draft) {
                    s = joined<false>(a.stats + (r * 2 + 1) * a.pieces, a.pieces, a.inv64);
                    q = d >= 0 && d < a.V ? exp(((double)a.draft[r * a.ld_d + d] - (double)s.m) * a.inv64) / s.s : 0.0;
                }
                const double p = d >= 0 && d < a.V ? exp(((double)a.target[r * a.ld_t + d] - (double)t.m) * a.inv64) / t.s : 0.0;
                stands = (double)a.u[r] * q < p; // with what is no number: no
            }
        }
        if (!stands) {
            fallen = j;
            if (lane == 0) atomicMin(&s_first, j);
        }
    }
    __syncthreads();
    const int taken = s_first;
    if (fallen == taken && lane == 0) s_p = t, s_q = s; // (one warp's)
    __syncthreads();
    t = s_p, s = s_q;
    const int64_t r = r0 + taken;
    if (GREEDY) {
        if (tid == 0) s_extra = t.s == 0.0 && t.m > -INFINITY ? t.at : -1;
    } else {
        drawn_row d{a.target + r * a.ld_t, nullptr, t.m, 0.f, 1.f, 0.f, -1};
        bool valid = t.s > 0.0;
        if (taken < drafts) {
            if (a.draft) {
                d.q = a.draft + r * a.ld_d, d.mq = s.m, d.sp = (float)(1.0 / t.s), d.sq = (float)(1.0 / s.s);
                valid = valid && s.s > 0.0;
            } else {
                d.without = a.drafted[r];
            }
        }
        const int64_t share = a.piece / kWarps; // a warp's part of a piece: a multiple of 4
        const int64_t v0 = blockIdx.x * a.piece + warp * share, v1 = min(a.V, v0 + share);
        double *sums = a.sums + (int64_t)seq * a.pieces * kWarps;
        double sum = 0.0;
        if (valid)
            for (int64_t b = v0; b < v1; b += 4 * 32 * kPasses) {
                float4 lp[kPasses], lq[kPasses];
                const int n = (int)min((int64_t)(4 * 32 * kPasses), v1 - b);
#pragma unroll
                for (int p = 0; p < kPasses; p++) {
                    lp[p] = lq[p] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (4 * 32 * p < n) {
                        lp[p] = load4(d.p + b, 4 * 32 * p + 4 * lane, n, a.vec_t);
                        if (d.q) lq[p] = load4(d.q + b, 4 * 32 * p + 4 * lane, n, a.vec_d);
                    }
                }
#pragma unroll
                for (int p = 0; p < kPasses; p++)
                    if (4 * 32 * p < n) sum += (double)weights(d, a.inv, lp[p], lq[p], b + 4 * 32 * p + 4 * lane);
            }
        sum = warp_sum_f64(sum);
        if (lane == 0) {
            sums[blockIdx.x * kWarps + warp] = sum;
            __threadfence();
        }
        __syncthreads();
        if (tid == 0) {
            s_last = atomicAdd(&a.done[seq], 1u) == gridDim.x - 1;
            s_extra = -1;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        // ---- the last one: the piece whose running sum exceeds u times the whole, then the warp's part of it; every warp finds the same
        double piece_sum[kMaxPieces / 32];
#pragma unroll
        for (int e = 0; e < kMaxPieces / 32; e++) {
            const int c = kMaxPieces / 32 * lane + e;
            piece_sum[e] = 0.0;
            if (c < a.pieces) {
                double x[kWarps];
#pragma unroll
                for (int w = 0; w < kWarps; w++) x[w] = __ldcg(sums + c * kWarps + w);
#pragma unroll
                for (int w = 0; w < kWarps; w++) piece_sum[e] += x[w];
            }
        }
        const double u = (double)a.u[r0 + drafts];
        int64_t b0 = 0, b1 = 0;
        double run = 0.0, to = u * place_of(piece_sum, 0.0, INFINITY).whole;
        const place piece = place_of(piece_sum, 0.0, to);
        if (valid && piece.at >= 0) {
            const double part[1] = {lane < kWarps ? __ldcg(sums + piece.at * kWarps + lane) : 0.0};
            const place in = place_of(part, piece.before, to);
            b0 = piece.at * a.piece + in.at * share, b1 = min(a.V, b0 + share), run = in.before;
        } else if (valid && (d.q || d.without >= 0)) { // rounding left nothing of p - q: from p, one sum over the whole row
            d.q = nullptr, d.without = -1, d.sp = 1.f;
            b1 = a.V, to = u * t.s;
        }
        // four numbers a thread at a time: the warps' sums in order, then the lanes' in the one where the running sum exceeds and the four numbers of that lane
        int turn = 0;
        for (int64_t b = b0; b < b1; b += 4 * kThreads, turn ^= 1) {
            const int64_t v = b + 4 * tid;
            const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            const int n = (int)min((int64_t)(4 * kThreads), b1 - b);
            const float4 lp = load4(d.p + b, 4 * tid, n, a.vec_t), lq = d.q ? load4(d.q + b, 4 * tid, n, a.vec_d) : none;
            const double mine[1] = {(double)weights(d, a.inv, lp, lq, v)}, all = warp_sum_f64(mine[0]);
            if (lane == 0) s_sum[turn][warp] = all;
            __syncthreads();
            const double part[1] = {lane < kWarps ? s_sum[turn][lane] : 0.0};
            const place block = place_of(part, run, to);
            if (block.at == warp) {
                const place four = place_of(mine, block.before, to);
                if (lane == four.at) {
                    double upto = four.before;
#pragma unroll 1
                    for (int e = 0; e < 4; e++) {
                        const float w = weight(d, a.inv, pick4(lp, e), pick4(lq, e), v + e);
                        if (!(w > 0.f)) continue;
                        s_extra = (int)(v + e); // the last one with a weight, so far
                        upto += (double)w;
                        if (upto > to) break;
                    }
                }
            }
            if (block.whole > to) break;
            run = block.whole;
            __syncthreads(); // (one block's place is written behind the one before)
        }
    }
    __syncthreads();
    for (int j = tid; j < rows; j += kThreads) a.tokens[r0 + j] = j < taken ? a.drafted[r0 + j] : j == taken ? s_extra : -1;
    if (tid == 0) a.accepted[seq] = taken;
}

} // namespace

extern "C" {

size_t ggb_draft_verify_scratch_bytes(int64_t R, int n_seq) {
    return (size_t)R * 2 * kMaxPieces * sizeof(piece_stats) + (size_t)n_seq * (kMaxPieces * kWarps * sizeof(double) + sizeof(unsigned));
}

int ggb_op_draft_verify(const float *target, int64_t ld_target, const float *draft, int64_t ld_draft, int64_t V, int64_t R, int n_seq, const int32_t *starts,
                        const int32_t *drafted, const float *u, float temperature, int32_t *tokens, int32_t *n_accepted, void *scratch, size_t scratch_bytes) {
    GGB_REQUIRE_INIT();
    GGB_CHECK_ARG(target && starts && drafted && (u || temperature == 0.f) && tokens && n_accepted && scratch, "draft_verify: a pointer is null");
    GGB_CHECK_ARG(V > 0 && V < (1ll << 31) - (1 << 20) && R > 0 && R <= 65535 && n_seq > 0 && n_seq <= 65535, "draft_verify: %lld rows of %lld numbers, %d sequences", (long long)R,
                  (long long)V, n_seq);
    GGB_CHECK_ARG(ld_target >= V && (!draft || ld_draft >= V), "draft_verify: rows of %lld numbers overlap", (long long)V);
    GGB_CHECK_ARG(temperature >= 0.f && temperature <= 3.0e38f && (temperature == 0.f || 1.5f / temperature <= 3.0e38f), "draft_verify: a temperature of %g", (double)temperature);
    GGB_CHECK_ARG((uintptr_t)scratch % 16 == 0 && scratch_bytes >= ggb_draft_verify_scratch_bytes(R, n_seq), "draft_verify: %zu bytes of scratch, %zu needed on a 16-byte boundary",
                  scratch_bytes, ggb_draft_verify_scratch_bytes(R, n_seq));
    const bool greedy = temperature == 0.f;
    const float *dr = greedy ? nullptr : draft;
    // pieces of 8192 numbers, a thread 32 of them in flight; smaller ones, down to 2048, where few rows leave SMs without work
    const int64_t sides = dr ? 2 : 1;
    int64_t piece = 8192;
    while (piece > 2048 && R * sides * ((V + piece - 1) / piece) < 2 * ggb_sm_count()) piece /= 2;
    piece = std::max(piece, ((V + kMaxPieces - 1) / kMaxPieces + 4 * kWarps - 1) / (4 * kWarps) * (4 * kWarps));
    verify_args a{};
    a.target = target, a.draft = dr, a.ld_t = ld_target, a.ld_d = ld_draft, a.V = V, a.R = R, a.piece = piece, a.n_seq = n_seq, a.pieces = (int)((V + piece - 1) / piece);
    a.starts = starts, a.drafted = drafted, a.u = u, a.inv = greedy ? 0.f : (float)(1.4426950408889634 / (double)temperature), a.inv64 = greedy ? 0.0 : 1.0 / (double)temperature, a.tokens = tokens,
    a.accepted = n_accepted;
    a.stats = (piece_stats *)scratch;
    a.sums = (double *)(a.stats + R * 2 * kMaxPieces);
    a.done = (unsigned *)(a.sums + (int64_t)n_seq * kMaxPieces * kWarps);
    a.vec_t = (uintptr_t)target % 16 == 0 && ld_target % 4 == 0, a.vec_d = (uintptr_t)dr % 16 == 0 && ld_draft % 4 == 0;
    const dim3 grid((unsigned)a.pieces, (unsigned)R, (unsigned)sides), pick(greedy ? 1u : (unsigned)a.pieces, (unsigned)n_seq);
    if (greedy) {
        GGB_CUDA(ggb_launch_step(verify_stats_kernel<true>, grid, dim3(kThreads), 0, a));
        GGB_LAUNCH_CHECK();
        GGB_CUDA(ggb_launch_step(verify_pick_kernel<true>, pick, dim3(kThreads), 0, a));
    } else {
        GGB_CUDA(ggb_launch_step(verify_stats_kernel<false>, grid, dim3(kThreads), 0, a));
        GGB_LAUNCH_CHECK();
        GGB_CUDA(ggb_launch_step(verify_pick_kernel<false>, pick, dim3(kThreads), 0, a));
    }
    GGB_LAUNCH_CHECK();
    return GGB_OK;
}

} // extern "C"
