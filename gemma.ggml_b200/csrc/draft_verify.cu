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
//           the token: the piece by the pieces' sums in order, then the place in it
//
// Exponentials in fp32 and sums of four of them; beyond that, sums, and the probabilities that judge a draft, in 64 bits.  A weight p - q is a 32-bit difference of
// 32-bit products: as far off as its exponentials are, and nothing where p and q are the same numbers.  So a decision is another one than in 64 bits throughout only
// where the numbers compared are within about 1e-7 of one another.  Sums are added in an order that the sizes alone set.
//
// What bounds it: the bytes of the logits, read once, and for the row that is drawn from once more out of L2; for a single sequence the two launches.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int kMaxPieces = 128, kThreads = 256;

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
    float inv; // 1 / temperature
    double inv64;
    int32_t *tokens, *accepted;
    piece_stats *stats; // [R][2][pieces]: target, draft
    double *sums;       // [n_seq][pieces]
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
__device__ __forceinline__ float4 load4(const float *row, int64_t v, int64_t end, bool vec) {
    if (vec && v + 4 <= end) return *reinterpret_cast<const float4 *>(row + v);
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = v + e < end ? row[v + e] : -INFINITY;
    return make_float4(x[0], x[1], x[2], x[3]);
}

// Each block of numbers waits in registers until the CTA's threads have their common maximum, so that a number costs one exponential and sums are scaled once a block
template <bool GREEDY> __global__ void __launch_bounds__(kThreads) verify_stats_kernel(const __grid_constant__ verify_args a) {
    __shared__ float s_m[2][kThreads / 32];
    __shared__ int s_at[kThreads / 32];
    __shared__ double s_s[kThreads / 32];
    step_wait();
    const int64_t r = blockIdx.y;
    const int side = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (r >= a.starts[a.n_seq]) return;
    const int seq = sequence_of(a.starts, a.n_seq, r);
    if (blockIdx.x == 0 && side == 0 && tid == 0 && r == a.starts[seq]) a.done[seq] = 0;
    if (side == 1 && r == a.starts[seq + 1] - 1) return; // nothing is judged by it
    const float *row = side ? a.draft + r * a.ld_d : a.target + r * a.ld_t;
    const bool vec = side ? a.vec_d : a.vec_t;
    const int64_t v0 = blockIdx.x * a.piece, v1 = min(a.V, v0 + a.piece); // pieces are multiples of 4
    float m = -INFINITY;
    int at = 0x7fffffff;
    double s = 0.0;
    bool odd = false;
    int turn = 0;
    for (int64_t b = v0; b < v1; b += kBlock, turn ^= 1) {
        float4 x[kPasses];
#pragma unroll
        for (int p = 0; p < kPasses; p++)
            x[p] = b + 4 * kThreads * p < v1 ? load4(row, b + 4 * kThreads * p + 4 * tid, v1, vec) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
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
            for (int w = 0; w < kThreads / 32; w++) best = fmaxf(best, s_m[turn][w]);
            if (best > m) s *= (double)expf((m - best) * a.inv); // m = -inf: 0
#pragma unroll
            for (int p = 0; p < kPasses; p++)
                if (b + 4 * kThreads * p < v1) {
                    auto power = [&](float y) { return y == -INFINITY ? 0.f : expf((y - best) * a.inv); }; // inf and NaN leave NaN
                    s += (double)((power(x[p].x) + power(x[p].y)) + (power(x[p].z) + power(x[p].w)));
                }
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
        for (int w = 1; w < kThreads / 32; w++) {
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
    piece_stats x[kMaxPieces / 32];
    float m = -INFINITY;
    int at = 0x7fffffff;
    double s = 0.0;
#pragma unroll
    for (int u = 0; u < kMaxPieces / 32; u++) {
        x[u] = lane + 32 * u < pieces ? p[lane + 32 * u] : piece_stats{-INFINITY, 0x7fffffff, 0.0};
        if (ahead(x[u].m, x[u].at, m, at)) at = x[u].at;
        m = fmaxf(m, x[u].m);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
        const int at2 = __shfl_xor_sync(0xffffffffu, at, off);
        if (ahead(m2, at2, m, at)) at = at2;
        m = fmaxf(m, m2);
    }
#pragma unroll
    for (int u = 0; u < kMaxPieces / 32; u++)
        if (32 * u < pieces) s += GREEDY || x[u].m == m ? x[u].s : x[u].s * exp(((double)x[u].m - (double)m) * inv); // of a piece of no numbers: NaN times 0
    return {m, at, warp_sum_f64(s)};
}

// the row that the token behind the draft is drawn from
struct drawn_row {
    const float *p, *q; // q: logits to take away from it, or null
    float mp, mq;
    float sp, sq;    // 1 / sum, where there is a q (p alone needs no division: the sums are in proportion)
    int64_t without; // a token that falls out, or -1
};
__device__ __forceinline__ float weight(const drawn_row &d, float inv, float lp, float lq, int64_t v) {
    float w = lp == -INFINITY ? 0.f : expf((lp - d.mp) * inv) * d.sp;
    if (d.q && lq != -INFINITY) w = __fsub_rn(w, __fmul_rn(expf((lq - d.mq) * inv), d.sq));
    return v == d.without || !(w > 0.f) ? 0.f : w;
}
// the weights of a block of numbers from b on, ahead of `end`: a thread's sums of four each, numbers b + 1024 p + 4 tid .. + 3
__device__ __forceinline__ void block_weights(const drawn_row &d, float inv, int64_t b, int64_t end, bool vec_t, bool vec_d, double (&sum)[kPasses]) {
    float4 lp[kPasses], lq[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; p++) {
        const int64_t v = b + 4 * kThreads * p + 4 * threadIdx.x;
        lp[p] = lq[p] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (b + 4 * kThreads * p < end) {
            lp[p] = load4(d.p, v, end, vec_t);
            if (d.q) lq[p] = load4(d.q, v, end, vec_d);
        }
    }
#pragma unroll
    for (int p = 0; p < kPasses; p++) {
        const int64_t v = b + 4 * kThreads * p + 4 * threadIdx.x;
        sum[p] = 0.0;
        if (b + 4 * kThreads * p < end)
            sum[p] = (double)((weight(d, inv, lp[p].x, lq[p].x, v) + weight(d, inv, lp[p].y, lq[p].y, v + 1)) +
                              (weight(d, inv, lp[p].z, lq[p].z, v + 2) + weight(d, inv, lp[p].w, lq[p].w, v + 3)));
    }
}

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
    constexpr int kWarps = kThreads / 32;
    __shared__ int s_first, s_extra;
    __shared__ bool s_last;
    __shared__ double s_sum[2][kPasses * kWarps];
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
        const int64_t v0 = blockIdx.x * a.piece, v1 = min(a.V, v0 + a.piece);
        double sum = 0.0, part[kPasses];
        if (valid)
            for (int64_t b = v0; b < v1; b += kBlock) {
                block_weights(d, a.inv, b, v1, a.vec_t, a.vec_d, part);
#pragma unroll
                for (int p = 0; p < kPasses; p++) sum += part[p];
            }
        sum = warp_sum_f64(sum);
        if (lane == 0) s_sum[0][warp] = sum;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kWarps; w++) sum += s_sum[0][w];
            a.sums[(int64_t)seq * a.pieces + blockIdx.x] = sum;
            __threadfence();
            s_last = atomicAdd(&a.done[seq], 1u) == gridDim.x - 1;
            s_extra = -1;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        // ---- the last one: the piece whose running sum exceeds u times the whole, then the place in it; every warp finds the same piece
        double piece_sum[kMaxPieces / 32];
#pragma unroll
        for (int e = 0; e < kMaxPieces / 32; e++) {
            const int c = kMaxPieces / 32 * lane + e;
            piece_sum[e] = c < a.pieces ? __ldcg(a.sums + (int64_t)seq * a.pieces + c) : 0.0;
        }
        const double u = (double)a.u[r0 + drafts];
        int64_t b0 = 0, b1 = 0;
        double run = 0.0, to = u * place_of(piece_sum, 0.0, 0.0).whole;
        const place in = place_of(piece_sum, 0.0, to);
        if (valid && in.at >= 0) {
            b0 = in.at * a.piece, b1 = min(a.V, b0 + a.piece), run = in.before;
        } else if (valid && (d.q || d.without >= 0)) { // rounding left nothing of p - q: from p, one sum over the whole row
            d.q = nullptr, d.without = -1, d.sp = 1.f;
            b1 = a.V, to = u * t.s;
        }
        // a block at a time: the sums of its passes and warps in order, then the lanes' in the one where the running sum exceeds and the four numbers of that lane
        int turn = 0;
        for (int64_t b = b0; b < b1; b += kBlock, turn ^= 1) {
            block_weights(d, a.inv, b, b1, a.vec_t, a.vec_d, part);
#pragma unroll
            for (int p = 0; p < kPasses; p++) {
                const double w = warp_sum_f64(part[p]);
                if (lane == 0) s_sum[turn][p * kWarps + warp] = w;
            }
            __syncthreads();
            const double two[2] = {s_sum[turn][2 * lane], s_sum[turn][2 * lane + 1]};
            const place block = place_of(two, run, to);
            if (block.at >= 0 && block.at % kWarps == warp) {
                double mine[1] = {0.0};
#pragma unroll
                for (int p = 0; p < kPasses; p++)
                    if (p == block.at / kWarps) mine[0] = part[p];
                const place four = place_of(mine, block.before, to);
                if (lane == four.at) {
                    double upto = four.before;
                    const int64_t v = b + 4 * kThreads * (block.at / kWarps) + 4 * tid;
                    const float4 lp = load4(d.p, v, b1, a.vec_t), lq = d.q ? load4(d.q, v, b1, a.vec_d) : lp;
                    const float x[4] = {lp.x, lp.y, lp.z, lp.w}, y[4] = {lq.x, lq.y, lq.z, lq.w};
                    for (int e = 0; e < 4; e++) {
                        const float w = weight(d, a.inv, x[e], y[e], v + e);
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
    return (size_t)R * 2 * kMaxPieces * sizeof(piece_stats) + (size_t)n_seq * (kMaxPieces * sizeof(double) + sizeof(unsigned));
}

int ggb_op_draft_verify(const float *target, int64_t ld_target, const float *draft, int64_t ld_draft, int64_t V, int64_t R, int n_seq, const int32_t *starts,
                        const int32_t *drafted, const float *u, float temperature, int32_t *tokens, int32_t *n_accepted, void *scratch, size_t scratch_bytes) {
    GGB_REQUIRE_INIT();
    GGB_CHECK_ARG(target && starts && drafted && u && tokens && n_accepted && scratch, "draft_verify: a pointer is null");
    GGB_CHECK_ARG(V > 0 && V < (1ll << 31) - (1 << 20) && R > 0 && R <= 65535 && n_seq > 0 && n_seq <= 65535, "draft_verify: %lld rows of %lld numbers, %d sequences", (long long)R,
                  (long long)V, n_seq);
    GGB_CHECK_ARG(ld_target >= V && (!draft || ld_draft >= V), "draft_verify: rows of %lld numbers overlap", (long long)V);
    GGB_CHECK_ARG(temperature >= 0.f && temperature <= 3.0e38f && (temperature == 0.f || 1.0f / temperature <= 3.0e38f), "draft_verify: a temperature of %g", (double)temperature);
    GGB_CHECK_ARG((uintptr_t)scratch % 16 == 0 && scratch_bytes >= ggb_draft_verify_scratch_bytes(R, n_seq), "draft_verify: %zu bytes of scratch, %zu needed on a 16-byte boundary",
                  scratch_bytes, ggb_draft_verify_scratch_bytes(R, n_seq));
    const bool greedy = temperature == 0.f;
    const float *dr = greedy ? nullptr : draft;
    // pieces of 8192 numbers, a thread 32 of them in flight; smaller ones, down to 2048, where few rows leave SMs without work
    const int64_t sides = dr ? 2 : 1;
    int64_t piece = 8192;
    while (piece > 2048 && R * sides * ((V + piece - 1) / piece) < 2 * ggb_sm_count()) piece /= 2;
    piece = std::max(piece, ((V + kMaxPieces - 1) / kMaxPieces + 3) / 4 * 4);
    verify_args a{};
    a.target = target, a.draft = dr, a.ld_t = ld_target, a.ld_d = ld_draft, a.V = V, a.R = R, a.piece = piece, a.n_seq = n_seq, a.pieces = (int)((V + piece - 1) / piece);
    a.starts = starts, a.drafted = drafted, a.u = u, a.inv = greedy ? 0.f : 1.0f / temperature, a.inv64 = greedy ? 0.0 : 1.0 / (double)temperature, a.tokens = tokens,
    a.accepted = n_accepted;
    a.stats = (piece_stats *)scratch;
    a.sums = (double *)(a.stats + R * 2 * kMaxPieces);
    a.done = (unsigned *)(a.sums + (int64_t)n_seq * kMaxPieces);
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
