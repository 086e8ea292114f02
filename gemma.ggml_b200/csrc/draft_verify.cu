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
// Exponentials in fp32, their sums in 64 bits from four numbers on, and probabilities, weights and running sums in 64 bits: a decision is another one than in 64
// bits throughout only where the numbers compared are within about 1e-7 of one another.  Sums are added in an order that the sizes alone set.
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

template <bool GREEDY> __global__ void __launch_bounds__(kThreads) verify_stats_kernel(const __grid_constant__ verify_args a) {
    __shared__ float s_m[kThreads / 32];
    __shared__ int s_at[kThreads / 32];
    __shared__ double s_s[kThreads / 32];
    step_wait();
    const int64_t r = blockIdx.y;
    const int side = blockIdx.z, tid = threadIdx.x;
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
    constexpr int U = 8; // 16-byte pieces in flight
    for (int64_t v = v0 + 4 * tid; v < v1; v += 4 * kThreads * U) {
        float x[U][4];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t w = v + 4 * kThreads * u;
            if (vec && w + 4 <= v1) {
                const float4 f = *reinterpret_cast<const float4 *>(row + w);
                x[u][0] = f.x, x[u][1] = f.y, x[u][2] = f.z, x[u][3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) x[u][e] = w + e < v1 ? row[w + e] : -INFINITY;
            }
        }
        float best = m;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (GREEDY) {
                    odd |= x[u][e] != x[u][e];
                    if (x[u][e] > best) at = (int)(v + 4 * kThreads * u) + e;
                }
                best = fmaxf(best, x[u][e]);
            }
        if (!GREEDY) {
            if (best > m) s *= (double)expf((m - best) * a.inv); // m = -inf: 0
#pragma unroll
            for (int u = 0; u < U; u++) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = x[u][e] == -INFINITY ? 0.f : expf((x[u][e] - best) * a.inv); // inf and NaN leave NaN
                s += (double)((w[0] + w[1]) + (w[2] + w[3]));
            }
        }
        m = best;
    }
    if (GREEDY && odd) s = NAN;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, off);
        const int at2 = __shfl_xor_sync(0xffffffffu, at, off);
        const double s2 = __shfl_xor_sync(0xffffffffu, s, off);
        if (GREEDY) {
            s += s2;
            if (ahead(m2, at2, m, at)) m = m2, at = at2;
        } else {
            const float big = fmaxf(m, m2);
            s = (m == big ? s : s * (double)expf((m - big) * a.inv)) + (m2 == big ? s2 : s2 * (double)expf((m2 - big) * a.inv));
            m = big;
        }
    }
    if ((tid & 31) == 0) s_m[tid >> 5] = m, s_at[tid >> 5] = at, s_s[tid >> 5] = s;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 32; w++) {
            if (GREEDY) {
                s += s_s[w];
                if (ahead(s_m[w], s_at[w], m, at)) m = s_m[w], at = s_at[w];
            } else {
                const float big = fmaxf(m, s_m[w]);
                s = (m == big ? s : s * (double)expf((m - big) * a.inv)) + (s_m[w] == big ? s_s[w] : s_s[w] * (double)expf((s_m[w] - big) * a.inv));
                m = big;
            }
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
    for (int u = 0; u < kMaxPieces / 32; u++) s += GREEDY || x[u].m == m ? x[u].s : x[u].s * exp(((double)x[u].m - (double)m) * inv); // of a piece of no numbers: NaN times 0
    return {m, at, warp_sum_f64(s)};
}

// the row that the token behind the draft is drawn from
struct drawn_row {
    const float *p, *q;   // q: logits to take away from it, or null
    float mp, mq;
    double sp, sq;        // 1 / sum
    int64_t without;      // a token that falls out, or -1
};
__device__ __forceinline__ double weight(const drawn_row &d, float inv, int64_t v) {
    const float lp = d.p[v];
    double w = lp == -INFINITY ? 0.0 : (double)expf((lp - d.mp) * inv) * d.sp;
    if (d.q) {
        const float lq = d.q[v];
        if (lq != -INFINITY) w -= (double)expf((lq - d.mq) * inv) * d.sq;
    }
    return v == d.without || !(w > 0.0) ? 0.0 : w;
}

template <bool GREEDY> __global__ void __launch_bounds__(kThreads) verify_pick_kernel(const __grid_constant__ verify_args a) {
    __shared__ int s_first, s_extra;
    __shared__ bool s_last;
    __shared__ double s_sum[kThreads / 32], s_base;
    __shared__ int s_piece;
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
    for (int j = warp; j < drafts; j += kThreads / 32) {
        const int64_t r = r0 + j, d = a.drafted[r];
        const row_stats t = joined<GREEDY>(a.stats + r * 2 * a.pieces, a.pieces, a.inv64);
        bool stands = false;
        if (GREEDY) {
            stands = t.s == 0.0 && t.m > -INFINITY && d == t.at;
        } else {
            double q = 1.0;
            if (a.draft) {
                const row_stats s = joined<false>(a.stats + (r * 2 + 1) * a.pieces, a.pieces, a.inv64);
                q = d >= 0 && d < a.V ? exp(((double)a.draft[r * a.ld_d + d] - (double)s.m) * a.inv64) / s.s : 0.0;
            }
            const double p = d >= 0 && d < a.V ? exp(((double)a.target[r * a.ld_t + d] - (double)t.m) * a.inv64) / t.s : 0.0;
            stands = (double)a.u[r] * q < p; // with what is no number: no
        }
        if (!stands && lane == 0) atomicMin(&s_first, j);
    }
    __syncthreads();
    const int taken = s_first;
    const int64_t r = r0 + taken;
    const row_stats t = joined<GREEDY>(a.stats + r * 2 * a.pieces, a.pieces, a.inv64);
    if (GREEDY) {
        if (tid == 0) s_extra = t.s == 0.0 && t.m > -INFINITY ? t.at : -1;
    } else {
        drawn_row d{a.target + r * a.ld_t, nullptr, t.m, 0.f, 1.0 / t.s, 0.0, -1};
        bool valid = t.s > 0.0;
        if (taken < drafts) {
            if (a.draft) {
                const row_stats s = joined<false>(a.stats + (r * 2 + 1) * a.pieces, a.pieces, a.inv64);
                d.q = a.draft + r * a.ld_d, d.mq = s.m, d.sq = 1.0 / s.s;
                valid = valid && s.s > 0.0;
            } else {
                d.without = a.drafted[r];
            }
        }
        const int64_t v0 = blockIdx.x * a.piece, v1 = min(a.V, v0 + a.piece);
        double sum = 0.0;
        if (valid)
            for (int64_t v = v0 + tid; v < v1; v += kThreads) sum += weight(d, a.inv, v);
        sum = warp_sum_f64(sum);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kThreads / 32; w++) sum += s_sum[w];
            a.sums[(int64_t)seq * a.pieces + blockIdx.x] = sum;
            __threadfence();
            s_last = atomicAdd(&a.done[seq], 1u) == gridDim.x - 1;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        // ---- the last one: the piece whose running sum exceeds u times the whole, then the place in it
        if (tid == 0) {
            const volatile double *sums = a.sums + (int64_t)seq * a.pieces;
            double whole = 0.0;
            for (int c = 0; c < a.pieces; c++) whole += sums[c];
            s_piece = -1;
            s_extra = -1;
            if (valid && !(whole > 0.0) && (d.q || d.without >= 0)) { // rounding left nothing of p - q: from p
                d.q = nullptr, d.without = -1;
                s_piece = -2;
            } else if (valid && whole > 0.0) {
                const double to = (double)a.u[r0 + drafts] * whole;
                double run = 0.0;
                for (int c = 0; c < a.pieces; c++) {
                    if (!(sums[c] > 0.0)) continue;
                    s_piece = c, s_base = to - run; // the last one with anything in it, should none exceed
                    run += sums[c];
                    if (run > to) break;
                }
            }
        }
        __syncthreads();
        int64_t b0 = 0, b1 = 0;
        double to = s_base;
        if (s_piece == -2) { // rare: one sum over the whole row
            d.q = nullptr, d.without = -1;
            b1 = a.V, to = (double)a.u[r0 + drafts];
        } else if (s_piece >= 0) {
            b0 = s_piece * a.piece, b1 = min(a.V, b0 + a.piece);
        }
        if (b1 > b0) {
            const int64_t each = (b1 - b0 + kThreads - 1) / kThreads, w0 = min(b1, b0 + tid * each), w1 = min(b1, w0 + each);
            double mine = 0.0;
            int last = -1;
            for (int64_t v = w0; v < w1; v++) {
                const double w = weight(d, a.inv, v);
                mine += w;
                if (w > 0.0) last = (int)v;
            }
            double run = mine; // inclusive over the warp, then over the CTA
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const double x = __shfl_up_sync(0xffffffffu, run, off);
                if (lane >= off) run += x;
            }
            __syncthreads();
            if (lane == 31) s_sum[warp] = run;
            if (tid == 0) s_first = 0x7fffffff;
            __syncthreads();
            double base = 0.0;
            for (int w = 0; w < warp; w++) base += s_sum[w];
            if (base + run > to && mine > 0.0) atomicMin(&s_first, tid);
            __syncthreads();
            if (s_first == 0x7fffffff) { // none exceeds: the last place with a weight
                if (last >= 0) atomicMax(&s_extra, last);
            } else if (s_first == tid) {
                double at = base + run - mine;
                for (int64_t v = w0; v < w1; v++) {
                    const double w = weight(d, a.inv, v);
                    if (w > 0.0) s_extra = (int)v;
                    at += w;
                    if (at > to && w > 0.0) break;
                }
            }
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
