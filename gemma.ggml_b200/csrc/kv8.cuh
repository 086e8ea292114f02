// kv8.cuh — the 8-bit paged cache: its layout, and codes to and from numbers.
//
// A page holds block_size positions of every key head: G records of kv8_record() bytes, each the codes of the keys [block_size][D], those of the
// values [block_size][Dv], the keys' scales [block_size / 16] and the values', in whole 128 bytes.  A number is its code times the scale of its
// group: 16 consecutive positions of one head, keys and values apart.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include <algorithm>

#include "dense.cuh"
#include "tc.cuh"

constexpr int kKv8Group = 16;    // positions that share a scale
constexpr int kKv8MaxHead = 256; // numbers of a key or value

__host__ __device__ inline int64_t kv8_record(int D, int Dv, int B) { return ((int64_t)B * (D + Dv) + 2 * (B / kKv8Group) * 4 + 127) / 128 * 128; }
inline bool kv8_sizes_fit(int code, int H, int G, int D, int Dv, int B) {
    return (code == GGB_KV8_INT8 || code == GGB_KV8_E4M3) && H > 0 && G > 0 && H % G == 0 && D > 0 && D % 16 == 0 && D <= kKv8MaxHead && Dv > 0 && Dv % 16 == 0 &&
           Dv <= kKv8MaxHead && B > 0 && B % kKv8Group == 0 && B <= (1 << 20);
}

#ifdef __CUDACC__
// of the sequences s < n_seq, whose first places at(s) do not fall, the last one with at(s) <= t: whole warps, all lanes the answer
template <typename AT> __device__ __forceinline__ int last_not_behind(int n_seq, int64_t t, AT at) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seq;
    while (n > 1) {
        const int step = (n + 31) / 32, k = lane * step;
        const unsigned yes = __ballot_sync(0xffffffffu, k < n && at(lo + k) <= t);
        const int last = max(0, __popc(yes) - 1) * step;
        lo += last;
        n = min(step, n - last);
    }
    return lo;
}

template <int CODE> struct kv8_code;
template <> struct kv8_code<GGB_KV8_INT8> {
    static constexpr float top = 127.f, inv_top = (float)(1.0 / 127.0);
    __device__ static __forceinline__ float decode(uint8_t c) { return (float)(int8_t)c; }
    __device__ static __forceinline__ uint8_t encode(float y) { return (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(y, -top), top)); }
};
template <> struct kv8_code<GGB_KV8_E4M3> {
    static constexpr float top = 448.f, inv_top = (float)(1.0 / 448.0);
    __device__ static __forceinline__ float decode(uint8_t c) {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)c, __NV_E4M3)));
    }
    __device__ static __forceinline__ uint8_t encode(float y) { return (uint8_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3); }
};

namespace kv8 {

struct attn_args {
    const float *q;
    const uint8_t *cache;
    const int32_t *tables;
    int64_t table_ld;
    int B, n_seq;
    const int32_t *starts, *pos0;
    int H, G, D, Dv;
    int64_t window, keep;
    float cap;
    const float *sink, *gate;
    int64_t ldg, record;
    void *out;
    int entries, groups; // places for the items of a key head (list_items); as many for every sequence, or 0
    int64_t rows_above, rows_up_to; // sequences of more rows (tokens x query heads of a key head) than the one, up to the other, are this kernel's
    float *part;    // pieces' sums [CTA][2][rows][Dv], or null: an item a CTA
    float2 *part_ml; // their maxima and denominators [CTA][2][rows]
    int4 *desc;     // [CTA][2], of an item that begins or goes on here and ends elsewhere: sequence (or -1), rows, key head, first row; first and last CTA that have it, first token
    int vec_q, vec_out, vec_gate; // queries, results, rows of the gate begin on a 16-byte boundary
    int64_t positions; // that a page table has room for
    int *wait_error;
};
// four codes as two pairs of fp16 numbers.  int8: code + 128 behind the bits of 1024, less 1152
template <int CODE> __device__ __forceinline__ void halves_of(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (CODE == GGB_KV8_INT8) {
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
    } else {
        asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
    }
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2 *>(&h)); }

// a power of two that brings m to [2^to, 2^(to + 1)); 1 for zero
__device__ __forceinline__ float power_for(float m, int to) {
    const int e = (int)(__float_as_uint(m) >> 23) - 127;
    return m == 0.f ? 1.f : __uint_as_float((uint32_t)(min(max(to - e, -126), 126) + 127) << 23);
}

// a row's sums, relative to 2^m, over the denominator (with the sink), times the gate
struct row_end {
    float f; // what the sums are multiplied by
    __device__ __forceinline__ row_end(const attn_args &a, int h, float m, float l) {
        if (a.sink) {
            const float s = a.sink[h], M = fmaxf(m, s * kLog2e), c = m == -INFINITY ? 0.f : exp2f(m - M);
            f = c / fmaf(l, c, s == -INFINITY ? 0.f : exp2f(fmaf(s, kLog2e, fmaf(s, kLog2eRest, -M))));
        } else {
            f = 1.f / l;
        }
    }
};
__device__ __forceinline__ float gated(const attn_args &a, float y, int64_t t, int64_t at) { return a.gate ? y / (1.f + expf(-a.gate[t * a.ldg + at])) : y; }

constexpr int kQueryParts = 2; // fp16 numbers that stand for an fp32 query: 22 bits
constexpr float kNone = -3e38f; // a maximum of nothing: a number, so that the differences to it are

// What goes into the products with the codes is 2^(s - m) times the group's value scale, as fp16 numbers.  These have 11 bits above 2^-14 and lose them below, so the products
// are brought to the upper part of the range: each row keeps a power of two 2^d that its products are multiplied by, such that the largest one that it has met (of what it
// sees: a scale says nothing without a weight) was at 2^kNewWeight when it was found, and lets it grow to 2^kMostWeight.  Any other is off by its last
// bit or by half of fp16's smallest step, 2^-25, which is 2^-32 of that.  Maxima are whole numbers, so 2^d stays what it is when they move.  The denominator is a sum of its own,
// of 2^(s - m).  (Relative to the largest scale of a tile instead, seen or not, a row whose own values are 10^5 times smaller came out 2 % off, 10^8 times: zero.)
constexpr int kNewWeight = 7, kMostWeight = 15;
// a whole number that a scale's logarithm is below; not below -110, so that d stays one that 2^d exists of
__device__ __forceinline__ int scale_exponent(float v) { return max((int)(__float_as_uint(v) >> 23) - 126, -110); }
// v 2^d, |d| <= 126; a number where it is beyond all of them (the scale of a group whose weights are nothing)
__device__ __forceinline__ float scale_times(float v, int d) { return fminf(v * __uint_as_float((uint32_t)(127 + d) << 23), 3e38f); }

// the rows of an item and the tiles that they see: [0, n_keep) in kt tiles, then [lo, i1] in tiles from position TILE * w0 on
struct item {
    int s, rg, row0, rows; // rows [row0, row0 + rows) of the sequence: its tokens x the query heads of a key head
    int p0, i0, i1;        // positions of its first token, of the item's first and last
    int lo, n_keep, kt, w0, n;
    int64_t t0;            // its first token
};
template <int R, int TILE> __device__ __forceinline__ item item_of(const attn_args &a, int s, int rg) {
    item x;
    const int hpg = a.H / a.G;
    x.s = s, x.rg = rg, x.n = 0;
    if (s >= a.n_seq) return x; // behind the last place
    x.t0 = a.starts[s], x.p0 = a.pos0[s], x.row0 = rg * R;
    const int64_t all = (a.starts[s + 1] - x.t0) * hpg;
    x.rows = (int)min((int64_t)R, all - x.row0);
    if (x.rows <= 0 || all <= a.rows_above || all > a.rows_up_to) return x;
    x.i0 = x.p0 + x.row0 / hpg, x.i1 = x.p0 + (x.row0 + x.rows - 1) / hpg;
    x.lo = a.window > 0 ? (int)max((int64_t)0, x.i0 - a.window + 1) : 0;
    x.n_keep = (int)min(a.keep, (int64_t)x.lo);
    x.kt = (x.n_keep + TILE - 1) / TILE, x.w0 = x.lo / TILE;
    x.n = x.kt + x.i1 / TILE - x.w0 + 1;
    return x;
}

// The tiles of a call lie in one row, head by head of every item, each with kBegin units of no work ahead of its tiles (what it costs to begin an item).  CTA b of N has U / N of these units, and one more where b < U % N.
struct deal {
    unsigned each, more;
    __device__ __forceinline__ deal(unsigned U, unsigned N) : each(U / N), more(U - U / N * N) {}
    __device__ __forceinline__ unsigned first(unsigned b) const { return b * each + min(b, more); }
    __device__ __forceinline__ unsigned owner(unsigned u) const { return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each; }
};
// what a CTA works on at a time: tiles [tile, tile + n) of an item and head
struct piece {
    item it;
    int entry, head, tile, n;
    unsigned u; // the head's first unit
};
// The places of a head's items, R rows each.  Either every sequence has as many as max_new tokens take, or sequence s those from starts[s] * (H / G) / R + s on, at least as many as
// its rows fill: whichever are fewer, since every CTA goes through all of them, and limits count them (512 sequences of which one brings 8,192 tokens, eight query heads a key head: 262,144 places
// of 128 rows, or 1,055)
template <int R> __device__ __forceinline__ int first_place(const attn_args &a, int s) { return (int)((int64_t)a.starts[s] * (a.H / a.G) / R) + s; }
template <int R, int TILE> __device__ __forceinline__ void to_entry(const attn_args &a, piece &x, int entry) {
    int s, rg;
    if (a.groups > 0) {
        s = entry / a.groups, rg = entry - s * a.groups;
    } else {
        int n = a.n_seq + 1; // the last place that is not behind
        for (s = 0; n > 1;) {
            const int half = n / 2;
            if (first_place<R>(a, s + half) <= entry) s += half, n -= half;
            else n = half;
        }
        rg = entry - first_place<R>(a, s);
    }
    x.entry = entry, x.it = item_of<R, TILE>(a, s, rg);
}
template <int R, int TILE> __device__ __forceinline__ void next_entry(const attn_args &a, piece &x) {
    int s = x.it.s, rg = x.it.rg + 1;
    x.entry++;
    if (s < a.n_seq && (a.groups > 0 ? rg == a.groups : x.entry == first_place<R>(a, s + 1))) s++, rg = 0;
    x.it = item_of<R, TILE>(a, s, rg);
}
// places of R rows for calls of up to T tokens, max_new a sequence
inline int64_t list_items(attn_args &a, int64_t T, int64_t max_new, int R) {
    const int64_t hpg = a.H / a.G, groups = (max_new * hpg + R - 1) / R, even = a.n_seq * groups, own = T * hpg / R + a.n_seq;
    a.groups = even <= own ? (int)groups : 0; // (no more than own, which is below 2^31 where it is used)
    return std::min(even, own);
}
// the first piece from unit `at` on, which lies in the head that begins at x.u; n 0: none ahead of `end`
template <int R, int TILE, int kBegin> __device__ __forceinline__ void piece_from(const attn_args &a, piece &x, unsigned at, unsigned end) {
    for (;;) {
        x.tile = max(0, (int)(at - x.u) - kBegin), x.n = (int)min((unsigned)(x.it.n + kBegin), end - x.u) - kBegin - x.tile;
        if (x.n > 0) return;
        x.n = 0, x.u += x.it.n + kBegin, at = x.u;
        if (at >= end) return;
        if (++x.head == a.G) {
            x.head = 0;
            do next_entry<R, TILE>(a, x);
            while (x.it.n == 0);
        }
    }
}

__device__ __forceinline__ uint4 lds_u4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds_u2(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
// the cache as lines of 128 bytes (a record is whole lines, and 16 rows of it are): boxes of a group's keys and of its values, piece c of line l of a box at place
// c ^ (l & 7), so that a quarter of a warp reads pieces of several rows from different banks
struct line_maps {
    CUtensorMap k, v;
};
__device__ __forceinline__ void request(const line_maps &m, uint32_t k_dst, uint32_t v_dst, int k_line, int v_line, uint32_t bytes, uint32_t bar) { // one lane
    mbar_expect_tx(bar, bytes);
    tma_load_2d(k_dst, &m.k, 0, k_line, bar);
    tma_load_2d(v_dst, &m.v, 0, v_line, bar);
}
__device__ __forceinline__ uint32_t in_box(int byte) { return (uint32_t)(byte & ~127) + ((((byte >> 4) & 7) ^ ((byte >> 7) & 7)) << 4) + (byte & 15); }
inline int make_line_maps(const attn_args &a, line_maps &m) { // (as many lines as a coordinate reaches: where the pool ends is the page tables' matter)
    const int rc = ggb_tensor_map_bf16(&m.k, a.cache, (1ll << 31) - 1, 64, 64, a.D / 8);
    return rc ? rc : ggb_tensor_map_bf16(&m.v, a.cache, (1ll << 31) - 1, 64, 64, a.Dv / 8);
}

} // namespace kv8
#endif
