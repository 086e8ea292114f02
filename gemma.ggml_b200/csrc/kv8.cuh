// kv8.cuh — the 8-bit paged cache: its layout, and codes to and from numbers.
//
// A page holds block_size positions of every key head: G records of kv8_record() bytes, each the codes of the keys [block_size][D], those of the
// values [block_size][Dv], the keys' scales [block_size / 16] and the values', in whole 128 bytes.  A number is its code times the scale of its
// group: 16 consecutive positions of one head, keys and values apart.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

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
    int groups;     // items of a sequence and key head, at most
    float *part;    // [CTA][2][rows][Dv + 2], or null: an item a CTA
    int4 *desc;     // [CTA][2], of an item that begins or goes on here and ends elsewhere: sequence (or -1), rows, key head, first row; first and last CTA that have it, first token
    int vec_q;      // queries begin on a 16-byte boundary
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

} // namespace kv8
#endif
