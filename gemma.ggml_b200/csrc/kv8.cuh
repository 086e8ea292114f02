// kv8.cuh — the 8-bit paged cache: its layout, and codes to and from numbers.
//
// A page holds block_size positions of every key head: G records of kv8_record() bytes, each the codes of the keys [block_size][D], those of the
// values [block_size][Dv], the keys' scales [block_size / 16] and the values', in whole 128 bytes.  A number is its code times the scale of its
// group: 16 consecutive positions of one head, keys and values apart.
#pragma once

#include <cuda_fp8.h>
#include <stdint.h>

#include "common.cuh"

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
#endif
