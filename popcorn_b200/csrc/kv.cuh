// What the paged 8-bit key/value cache's kernels share: element types,
// sequence lookup and the error bits of out-of-range pages and positions.
#ifndef POPCORN_B200_KV_CUH
#define POPCORN_B200_KV_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "popcorn_serve.h"

namespace pcb {

// A block scale below this counts as zero (and its codes are zero).
constexpr float kKvSmallestScale = 8.271806125530277e-25f;  // 2^-80

// Error bits (popcornB200DeviceErrors, shifted by 16).
constexpr unsigned int kKvErrAppend = 0x2000u;
constexpr unsigned int kKvErrAttention = 0x4000u;

// Whether the cache's own sizes and alignment are ones that the kernels take.
inline bool kv_cache_supported(const popcornKvCache_t& c) {
    const int64_t p = c.page_size;
    return c.pages > 0 && c.pages <= INT32_MAX && c.heads > 0 && c.heads <= 65535 && p >= 16 && p <= 256 &&
           (p & (p - 1)) == 0 && c.dim >= 16 && c.dim <= 256 && c.dim % 16 == 0 && aligned16(c.k) && aligned16(c.v);
}

inline bool kv_type_supported(popcornType_t t) {
    return t == POPCORN_TYPE_F32 || t == POPCORN_TYPE_F16 || t == POPCORN_TYPE_BF16;
}

inline int64_t kv_type_size(popcornType_t t) { return t == POPCORN_TYPE_F32 ? 4 : 2; }

inline int log2_of(int64_t p) {
    int s = 0;
    while ((int64_t{1} << s) < p) ++s;
    return s;
}

#ifdef __CUDACC__
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four consecutive elements: one load where the caller knows that p is
// aligned to four elements (vec), else four.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float (&v)[4]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(p);
            const T* h = reinterpret_cast<const T*>(&a);
            #pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = to_f32(h[i]);
        }
    } else {
        #pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32(p[i]);
    }
}

// The counterpart of load4, each value rounded once.
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, const float (&v)[4]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint2 a;
            T* h = reinterpret_cast<T*>(&a);
            #pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = from_f32<T>(v[i]);
            *reinterpret_cast<uint2*>(p) = a;
        }
    } else {
        #pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = from_f32<T>(v[i]);
    }
}

// The sequence whose rows first[b] .. first[b + 1] - 1 hold row t: the number
// of entries first[1 ..] that are <= t, counted 32 at a time by the warp (one
// memory latency for 32 sequences, where a binary search takes one per step).
// All lanes call it with the same t; the result is at most seqs.
__device__ __forceinline__ int64_t sequence_of(const int32_t* first, int64_t seqs, int64_t t, int lane) {
    int64_t b = 0;
    for (int64_t i = 0; i < seqs; i += 32) {
        const bool below = i + lane < seqs && first[i + lane + 1] <= t;
        b += __popc(__ballot_sync(0xffffffffu, below));
    }
    return b;
}
#endif

}  // namespace pcb

#endif  // POPCORN_B200_KV_CUH
