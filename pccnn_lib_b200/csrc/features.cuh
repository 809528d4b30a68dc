// Loads and stores of feature vectors in float32 or bfloat16: V consecutive elements (1, 2, 4 or 8) as accesses of up to 16
// bytes, which the address has to be aligned to.  Arithmetic is 32-bit throughout.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace pccnn {

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

#ifdef __CUDACC__

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
// The one rounding of a bf16 result: to nearest, from a 32-bit value.
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <class T, int V>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&v)[V]) {
    if constexpr (sizeof(T) == 4 && V % 4 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 r = *reinterpret_cast<const float4*>(p + i);
            v[i] = r.x, v[i + 1] = r.y, v[i + 2] = r.z, v[i + 3] = r.w;
        }
    } else if constexpr (sizeof(T) == 2 && V == 8) {
        const uint4 r = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else if constexpr (sizeof(T) == 4 && V == 2) {
        const float2 r = *reinterpret_cast<const float2*>(p);
        v[0] = r.x, v[1] = r.y;
    } else if constexpr (sizeof(T) == 2 && V == 4) {
        const uint2 r = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(r.x << 16), v[1] = __uint_as_float(r.x & 0xffff0000u);
        v[2] = __uint_as_float(r.y << 16), v[3] = __uint_as_float(r.y & 0xffff0000u);
    } else if constexpr (sizeof(T) == 2 && V == 2) {
        const uint32_t r = *reinterpret_cast<const uint32_t*>(p);
        v[0] = __uint_as_float(r << 16), v[1] = __uint_as_float(r & 0xffff0000u);
    } else {
        static_assert(V == 1, "1, 2, 4 or 8 elements");
        v[0] = to_float(p[0]);
    }
}

// The same vector as it lies in memory, for loads that stay in flight while other rows are worked on.
template <int BYTES> struct RawBytes;
template <> struct RawBytes<16> { using type = uint4; };
template <> struct RawBytes<8> { using type = uint2; };
template <> struct RawBytes<4> { using type = uint32_t; };
template <> struct RawBytes<2> { using type = uint16_t; };
template <class T, int V>
struct RawVec {
    typename RawBytes<V * sizeof(T)>::type v;
    __device__ __forceinline__ void load(const T* __restrict__ p) { v = *reinterpret_cast<const decltype(v)*>(p); }
    __device__ __forceinline__ void clear() { v = decltype(v)(); }
    __device__ __forceinline__ void widen(float (&x)[V]) const {
        constexpr int kWords = V * sizeof(T) < 4 ? 1 : V * sizeof(T) / 4;
        uint32_t w[kWords];
        if constexpr (sizeof(v) == 16) w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        else if constexpr (sizeof(v) == 8) w[0] = v.x, w[1] = v.y;
        else w[0] = v;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                x[i] = __uint_as_float(w[i]);
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                if constexpr (V > 1) x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <class T, int V>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&v)[V]) {
    if constexpr (sizeof(T) == 4 && V % 4 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if constexpr (sizeof(T) == 2 && V == 8) {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    } else if constexpr (sizeof(T) == 4 && V == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else if constexpr (sizeof(T) == 2 && V == 4) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else if constexpr (sizeof(T) == 2 && V == 2) {
        *reinterpret_cast<uint32_t*>(p) = pack_bf16(v[0], v[1]);
    } else {
        static_assert(V == 1, "1, 2, 4 or 8 elements");
        p[0] = from_float<T>(v[0]);
    }
}

#endif  // __CUDACC__

}  // namespace pccnn
