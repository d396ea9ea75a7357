// Element types of the row operators (frx.h: FRX_F32, FRX_BF16, FRX_F16) and rows read and written in vectors.
#pragma once

#include <cuda_bf16.h>

#include "frx_common.cuh"

namespace frx {

inline int dtype_size(int dtype) { return dtype == FRX_F32 ? 4 : (dtype == FRX_BF16 || dtype == FRX_F16) ? 2 : 0; }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements, moved in one access (16 bytes, or a single element where rows do not allow more)
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

// A vector that is not needed again after this read: its lines are the first to leave the L2.
template <class V>
__device__ __forceinline__ V load_last(const V* p) {
    if constexpr (sizeof(V) == 16) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
        return *reinterpret_cast<const V*>(&u);
    } else {
        return *p;
    }
}

// Whether rows of n elements at `p`, `ld` elements apart, can be moved 16 bytes at a time.
inline bool rows_vec16(const void* p, int64_t ld, int n, int size) {
    return (reinterpret_cast<uintptr_t>(p) % 16) == 0 && (ld * size) % 16 == 0 && (int64_t(n) * size) % 16 == 0;
}
inline bool rows_aligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// f(T(), integral constant N): the element type and how many of them are moved at a time
template <class F>
inline void with_rows(int dtype, bool vec, F f) {
    if (dtype == FRX_F32) {
        if (vec)
            f(float{}, std::integral_constant<int, 4>{});
        else
            f(float{}, std::integral_constant<int, 1>{});
    } else if (dtype == FRX_BF16) {
        if (vec)
            f(__nv_bfloat16{}, std::integral_constant<int, 8>{});
        else
            f(__nv_bfloat16{}, std::integral_constant<int, 1>{});
    } else {
        if (vec)
            f(__half{}, std::integral_constant<int, 8>{});
        else
            f(__half{}, std::integral_constant<int, 1>{});
    }
}

}  // namespace frx
