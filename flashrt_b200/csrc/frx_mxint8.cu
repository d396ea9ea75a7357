// MXINT8: activations kept in 8 bits for a backward pass. Rows to 8 bits and back, SwiGLU that keeps its gate and up rows in 8 bits in the same pass, and its
// gradient from what was kept (frx_mxint8_* in frx.h).
#include <algorithm>
#include <type_traits>

#include "frx_mx.cuh"
#include "frx_rows.cuh"

namespace frx {
namespace {

constexpr int kPer = 8;   // values a thread takes at a time: 16 bytes of 16-bit elements; four threads a block of 32

// kPer values from (or to) consecutive elements: in accesses of 16 bytes where rows allow it (VEC), else element by element
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* p, T (&v)[kPer]) {
    constexpr int N = VEC ? 16 / int(sizeof(T)) : 1;
#pragma unroll
    for (int j = 0; j < kPer; j += N) *reinterpret_cast<Vec<T, N>*>(v + j) = load_last(reinterpret_cast<const Vec<T, N>*>(p + j));
}
template <class T, bool VEC>
__device__ __forceinline__ void put8(T* p, const float (&f)[kPer]) {
    constexpr int N = VEC ? 16 / int(sizeof(T)) : 1;
#pragma unroll
    for (int j = 0; j < kPer; j += N) {
        Vec<T, N> o;
#pragma unroll
        for (int k = 0; k < N; ++k) o.v[k] = from_float<T>(f[j + k]);
        *reinterpret_cast<Vec<T, N>*>(p + j) = o;
    }
}

// The bits of the largest magnitude of a thread's values as a 32-bit float, infinity above all numbers and NaN above that. Pairs of 16-bit elements are compared as they are.
template <class T>
__device__ __forceinline__ uint32_t largest(const T (&v)[kPer]) {
    if constexpr (sizeof(T) == 4) {
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
        return amax;
    } else {
        using Two = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
        const Two* two = reinterpret_cast<const Two*>(v);
        Two top = __habs2(two[0]);
#pragma unroll
        for (int j = 1; j < kPer / 2; ++j) top = __hmax2_nan(top, __habs2(two[j]));
        return __float_as_uint(to_float(__hmax_nan(top.x, top.y))) & 0x7fffffffu;
    }
}

// A quarter of a block of 32 to its codes; amax: `largest` of the quarter. The block's four lanes get the scale byte, the exponent field of its largest magnitude (0 for a subnormal one:
// 2^-127), 255 where there is a NaN or an infinity. One rounding: the value times 2^(6 - e), plus 1.5 * 2^23, is rounded to an integer, ties to even, in one fused step, and the code is its low
// byte (the conversion instructions have a quarter of the rate). A magnitude beyond 127.5 steps gives 128, the byte 0x80, which no other value has: these few are formed again, within +-127.
__device__ __forceinline__ uint2 codes8(const float (&f)[kPer], uint32_t amax, uint32_t& byte) {
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    byte = amax >> 23;
    if (byte == 255u) return make_uint2(0u, 0u);
    constexpr float kRound = 12582912.0f;   // 1.5 * 2^23
    const float inv = __uint_as_float((260u - max(byte, 6u)) << 23);   // 2^(133 - byte), which 32 bits hold from a byte of 6 on
    float v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = fmaf(f[j], inv, kRound);
    auto word = [&](int j) {
        return __byte_perm(__byte_perm(__float_as_uint(v[j]), __float_as_uint(v[j + 1]), 0x0040), __byte_perm(__float_as_uint(v[j + 2]), __float_as_uint(v[j + 3]), 0x0040), 0x5410);
    };
    uint2 w = make_uint2(word(0), word(4));
    auto minus128 = [](uint32_t x) { return x & ~((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) & 0x80808080u; };   // a byte's top bit where the byte is 0x80
    if (byte < 6u || (minus128(w.x) | minus128(w.y)) != 0) {
        const float two = byte < 6u ? __uint_as_float((254u - byte) << 23) : 1.0f, one = byte < 6u ? 64.0f : inv;   // (two exact steps for a scale of the lowest ones)
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = fminf(fmaxf(fmaf(f[j] * two, one, kRound), kRound - 127.0f), kRound + 127.0f);
        w = make_uint2(word(0), word(4));
    }
    return w;
}
// and back: q * 2^(byte - 133), exact
__device__ __forceinline__ void values8(uint2 codes, uint32_t byte, float (&f)[kPer]) {
    const float s = mx_scale(byte) * 0.015625f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = float(int8_t((j < 4 ? codes.x : codes.y) >> (8 * (j & 3)))) * s;
}

// s = 1 / (1 + exp(-g)) and c = 1 - s, neither by a difference. For 16-bit results the hardware's exponential and reciprocal: relative errors of 2^-22 + |g| 1.25 * 2^-24 and 2^-23; 0 where exp(-|g|)
// is below 2^-126. (The passes are bounded by memory only as long as a pair of values takes some 40 instructions, of which every one counts: with five more, and conversion instructions for the codes, SwiGLU took 60
// us instead of 53; for 32-bit results, which move twice the bytes, the functions of the library.)
template <class T>
__device__ __forceinline__ void sigmoid(float g, float& s, float& c) {
    float e, r;
    if constexpr (sizeof(T) == 4) {
        e = expf(-fabsf(g));
        r = __fdiv_rn(1.0f, 1.0f + e);
    } else {
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(g) * -1.44269504f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    }
    const float er = e * r;
    s = g >= 0.0f ? r : er;
    c = g >= 0.0f ? er : r;
}

// Per value of x 4, 2 or 2 bytes in, 33 / 32 out: memory bounds it. U pieces a thread in flight. (Inputs are not __restrict__: the kernel in front may still write them when this one starts, so
// their loads must stay behind pdl_wait().)
template <class T, bool VEC, int U>
__global__ void __launch_bounds__(256) k_int8_quantize(const T* x, int64_t ldx, uint32_t pieces, uint32_t per_row, uint2* __restrict__ codes, uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    alignas(16) T v[U][kPer];
    const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = min(i0 + q * 256u, pieces - 1u), t = i / per_row;
        load8<T, VEC>(x + int64_t(t) * ldx + (i - t * per_row) * kPer, v[q]);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = i0 + q * 256u;
        float f[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) f[j] = to_float(v[q][j]);
        uint32_t byte;
        const uint2 c = codes8(f, largest(v[q]), byte);   // (whole blocks: pieces is a multiple of four)
        if (i < pieces) {
            codes[i] = c;
            if ((i & 3u) == 0) scales[i >> 2] = uint8_t(byte);
        }
    }
}

template <class T, bool VEC, int U>
__global__ void __launch_bounds__(256) k_int8_dequantize(const uint2* codes, const uint8_t* scales, uint32_t pieces, uint32_t per_row, T* __restrict__ x, int64_t ldx) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
    uint2 c[U];
    uint32_t byte[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = min(i0 + q * 256u, pieces - 1u);
        c[q] = __ldcs(codes + i);
        byte[q] = __ldcs(scales + (i >> 2));
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = i0 + q * 256u;
        if (i >= pieces) return;
        const uint32_t t = i / per_row;
        float f[kPer];
        values8(c[q], byte[q], f);
        put8<T, VEC>(x + int64_t(t) * ldx + (i - t * per_row) * kPer, f);
    }
}

// h = g s(g) u of rows [g | u], which are kept in 8 bits: per pair two elements in, one and 33 / 16 bytes out
template <class T, bool VEC, int U>
__global__ void __launch_bounds__(256) k_int8_swiglu(const T* gu, int64_t ldgu, uint32_t pieces, uint32_t per_row, uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                                                     T* __restrict__ h, int64_t ldh) {
    pdl_wait();
    pdl_trigger();
    alignas(16) T v[U][2][kPer];
    const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = min(i0 + q * 256u, pieces - 1u), t = i / per_row;
        const T* row = gu + int64_t(t) * ldgu + (i - t * per_row) * kPer;
        load8<T, VEC>(row, v[q][0]);
        load8<T, VEC>(row + per_row * kPer, v[q][1]);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = i0 + q * 256u, t = i / per_row, c = i - t * per_row;
        float g[kPer], u[kPer], o[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            g[j] = to_float(v[q][0][j]);
            u[j] = to_float(v[q][1][j]);
            float s, rest;
            sigmoid<T>(g[j], s, rest);
            o[j] = g[j] * s * u[j];
        }
        uint32_t byte_g, byte_u;
        const uint2 cg = codes8(g, largest(v[q][0]), byte_g), cu = codes8(u, largest(v[q][1]), byte_u);
        if (i < pieces) {
            put8<T, VEC>(h + int64_t(t) * ldh + c * kPer, o);
            const size_t at = size_t(t) * 2 * per_row + c;   // in pieces
            codes[at] = cg;
            codes[at + per_row] = cu;
            if ((c & 3u) == 0) {
                scales[at >> 2] = uint8_t(byte_g);
                scales[(at + per_row) >> 2] = uint8_t(byte_u);
            }
        }
    }
}

// From what was kept and gh, the gradient of h:  gg = gh u s (1 + g (1 - s)),  gu = gh g s,  and h again where it is asked for (for the gradient of the next matrix)
template <class T, bool VEC, int U>
__global__ void __launch_bounds__(256) k_int8_swiglu_grad(const T* gh, int64_t ldgh, const uint2* codes, const uint8_t* scales, uint32_t pieces, uint32_t per_row, T* __restrict__ ggu,
                                                          int64_t ldggu, T* __restrict__ h, int64_t ldh) {
    pdl_wait();
    pdl_trigger();
    alignas(16) T v[U][kPer];
    uint2 code[U][2];
    uint32_t byte[U][2];
    const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = min(i0 + q * 256u, pieces - 1u), t = i / per_row, c = i - t * per_row;
        const size_t at = size_t(t) * 2 * per_row + c;
        load8<T, VEC>(gh + int64_t(t) * ldgh + c * kPer, v[q]);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            code[q][m] = __ldcs(codes + at + m * per_row);
            byte[q][m] = __ldcs(scales + ((at + m * per_row) >> 2));
        }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = i0 + q * 256u, t = i / per_row, c = i - t * per_row;
        if (i >= pieces) return;
        float g[kPer], u[kPer], o[kPer];
        values8(code[q][0], byte[q][0], g);
        values8(code[q][1], byte[q][1], u);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            float s, rest;
            sigmoid<T>(g[j], s, rest);
            const float d = to_float(v[q][j]), gs = g[j] * s, us = u[j] * s;
            o[j] = gs * u[j];
            u[j] = d * gs;
            g[j] = d * us * (1.0f + g[j] * rest);
        }
        T* row = ggu + int64_t(t) * ldggu + c * kPer;
        put8<T, VEC>(row, g);
        put8<T, VEC>(row + per_row * kPer, u);
        if (h) put8<T, VEC>(h + int64_t(t) * ldh + c * kPer, o);
    }
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// f(T(), whether accesses of 16 bytes are possible, how many pieces a thread has in flight): of 16-bit elements four where that leaves blocks enough for every SM, of 32-bit ones two.
// 81,920 rows of 2 x 512 bf16: SwiGLU 53 us, its gradient 67 (70 with two; 6.3 TB/s of what has to move, a copy 6.4); f32 89 and 116 (6.6 TB/s; with four 120 and 120).
template <class F>
void with_type(int dtype, bool vec, uint64_t pieces, F f) {
    auto flight = [&](auto v, auto wide) {
        if (pieces >= (uint64_t(1) << 19))
            f(v, wide, std::integral_constant<int, sizeof(v) == 2 ? 4 : 2>{});
        else
            f(v, wide, std::integral_constant<int, 1>{});
    };
    auto typed = [&](auto v) { vec ? flight(v, std::true_type{}) : flight(v, std::false_type{}); };
    if (dtype == FRX_F32)
        typed(float{});
    else if (dtype == FRX_BF16)
        typed(__nv_bfloat16{});
    else
        typed(__half{});
}

int sizes(const char* who, int dtype, int T, int n) {
    if (T < 0 || n < 0) return fail(FRX_ERR_ARG, "%s: %d rows of %d values", who, T, n);
    if (n % kMxBlock || n > (1 << 30)) return fail(FRX_ERR_SHAPE, "%s: rows of %d values are not whole blocks of 32", who, n);
    if (!dtype_size(dtype)) return fail(FRX_ERR_ARG, "%s: element type %d", who, dtype);
    if (uint64_t(T) * uint64_t(n / kPer) > 0xffffff00ull) return fail(FRX_ERR_SHAPE, "%s: %d rows of %d values", who, T, n);
    return FRX_OK;
}
int rows_arg(const char* who, const char* what, const void* x, int64_t ld, int64_t n, int dtype) {
    if (!x) return fail(FRX_ERR_ARG, "%s: null pointer (%s)", who, what);
    if (ld < n) return fail(FRX_ERR_ARG, "%s: rows of %s are %lld elements apart and %lld long", who, what, (long long)ld, (long long)n);
    if (!rows_aligned(x, dtype_size(dtype))) return fail(FRX_ERR_ARG, "%s: misaligned pointer (%s)", who, what);
    return FRX_OK;
}
int codes_arg(const char* who, const void* codes, const void* scales) {
    if (!codes || !scales) return fail(FRX_ERR_ARG, "%s: null pointer (codes, scales)", who);
    if (!aligned(codes, 8)) return fail(FRX_ERR_ARG, "%s: misaligned pointer (codes)", who);
    return FRX_OK;
}
template <int U>
dim3 grid_of(uint64_t pieces) { return dim3(unsigned((pieces + 256 * U - 1) / (256 * U))); }

}  // namespace
}  // namespace frx

using namespace frx;

extern "C" {

int frx_mxint8_quantize(frx_stream_t stream, const void* x, int64_t ldx, int dtype, int T, int n, void* codes, void* scales) {
    const char* who = "frx_mxint8_quantize";
    int rc = sizes(who, dtype, T, n);
    if (rc != FRX_OK || T == 0 || n == 0) return rc;
    if ((rc = rows_arg(who, "x", x, ldx, n, dtype)) != FRX_OK || (rc = codes_arg(who, codes, scales)) != FRX_OK) return rc;
    const uint64_t pieces = uint64_t(T) * uint64_t(n / kPer);
    with_type(dtype, rows_vec16(x, ldx, n, dtype_size(dtype)), pieces, [&](auto v, auto vec, auto u) {
        using V = decltype(v);
        constexpr int U = decltype(u)::value;
        FRX_LAUNCH(kKQuant, stream, launch_pdl(k_int8_quantize<V, decltype(vec)::value, U>, grid_of<U>(pieces), dim3(256), 0, stream, static_cast<const V*>(x), ldx, uint32_t(pieces),
                                               uint32_t(n / kPer), static_cast<uint2*>(codes), static_cast<uint8_t*>(scales)));
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_mxint8_dequantize(frx_stream_t stream, const void* codes, const void* scales, int T, int n, int dtype, void* x, int64_t ldx) {
    const char* who = "frx_mxint8_dequantize";
    int rc = sizes(who, dtype, T, n);
    if (rc != FRX_OK || T == 0 || n == 0) return rc;
    if ((rc = rows_arg(who, "x", x, ldx, n, dtype)) != FRX_OK || (rc = codes_arg(who, codes, scales)) != FRX_OK) return rc;
    const uint64_t pieces = uint64_t(T) * uint64_t(n / kPer);
    with_type(dtype, rows_vec16(x, ldx, n, dtype_size(dtype)), pieces, [&](auto v, auto vec, auto u) {
        using V = decltype(v);
        constexpr int U = decltype(u)::value;
        FRX_LAUNCH(kKQuant, stream, launch_pdl(k_int8_dequantize<V, decltype(vec)::value, U>, grid_of<U>(pieces), dim3(256), 0, stream, static_cast<const uint2*>(codes),
                                               static_cast<const uint8_t*>(scales), uint32_t(pieces), uint32_t(n / kPer), static_cast<V*>(x), ldx));
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_mxint8_swiglu(frx_stream_t stream, const void* gu, int64_t ldgu, int dtype, int T, int ff, void* codes, void* scales, void* h, int64_t ldh) {
    const char* who = "frx_mxint8_swiglu";
    int rc = sizes(who, dtype, T, ff);
    if (rc != FRX_OK || T == 0 || ff == 0) return rc;
    if ((rc = rows_arg(who, "gu", gu, ldgu, int64_t(2) * ff, dtype)) != FRX_OK || (rc = rows_arg(who, "h", h, ldh, ff, dtype)) != FRX_OK || (rc = codes_arg(who, codes, scales)) != FRX_OK) return rc;
    const uint64_t pieces = uint64_t(T) * uint64_t(ff / kPer);
    const int size = dtype_size(dtype);
    with_type(dtype, rows_vec16(gu, ldgu, ff, size) && rows_vec16(h, ldh, ff, size), pieces, [&](auto v, auto vec, auto u) {
        using V = decltype(v);
        constexpr int U = decltype(u)::value;
        FRX_LAUNCH(kKSwiglu, stream, launch_pdl(k_int8_swiglu<V, decltype(vec)::value, U>, grid_of<U>(pieces), dim3(256), 0, stream, static_cast<const V*>(gu), ldgu, uint32_t(pieces),
                                               uint32_t(ff / kPer), static_cast<uint2*>(codes), static_cast<uint8_t*>(scales), static_cast<V*>(h), ldh));
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_mxint8_swiglu_backward(frx_stream_t stream, const void* gh, int64_t ldgh, const void* codes, const void* scales, int dtype, int T, int ff, void* ggu, int64_t ldggu, void* h,
                               int64_t ldh) {
    const char* who = "frx_mxint8_swiglu_backward";
    int rc = sizes(who, dtype, T, ff);
    if (rc != FRX_OK || T == 0 || ff == 0) return rc;
    if ((rc = rows_arg(who, "gh", gh, ldgh, ff, dtype)) != FRX_OK || (rc = codes_arg(who, codes, scales)) != FRX_OK ||
        (rc = rows_arg(who, "ggu", ggu, ldggu, int64_t(2) * ff, dtype)) != FRX_OK || (h && (rc = rows_arg(who, "h", h, ldh, ff, dtype)) != FRX_OK))
        return rc;
    const uint64_t pieces = uint64_t(T) * uint64_t(ff / kPer);
    const int size = dtype_size(dtype);
    with_type(dtype, rows_vec16(gh, ldgh, ff, size) && rows_vec16(ggu, ldggu, ff, size) && (!h || rows_vec16(h, ldh, ff, size)), pieces, [&](auto v, auto vec, auto u) {
        using V = decltype(v);
        constexpr int U = decltype(u)::value;
        FRX_LAUNCH(kKSwiglu, stream, launch_pdl(k_int8_swiglu_grad<V, decltype(vec)::value, U>, grid_of<U>(pieces), dim3(256), 0, stream, static_cast<const V*>(gh), ldgh,
                                               static_cast<const uint2*>(codes), static_cast<const uint8_t*>(scales), uint32_t(pieces), uint32_t(ff / kPer), static_cast<V*>(ggu), ldggu,
                                               static_cast<V*>(h), ldh));
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

}  // extern "C"
