// MXFP4: the quantizer, the way back, the layout that the product reads, the product (dense, and grouped by expert), and
// the expert layer made of them.
#include <algorithm>
#include <type_traits>

#include "frx_mx.cuh"
#include "frx_rows.cuh"
#include "frx_sort.cuh"

namespace frx {
namespace {

// ---- quantizer. A thread takes 16 values (two threads a block of 32): per value 2 or 4 bytes in, 17 / 32 out, so bandwidth bounds it.
template <class T>
__global__ void __launch_bounds__(256) k_mx_quantize(const T* __restrict__ x, int64_t ldx, uint32_t pieces, uint32_t per_row, uint2* __restrict__ codes,
                                                     uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;   // (pairs of threads are whole: pieces is even)
    if (i >= pieces) return;
    const uint32_t t = i / per_row, c = i - t * per_row;
    constexpr int kPer = 16 / int(sizeof(T));
    Vec<T, kPer> v[16 / kPer];
#pragma unroll
    for (int j = 0; j < 16 / kPer; ++j) v[j] = *reinterpret_cast<const Vec<T, kPer>*>(x + int64_t(t) * ldx + c * 16 + j * kPer);
    float f[2][8];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        f[j / 8][j % 8] = to_float(v[j / kPer].v[j % kPer]);
        amax = max(amax, __float_as_uint(f[j / 8][j % 8]) & 0x7fffffffu);   // (the bits of magnitudes are in their order, infinity and NaN on top)
    }
    amax = max(amax, __shfl_xor_sync(__activemask(), amax, 1));
    const uint32_t byte = mx_scale_byte(amax);
    const float inv = mx_inverse(min(byte, 253u));
#pragma unroll
    for (int j = 0; j < 16; ++j) f[j / 8][j % 8] *= inv;
    uint2 out = make_uint2(mx_codes8(f[0]), mx_codes8(f[1]));
    if (byte == 255u) out = make_uint2(0u, 0u);
    codes[i] = out;
    if ((i & 1u) == 0) scales[i >> 1] = uint8_t(byte);
}
// rows that do not start on 16 bytes: a warp per block of 32, a lane per value
template <class T>
__global__ void __launch_bounds__(256) k_mx_quantize_any(const T* __restrict__ x, int64_t ldx, uint32_t blocks, uint32_t per_row, uint32_t* __restrict__ codes,
                                                         uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    const uint32_t b = blockIdx.x * 8u + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
    if (b >= blocks) return;
    const uint32_t t = b / per_row;
    const float v = to_float(x[int64_t(t) * ldx + (b - t * per_row) * kMxBlock + lane]);
    const uint32_t byte = mx_scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
    const float mine = v * mx_inverse(min(byte, 253u));
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __shfl_sync(0xffffffffu, mine, (lane & ~7u) + j);
    const uint32_t w = byte == 255u ? 0u : mx_codes8(f);
    if ((lane & 7u) == 0) codes[size_t(b) * 4 + lane / 8] = w;
    if (lane == 0) scales[b] = uint8_t(byte);
}

template <class T, int N>
__global__ void __launch_bounds__(256) k_mx_dequantize(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t pieces, uint32_t per_row, T* __restrict__ x,
                                                       int64_t ldx) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;   // eight values
    if (i >= pieces) return;
    const uint32_t t = i / per_row, c = i - t * per_row;
    float f[8];
    mx_values8(codes[i], f);
    const float s = mx_scale(scales[i >> 2]);
    T* out = x + int64_t(t) * ldx + c * 8;
#pragma unroll
    for (int j = 0; j < 8; j += N) {
        Vec<T, N> o;
#pragma unroll
        for (int k = 0; k < N; ++k) o.v[k] = from_float<T>(f[j + k] * s);
        *reinterpret_cast<Vec<T, N>*>(out + j) = o;
    }
}

// ---- layout (frx_mxfp4_pack in frx.h): a block per unit of 128 rows x 128 columns, a thread per row
template <bool PACK>
__global__ void __launch_bounds__(kMxTileRows) k_mx_pack(uint4* __restrict__ codes, uint32_t* __restrict__ scales, int rows, int units, int tiles, uint8_t* __restrict__ packed) {
    const int r = threadIdx.x, u = blockIdx.x % units;
    const int64_t et = blockIdx.x / units;   // tile of all matrices
    const int row = int(et % tiles) * kMxTileRows + r;
    const bool have = row < rows;
    uint8_t* unit = packed + size_t(blockIdx.x) * kMxUnitBytes;
    uint4* plane = reinterpret_cast<uint4*>(unit) + r;
    uint32_t* scale = reinterpret_cast<uint32_t*>(unit + kMxUnitCode + (r % 32) * 16 + (r / 32) * 4);
    const size_t at = (size_t(et / tiles) * rows + row) * units + u;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (PACK)
            plane[c * kMxTileRows] = have ? codes[at * 4 + c] : make_uint4(0u, 0u, 0u, 0u);
        else if (have)
            codes[at * 4 + c] = plane[c * kMxTileRows];
    }
    if (PACK)
        *scale = have ? scales[at] : 0x7f7f7f7fu;   // rows that fill a tile up are zeros times 1
    else if (have)
        scales[at] = *scale;
}

// ---- product
struct MxProduct {
    const uint8_t* w;        // packed matrices
    const uint8_t* codes;    // activations [x_rows][n / 2]
    const uint8_t* scales;   // [x_rows][n / 32]
    const int32_t* offsets;  // [E + 1] rows of every expert; null: one matrix, all rows
    const int32_t* slot_of;  // the x row of sorted row r is slot_of[r] / K; null: r
    void* y;
    int64_t ldy;
    int E, rows, n, K, x_rows, S;   // rows: of a matrix; S: rows of y
    int y_type;
};

__device__ __forceinline__ void store_y(const MxProduct& p, int64_t r, int row, float v) {
    if (p.y_type == FRX_F32)
        static_cast<float*>(p.y)[r * p.ldy + row] = v;
    else if (p.y_type == FRX_BF16)
        static_cast<__nv_bfloat16*>(p.y)[r * p.ldy + row] = __float2bfloat16_rn(v);
    else
        static_cast<__half*>(p.y)[r * p.ldy + row] = __float2half_rn(v);
}

// A thread per matrix row and eight y rows.
__global__ void __launch_bounds__(kMxTileRows) k_mx_product(const MxProduct p) {
    __shared__ int item[3];
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) {
        int left = int(blockIdx.x), e = 0, a = 0, b = p.offsets ? 0 : p.S;
        item[0] = -1;
        for (; e < p.E; ++e) {
            if (p.offsets) {
                a = min(max(p.offsets[e], 0), p.S);
                b = min(max(p.offsets[e + 1], a), p.S);
            }
            const int items = (b - a + 7) / 8;
            if (left < items) {
                item[0] = e;
                item[1] = a + left * 8;
                item[2] = min(8, b - item[1]);
                break;
            }
            left -= items;
        }
    }
    __syncthreads();
    if (item[0] < 0) return;
    const int units = p.n / kMxUnitK, tiles = (p.rows + kMxTileRows - 1) / kMxTileRows, r = threadIdx.x, row = blockIdx.y * kMxTileRows + r;
    const uint8_t* w = p.w + (size_t(item[0]) * tiles + blockIdx.y) * units * kMxUnitBytes;
    float acc[8] = {};
    for (int u = 0; u < units; ++u, w += kMxUnitBytes)
        for (int c = 0; c < 4; ++c) {   // a block of 32
            const uint32_t ws = w[kMxUnitCode + (r % 32) * 16 + (r / 32) * 4 + c];
            const uint4 wc = reinterpret_cast<const uint4*>(w)[c * kMxTileRows + r];
            const uint32_t ww[4] = {wc.x, wc.y, wc.z, wc.w};
            for (int j = 0; j < item[2]; ++j) {
                const int slot = p.slot_of ? p.slot_of[item[1] + j] : (item[1] + j) * p.K;
                const int t = slot / p.K;
                if (slot < 0 || t >= p.x_rows) continue;
                const size_t at = size_t(t) * (p.n / kMxBlock) + u * 4 + c;
                float sum = 0.0f;
                for (int q = 0; q < 4; ++q) {
                    float a[8], b[8];
                    mx_values8(ww[q], a);
                    mx_values8(reinterpret_cast<const uint32_t*>(p.codes)[at * 4 + q], b);
                    for (int i = 0; i < 8; ++i) sum = fmaf(a[i], b[i], sum);
                }
                acc[j] = fmaf(sum * mx_scale(ws), mx_scale(p.scales[at]), acc[j]);
            }
        }
    if (row < p.rows)
        for (int j = 0; j < item[2]; ++j) store_y(p, item[1] + j, row, acc[j]);
}

int launch_product(const MxProduct& p, cudaStream_t stream, int cls) {
    const int tiles = (p.rows + kMxTileRows - 1) / kMxTileRows;
    const dim3 grid(unsigned((int64_t(p.S) + 7) / 8 + (p.offsets ? p.E : 0)), unsigned(tiles));
    FRX_LAUNCH(cls, stream, launch_pdl(k_mx_product, grid, dim3(kMxTileRows), 0, stream, p));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

// h = silu(g) * u of the rows that experts have, to MXFP4: a warp per block of 32
__global__ void __launch_bounds__(256) k_mx_swiglu(const float* __restrict__ g, const float* __restrict__ u, const int32_t* __restrict__ n_rows, int ff, uint32_t* __restrict__ codes,
                                                   uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    const size_t b = size_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31u;
    if (b >= size_t(*n_rows) * (ff / kMxBlock)) return;
    const float a = g[b * kMxBlock + lane], v = a / (1.0f + expf(-a)) * u[b * kMxBlock + lane];
    const uint32_t byte = mx_scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
    const float mine = v * mx_inverse(min(byte, 253u));
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __shfl_sync(0xffffffffu, mine, (lane & ~7u) + j);
    const uint32_t w = byte == 255u ? 0u : mx_codes8(f);
    if ((lane & 7u) == 0) codes[b * 4 + lane / 8] = w;
    if (lane == 0) scales[b] = uint8_t(byte);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// where the layer keeps what it forms, in its workspace
struct LayerBuffers {
    size_t offsets, slot_of, row_of, sort, xq, xs, hq, hs, g, u, y, total;
};
LayerBuffers layer_buffers(int T, int K, int n, int ff, int E) {
    LayerBuffers b{};
    const size_t S = size_t(T) * K;
    size_t at = kAlign;
    auto take = [&](size_t& where, size_t bytes) {
        where = at;
        at += align_up(bytes);
    };
    take(b.offsets, (size_t(E) + 1) * 4);
    take(b.slot_of, S * 4);
    take(b.row_of, S * 4);
    take(b.sort, sort_scratch_bytes((long long)S, E));
    take(b.xq, size_t(T) * n / 2);
    take(b.xs, size_t(T) * n / kMxBlock);
    take(b.hq, S * ff / 2);
    take(b.hs, S * ff / kMxBlock);
    take(b.g, S * ff * 4);
    take(b.u, S * ff * 4);
    take(b.y, S * n * 4);
    b.total = at;
    return b;
}

int quantize(const char* who, const void* x, int64_t ldx, int dtype, int T, int n, void* codes, void* scales, cudaStream_t stream) {
    if (T < 0 || n < 0 || n % kMxBlock) return fail(T < 0 || n < 0 ? FRX_ERR_ARG : FRX_ERR_SHAPE, "%s: T %d, n %d (blocks of 32)", who, T, n);
    const int size = dtype_size(dtype);
    if (!size) return fail(FRX_ERR_ARG, "%s: element type %d", who, dtype);
    if (T == 0 || n == 0) return FRX_OK;
    if (!x || !codes || !scales) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (ldx < n) return fail(FRX_ERR_ARG, "%s: rows of x are %lld elements apart and %d long", who, (long long)ldx, n);
    if (!rows_aligned(x, size) || !aligned(codes, 16)) return fail(FRX_ERR_ARG, "%s: misaligned pointer", who);
    const uint64_t pieces = uint64_t(T) * uint64_t(n / 16);
    if (pieces > 0xffffff00ull) return fail(FRX_ERR_SHAPE, "%s: T %d, n %d", who, T, n);
    with_rows(dtype, true, [&](auto v, auto) {
        using T_ = decltype(v);
        if (rows_vec16(x, ldx, n, size))
            FRX_LAUNCH(kKQuant, stream, launch_pdl(k_mx_quantize<T_>, dim3(unsigned((pieces + 255) / 256)), dim3(256), 0, stream, static_cast<const T_*>(x), ldx, uint32_t(pieces),
                                                   uint32_t(n / 16), static_cast<uint2*>(codes), static_cast<uint8_t*>(scales)));
        else
            FRX_LAUNCH(kKQuant, stream, launch_pdl(k_mx_quantize_any<T_>, dim3(unsigned((pieces / 2 + 7) / 8)), dim3(256), 0, stream, static_cast<const T_*>(x), ldx,
                                                   uint32_t(pieces / 2), uint32_t(n / kMxBlock), static_cast<uint32_t*>(codes), static_cast<uint8_t*>(scales)));
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int product_args(const char* who, const void* codes, const void* scales, const void* w, int x_rows, int n, int E, int rows, const void* y, int64_t ldy, int y_type) {
    if (!codes || !scales || !w || !y) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (!dtype_size(y_type)) return fail(FRX_ERR_ARG, "%s: element type %d", who, y_type);
    if (x_rows < 0) return fail(FRX_ERR_ARG, "%s: %d rows of x", who, x_rows);
    if (n < kMxUnitK || n % kMxUnitK || rows < 1 || rows > 65535 * kMxTileRows || E < 1 || E > 4096)
        return fail(FRX_ERR_SHAPE, "%s: unsupported shape E %d, rows %d, n %d (n a multiple of 128)", who, E, rows, n);
    if (ldy < rows) return fail(FRX_ERR_ARG, "%s: rows of y are %lld elements apart and %d long", who, (long long)ldy, rows);
    if (!aligned(codes, 16) || !aligned(scales, 4) || !aligned(w, 16) || !rows_aligned(y, dtype_size(y_type))) return fail(FRX_ERR_ARG, "%s: misaligned pointer", who);
    return FRX_OK;
}

}  // namespace
}  // namespace frx

using namespace frx;

extern "C" {

int frx_mxfp4_quantize(frx_stream_t stream, const void* x, int64_t ldx, int dtype, int T, int n, void* codes, void* scales) {
    return quantize("frx_mxfp4_quantize", x, ldx, dtype, T, n, codes, scales, stream);
}

int frx_mxfp4_dequantize(frx_stream_t stream, const void* codes, const void* scales, int T, int n, int dtype, void* x, int64_t ldx) {
    const char* who = "frx_mxfp4_dequantize";
    if (T < 0 || n < 0 || n % kMxBlock) return fail(T < 0 || n < 0 ? FRX_ERR_ARG : FRX_ERR_SHAPE, "%s: T %d, n %d (blocks of 32)", who, T, n);
    if (dtype != FRX_F32 && dtype != FRX_BF16) return fail(FRX_ERR_ARG, "%s: element type %d (float32 and bfloat16 hold every value)", who, dtype);
    if (T == 0 || n == 0) return FRX_OK;
    if (!x || !codes || !scales) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (ldx < n) return fail(FRX_ERR_ARG, "%s: rows of x are %lld elements apart and %d long", who, (long long)ldx, n);
    const int size = dtype_size(dtype);
    if (!rows_aligned(x, size) || !aligned(codes, 4)) return fail(FRX_ERR_ARG, "%s: misaligned pointer", who);
    const uint64_t pieces = uint64_t(T) * uint64_t(n / 8);
    if (pieces > 0xffffff00ull) return fail(FRX_ERR_SHAPE, "%s: T %d, n %d", who, T, n);
    const dim3 grid(unsigned((pieces + 255) / 256));
    with_rows(dtype, rows_vec16(x, ldx, n, size), [&](auto v, auto width) {
        using T_ = decltype(v);
        FRX_LAUNCH(kKQuant, stream, launch_pdl(k_mx_dequantize<T_, decltype(width)::value>, grid, dim3(256), 0, stream, static_cast<const uint32_t*>(codes),
                                               static_cast<const uint8_t*>(scales), uint32_t(pieces), uint32_t(n / 8), static_cast<T_*>(x), ldx));
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

size_t frx_mxfp4_packed_bytes(int rows, int n) {
    if (rows < 1 || rows > 65535 * kMxTileRows || n < kMxUnitK || n % kMxUnitK) return 0;
    return size_t((rows + kMxTileRows - 1) / kMxTileRows) * size_t(n / kMxUnitK) * kMxUnitBytes;
}

static int pack_args(const char* who, const void* codes, const void* scales, const void* packed, int E, int rows, int n) {
    if (E < 0) return fail(FRX_ERR_ARG, "%s: E %d", who, E);
    if (!frx_mxfp4_packed_bytes(rows, n)) return fail(FRX_ERR_SHAPE, "%s: unsupported shape rows %d, n %d (n a multiple of 128)", who, rows, n);
    if (E == 0) return FRX_OK;
    if (!codes || !scales || !packed) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (!aligned(codes, 16) || !aligned(scales, 4) || !aligned(packed, 16)) return fail(FRX_ERR_ARG, "%s: misaligned pointer", who);
    if (uint64_t(E) * (frx_mxfp4_packed_bytes(rows, n) / kMxUnitBytes) > 0x7fffffffull) return fail(FRX_ERR_SHAPE, "%s: E %d, rows %d, n %d", who, E, rows, n);
    return FRX_OK;
}
static dim3 pack_grid(int E, int rows, int n) { return dim3(unsigned(size_t(E) * (frx_mxfp4_packed_bytes(rows, n) / kMxUnitBytes))); }

int frx_mxfp4_pack(frx_stream_t stream, const void* codes, const void* scales, int E, int rows, int n, void* packed) {
    const int rc = pack_args("frx_mxfp4_pack", codes, scales, packed, E, rows, n);
    if (rc != FRX_OK || E == 0) return rc;
    FRX_LAUNCH(kKLayout, stream, k_mx_pack<true><<<pack_grid(E, rows, n), kMxTileRows, 0, stream>>>(
                                     static_cast<uint4*>(const_cast<void*>(codes)), static_cast<uint32_t*>(const_cast<void*>(scales)), rows, n / kMxUnitK,
                                     (rows + kMxTileRows - 1) / kMxTileRows, static_cast<uint8_t*>(packed)));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_mxfp4_unpack(frx_stream_t stream, const void* packed, int E, int rows, int n, void* codes, void* scales) {
    const int rc = pack_args("frx_mxfp4_unpack", codes, scales, packed, E, rows, n);
    if (rc != FRX_OK || E == 0) return rc;
    FRX_LAUNCH(kKLayout, stream, k_mx_pack<false><<<pack_grid(E, rows, n), kMxTileRows, 0, stream>>>(
                                     static_cast<uint4*>(codes), static_cast<uint32_t*>(scales), rows, n / kMxUnitK, (rows + kMxTileRows - 1) / kMxTileRows,
                                     static_cast<uint8_t*>(const_cast<void*>(packed))));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_mxfp4_matmul(frx_stream_t stream, const void* codes, const void* scales, int T, int n, const void* packed, int rows, void* y, int64_t ldy, int dtype) {
    const char* who = "frx_mxfp4_matmul";
    if (T == 0 && n > 0 && n % kMxUnitK == 0 && rows > 0 && dtype_size(dtype)) return FRX_OK;
    const int rc = product_args(who, codes, scales, packed, T, n, 1, rows, y, ldy, dtype);
    if (rc != FRX_OK) return rc;
    MxProduct p{};
    p.w = static_cast<const uint8_t*>(packed);
    p.codes = static_cast<const uint8_t*>(codes);
    p.scales = static_cast<const uint8_t*>(scales);
    p.y = y;
    p.ldy = ldy;
    p.E = 1;
    p.rows = rows;
    p.n = n;
    p.K = 1;
    p.x_rows = T;
    p.S = T;
    p.y_type = dtype;
    return launch_product(p, stream, kKGateUp);
}

int frx_mxfp4_moe_matmul(frx_stream_t stream, const void* codes, const void* scales, int T, int n, const void* packed, int E, int rows, const int32_t* offsets,
                         const int32_t* slot_of, int K, int S, void* y, int64_t ldy, int dtype) {
    const char* who = "frx_mxfp4_moe_matmul";
    if (S < 0 || T < 0 || K < 1) return fail(FRX_ERR_ARG, "%s: S %d, T %d, K %d", who, S, T, K);
    if (!slot_of && (K != 1 || T < S)) return fail(FRX_ERR_ARG, "%s: %d rows of x for %d sorted rows (without slot_of row r of y is of row r of x, K 1)", who, T, S);
    if (S == 0 && n > 0 && n % kMxUnitK == 0 && rows > 0 && dtype_size(dtype)) return FRX_OK;
    const int rc = product_args(who, codes, scales, packed, T, n, E, rows, y, ldy, dtype);
    if (rc != FRX_OK) return rc;
    if (!offsets) return fail(FRX_ERR_ARG, "%s: null pointer (offsets)", who);
    MxProduct p{};
    p.w = static_cast<const uint8_t*>(packed);
    p.codes = static_cast<const uint8_t*>(codes);
    p.scales = static_cast<const uint8_t*>(scales);
    p.offsets = offsets;
    p.slot_of = slot_of;
    p.y = y;
    p.ldy = ldy;
    p.E = E;
    p.rows = rows;
    p.n = n;
    p.K = K;
    p.x_rows = T;
    p.S = S;
    p.y_type = dtype;
    return launch_product(p, stream, kKGateUp);
}

size_t frx_mxfp4_moe_layer_workspace_bytes(int T, int K, int n, int ff, int E) {
    if (T < 0 || K < 1 || K > 32 || E < 1 || E > 4096 || n < 128 || ff < 128 || n % 128 || ff % 128 || n > (1 << 20) || ff > (1 << 20) || (long long)T * K > 0x7fffffffLL) return 0;
    return layer_buffers(T, K, n, ff, E).total;
}

int frx_mxfp4_moe_layer(frx_stream_t stream, const void* w_gate, const void* w_up, const void* w_down, int E, int n, int ff, const void* x, int64_t ldx, int x_dtype,
                        const int32_t* ids, const float* wts, int T, int K, void* out, int64_t ldo, int out_dtype, void* ws, size_t ws_bytes) {
    const char* who = "frx_mxfp4_moe_layer";
    if (T < 0) return fail(FRX_ERR_ARG, "%s: T %d", who, T);
    const size_t need = frx_mxfp4_moe_layer_workspace_bytes(T, K, n, ff, E);
    if (!need) return fail(FRX_ERR_SHAPE, "%s: unsupported shape T %d, K %d, n %d, ff %d, E %d", who, T, K, n, ff, E);
    if (!dtype_size(x_dtype) || !dtype_size(out_dtype)) return fail(FRX_ERR_ARG, "%s: element types %d, %d", who, x_dtype, out_dtype);
    if (T == 0) return FRX_OK;
    if (!w_gate || !w_up || !w_down || !x || !ids || !wts || !out || !ws) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (ldx < n || ldo < n) return fail(FRX_ERR_ARG, "%s: rows of x and out are %lld and %lld elements apart and %d long", who, (long long)ldx, (long long)ldo, n);
    if (!aligned(w_gate, 16) || !aligned(w_up, 16) || !aligned(w_down, 16) || !aligned(ws, 16) || !rows_aligned(x, dtype_size(x_dtype)) || !rows_aligned(out, dtype_size(out_dtype)))
        return fail(FRX_ERR_ARG, "%s: misaligned pointer", who);
    if (ws_bytes < need) return fail(FRX_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, need);
    const LayerBuffers b = layer_buffers(T, K, n, ff, E);
    uint8_t* base = static_cast<uint8_t*>(ws);
    const int S = T * K;
    int32_t *offsets = reinterpret_cast<int32_t*>(base + b.offsets), *slot_of = reinterpret_cast<int32_t*>(base + b.slot_of), *row_of = reinterpret_cast<int32_t*>(base + b.row_of);
    int rc = quantize(who, x, ldx, x_dtype, T, n, base + b.xq, base + b.xs, stream);
    if (rc != FRX_OK) return rc;
    rc = sort_slots(ids, S, E, offsets, slot_of, row_of, reinterpret_cast<int*>(base), reinterpret_cast<int*>(base + b.sort), stream);
    if (rc != FRX_OK) return rc;
    MxProduct p{};
    p.codes = base + b.xq;
    p.scales = base + b.xs;
    p.offsets = offsets;
    p.slot_of = slot_of;
    p.E = E;
    p.rows = ff;
    p.n = n;
    p.K = K;
    p.x_rows = T;
    p.S = S;
    p.y_type = FRX_F32;
    p.ldy = ff;
    for (int i = 0; i < 2; ++i) {
        p.w = static_cast<const uint8_t*>(i ? w_up : w_gate);
        p.y = base + (i ? b.u : b.g);
        if ((rc = launch_product(p, stream, kKGateUp)) != FRX_OK) return rc;
    }
    FRX_LAUNCH(kKQuant, stream, launch_pdl(k_mx_swiglu, dim3(unsigned((size_t(S) * (ff / 32) + 7) / 8)), dim3(256), 0, stream, reinterpret_cast<const float*>(base + b.g),
                                           reinterpret_cast<const float*>(base + b.u), (const int32_t*)(offsets + E), ff, reinterpret_cast<uint32_t*>(base + b.hq), base + b.hs));
    // an expert's rows are kept in bfloat16 on their way to a bfloat16 sum: that rounding is half of what such a sum is rounded to anyway,
    // and the rows are the largest thing that the layer writes and reads
    p.w = static_cast<const uint8_t*>(w_down);
    p.codes = base + b.hq;
    p.scales = base + b.hs;
    p.slot_of = nullptr;
    p.rows = n;
    p.n = ff;
    p.K = 1;
    p.x_rows = S;
    p.y = base + b.y;
    p.ldy = n;
    p.y_type = out_dtype == FRX_BF16 ? FRX_BF16 : FRX_F32;
    if ((rc = launch_product(p, stream, kKDown)) != FRX_OK) return rc;
    return rows_back(base + b.y, n, p.y_type, wts, row_of, S, T, K, n, out, ldo, out_dtype, stream);
}

}  // extern "C"
