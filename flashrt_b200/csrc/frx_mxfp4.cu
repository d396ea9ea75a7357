// MXFP4: the quantizer, the way back, the layout that the product reads, the product (dense, and grouped by expert), and
// the expert layer made of them.
#include <algorithm>
#include <type_traits>

#include "frx_groups.cuh"
#include "frx_mx.cuh"
#include "frx_rows.cuh"
#include "frx_sort.cuh"
#include "frx_umma.cuh"

namespace frx {
namespace {

// ---- quantizer. A thread takes 16 values (two threads a block of 32), U times: per value 2 or 4 bytes in, 17 / 32 out, so bandwidth bounds it, and U
// is how many loads a thread has in flight. (x is not __restrict__: the kernel in front may still write it when this one starts, so its loads must stay
// behind pdl_wait().)
template <class T, int U>
__global__ void __launch_bounds__(256) k_mx_quantize(const T* x, int64_t ldx, uint32_t pieces, uint32_t per_row, uint2* __restrict__ codes,
                                                     uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_trigger();
    constexpr int kPer = 16 / int(sizeof(T));
    Vec<T, kPer> v[U][16 / kPer];
    const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = min(i0 + q * 256u, pieces - 1u), t = i / per_row, c = i - t * per_row;
#pragma unroll
        for (int j = 0; j < 16 / kPer; ++j) v[q][j] = *reinterpret_cast<const Vec<T, kPer>*>(x + int64_t(t) * ldx + c * 16 + j * kPer);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = i0 + q * 256u;
        float f[2][8];
        uint32_t amax = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            f[j / 8][j % 8] = to_float(v[q][j / kPer].v[j % kPer]);
            amax = max(amax, __float_as_uint(f[j / 8][j % 8]) & 0x7fffffffu);   // (the bits of magnitudes are in their order, infinity and NaN on top)
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));   // (pairs are whole: pieces is even)
        const uint32_t byte = mx_scale_byte(amax);
        const float inv = mx_inverse(min(byte, 253u));
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j / 8][j % 8] *= inv;
        uint2 out = make_uint2(mx_codes8(f[0]), mx_codes8(f[1]));
        if (byte == 255u) out = make_uint2(0u, 0u);
        if (i < pieces) {
            codes[i] = out;
            if ((i & 1u) == 0) scales[i >> 1] = uint8_t(byte);
        }
    }
}
// rows that do not start on 16 bytes: a warp per block of 32, a lane per value
template <class T>
__global__ void __launch_bounds__(256) k_mx_quantize_any(const T* x, int64_t ldx, uint32_t blocks, uint32_t per_row, uint32_t* __restrict__ codes,
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

// eight values a thread, U times
template <class T, int N, int U>
__global__ void __launch_bounds__(256) k_mx_dequantize(const uint32_t* codes, const uint8_t* scales, uint32_t pieces, uint32_t per_row, T* __restrict__ x,
                                                       int64_t ldx) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i0 = blockIdx.x * (256u * U) + threadIdx.x;
    uint32_t c8[U], sb[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = min(i0 + q * 256u, pieces - 1u);
        c8[q] = codes[i];
        sb[q] = scales[i >> 2];
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
        const uint32_t i = i0 + q * 256u;
        if (i >= pieces) return;
        const uint32_t t = i / per_row, c = i - t * per_row;
        float f[8];
        mx_values8(c8[q], f);
        const float s = mx_scale(sb[q]);
        T* out = x + int64_t(t) * ldx + c * 8;
#pragma unroll
        for (int j = 0; j < 8; j += N) {
            Vec<T, N> o;
#pragma unroll
            for (int k = 0; k < N; ++k) o.v[k] = from_float<T>(f[j + k] * s);
            *reinterpret_cast<Vec<T, N>*>(out + j) = o;
        }
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

// ---- product on the tensor cores
//
// y[r] = sum over blocks b of 32 columns of 2^(ew[b] + ex[b]) * (sum of the 32 products of elements): kind::mxf4 does 64 columns, both scales included, per
// instruction. A tile is 256 matrix rows (two row tiles of 128: the M of the instruction, or the gate and the up tile of 128 hidden rows) by
// up to 112 y rows of one expert (its N), so weights are read once per 112 rows and an expert with few rows costs what its weights
// cost. A stage of the ring is 256 columns:
// per row tile two 8,704-byte units of the packed layout, brought by one bulk copy, and 128 bytes of codes of each y row, by
// TMA into the 128-byte swizzle. The y rows' scale words, 4 bytes a row and unit, come in segments of 16 units
// through registers. Tensor memory: two sets of accumulators (2 x 2 x 112 columns), so that a tile's epilogue runs beside the next
// tile's products, and four sets of scales (16 columns each).
//
// What bounds it. Up to a few rows an expert: the weights. 64 tokens of ten experts out of 512 (2048 / 512; gate and up): 408 MB from DRAM in 61 us between
// launches, 6.7 TB/s (reads alone; a copy reaches 6.55); 10 us of the layer's 110 are the start of the two products and their uneven ends. 4,096 tokens: 100 us for 570 MB of weights. 16,384 tokens
// (three blocks of 107 rows an expert): 262 us for 687 GFLOP at full clocks, the thread that issues (a stage's hand-offs, six copies of scales and eight MMAs take
// 900 clocks, of which the MMAs are 464) and the L2, which delivers 55 bytes a clock and SM without any MMA; in a stream of such layers the GPU is at its power
// limit (1,000 W) and at 1,650 MHz. The down product of these tokens writes 1.34 GB of rows in 32 bits: 333 us, 218 in bfloat16 (4,096 tokens 109 and 87).
constexpr int kTok = 112;                 // y rows of a tile at most
constexpr int kRowTiles = 2;              // row tiles of a tile
constexpr int kStageUnits = 2;            // units of a stage
constexpr int kTileW = kStageUnits * kMxUnitBytes, kStageW = kRowTiles * kTileW, kRowB = kStageUnits * kMxUnitK / 2, kStageBytes = kStageW + kTok * kRowB;
constexpr int kSegUnits = 16, kSegBytes = kSegUnits * 512, kSegs = 2;   // scale words of y rows: units of a segment, and segments
constexpr int kMaxStages = 4;
constexpr int kWarpsEpi = 16, kWarpW = 16, kWarpMma = 17, kWarpAct = 18, kWarpsAct = 8;
constexpr int kMxThreads = 32 * (kWarpAct + kWarpsAct);
constexpr int kColsAcc = kRowTiles * kTok, kColScale = 2 * kColsAcc, kScaleSets = 4, kColsScale = 16;
static_assert(kColScale + kScaleSets * kColsScale <= 512, "tensor memory has 512 columns");
static_assert(kTok % 16 == 0 && kTok <= 128, "the tokens' scales of a unit are one block of 512 bytes");
static_assert(kRowB == 128 && kStageW % 1024 == 0 && kStageBytes % 1024 == 0, "rows of the 128-byte swizzle, in groups of eight");
static_assert(kSegUnits % kStageUnits == 0, "a stage has its scales in one segment");
static_assert(kTok <= 16 * kWarpsAct, "sixteen rows a warp");
// barriers, 8 bytes each, then the abort flag, the address of the tensor memory and the scan's sums
constexpr int kBarFull = 0, kBarFree = kMaxStages, kBarDFull = 2 * kMaxStages, kBarDFree = kBarDFull + 2, kBarSFull = kBarDFree + 2, kBarSFree = kBarSFull + kSegs,
              kBars = kBarSFree + kSegs;
static_assert(256 + 8 * kMxThreads / 32 <= 1024, "the scan's sums");
constexpr int kSmemSegs = 1024, kSmemHead = kSmemSegs + kSegs * kSegBytes;   // the scale segments, then the stages

enum { kYswiglu = 3 };   // beside the element types of y

struct MxProduct {
    const uint8_t* w[2];     // packed matrices; the second: the up matrices of the SwiGLU form
    const uint8_t* codes;    // activations [x_rows][n / 2]
    const uint8_t* scales;   // [x_rows][n / 32]
    const int32_t* offsets;  // [E + 1] rows of every expert; null: one matrix, all rows
    const int32_t* slot_of;  // the x row of sorted row r is slot_of[r] / K; null: r
    void* y;
    uint8_t* y_scales;       // SwiGLU form
    int64_t ldy;
    int* status;             // of a workspace, or null
    unsigned long long wait_ns;
    int E, rows, n, K, x_rows, S;   // rows: of a matrix; S: rows of y
    int stages;
    int single;              // tiles of one row tile instead of two
    int most;                // tiles of any plan whose experts' rows do not overlap
    int early;               // the plan was complete before the kernel in front began: it and the weights are read before the wait for that kernel
};

// Four rows of the map's box width from column x (bytes here) on, one below the other in shared memory; completion counted on an mbarrier.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, const int (&row)[4], uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(bar)
                 : "memory");
}
// sixteen consecutive rows
__device__ __forceinline__ void tma_rows16(uint32_t dst, const CUtensorMap* map, int x, int row, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(bar) : "memory");
}
// Instruction descriptor of kind::mxf4 with scales of 32: A and B E2M1 (1), scales UE8M0, both K-major, D fp32 128 x n; the byte pair of
// the scale words that belongs to these 64 columns is part of it.
__device__ __forceinline__ uint32_t mx_idesc(int n, int pair) {
    return (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (1u << 23) | (uint32_t(kMxTileRows >> 4) << 24) | (uint32_t(2 * pair) << 4) | (uint32_t(2 * pair) << 29);
}
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
}
// 512 bytes (32 rows of 16) to four columns of tensor memory, the same in all four quarters of its lanes. In order with the MMAs of the issuing thread.
__device__ __forceinline__ void tmem_copy_scales(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// 8 columns of this warp's lanes from two places, complete on return
__device__ __forceinline__ void tmem_ld8x2(uint32_t a0, uint32_t a1, uint32_t (&v)[8], uint32_t (&w)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]),
          "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
        : "r"(a0), "r"(a1)
        : "memory");
}

// The scale words of units u .. u + 7 of a row (as far as there are so many). Of scattered rows every access costs one a row, whatever its width.
__device__ __forceinline__ void load_words(uint32_t (&w)[8], const uint8_t* row, int u, int units, bool wide, bool on) {
    if (!on) return;
    if (wide) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (u + 4 * i < units) {
                const uint4 v = __ldcg(reinterpret_cast<const uint4*>(row + (u + 4 * i) * 4));
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (u + j < units) w[j] = __ldcg(reinterpret_cast<const uint32_t*>(row + (u + j) * 4));
    }
}

// silu(g) * u of eight y rows for one hidden row a lane; the warp's 32 hidden rows are one block. codes: where this lane's word goes,
// four bytes (eight hidden rows) of y row lane % 8; scale: that row's scale byte, of lane < 8.
__device__ __forceinline__ void swiglu8(const uint32_t (&g)[8], const uint32_t (&u)[8], uint32_t& codes, uint32_t& scale) {
    const unsigned lane = threadIdx.x & 31u;
    float h[8];
    uint32_t top[8], mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // The exponential's relative error is 2^-22 and |g| * 1.25 * 2^-24 of its rounded argument, which is what a sum g that is itself rounded to 32 bits
        // leaves open; the reciprocal's is 2^-23 (2^-21 as a subnormal, below g = -87.3; 0 below -88.7).
        const float a = __uint_as_float(g[i]);
        float e, r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a * -1.44269504f));
        asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));   // (a subnormal from 2^126 on: the product with a is not one)
        h[i] = a * r * __uint_as_float(u[i]);
        top[i] = __reduce_max_sync(0xffffffffu, __float_as_uint(h[i]) & 0x7fffffffu);
        mine = (lane & 7u) == unsigned(i) ? top[i] : mine;
    }
    scale = mx_scale_byte(mine);
    if (__any_sync(0xffffffffu, mine - (3u << 23) >= (252u << 23))) {   // a block whose scale is at its lowest, or with a NaN or an infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t byte = mx_scale_byte(top[i]);
            h[i] = byte == 255u ? 0.0f : h[i] * mx_inverse(byte);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] *= __uint_as_float((256u << 23) - (top[i] & 0x7f800000u));   // mx_inverse of the byte e - 2
    }
    // lane l has the codes of row l for eight y rows, one a nibble; wanted: y row l % 8 for the eight hidden rows of its lanes
    uint32_t w = mx_codes8(h), other = __shfl_xor_sync(0xffffffffu, w, 4);
    w = __byte_perm(w, other, lane & 4u ? 0x3276 : 0x5410);
    other = __shfl_xor_sync(0xffffffffu, w, 2);
    w = __byte_perm(w, other, lane & 2u ? 0x3715 : 0x6240);
    other = __shfl_xor_sync(0xffffffffu, w, 1);
    codes = lane & 1u ? ((other >> 4) & 0x0f0f0f0fu) | (w & 0xf0f0f0f0u) : (w & 0x0f0f0f0fu) | ((other & 0x0f0f0f0fu) << 4);
}

template <int MODE>
__global__ void __launch_bounds__(kMxThreads, 1) k_mx_product(const MxProduct p, const __grid_constant__ CUtensorMap codes_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t s0 = smem_u32(smem), stages0 = s0 + kSmemHead, bars = s0, abort = s0 + 240;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 240);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 244);
    long long* warp_sums = reinterpret_cast<long long*>(smem + 256);   // one a warp
    const uint32_t n_stages = uint32_t(p.stages);
    GroupTables tab;
    tab.tile_end = reinterpret_cast<int*>(smem + kSmemHead + n_stages * kStageBytes);
    tab.first = tab.tile_end + p.E;
    tab.count = tab.first + p.E;
    tab.blocks = tab.count + p.E;
    const int units = p.n / kMxUnitK;
    const int row_tiles = (p.rows + kMxTileRows - 1) / kMxTileRows, row_pairs = MODE == kYswiglu || p.single ? row_tiles : (row_tiles + 1) / 2;
    // first row tile of a tile's row pair, and whether it has a second one
    auto row_tile = [&](int rp) { return MODE == kYswiglu || p.single ? rp : 2 * rp; };
    auto has_second = [&](int rp) { return MODE == kYswiglu || (!p.single && 2 * rp + 1 < row_tiles); };
    static_assert(kBars * 8 <= 240, "the barriers' block");

    if (threadIdx.x == 0) {
        uint64_t* b = reinterpret_cast<uint64_t*>(smem);
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(b + kBarFull + i, 1 + kWarpsAct);   // the weights' warp with the bytes of both, and every gathering warp
            mbar_init(b + kBarFree + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b + kBarDFull + i, 1);
            mbar_init(b + kBarDFree + i, kWarpsEpi);
        }
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(b + kBarSFull + i, kWarpsAct);
            mbar_init(b + kBarSFree + i, 1);
        }
        asm volatile("prefetch.tensormap [%0];" ::"l"(&codes_map) : "memory");
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kWarpMma) tmem_alloc(tmem_slot, 512);
    // With the plan known early only the warps that read activations or write y wait for the kernel in front, and let the next one in. (That kernel's blocks,
    // which let this one in, had waited for the ones that made the plan, so these had completed.) One token: 2.1 us from the end of a kernel to
    // the return of its dependents' wait, 1.4 for the tables and 2 to the first weights, now side by side.
    if (!p.early) {
        pdl_wait();
        pdl_trigger();
    }
    // offsets that are not ascending: nothing is computed
    const int experts = group_tables<kMxThreads>(tab, p.offsets, p.E, p.S, kTok, row_pairs, warp_sums) > p.most ? 0 : p.E;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    GroupWalk t;
    t.begin(tab, experts);

    // "free" barriers are waited on with the parity of the phase before the one about to be used, which a fresh barrier reports as complete
    if (warp == kWarpW) {
        // ---------------- weights: one lane, a bulk copy per row tile and stage
        uint32_t st = 0, phase = 1;
        const size_t tile_bytes = size_t(units) * kMxUnitBytes;
        // Weights that no other tile reads leave the L2 first: they would push out what is read again (hidden rows, y). A layer of 64 tokens 111.5 -> 107.5 us, of 4,096
        // 244 -> 238.
        const uint64_t once = l2_policy_evict_first(), again = l2_policy_evict_normal();
        bool ok = true;
        while (ok && t.next()) {
            const uint8_t *w0, *w1;
            bool second = true;
            if (MODE == kYswiglu) {
                const size_t at = (size_t(t.e) * row_tiles + t.rp) * tile_bytes;
                w0 = p.w[0] + at;
                w1 = p.w[1] + at;
            } else {
                w0 = p.w[0] + (size_t(t.e) * row_tiles + row_tile(t.rp)) * tile_bytes;
                w1 = w0 + tile_bytes;
                second = has_second(t.rp);
            }
            for (int u = 0; u < units; u += kStageUnits) {
                const uint32_t full = bars + (kBarFull + st) * 8, dst = stages0 + st * kStageBytes, bytes = uint32_t(min(kStageUnits, units - u)) * kMxUnitBytes;
                if (!(ok = warp_wait(bars + (kBarFree + st) * 8, phase, abort, p.wait_ns))) break;
                if (lane == 0) {
                    mbar_expect_tx(full, (second ? 2 * bytes : bytes) + uint32_t(t.width) * kRowB);   // the gathered rows' bytes too
                    bulk_g2s_hint(dst, w0, bytes, full, t.alone ? once : again);
                    if (second) bulk_g2s_hint(dst + kTileW, w1, bytes, full, t.alone ? once : again);
                }
                __syncwarp();
                w0 += kTileW;
                w1 += kTileW;
                if (++st == n_stages) st = 0, phase ^= 1u;
            }
        }
    } else if (warp >= kWarpAct) {
        // ---------------- activations. Codes: rows that follow one another come sixteen at a time, others are gathered by lanes 0 to 3 of a warp, four
        // rows each (36 clocks a four: 14 bytes a clock; by cp.async, 512 bytes an instruction, they came at 11). Scales: a lane has
        // one of the warp's sixteen rows and half of a segment's units. A tile begins with dependent loads (slots, then scale words), which
        // are made during the tile in front.
        const int aw = warp - kWarpAct;
        const size_t row_scales = size_t(p.n / kMxBlock);
        const bool s_wide = units % 4 == 0 && reinterpret_cast<uintptr_t>(p.scales) % 16 == 0;
        const int four = aw + (lane & 3) * kWarpsAct;                    // the lane's four rows
        const int stok = aw * 16 + (lane & 15), shalf = lane >> 4;       // the lane's row and half segment of scale words
        const uint32_t sdst = s0 + kSmemSegs + shalf * (kSegBytes / 2) + (stok & 31) * 16 + (stok >> 5) * 4;
        uint32_t st = 0, phase = 1, sg = 0, sphase = 1;
        int slot[4], sslot = 0;   // of the rows (beyond the live ones the last again): their slots, or themselves
        auto look_up = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = t.row0 + min(four * 4 + i, t.live - 1);
                slot[i] = p.slot_of ? __ldcg(p.slot_of + r) : r;
            }
            const int r = t.row0 + min(stok, t.live - 1);
            sslot = p.slot_of ? __ldcg(p.slot_of + r) : r;
        };
        auto x_row = [&](int s) {
            const int x = p.slot_of ? (s < 0 ? 0 : int(unsigned(s) / unsigned(p.K))) : s;
            return x < p.x_rows ? x : 0;
        };
        uint32_t words[8];   // the lane's half of the tile's first segment
        int row[4];
        const uint8_t* ssrc = nullptr;
        auto take_up = [&]() {
#pragma unroll
            for (int i = 0; i < 4; ++i) row[i] = x_row(slot[i]);
            ssrc = p.scales + size_t(x_row(sslot)) * row_scales;
            load_words(words, ssrc, shalf * (kSegUnits / 2), units, s_wide, stok < t.width);
        };
        bool more = t.next(), ok = true;
        if (more) look_up();
        if (p.early) {
            pdl_wait();
            pdl_trigger();
        }
        if (more) take_up();
        while (more && ok) {
            const int width = t.width, row0 = t.row0;
            int now[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) now[i] = row[i];
            const uint8_t* snow = ssrc;
            const bool s_on = stok < width;
            // A warp without rows in the tile takes part in every stage all the same: whoever is more than a ring ahead of the MMAs or behind
            // them can no longer tell the barriers' phases by their parity.
            const bool mine = p.slot_of ? lane < 4 && four * 4 < width : lane == 0 && aw * 16 < width;
            more = t.next();
            if (more) look_up();
            const int last = (units - 1) / kStageUnits * kStageUnits, ahead = min(2 * kStageUnits, last);   // the stage behind which the next tile's rows are taken up
            for (int u = 0; u < units; u += kStageUnits) {
                if (u % kSegUnits == 0) {
                    if (u) load_words(words, snow, u + shalf * (kSegUnits / 2), units, s_wide, s_on);
                    if (!(ok = warp_wait(bars + (kBarSFree + sg) * 8, sphase, abort, p.wait_ns))) break;
#pragma unroll
                    for (int j = 0; j < kSegUnits / 2; ++j)
                        if (s_on && u + shalf * (kSegUnits / 2) + j < units) sts32(sdst + sg * kSegBytes + j * 512, words[j]);
                    fence_async_smem();   // generic-proxy writes: visible to the tensor core before the arrival
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + (kBarSFull + sg) * 8);
                    if (++sg == kSegs) sg = 0, sphase ^= 1u;
                }
                if (!(ok = warp_wait(bars + (kBarFree + st) * 8, phase, abort, p.wait_ns))) break;
                const uint32_t dst = stages0 + st * kStageBytes + kStageW, full = bars + (kBarFull + st) * 8;
                if (mine) {
                    if (p.slot_of)
                        tma_gather4(dst + four * 4 * kRowB, &codes_map, u * (kMxUnitK / 2), now, full);
                    else
                        tma_rows16(dst + aw * 16 * kRowB, &codes_map, u * (kMxUnitK / 2), row0 + aw * 16, full);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(full);
                if (++st == n_stages) st = 0, phase ^= 1u;
                if (u == ahead && more && last < kSegUnits) take_up();   // (a tile of several segments has used its words by the last stage)
            }
            if (ok && more && last >= kSegUnits) take_up();
        }
    } else if (warp == kWarpMma) {
        // ---------------- MMA: one elected lane issues
        uint32_t st = 0, phase = 0, set = 0, sc = 0, dphase = 1, sg = 0, sphase = 0;
        bool ok = true;
        while (ok && t.next()) {
            const uint32_t id0 = mx_idesc(t.width, 0), id1 = mx_idesc(t.width, 1);
            const bool second = has_second(t.rp);
            if (!(ok = warp_wait(bars + (kBarDFree + set) * 8, dphase, abort, p.wait_ns))) break;
            tc_fence_after_sync();   // behind the epilogue's loads of these accumulators
            const uint32_t acc = tmem + set * kColsAcc;
            for (int u = 0; u < units; u += kStageUnits) {
                if (u % kSegUnits == 0 && !(ok = warp_wait(bars + (kBarSFull + sg) * 8, sphase, abort, p.wait_ns))) break;
                if (!(ok = warp_wait(bars + (kBarFull + st) * 8, phase, abort, p.wait_ns))) break;
                const uint32_t base = stages0 + st * kStageBytes;
                const uint64_t da0 = umma_desc(base, 2048, 128), db0 = umma_desc_sw128(base + kStageW);
                const uint64_t dsa = umma_desc(base + kMxUnitCode, 128, 128), dsb = umma_desc(s0 + kSmemSegs + sg * kSegBytes + (u % kSegUnits) * 512, 128, 128);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kStageUnits; ++k) {
                        if (u + k >= units) break;
                        const uint32_t sf = tmem + kColScale + (sc + k) * kColsScale;
                        tmem_copy_scales(sf, dsa + uint64_t(k * kMxUnitBytes >> 4));
                        if (second) tmem_copy_scales(sf + 4, dsa + uint64_t((kTileW + k * kMxUnitBytes) >> 4));
                        tmem_copy_scales(sf + 8, dsb + uint64_t(k * 512 >> 4));
                    }
#pragma unroll
                    for (int k = 0; k < kStageUnits; ++k) {
                        if (u + k >= units) break;
                        const uint32_t sf = tmem + kColScale + (sc + k) * kColsScale;
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const uint64_t db = db0 + uint64_t((k * 64 + s * 32) >> 4);
                            const uint32_t on = u + k + s > 0;
                            umma_mxf4(acc, da0 + uint64_t((k * kMxUnitBytes + s * 4096) >> 4), db, s ? id1 : id0, sf, sf + 8, on);
                            if (second) umma_mxf4(acc + kTok, da0 + uint64_t((kTileW + k * kMxUnitBytes + s * 4096) >> 4), db, s ? id1 : id0, sf + 4, sf + 8, on);
                        }
                    }
                    umma_commit(bars + (kBarFree + st) * 8);
                    if (u + kStageUnits >= units || (u + kStageUnits) % kSegUnits == 0) umma_commit(bars + (kBarSFree + sg) * 8);
                    if (u + kStageUnits >= units) umma_commit(bars + (kBarDFull + set) * 8);
                }
                __syncwarp();
                if (++st == n_stages) st = 0, phase ^= 1u;
                sc = (sc + kStageUnits) % kScaleSets;
                if (u + kStageUnits >= units || (u + kStageUnits) % kSegUnits == 0)
                    if (++sg == kSegs) sg = 0, sphase ^= 1u;
            }
            set ^= 1u;
            if (set == 0) dphase ^= 1u;
        }
    } else {
        // ---------------- epilogue: a warp has a quarter of the lanes (32 matrix rows of either row tile) and every fourth eight of the y rows.
        // Chains of dependent steps (load, SwiGLU, maximum over the warp, codes, exchange, store): it takes four warps a scheduler to hide them.
        const int quarter = warp & 3, part = warp >> 2, r = quarter * 32 + lane;
        constexpr int kParts = kWarpsEpi / 4;
        uint32_t set = 0, phase = 0;
        if (p.early) pdl_wait();
        const bool pairs = MODE != FRX_F32 && p.rows % 2 == 0 && p.ldy % 2 == 0 && reinterpret_cast<uintptr_t>(p.y) % 4 == 0;
        // A wait ran out: NaN, not a wrong number, and no more waits. (Of the uses of a set of accumulators behind the lost one, every second would find the
        // parity of the last complete one, and take sums that nobody has finished.)
        bool lost = false;
        while (t.next()) {
            lost = lost || !warp_wait(bars + (kBarDFull + set) * 8, phase, abort, p.wait_ns);
            tc_fence_after_sync();
            const uint32_t acc = tmem + (uint32_t(quarter * 32) << 16) + set * kColsAcc;
            const int eights = t.width >> 3;
            for (int c = part; c < eights; c += kParts) {
                uint32_t v[2][8];
                if (lost) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[0][i] = v[1][i] = 0x7fffffffu;
                } else {
                    tmem_ld8x2(acc + c * 8, acc + kTok + c * 8, v[0], v[1]);
                }
                if (c + kParts >= eights && !lost) {   // the sums are all in registers: the accumulators go back
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + (kBarDFree + set) * 8);
                }
                const int live = t.live - c * 8;
                const int64_t y0 = t.row0 + c * 8;
                if (MODE == kYswiglu) {
                    uint32_t codes, scale;
                    swiglu8(v[0], v[1], codes, scale);
                    const size_t y = size_t(y0) + (lane & 7);
                    const uint32_t at = uint32_t(t.rp) * kMxTileRows + quarter * 32;   // the block's first hidden row
                    if (int(lane & 7) < live) {
                        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.y) + y * (p.rows / 2) + at / 2 + (lane >> 3) * 4) = codes;
                        if (lane < 8) p.y_scales[y * (p.rows / kMxBlock) + at / kMxBlock] = uint8_t(scale);
                    }
                } else {
                    constexpr int size = MODE == FRX_F32 ? 4 : 2;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const int row = (row_tile(t.rp) + m) * kMxTileRows + r;
                        store8<MODE>(v[m], static_cast<uint8_t*>(p.y) + (y0 * p.ldy + row) * size, p.ldy, live, row < p.rows && (m == 0 || has_second(t.rp)), pairs);
                    }
                }
            }
            if (part >= eights && !lost) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bars + (kBarDFree + set) * 8);
            }
            set ^= 1u;
            if (set == 0) phase ^= 1u;
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        // A wait ran out: copies and MMAs may still be in flight. Give them time to land before tensor memory and the block's
        // shared memory are released.
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) {
        }
        __syncthreads();
        if (threadIdx.x == 0 && p.status) p.status[0] = kDevWaitTimeout;
    }
    if (warp == kWarpMma) tmem_free(tmem, 512);
}

// The codes [rows][n / 2] as a tensor map whose box is 128 bytes of one row (gathered) or of sixteen, in the 128-byte swizzle; what lies beyond the rows is zeros.
int codes_tensor_map(CUtensorMap& map, const void* codes, int rows, int n, bool gathered) {
    const cuuint64_t dims[2] = {cuuint64_t(n / 2), cuuint64_t(rows)}, strides[1] = {cuuint64_t(n / 2)};
    const cuuint32_t box[2] = {cuuint32_t(kRowB), gathered ? 1u : 16u};
    return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box);
}

template <int MODE>
int launch_mode(MxProduct& p, cudaStream_t stream, int cls) {
    const size_t tables = size_t(p.E) * 4 * 4;
    // Two row tiles a tile halve how often y rows' activations are read; where single ones still find an SM each, they halve the time that an SM takes for its weights
    // (1,024 x 2,048 by one token: 7.1 us a call instead of 7.7).
    const int64_t row_tiles = (p.rows + kMxTileRows - 1) / kMxTileRows, blocks = int64_t(p.S) / kTok + std::min(p.E, p.S);   // blocks of y rows at most
    p.single = MODE != kYswiglu && row_tiles * blocks <= sm_count();
    const int64_t pairs = MODE == kYswiglu || p.single ? row_tiles : (row_tiles + 1) / 2;
    if ((int64_t(p.S) + kTok - 1) / kTok >= (1 << 24) || (int64_t(p.S) / kTok + p.E) * pairs > 0x7fff0000) return fail(FRX_ERR_SHAPE, "MXFP4 product: %d rows by %d is more than 2^31 tiles", p.S, p.rows);
    int rc = allow_smem<k_mx_product<MODE>>();
    if (rc != FRX_OK) return rc;
    p.stages = int(std::min<size_t>(kMaxStages, (kSmemMost - kSmemHead - tables) / kStageBytes));
    static_assert((kSmemMost - kSmemHead - 4096 * 4 * 4) / kStageBytes >= 2, "stages beside the tables of 4096 experts");
    p.wait_ns = wait_limit_ns();
    CUtensorMap map;
    rc = codes_tensor_map(map, p.codes, p.x_rows, p.n, p.slot_of != nullptr);
    if (rc != FRX_OK) return rc;
    const int64_t most = blocks * pairs;
    p.most = int(most);
    const unsigned grid = unsigned(std::min<int64_t>(sm_count(), std::max<int64_t>(1, most)));
    FRX_LAUNCH(cls, stream, launch_pdl(k_mx_product<MODE>, dim3(grid), dim3(kMxThreads), kSmemHead + size_t(p.stages) * kStageBytes + tables, stream, p, map));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}
int launch_product(MxProduct& p, int mode, cudaStream_t stream, int cls) {
    switch (mode) {
        case FRX_F32: return launch_mode<FRX_F32>(p, stream, cls);
        case FRX_BF16: return launch_mode<FRX_BF16>(p, stream, cls);
        case FRX_F16: return launch_mode<FRX_F16>(p, stream, cls);
        default: return launch_mode<kYswiglu>(p, stream, cls);
    }
}

// where the layer keeps what it forms, in its workspace
struct LayerBuffers {
    size_t offsets, slot_of, row_of, sort, xq, xs, hq, hs, y, total;
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
    take(b.y, S * n * 4);
    b.total = at;
    return b;
}

// From so many pieces of 16 values on (enough blocks for every SM all the same) a thread has several in flight. 16,384 rows of 2,048 bf16 values: quantized in
// 14.8 / 14.0 / 14.6 us with 1 / 2 / 4 of 16 values, back in 20.4 / 15.7 / 14.9 with 1 / 2 / 4 of eight (5.7 to 6.1 TB/s).
constexpr uint64_t kMxMany = 1 << 19;
template <class T, int U>
void quantize_launch(const void* x, int64_t ldx, uint64_t pieces, int n, void* codes, void* scales, cudaStream_t stream) {
    FRX_LAUNCH(kKQuant, stream, launch_pdl(k_mx_quantize<T, U>, dim3(unsigned((pieces + 256 * U - 1) / (256 * U))), dim3(256), 0, stream, static_cast<const T*>(x), ldx,
                                           uint32_t(pieces), uint32_t(n / 16), static_cast<uint2*>(codes), static_cast<uint8_t*>(scales)));
}
template <class T, int N, int U>
void dequantize_launch(const void* codes, const void* scales, uint64_t pieces, int n, void* x, int64_t ldx, cudaStream_t stream) {
    FRX_LAUNCH(kKQuant, stream, launch_pdl(k_mx_dequantize<T, N, U>, dim3(unsigned((pieces + 256 * U - 1) / (256 * U))), dim3(256), 0, stream,
                                           static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales), uint32_t(pieces), uint32_t(n / 8), static_cast<T*>(x), ldx));
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
            pieces >= kMxMany ? quantize_launch<T_, 2>(x, ldx, pieces, n, codes, scales, stream) : quantize_launch<T_, 1>(x, ldx, pieces, n, codes, scales, stream);
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
    with_rows(dtype, rows_vec16(x, ldx, n, size), [&](auto v, auto width) {
        using T_ = decltype(v);
        constexpr int N = decltype(width)::value;
        pieces >= 2 * kMxMany ? dequantize_launch<T_, N, 4>(codes, scales, pieces, n, x, ldx, stream) : dequantize_launch<T_, N, 1>(codes, scales, pieces, n, x, ldx, stream);
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
    p.w[0] = static_cast<const uint8_t*>(packed);
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
    return launch_product(p, dtype, stream, kKGateUp);
}

int frx_mxfp4_moe_matmul(frx_stream_t stream, const void* codes, const void* scales, int T, int n, const void* packed, int E, int rows, const int32_t* offsets,
                         const int32_t* slot_of, int K, int S, void* y, int64_t ldy, int dtype) {
    const char* who = "frx_mxfp4_moe_matmul";
    if (S < 0 || T < 0 || K < 1) return fail(FRX_ERR_ARG, "%s: S %d, T %d, K %d", who, S, T, K);
    if (!slot_of && (K != 1 || T < S)) return fail(FRX_ERR_ARG, "%s: %d rows of x for %d sorted rows (without slot_of row r of y is of row r of x, K 1)", who, T, S);
    if ((S == 0 || T == 0) && n > 0 && n % kMxUnitK == 0 && rows > 0 && dtype_size(dtype)) return FRX_OK;
    const int rc = product_args(who, codes, scales, packed, T, n, E, rows, y, ldy, dtype);
    if (rc != FRX_OK) return rc;
    if (!offsets) return fail(FRX_ERR_ARG, "%s: null pointer (offsets)", who);
    MxProduct p{};
    p.w[0] = static_cast<const uint8_t*>(packed);
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
    return launch_product(p, dtype, stream, kKGateUp);
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
    // Rows of the experts in 32 bits, unless the caller asks for fewer: rounded to bfloat16 as well as out, they leave it 1.41 times as far
    // from the sums. In 32 bits a layer of 64 tokens takes as long (110 us), of 4,096 316 us instead of 280, of 16,384 927 instead of 747.
    const bool rows_bf16 = out_dtype == (FRX_BF16 | FRX_ROWS_BF16);
    if (rows_bf16) out_dtype = FRX_BF16;
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
    // the sort before the quantizer: the products then find the plan made by a kernel that is not the one in front of them
    int rc = sort_slots(ids, S, E, offsets, slot_of, row_of, reinterpret_cast<int*>(base), reinterpret_cast<int*>(base + b.sort), stream);
    if (rc != FRX_OK) return rc;
    rc = quantize(who, x, ldx, x_dtype, T, n, base + b.xq, base + b.xs, stream);
    if (rc != FRX_OK) return rc;
    MxProduct p{};
    p.codes = base + b.xq;
    p.scales = base + b.xs;
    p.offsets = offsets;
    p.slot_of = slot_of;   // (sorted copies of the rows instead, which the product reads 16 at a time: 16,384 tokens 219 instead of 248 us where the two were compared, but 24 more in
    p.E = E;               // the quantizer; 4,096 tokens 113 instead of 103)
    p.rows = ff;
    p.n = n;
    p.K = K;
    p.x_rows = T;
    p.S = S;
    p.w[0] = static_cast<const uint8_t*>(w_gate);
    p.w[1] = static_cast<const uint8_t*>(w_up);
    p.y = base + b.hq;
    p.y_scales = base + b.hs;
    p.status = reinterpret_cast<int*>(base);
    p.early = 1;
    if ((rc = launch_product(p, kYswiglu, stream, kKGateUp)) != FRX_OK) return rc;
    // (the rows are the largest thing that the layer writes and reads)
    p.w[0] = static_cast<const uint8_t*>(w_down);
    p.codes = base + b.hq;
    p.scales = base + b.hs;
    p.slot_of = nullptr;
    p.rows = n;
    p.n = ff;
    p.K = 1;
    p.x_rows = S;
    p.y = base + b.y;
    p.ldy = n;
    const int y_type = rows_bf16 ? FRX_BF16 : FRX_F32;
    if ((rc = launch_product(p, y_type, stream, kKDown)) != FRX_OK) return rc;
    return rows_back(base + b.y, n, y_type, wts, row_of, S, T, K, n, out, ldo, out_dtype, true, stream);
}

}  // extern "C"
