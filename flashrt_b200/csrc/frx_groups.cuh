// What the products by expert share (frx_mxfp4.cu, frx_experts.cu): their tiles, waits, tensor maps and the stores of their epilogues.
#pragma once

#include <cuda.h>

#include <atomic>
#include <mutex>

#include "frx_rows.cuh"
#include "frx_umma.cuh"

namespace frx {

// A bounded wait of a whole warp: false, in all its lanes, when it, or another one of the block, ran out. The role then leaves its loop: what is
// issued behind a wait that was given up could run the barriers' byte counts over.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint32_t abort, uint64_t limit_ns) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) {
        uint64_t t0 = 0;
        for (uint32_t polls = 1; !(ok = mbar_try_wait(bar, parity)); ++polls) {   // (a poll suspends the thread for microseconds by itself)
            if (polls & 7u) continue;
            if (lds32(abort)) break;
            const uint64_t now = global_ns();
            if (t0 == 0) {
                t0 = now;
            } else if (now - t0 > limit_ns) {
                sts32(abort, 1u);
                break;
            }
        }
    }
    return __all_sync(0xffffffffu, ok);
}
// umma_desc for rows of 128 bytes in the 128-byte swizzle (the 16-byte pieces of row r in the order piece ^ (r % 8)), groups of eight rows 1024 bytes
// apart; a column offset is added to the address
__device__ __forceinline__ uint64_t umma_desc_sw128(uint32_t smem_addr) { return umma_desc(smem_addr, 16, 1024) | (uint64_t(2) << 61); }


// The tiles of a block, one after the other: expert after expert, within one row pair after row pair, within these the blocks of y rows
// (so that blocks that share weights run at the same time).
struct GroupTables {
    int *tile_end, *first, *count, *blocks;   // per expert: tiles up to it, its first row, its rows, blocks of y rows | width / 16 << 24
};
struct GroupWalk {
    GroupTables tab;
    int E, tile, e;
    int rp, row0, live, width;   // row pair, first y row, y rows, their number rounded up to 16
    bool alone;                  // the expert has one block of y rows: this tile's weights are read by no other
    __device__ __forceinline__ void begin(const GroupTables& tables, int experts) {
        tab = tables;
        E = experts;
        tile = int(blockIdx.x) - int(gridDim.x);
        e = 0;
    }
    __device__ __forceinline__ bool next() {
        tile += int(gridDim.x);
        const int lane = threadIdx.x & 31;
        // 32 experts at a time, those that end at or before the tile: from the last one on, then, if all of these do, over the whole list
        // in 32 steps
        unsigned done = __ballot_sync(0xffffffffu, e + lane < E && tab.tile_end[e + lane] <= tile);
        e += __popc(done);
        if (done == 0xffffffffu) {
            const int step = (E + 31) >> 5, at = min(E, (lane + 1) * step);
            e = max(e, __popc(__ballot_sync(0xffffffffu, tab.tile_end[at - 1] <= tile)) * step);
            while (e < E) {
                done = __ballot_sync(0xffffffffu, e + lane < E && tab.tile_end[e + lane] <= tile);
                e += __popc(done);
                if (done != 0xffffffffu) break;
            }
        }
        if (e >= E) return false;
        const int local = tile - (e ? tab.tile_end[e - 1] : 0), bw = tab.blocks[e], w = int(unsigned(bw) >> 24) * 16, blocks = bw & 0xffffff;
        alone = blocks == 1;
        rp = blocks == 1 ? local : int(unsigned(local) / unsigned(blocks));
        const int b = local - rp * blocks;
        row0 = tab.first[e] + b * w;
        live = min(w, tab.count[e] - b * w);
        width = (live + 15) & ~15;
        // (the shuffles tell the compiler that the values are the same in all lanes)
        width = __shfl_sync(0xffffffffu, width, 0);
        return true;
    }
};

// Fills the tables: a thread takes a few experts in a row. blocks: tiles across the matrix; width: y rows of a tile at most (a multiple of 16, up to 256). Returns the number of
// tiles, which is more than there can be where offsets do not ascend. All THREADS threads of the block; sums: one a warp. The tables are
// complete behind the next barrier of the block.
template <int THREADS>
__device__ __forceinline__ long long group_tables(const GroupTables& tab, const int32_t* offsets, int E, int S, int width, int across, long long* sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (E + THREADS - 1) / THREADS, e0 = min(E, int(threadIdx.x) * per), e1 = min(E, e0 + per);
    long long sum = 0;
    for (int e = e0; e < e1; ++e) {
        int a = 0, b = S;
        if (offsets) {   // (what a plan says beyond the rows that there are is left out)
            a = min(max(__ldcg(offsets + e), 0), S);
            b = min(max(__ldcg(offsets + e + 1), a), S);
        }
        const int count = b - a, blocks = (count + width - 1) / width;
        const int w16 = blocks ? ((count + blocks - 1) / blocks + 15) >> 4 : 0;   // as even as multiples of 16 allow
        tab.first[e] = a;
        tab.count[e] = count;
        tab.blocks[e] = blocks | w16 << 24;
        sum += (long long)blocks * across;
        tab.tile_end[e] = int(sum);
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    long long before = inc - sum, total = 0;
    for (int i = 0; i < THREADS / 32; ++i) {
        before += i < warp ? sums[i] : 0;
        total += sums[i];
    }
    for (int e = e0; e < e1; ++e) tab.tile_end[e] += int(before);
    return total;
}

// y of eight y rows for one matrix row a lane: y points at the matrix row's element of the first y row
template <int MODE>
__device__ __forceinline__ void store8(const uint32_t (&v)[8], void* y, int64_t ldy, int live, bool have, bool pairs) {
    if (MODE == FRX_F32) {
        float* p = static_cast<float*>(y);
#pragma unroll
        for (int i = 0; i < 8; ++i, p += ldy)
            if (i < live && have) *p = __uint_as_float(v[i]);
        return;
    }
    const bool odd = threadIdx.x & 1;
    if (pairs) {   // two lanes exchange a value so that each has two neighbouring matrix rows of one y row
        uint16_t* p = static_cast<uint16_t*>(y) + (odd ? ldy - 1 : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i, p += 2 * ldy) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? v[2 * i] : v[2 * i + 1], 1);
            const float lo = __uint_as_float(odd ? got : v[2 * i]), hi = __uint_as_float(odd ? v[2 * i + 1] : got);
            uint32_t w;
            if (MODE == FRX_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
                w = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(lo, hi);
                w = *reinterpret_cast<const uint32_t*>(&h);
            }
            if (2 * i + int(odd) < live && have) *reinterpret_cast<uint32_t*>(p) = w;
        }
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(y);
#pragma unroll
    for (int i = 0; i < 8; ++i, p += ldy)
        if (i < live && have) {
            if (MODE == FRX_BF16)
                *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(__uint_as_float(v[i]));
            else
                *reinterpret_cast<__half*>(p) = __float2half_rn(__uint_as_float(v[i]));
        }
}

// ---- host side

// A tensor map with the 128-byte swizzle (box[0] elements are 128 bytes) over rows of dims[0] elements; strides in bytes, of the dimensions from the second on. What
// lies outside reads as zeros.
inline int encode_tensor_map(CUtensorMap& map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<void*> entry{nullptr};   // the driver's function: looked up once
    void* fn = entry.load(std::memory_order_acquire);
    if (!fn) {
        cudaDriverEntryPointQueryResult found;
        FRX_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !fn) return fail(FRX_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        entry.store(fn, std::memory_order_release);
    }
    const cuuint32_t steps[3] = {1, 1, 1};
    const CUresult r = reinterpret_cast<Encode>(fn)(&map, type, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? FRX_OK : fail(FRX_ERR_CUDA, "cuTensorMapEncodeTiled: error %d (%llu rows of %llu elements)", int(r), (unsigned long long)dims[1], (unsigned long long)dims[0]);
}

constexpr size_t kSmemMost = 227 * 1024;   // dynamic shared memory of a block at most
// Raises a kernel's limit of shared memory to that, once a device.
template <auto Kernel>
inline int allow_smem() {
    static std::mutex mu;
    static bool done[64] = {};
    int dev = 0;
    FRX_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 0 || dev >= 64 || !done[dev]) FRX_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemMost)));
    if (dev >= 0 && dev < 64) done[dev] = true;
    return FRX_OK;
}

}  // namespace frx
