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
    int stride;                  // tiles between two of this block: as many as there are blocks, or pairs of them
    __device__ __forceinline__ void begin(const GroupTables& tables, int experts, int block = int(blockIdx.x), int blocks = int(gridDim.x)) {
        tab = tables;
        E = experts;
        tile = block - blocks;
        stride = blocks;
        e = 0;
    }
    __device__ __forceinline__ bool next() {
        tile += stride;
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

// Fills the tables: a thread takes a few experts in a row. blocks: tiles across the matrix; width: y rows of a tile at most (a multiple of UNIT, up to 256). Returns the number of
// tiles, which is more than there can be where offsets do not ascend. All THREADS threads of the block; sums: one a warp. The tables are
// complete behind the next barrier of the block.
template <int THREADS, int UNIT = 16>
__device__ __forceinline__ long long group_tables(const GroupTables& tab, const int32_t* offsets, int E, int S, int width, int across, long long* sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (E + THREADS - 1) / THREADS, e0 = min(E, int(threadIdx.x) * per), e1 = min(E, e0 + per);
    constexpr int kFirst = 2;   // experts of a thread whose offsets are read at once (512 experts and 352 threads: 0.5 us less than one after the other)
    int first[kFirst + 1];
#pragma unroll
    for (int i = 0; i <= kFirst; ++i) first[i] = offsets && e0 + i <= e1 ? __ldcg(offsets + e0 + i) : 0;
    long long sum = 0;
    for (int e = e0; e < e1; ++e) {
        int a = 0, b = S;
        if (offsets) {   // (what a plan says beyond the rows that there are is left out)
            const int i = e - e0;
            a = i == 0 ? first[0] : i == 1 ? first[1] : __ldcg(offsets + e);
            b = i == 0 ? first[1] : i == 1 ? first[2] : __ldcg(offsets + e + 1);
            a = min(max(a, 0), S);
            b = min(max(b, a), S);
        }
        const int count = b - a, blocks = (count + width - 1) / width;
        const int w16 = blocks ? ((count + blocks - 1) / blocks + UNIT - 1) / UNIT * (UNIT / 16) : 0;   // as even as multiples of UNIT allow
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

// An element of rows that are added to, of which nothing is waited for here (as a conditional assignment the load becomes a branch that is waited for)
template <int TYPE>
__device__ __forceinline__ void load_one_if(uint32_t& w, const void* p, bool on) {
    if (TYPE == FRX_F32)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.u32 %0, [%1];\n\t}" : "+r"(w) : "l"(p), "r"(uint32_t(on)));
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.u16 %0, [%1];\n\t}" : "+r"(w) : "l"(p), "r"(uint32_t(on)));
}
template <int TYPE>
__device__ __forceinline__ float wide(uint32_t bits) {   // of the low half
    if (TYPE == FRX_BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half(uint16_t(bits)));
}

// ---- blocks of a cluster

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_peer(uint32_t addr) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory"); }
__device__ __forceinline__ void mbar_arrive_peer_relaxed(uint32_t addr) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory"); }
// warp_wait for what other blocks of the cluster have written
__device__ __forceinline__ bool warp_wait_cluster(uint32_t bar, uint32_t parity, uint32_t abort, uint64_t limit_ns) {
    if (!warp_wait(bar, parity, abort, limit_ns)) return false;
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}

// ---- 16-bit operands

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// A whole tile's step of 16 of depth, both operands in shared memory, issued by one thread
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 16 columns of this warp's lanes, complete on return
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[2][8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0][0]), "=r"(v[0][1]), "=r"(v[0][2]), "=r"(v[0][3]), "=r"(v[0][4]), "=r"(v[0][5]), "=r"(v[0][6]), "=r"(v[0][7]), "=r"(v[1][0]), "=r"(v[1][1]),
          "=r"(v[1][2]), "=r"(v[1][3]), "=r"(v[1][4]), "=r"(v[1][5]), "=r"(v[1][6]), "=r"(v[1][7])
        : "r"(addr)
        : "memory");
}

// ---- host side

// A tensor map with the 128-byte swizzle (box[0] elements are 128 bytes) over rows of dims[0] elements; strides in bytes, of the dimensions from the second on. What
// lies outside reads as zeros.
inline int encode_tensor_map(CUtensorMap& map, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                             CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_128B) {
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
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    const CUresult r = reinterpret_cast<Encode>(fn)(&map, type, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                    CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
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

// Instruction descriptor of kind::f16 without N: sums in 32 bits, both operands of one type (0 fp16, 1 bf16), `mn` bits where an operand is MN-major
inline uint32_t f16_idesc(int dtype, bool lanes_mn, bool cols_mn, int lanes = 128) {
    const uint32_t type = dtype == FRX_BF16;
    return (1u << 4) | type << 7 | type << 10 | uint32_t(lanes_mn) << 15 | uint32_t(cols_mn) << 16 | uint32_t(lanes >> 4) << 24;
}
// A map of 16-bit elements. The 128 bytes of a row that a box brings come into the L2 with their neighbours, which the next stage reads (1.5 GB of matrices by a row or two each 247 -> 228 us, by
// sixty 151 -> 140).
inline int encode_16(CUtensorMap& map, int dtype, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    return encode_tensor_map(map, dtype == FRX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, base, dims, strides, box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

// rows of n elements, `box` of them a load
inline int rows_map(CUtensorMap& map, const void* x, int64_t ld, int dtype, int rows, int n, int box) {
    const cuuint64_t dims[2] = {cuuint64_t(n), cuuint64_t(rows)}, strides[1] = {cuuint64_t(ld) * 2};
    const cuuint32_t boxes[2] = {64, cuuint32_t(box)};
    return encode_16(map, dtype, 2, x, dims, strides, boxes);
}
inline int matrices_map(CUtensorMap& map, const void* w, int64_t ldw, int64_t lde, int dtype, int E, int rows, int n, int box) {
    const cuuint64_t dims[3] = {cuuint64_t(n), cuuint64_t(rows), cuuint64_t(E)}, strides[2] = {cuuint64_t(ldw) * 2, cuuint64_t(lde) * 2};
    const cuuint32_t boxes[3] = {64, cuuint32_t(box), 1};
    return encode_16(map, dtype, 3, w, dims, strides, boxes);
}

inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// What TMA reads of 16-bit elements: rows `ld` apart, at least n long, on 16-byte boundaries. One row alone has no distance to the next.
inline int operand(const char* who, const char* what, const void* x, int64_t& ld, int64_t rows, int64_t n) {
    if (!x) return fail(FRX_ERR_ARG, "%s: null pointer (%s)", who, what);
    if (ld < n) return fail(FRX_ERR_ARG, "%s: rows of %s are %lld elements apart and %lld long", who, what, (long long)ld, (long long)n);
    if (rows == 1) ld = (n + 7) / 8 * 8;
    if (!aligned(x, 16) || ld % 8 || ld >= (int64_t(1) << 38))
        return fail(FRX_ERR_ARG, "%s: rows of %s must begin on 16-byte boundaries (they are %lld elements apart)", who, what, (long long)ld);
    return FRX_OK;
}
}  // namespace frx
