// Products of sorted rows with their experts' matrices in 16 bits, and their gradients (frx_moe_matmul, _backward_x, _backward_w in frx.h).
#include <algorithm>

#include "frx_groups.cuh"

namespace frx {
namespace {

// Three forms of one kernel. D is the tensor core's 256 x N block of sums (N a multiple of 32 up to 256); its lanes are the index that is contiguous in what
// is written, so that a warp's stores of a column are whole sectors and need no exchange through shared memory:
//   forward  y[r][m]     = sum_k W_e[m][k] x[r][k]     lanes: matrix rows m, columns: rows r of expert e, depth: n
//   grad x   gx[r][m]    = sum_k W_e[k][m] gy[r][k]    lanes: matrix columns m, columns: rows r of expert e, depth: rows of the matrix
//   grad w   gW_e[c][m]  = sum_t gy[t][c] x[t][m]      lanes: matrix columns m, columns: matrix rows c, depth: the rows t of expert e
// The rows of an expert are the N side in the first two, so that few rows waste little (N is that of the tile, not of the kernel), and the matrix is read once per 256 of
// them. Operands come by TMA in the 128-byte swizzle as they lie in memory: a side whose index is contiguous there is the instruction's MN-major form, which is as fast, so no
// operand is ever transposed. A stage is 64 of depth. What lies beyond a matrix, or beyond all rows, arrives as zeros. Rows of the next expert that a box brings along fill
// columns of D that are not stored; in the third form, where they would be summed, they are zeroed in shared memory first.
//
// Two blocks on neighbouring SMs (a cluster) share a tile of 256 lanes by up to 256 columns: the instruction (cta_group::2) takes 128 lanes and half of the columns from the shared memory of
// each and leaves 128 lanes of all columns in the tensor memory of each: 32 KB a stage and SM for 512 clocks of products where one block's tile of 128 x 256 takes 48. The
// first block of a pair issues; both load their own operands, whose bytes are counted on the first one's barriers, and both write their own lanes. 131,072 rows of 2,048 by 1,024: 712 us with
// single blocks, 593 with pairs, 521 with two loads a stage instead of five.
//
// What bounds it. 65,536 rows of 64 equal experts, 2,048 by 1,024: 212 us, gradients 221 and 216 (1,300, 1,240 and 1,270 TFLOP/s; the library's batched product of the same matrices, equal
// experts alone, takes 202): some 17,300 clocks a tile of 16,400 that the tensor cores need, at 1.1 to 1.3 GHz, which is what the power limit leaves. Experts of 1,030 rows instead of 1,024, whose five
// tiles of 224 columns wait for their loads: 244, 254 and 253. 131,072 rows of 128 experts of a skewed routing: 542, 28 % more than twice the 212. A row or two an expert: the matrices. 64 tokens of
// ten experts out of 512: 1.54 GB in 226 us, 6.8 TB/s of what has to move. One token: 40 tiles, 8.5 of 15 us for 512 KB a block, the rest is start, tables and end. Gradients of matrices with few rows:
// what is written (128 of 2,560 by 1,280 in 32 bits, 1.68 GB, 280 us). Added to what is there (65,536 rows): 297 us, in 32 bits 396 instead of 265: a lane's 16 elements are read at once, but
// none before the sums are there.
enum Form { kForward, kGradX, kGradW };

constexpr int kTileM = 256, kLanes = 128, kDepth = 64, kTileN = 256, kUnitN = 32;   // lanes of a tile, of a block; columns of a tile at most, what they are a multiple of
constexpr int kStageA = kLanes * kDepth * 2, kChunk = 64 * kDepth * 2;   // bytes of a stage's lanes side; of 64 contiguous elements x 64 of an MN-major side
constexpr int kMaxStages = 10, kMaxSets = 8;
constexpr int kWarpsEpi = 8, kWarpLoad = 8, kWarpMma = 9, kWarpTail = 10, kThreads = 32 * 11;
constexpr int kBarFull = 0, kBarFree = kMaxStages, kBarDFull = 2 * kMaxStages, kBarDFree = kBarDFull + kMaxSets, kBarTail = kBarDFree + kMaxSets, kBarTailPeer = kBarTail + kMaxStages, kBars = kBarTailPeer + kMaxStages;
constexpr int kAbort = 512, kSlot = 516, kSums = 640, kHead = 1024;
static_assert(kBars * 8 <= kAbort && kSums + 8 * kThreads / 32 <= kHead, "the block's head");

struct Product {
    const int32_t* offsets;   // [E + 1]
    void* y;
    int64_t ldy, ldye;        // elements between y's rows, and in the third form between its matrices
    unsigned long long wait_ns;
    int E, S;
    int lanes, cols, depth;   // extents: of the lanes side; of the columns side in the third form; of the depth in the other two
    int width, box, box_small;   // columns of a tile at most; rows of a load of the columns side in the first two forms, and of a small one
    int unit;                 // columns of a tile are a multiple of this
    int lanes_chunks, cols_chunks;   // chunks of 64 a load of an MN-major side brings
    int stages, stage_bytes;
    int most;                 // tiles of any plan whose experts' rows do not overlap
    uint32_t idesc;           // the instruction descriptor without N
    int run;                  // stages whose products are summed by the tensor cores
    int sets;                 // of accumulators, `width` columns each
    int add;                  // third form: added to what is there
};

// Shared-memory descriptor of an operand whose rows of 128 bytes run along its own index (64 elements) and not along the depth: 128-byte swizzle, eight of depth
// 1024 bytes apart, the next 64 elements a chunk further.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr) { return umma_desc(smem_addr, kChunk, 1024) | (uint64_t(2) << 61); }

// Loads of a pair: into this block's shared memory, counted on a barrier of the first block (at its address in the cluster)
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_4d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int u, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(u),
                 "r"(bar)
                 : "memory");
}
// 256 lanes x N x 16 of depth, operands at the same places in both blocks' shared memory
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// An arrival at this barrier of both blocks when every MMA issued so far by this thread has completed
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_result, uint32_t cols) {   // by one warp of each block
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t base, uint32_t cols) { asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory"); }

// what is there, added to 16 columns of this lane (32 bits, before the one rounding): all of them are on their way at once
template <int TYPE>
__device__ __forceinline__ void add16(uint32_t (&v)[2][8], const uint8_t* y, int64_t ldy, int live, bool have) {
    constexpr int size = TYPE == FRX_F32 ? 4 : 2;
    uint32_t old[16] = {};
#pragma unroll
    for (int i = 0; i < 16; ++i) load_one_if<TYPE>(old[i], y + i * ldy * size, i < live && have);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = __float_as_uint(__uint_as_float(v[i / 8][i % 8]) + (TYPE == FRX_F32 ? __uint_as_float(old[i]) : wide<TYPE>(old[i])));
}

// The tiles of a block. First two forms: those of GroupWalk (expert, lanes tile, block of its rows). Third form: every matrix has as many.
template <int FORM>
struct Tiles {
    GroupWalk g;
    int tile, per, across;   // third form: the tile, tiles of a matrix, of them along the columns
    int e, lane0, col0, live, width;   // expert; first of the tile's lanes side; first column, columns, their number rounded up to 32
    int row0, steps, last;   // first row of the expert; stages; depth of the last one
    __device__ __forceinline__ void begin(const Product& p, const GroupTables& tab, int experts) {
        if (FORM == kGradW) {
            g.tab = tab;
            across = (p.cols + kTileN - 1) / kTileN;
            per = across * ((p.lanes + kTileM - 1) / kTileM);
            tile = int(blockIdx.x >> 1) - int(gridDim.x >> 1);
        } else {
            g.begin(tab, experts, int(blockIdx.x >> 1), int(gridDim.x >> 1));
            steps = (p.depth + kDepth - 1) / kDepth;
            last = p.depth - (steps - 1) * kDepth;
        }
    }
    __device__ __forceinline__ bool next(const Product& p) {
        if (FORM == kGradW) {
            tile += int(gridDim.x >> 1);
            e = tile / per;
            if (e >= p.E) return false;
            const int local = tile - e * per, m = local / across;
            lane0 = m * kTileM;
            col0 = (local - m * across) * kTileN;
            live = min(kTileN, p.cols - col0);
            width = (live + p.unit - 1) & -p.unit;
            row0 = g.tab.first[e];
            const int count = g.tab.count[e];
            steps = (count + kDepth - 1) / kDepth;
            last = count - (steps - 1) * kDepth;
            return true;
        }
        if (!g.next()) return false;
        e = g.e;
        lane0 = g.rp * kTileM;
        row0 = col0 = g.row0;
        live = g.live;
        width = __shfl_sync(0xffffffffu, (live + kUnitN - 1) & -kUnitN, 0);
        return true;
    }
};

template <int FORM, int TYPE>
__global__ void __launch_bounds__(kThreads, 1) k_moe_product(const Product p, const __grid_constant__ CUtensorMap lanes_map, const __grid_constant__ CUtensorMap cols_map,
                                                              const __grid_constant__ CUtensorMap small_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t s0 = smem_u32(smem), stages0 = s0 + kHead, bars = s0, abort = s0 + kAbort, n_stages = uint32_t(p.stages), stage_bytes = uint32_t(p.stage_bytes);
    const uint32_t rank = cluster_rank(), bars_first = peer_addr(bars, 0);   // the barriers of the pair's first block
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kAbort);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSlot);
    GroupTables tab;
    tab.tile_end = reinterpret_cast<int*>(smem + kHead + n_stages * stage_bytes);
    tab.first = tab.tile_end + p.E;
    tab.count = tab.first + p.E;
    tab.blocks = tab.count + p.E;
    if (threadIdx.x == 0) {
        uint64_t* b = reinterpret_cast<uint64_t*>(smem);
        for (int i = 0; i < kMaxStages; ++i) {
            mbar_init(b + kBarFull + i, 1);   // the first block, with the bytes of both
            mbar_init(b + kBarFree + i, 1);
            mbar_init(b + kBarTail + i, 1);
            mbar_init(b + kBarTailPeer + i, 1);
        }
        for (int i = 0; i < kMaxSets; ++i) {
            mbar_init(b + kBarDFull + i, 1);
            mbar_init(b + kBarDFree + i, 2 * kWarpsEpi);
        }
        asm volatile("prefetch.tensormap [%0];" ::"l"(&lanes_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&cols_map) : "memory");
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kWarpMma) tmem_alloc_pair(tmem_slot, 512);
    __syncwarp();
    cluster_sync_all();   // the barriers of both blocks are there
    pdl_wait();
    pdl_trigger();
    const long long tiles = group_tables<kThreads, kUnitN>(tab, p.offsets, p.E, p.S, p.width, (p.lanes + kTileM - 1) / kTileM, reinterpret_cast<long long*>(smem + kSums));
    const int experts = FORM != kGradW && tiles > p.most ? 0 : p.E;   // offsets that do not ascend: nothing is computed
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    Tiles<FORM> t;
    t.begin(p, tab, experts);

    // "free" barriers are waited on with the parity of the phase before the one about to be used, which a fresh barrier reports as complete
    if (warp == kWarpLoad) {
        // ---------------- loads: this block's 128 lanes and its half of the columns, in as few as possible (each costs the issuing thread some 100 clocks, whatever its size: with
        // 5 of them a stage took 750 clocks, with two 520)
        uint32_t st = 0, phase = 1;
        bool ok = true;
        while (ok && t.next(p)) {
            const int half = t.width / 2, lane0 = t.lane0 + int(rank) * kLanes, col0 = t.col0 + int(rank) * half;
            const bool small = FORM != kGradW && half <= 3 * p.box_small;
            const int box = FORM == kGradW ? 64 * p.cols_chunks : small ? p.box_small : p.box, boxes = (half + box - 1) / box, box_bytes = box * 128;
            const CUtensorMap* const cols = small ? &small_map : &cols_map;
            const uint32_t bytes = uint32_t(kStageA + boxes * box_bytes);
            for (int s = 0; s < t.steps; ++s) {
                if (!(ok = warp_wait(bars + (kBarFree + st) * 8, phase, abort, p.wait_ns))) break;
                const uint32_t a = stages0 + st * stage_bytes, b = a + kStageA;
                // rows of the next expert have to be zeroed in the last stage: its bytes are counted here, and kWarpTail reports
                const bool tail = FORM == kGradW && s + 1 == t.steps && t.last % 16 != 0;
                const uint32_t full = tail ? peer_addr(bars + (kBarTail + st) * 8, rank) : bars_first + (kBarFull + st) * 8;
                if (lane == 0) {
                    if (tail)
                        mbar_expect_tx(bars + (kBarTail + st) * 8, bytes);
                    else if (rank == 0)
                        mbar_expect_tx(bars + (kBarFull + st) * 8, 2 * bytes);
                    if (FORM == kForward) {
                        tma_3d_pair(a, &lanes_map, s * kDepth, lane0, t.e, full);
                    } else if (p.lanes_chunks == 2) {
                        if (FORM == kGradX)
                            tma_4d_pair(a, &lanes_map, 0, s * kDepth, lane0 / 64, t.e, full);
                        else
                            tma_3d_pair(a, &lanes_map, 0, t.row0 + s * kDepth, lane0 / 64, full);
                    } else {
                        for (int i = 0; i < 2; ++i) {
                            if (FORM == kGradX)
                                tma_3d_pair(a + i * kChunk, &lanes_map, lane0 + 64 * i, s * kDepth, t.e, full);
                            else
                                tma_2d_pair(a + i * kChunk, &lanes_map, lane0 + 64 * i, t.row0 + s * kDepth, full);
                        }
                    }
                    if (FORM == kGradW && p.cols_chunks == 2)
                        tma_3d_pair(b, &cols_map, 0, t.row0 + s * kDepth, col0 / 64, full);
                    else
                        for (int i = 0; i < boxes; ++i) {
                            if (FORM == kGradW)
                                tma_2d_pair(b + i * kChunk, &cols_map, col0 + 64 * i, t.row0 + s * kDepth, full);
                            else
                                tma_2d_pair(b + i * box_bytes, cols, s * kDepth, col0 + i * box, full);
                        }
                }
                __syncwarp();
                if (++st == n_stages) st = 0, phase ^= 1u;
            }
        }
    } else if (warp == kWarpTail) {
        // ---------------- third form: the rows behind the expert's last one, up to the next 16, to zeros in both operands (a row of depth is 128 bytes in every chunk, whatever the swizzle)
        if (FORM == kGradW) {
            uint32_t st = 0, phases = 0;   // a stage's barriers are used again only when its products are done: a phase bit each (one barrier for all stages could run two phases ahead of its waiter)
            while (t.next(p)) {
                st += uint32_t(t.steps);
                if (t.steps && t.last % 16) {
                    const uint32_t stage = (st - 1) % n_stages;
                    if (!warp_wait(bars + (kBarTail + stage) * 8, phases >> stage & 1u, abort, p.wait_ns)) break;
                    const uint32_t a = stages0 + stage * stage_bytes;
                    const int extra = 16 - t.last % 16, chunks = 2 + (t.width / 2 + 63) / 64;
                    for (int i = lane; i < chunks * extra * 8; i += 32) {
                        const int r = i >> 3, c = r / extra;
                        const uint32_t at = a + uint32_t(c * kChunk + (t.last + r - c * extra) * 128 + (i & 7) * 16);   // (the lanes side's two chunks, then the columns')
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                    }
                    fence_async_smem();   // generic-proxy writes: visible to the tensor core
                    __syncwarp();
                    if (rank == 0 && !warp_wait_cluster(bars + (kBarTailPeer + stage) * 8, phases >> stage & 1u, abort, p.wait_ns)) break;
                    if (lane == 0) mbar_arrive_peer(bars_first + ((rank ? kBarTailPeer : kBarFull) + stage) * 8);
                    phases ^= 1u << stage;
                }
                st %= n_stages;
            }
        }
    } else if (warp == kWarpMma) {
        // ---------------- MMA: the first block's warp, one elected lane
        uint32_t st = 0, phase = 0, set = 0, dphase = 1;
        bool ok = rank == 0;
        while (ok && t.next(p)) {
            const uint32_t idesc = p.idesc | uint32_t(t.width >> 3) << 17;
            for (int first = 0; first == 0 || first < t.steps; first += p.run) {   // (an expert without rows has one run of nothing)
                if (!(ok = warp_wait(bars + (kBarDFree + set) * 8, dphase, abort, p.wait_ns))) break;
                tc_fence_after_sync();   // behind the epilogues' loads of these accumulators
                const uint32_t acc = tmem + set * uint32_t(p.width);
                const int end = min(t.steps, first + p.run);
                for (int s = first; s < end; ++s) {
                    if (!(ok = warp_wait_cluster(bars + (kBarFull + st) * 8, phase, abort, p.wait_ns))) break;
                    const uint32_t a = stages0 + st * stage_bytes, b = a + kStageA;
                    const int depth = s + 1 < t.steps ? kDepth : t.last;
                    if (elect_one()) {
                        const uint64_t da = FORM == kForward ? umma_desc_sw128(a) : umma_desc_mn(a), db = FORM == kGradW ? umma_desc_mn(b) : umma_desc_sw128(b);
                        constexpr uint64_t kStepK = 32 >> 4, kStepMn = 16 * 128 >> 4;   // 16 of depth
#pragma unroll
                        for (int k = 0; k < kDepth / 16; ++k) {
                            if (k * 16 >= depth) break;
                            umma_f16_pair(acc, da + k * (FORM == kForward ? kStepK : kStepMn), db + k * (FORM == kGradW ? kStepMn : kStepK), idesc, s - first + k > 0);
                        }
                        umma_commit_pair(bars + (kBarFree + st) * 8);
                    }
                    __syncwarp();
                    if (++st == n_stages) st = 0, phase ^= 1u;
                }
                if (!ok) break;
                if (elect_one()) umma_commit_pair(bars + (kBarDFull + set) * 8);
                __syncwarp();
                if (++set == uint32_t(p.sets)) set = 0, dphase ^= 1u;
            }
        }
    } else {
        // ---------------- epilogue: a warp has a quarter of the lanes and every second 16 columns, whose sums it keeps in registers
        const int quarter = warp & 3, part = warp >> 2, m = quarter * 32 + lane;
        constexpr int size = TYPE == FRX_F32 ? 4 : 2, kSixteens = kTileN / 32;
        uint32_t set = 0, phase = 0;
        const bool pairs = TYPE != FRX_F32 && p.lanes % 2 == 0 && p.ldy % 2 == 0 && (FORM != kGradW || p.ldye % 2 == 0) && reinterpret_cast<uintptr_t>(p.y) % 4 == 0;
        bool lost = false;   // a wait ran out: NaN, not a wrong number, and no more waits
        // a run's sums are there; they have been read
        auto wait_for_sums = [&]() {
            lost = lost || !warp_wait(bars + (kBarDFull + set) * 8, phase, abort, p.wait_ns);
            tc_fence_after_sync();
            return tmem + (uint32_t(quarter * 32) << 16) + set * uint32_t(p.width);
        };
        auto give_back = [&]() {
            if (!lost) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_peer_relaxed(bars_first + (kBarDFree + set) * 8);   // (tensor memory alone has been read: nothing of memory to wait for)
            }
            if (++set == uint32_t(p.sets)) set = 0, phase ^= 1u;
        };
        while (t.next(p)) {
            const int at_lane = t.lane0 + int(rank) * kLanes + m;
            const bool have = at_lane < p.lanes;
            uint8_t* y = static_cast<uint8_t*>(p.y) + ((FORM == kGradW ? t.e * p.ldye : 0) + t.col0 * p.ldy + at_lane) * size;
            auto store16 = [&](uint32_t (&v)[2][8], int c) {
                if (lost) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = 0x7fffffffu;
                }
                if (FORM == kGradW && p.add) add16<TYPE>(v, y + c * p.ldy * size, p.ldy, t.live - c, have);
#pragma unroll
                for (int h = 0; h < 2; ++h) store8<TYPE>(v[h], y + (c + 8 * h) * p.ldy * size, p.ldy, t.live - c - 8 * h, have, pairs);
            };
            if (t.steps <= p.run) {   // one run: from tensor memory to y
                const uint32_t acc = wait_for_sums();
                const bool empty = FORM == kGradW && t.steps == 0;
                for (int c = part * 16; c < t.width && !(empty && p.add && !lost); c += 32) {
                    uint32_t v[2][8] = {};
                    if (!lost && !empty) tmem_ld16(acc + c, v);
                    store16(v, c);
                }
                give_back();
                continue;
            }
            uint32_t sums[kSixteens][2][8] = {};
            for (int first = 0; first < t.steps; first += p.run) {
                const uint32_t acc = wait_for_sums();
#pragma unroll
                for (int c = 0; c < kSixteens; ++c) {
                    if (c * 32 + part * 16 >= t.width || lost) break;
                    uint32_t v[2][8];
                    tmem_ld16(acc + c * 32 + part * 16, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) sums[c][i / 8][i % 8] = __float_as_uint(__uint_as_float(sums[c][i / 8][i % 8]) + __uint_as_float(v[i / 8][i % 8]));
                }
                give_back();
            }
#pragma unroll
            for (int c = 0; c < kSixteens; ++c) {
                if (c * 32 + part * 16 >= t.width) break;   // (instructions that are not reached are not fetched either)
                store16(sums[c], c * 32 + part * 16);
            }
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
    }
    cluster_sync_all();   // neither block's shared or tensor memory is used by the other any more
    if (warp == kWarpMma) tmem_free_pair(tmem, 512);
}

template <int FORM, int TYPE>
int launch_typed(Product& p, const CUtensorMap& lanes_map, const CUtensorMap& cols_map, const CUtensorMap& small_map, cudaStream_t stream) {
    const size_t tables = size_t(p.E) * 16;
    int rc = allow_smem<k_moe_product<FORM, TYPE>>();
    if (rc != FRX_OK) return rc;
    const int64_t lane_tiles = (p.lanes + kTileM - 1) / kTileM;
    const int64_t most = FORM == kGradW ? lane_tiles * ((p.cols + kTileN - 1) / kTileN) * p.E : lane_tiles * (int64_t(p.S) / p.width + std::min(p.E, p.S));
    if (most > 0x7fff0000 || p.S / 16 >= (1 << 24)) return fail(FRX_ERR_SHAPE, "product by expert: %lld tiles of %d rows", (long long)most, p.S);
    p.most = int(most);
    p.stages = int(std::min<size_t>(kMaxStages, (kSmemMost - kHead - tables) / size_t(p.stage_bytes)));
    static_assert((kSmemMost - kHead - 4096 * 16) / (kStageA + kTileN / 2 * kDepth * 2) >= 4, "stages beside the tables of 4096 experts");
    // The tensor cores add to their sums by cutting off, half a step of 2^-23 of the sum so far on average and always towards zero: 128 additions (2,048 of depth) leave a relative error of
    // 2.1e-6 in the root mean square. So they sum over a part of the depth at a time, and the epilogue adds these sums up rounded to nearest. What is returned in 32 bits: 256 of depth, 2.4e-7 (a plain
    // sum in 32 bits leaves 1e-7 to 1e-6, by its order and depth). What is rounded to 16 bits afterwards, by up to 2^-8 or 2^-11: 1,024 of depth, 1.0e-6. It costs nothing where matrices are the
    // traffic; where the tensor cores are busy a tenth in 32 bits (131,072 rows of 2,048 by 1,024 523 instead of 469 us) and 1 to 2 % in 16 (the same 545 instead of 538 in a stream of such, 65,536 rows 211
    // instead of 207; with 512 of depth 550 and 217: an epilogue that writes has two runs' time before the tensor cores wait for it).
    p.run = TYPE == FRX_F32 ? 4 : 16;
    p.sets = std::min(kMaxSets, 512 / p.width);
    p.wait_ns = wait_limit_ns();
    const unsigned pairs = unsigned(std::min<int64_t>(std::max(1, sm_count() / 2), std::max<int64_t>(1, most)));
    FRX_LAUNCH(kKProduct, stream,
               launch_pdl_cluster(k_moe_product<FORM, TYPE>, dim3(2 * pairs), dim3(kThreads), kHead + size_t(p.stages) * p.stage_bytes + tables, stream, 2u, p, lanes_map, cols_map, small_map));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}
template <int FORM>
int launch(Product& p, int type, const CUtensorMap& lanes_map, const CUtensorMap& cols_map, const CUtensorMap& small_map, cudaStream_t stream) {
    switch (type) {
        case FRX_F32: return launch_typed<FORM, FRX_F32>(p, lanes_map, cols_map, small_map, stream);
        case FRX_BF16: return launch_typed<FORM, FRX_BF16>(p, lanes_map, cols_map, small_map, stream);
        default: return launch_typed<FORM, FRX_F16>(p, lanes_map, cols_map, small_map, stream);
    }
}

// Sides whose index is contiguous in memory, 64 of depth a load: two chunks of 64 at once where the extent is whole chunks (the chunk is a dimension of the map then), else one
int depth_rows_map(CUtensorMap& map, const void* x, int64_t ld, int dtype, int rows, int n, int chunks) {
    if (chunks == 1) return rows_map(map, x, ld, dtype, rows, n, kDepth);
    const cuuint64_t dims[3] = {64, cuuint64_t(rows), cuuint64_t(n / 64)}, strides[2] = {cuuint64_t(ld) * 2, 128};
    const cuuint32_t boxes[3] = {64, kDepth, cuuint32_t(chunks)};
    return encode_16(map, dtype, 3, x, dims, strides, boxes);
}
int depth_matrices_map(CUtensorMap& map, const void* w, int64_t ldw, int64_t lde, int dtype, int E, int rows, int n, int chunks) {
    if (chunks == 1) return matrices_map(map, w, ldw, lde, dtype, E, rows, n, kDepth);
    const cuuint64_t dims[4] = {64, cuuint64_t(rows), cuuint64_t(n / 64), cuuint64_t(E)}, strides[3] = {cuuint64_t(ldw) * 2, 128, cuuint64_t(lde) * 2};
    const cuuint32_t boxes[4] = {64, kDepth, cuuint32_t(chunks), 1};
    return encode_16(map, dtype, 4, w, dims, strides, boxes);
}

int shape(const char* who, int dtype, int out_dtype, int E, int rows, int n, int S) {
    if (S < 0) return fail(FRX_ERR_ARG, "%s: %d rows", who, S);
    if (dtype != FRX_BF16 && dtype != FRX_F16) return fail(FRX_ERR_ARG, "%s: element type %d (bfloat16 or float16)", who, dtype);
    if (!dtype_size(out_dtype)) return fail(FRX_ERR_ARG, "%s: element type %d", who, out_dtype);
    if (E < 1 || E > 4096 || rows < 1 || n < 1 || rows > (1 << 20) || n > (1 << 20)) return fail(FRX_ERR_SHAPE, "%s: unsupported shape E %d, rows %d, n %d", who, E, rows, n);
    return FRX_OK;
}
int result(const char* who, const char* what, const void* y, int64_t ld, int64_t n, int out_dtype) {
    if (!y) return fail(FRX_ERR_ARG, "%s: null pointer (%s)", who, what);
    if (ld < n) return fail(FRX_ERR_ARG, "%s: rows of %s are %lld elements apart and %lld long", who, what, (long long)ld, (long long)n);
    if (!rows_aligned(y, dtype_size(out_dtype))) return fail(FRX_ERR_ARG, "%s: misaligned pointer (%s)", who, what);
    return FRX_OK;
}

// Columns of a tile of rows: twice what an expert has on average, so that most experts' rows are one tile, and no more, so that a stage of few rows is mostly matrix and many are in
// flight.
void row_tiles(Product& p) {
    const int average = (p.S + p.E - 1) / p.E;
    p.width = kUnitN;
    while (p.width < kTileN && p.width < 2 * average) p.width *= 2;
    p.box = p.width / 2;
    p.box_small = std::max(16, p.width / 8);
    p.stage_bytes = kStageA + p.width / 2 * kDepth * 2;
}

}  // namespace
}  // namespace frx

using namespace frx;

extern "C" {

int frx_moe_matmul(frx_stream_t stream, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t lde, int dtype, const int32_t* offsets, int E, int rows, int n, int S,
                   void* y, int64_t ldy, int out_dtype) {
    const char* who = "frx_moe_matmul";
    int rc = shape(who, dtype, out_dtype, E, rows, n, S);
    if (rc != FRX_OK || S == 0) return rc;
    if ((rc = operand(who, "x", x, ldx, S, n)) != FRX_OK || (rc = operand(who, "w", w, ldw, rows, n)) != FRX_OK || (rc = result(who, "y", y, ldy, rows, out_dtype)) != FRX_OK) return rc;
    if ((rc = operand(who, "w (its matrices)", w, lde, E, (rows - 1) * ldw + n)) != FRX_OK) return rc;
    if (!offsets) return fail(FRX_ERR_ARG, "%s: null pointer (offsets)", who);
    Product p{};
    p.offsets = offsets;
    p.y = y;
    p.ldy = ldy;
    p.E = E;
    p.S = S;
    p.lanes = rows;
    p.depth = n;
    row_tiles(p);
    p.idesc = f16_idesc(dtype, false, false, kTileM);
    CUtensorMap wm, xm, small;
    if ((rc = matrices_map(wm, w, ldw, lde, dtype, E, rows, n, kLanes)) != FRX_OK || (rc = rows_map(xm, x, ldx, dtype, S, n, p.box)) != FRX_OK ||
        (rc = rows_map(small, x, ldx, dtype, S, n, p.box_small)) != FRX_OK)
        return rc;
    return launch<kForward>(p, out_dtype, wm, xm, small, stream);
}

int frx_moe_matmul_backward_x(frx_stream_t stream, const void* gy, int64_t ldgy, const void* w, int64_t ldw, int64_t lde, int dtype, const int32_t* offsets, int E, int rows, int n,
                              int S, void* gx, int64_t ldgx, int out_dtype) {
    const char* who = "frx_moe_matmul_backward_x";
    int rc = shape(who, dtype, out_dtype, E, rows, n, S);
    if (rc != FRX_OK || S == 0) return rc;
    if ((rc = operand(who, "gy", gy, ldgy, S, rows)) != FRX_OK || (rc = operand(who, "w", w, ldw, rows, n)) != FRX_OK || (rc = result(who, "gx", gx, ldgx, n, out_dtype)) != FRX_OK)
        return rc;
    if ((rc = operand(who, "w (its matrices)", w, lde, E, (rows - 1) * ldw + n)) != FRX_OK) return rc;
    if (!offsets) return fail(FRX_ERR_ARG, "%s: null pointer (offsets)", who);
    Product p{};
    p.offsets = offsets;
    p.y = gx;
    p.ldy = ldgx;
    p.E = E;
    p.S = S;
    p.lanes = n;
    p.depth = rows;
    row_tiles(p);
    p.idesc = f16_idesc(dtype, true, false, kTileM);
    p.lanes_chunks = n % 64 == 0 ? 2 : 1;
    CUtensorMap wm, gm, small;
    if ((rc = depth_matrices_map(wm, w, ldw, lde, dtype, E, rows, n, p.lanes_chunks)) != FRX_OK || (rc = rows_map(gm, gy, ldgy, dtype, S, rows, p.box)) != FRX_OK ||
        (rc = rows_map(small, gy, ldgy, dtype, S, rows, p.box_small)) != FRX_OK)
        return rc;
    return launch<kGradX>(p, out_dtype, wm, gm, small, stream);
}

int frx_moe_matmul_backward_w(frx_stream_t stream, const void* gy, int64_t ldgy, const void* x, int64_t ldx, int dtype, const int32_t* offsets, int E, int rows, int n, int S, void* gw,
                              int64_t ldgw, int64_t ldge, int out_dtype, int add) {
    const char* who = "frx_moe_matmul_backward_w";
    int rc = shape(who, dtype, out_dtype, E, rows, n, S);
    if (rc != FRX_OK) return rc;
    if ((rc = result(who, "gw", gw, ldgw, n, out_dtype)) != FRX_OK) return rc;
    if (E > 1 && ldge < (rows - 1) * ldgw + n) return fail(FRX_ERR_ARG, "%s: matrices of gw are %lld elements apart and overlap", who, (long long)ldge);
    if (S == 0) {   // no rows: the gradient of every matrix is 0
        const size_t size = size_t(dtype_size(out_dtype));
        for (int e = 0; e < E && !add; ++e)
            FRX_CUDA(cudaMemset2DAsync(static_cast<uint8_t*>(gw) + size_t(e) * ldge * size, size_t(ldgw) * size, 0, size_t(n) * size, size_t(rows), stream));
        return FRX_OK;
    }
    if ((rc = operand(who, "gy", gy, ldgy, S, rows)) != FRX_OK || (rc = operand(who, "x", x, ldx, S, n)) != FRX_OK) return rc;
    if (!offsets) return fail(FRX_ERR_ARG, "%s: null pointer (offsets)", who);
    Product p{};
    p.offsets = offsets;
    p.y = gw;
    p.ldy = ldgw;
    p.ldye = ldge;
    p.E = E;
    p.S = S;
    p.lanes = n;
    p.cols = rows;
    p.width = kTileN;
    p.add = add != 0;
    p.stage_bytes = kStageA + std::min((rows + 127) / 128, kTileN / 128) * kChunk;
    p.idesc = f16_idesc(dtype, true, true, kTileM);
    p.lanes_chunks = n % 64 == 0 ? 2 : 1;
    p.cols_chunks = rows % 64 == 0 && rows > 128 ? 2 : 1;
    p.unit = p.cols_chunks == 2 ? 128 : kUnitN;   // (a block's half begins with a chunk)
    CUtensorMap xm, gm;
    if ((rc = depth_rows_map(xm, x, ldx, dtype, S, n, p.lanes_chunks)) != FRX_OK || (rc = depth_rows_map(gm, gy, ldgy, dtype, S, rows, p.cols_chunks)) != FRX_OK) return rc;
    return launch<kGradW>(p, out_dtype, xm, gm, gm, stream);
}

}  // extern "C"
