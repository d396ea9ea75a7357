// Products of sorted rows with their experts' matrices in 16 bits, and their gradients (frx_moe_matmul, _backward_x, _backward_w in frx.h).
#include <algorithm>

#include "frx_groups.cuh"

namespace frx {
namespace {

// Three forms of one kernel. D is the tensor core's 128 x N block of sums (N a multiple of 16 up to 256); its lanes are the index that is contiguous in what
// is written, so that a warp's stores of a column are whole sectors and need no exchange through shared memory:
//   forward  y[r][m]     = sum_k W_e[m][k] x[r][k]     lanes: matrix rows m, columns: rows r of expert e, depth: n
//   grad x   gx[r][m]    = sum_k W_e[k][m] gy[r][k]    lanes: matrix columns m, columns: rows r of expert e, depth: rows of the matrix
//   grad w   gW_e[c][m]  = sum_t gy[t][c] x[t][m]      lanes: matrix columns m, columns: matrix rows c, depth: the rows t of expert e
// The rows of an expert are the N side in the first two, so that few rows waste nothing (N is that of the tile, not of the kernel), and the matrix is read once per 256 of
// them. Operands come by TMA in the 128-byte swizzle as they lie in memory: a side whose index is contiguous there is the instruction's MN-major form, so no
// operand is ever transposed. A stage is 64 of depth. What lies beyond a matrix, or beyond all rows, arrives as zeros. Rows of the next expert that a box brings along fill
// columns of D that are not stored; in the third form, where they would be summed, they are zeroed in shared memory first.
enum Form { kForward, kGradX, kGradW };

constexpr int kTileM = 128, kDepth = 64, kTileN = 256;
constexpr int kStageA = kTileM * kDepth * 2, kChunk = 64 * kDepth * 2;   // bytes of a stage's lanes side; of 64 contiguous elements x 64 of an MN-major side
constexpr int kMaxStages = 10;
constexpr int kWarpsEpi = 8, kWarpLoad = 8, kWarpMma = 9, kThreads = 32 * 10;
constexpr int kBarFull = 0, kBarFree = kMaxStages, kBarDFull = 2 * kMaxStages, kBarDFree = kBarDFull + 2, kBars = kBarDFree + 2;
constexpr int kAbort = 512, kSlot = 516, kSums = 640, kHead = 1024;
static_assert(kBars * 8 <= kAbort && kSums + 8 * kThreads / 32 <= kHead, "the block's head");

struct Product {
    const int32_t* offsets;   // [E + 1]
    void* y;
    int64_t ldy, ldye;        // elements between y's rows, and in the third form between its matrices
    unsigned long long wait_ns;
    int E, S;
    int lanes, cols, depth;   // extents: of the lanes side; of the columns side in the third form; of the depth in the other two
    int width, box;           // columns of a tile at most; rows of a load of the columns side in the first two forms
    int stages, stage_bytes;
    int most;                 // tiles of any plan whose experts' rows do not overlap
    uint32_t idesc;           // the instruction descriptor without N
    int add;                  // third form: added to what is there
};

// Shared-memory descriptor of an operand whose rows of 128 bytes run along its own index (64 elements) and not along the depth: 128-byte swizzle, eight of depth
// 1024 bytes apart, the next 64 elements a chunk further.
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr) { return umma_desc(smem_addr, kChunk, 1024) | (uint64_t(2) << 61); }

// what is there, added to eight columns of this lane (32 bits, before the one rounding)
template <int TYPE>
__device__ __forceinline__ void add8(uint32_t (&v)[8], const void* y, int64_t ldy, int live, bool have) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < live && have) {
            float old;
            if (TYPE == FRX_F32)
                old = static_cast<const float*>(y)[i * ldy];
            else if (TYPE == FRX_BF16)
                old = __bfloat162float(static_cast<const __nv_bfloat16*>(y)[i * ldy]);
            else
                old = __half2float(static_cast<const __half*>(y)[i * ldy]);
            v[i] = __float_as_uint(__uint_as_float(v[i]) + old);
        }
}

// The tiles of a block. First two forms: those of GroupWalk (expert, lanes tile, block of its rows). Third form: every matrix has as many.
template <int FORM>
struct Tiles {
    GroupWalk g;
    int tile, per, across;   // third form: the tile, tiles of a matrix, of them along the columns
    int e, lane0, col0, live, width;   // expert; first of the lanes side; first column, columns, their number rounded up to 16
    int row0, steps, last;   // first row of the expert; stages; depth of the last one
    __device__ __forceinline__ void begin(const Product& p, const GroupTables& tab, int experts) {
        if (FORM == kGradW) {
            g.tab = tab;
            across = (p.cols + kTileN - 1) / kTileN;
            per = across * ((p.lanes + kTileM - 1) / kTileM);
            tile = int(blockIdx.x) - int(gridDim.x);
        } else {
            g.begin(tab, experts);
            steps = (p.depth + kDepth - 1) / kDepth;
            last = p.depth - (steps - 1) * kDepth;
        }
    }
    __device__ __forceinline__ bool next(const Product& p) {
        if (FORM == kGradW) {
            tile += int(gridDim.x);
            e = tile / per;
            if (e >= p.E) return false;
            const int local = tile - e * per, m = local / across;
            lane0 = m * kTileM;
            col0 = (local - m * across) * kTileN;
            live = min(kTileN, p.cols - col0);
            width = (live + 15) & ~15;
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
        width = g.width;
        return true;
    }
};

template <int FORM, int TYPE>
__global__ void __launch_bounds__(kThreads, 1) k_moe_product(const Product p, const __grid_constant__ CUtensorMap lanes_map, const __grid_constant__ CUtensorMap cols_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t s0 = smem_u32(smem), stages0 = s0 + kHead, bars = s0, abort = s0 + kAbort, n_stages = uint32_t(p.stages), stage_bytes = uint32_t(p.stage_bytes);
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
            mbar_init(b + kBarFull + i, 1);
            mbar_init(b + kBarFree + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b + kBarDFull + i, 1);
            mbar_init(b + kBarDFree + i, kWarpsEpi);
        }
        asm volatile("prefetch.tensormap [%0];" ::"l"(&lanes_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&cols_map) : "memory");
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kWarpMma) tmem_alloc(tmem_slot, 512);
    pdl_wait();
    pdl_trigger();
    const long long tiles = group_tables<kThreads>(tab, p.offsets, p.E, p.S, p.width, (p.lanes + kTileM - 1) / kTileM, reinterpret_cast<long long*>(smem + kSums));
    const int experts = FORM != kGradW && tiles > p.most ? 0 : p.E;   // offsets that do not ascend: nothing is computed
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    Tiles<FORM> t;
    t.begin(p, tab, experts);

    // "free" barriers are waited on with the parity of the phase before the one about to be used, which a fresh barrier reports as complete
    if (warp == kWarpLoad) {
        uint32_t st = 0, phase = 1;
        bool ok = true;
        while (ok && t.next(p)) {
            const int box = FORM == kGradW ? 64 : p.box, boxes = (t.width + box - 1) / box, box_bytes = box * 128;
            const int halves = FORM == kForward || p.lanes - t.lane0 <= 64 ? 1 : 2;   // chunks of the lanes side
            const uint32_t bytes = (FORM == kForward ? kStageA : uint32_t(halves * kChunk)) + uint32_t(boxes * box_bytes);
            for (int s = 0; s < t.steps; ++s) {
                if (!(ok = warp_wait(bars + (kBarFree + st) * 8, phase, abort, p.wait_ns))) break;
                const uint32_t full = bars + (kBarFull + st) * 8, a = stages0 + st * stage_bytes, b = a + kStageA;
                if (lane == 0) {
                    mbar_expect_tx(full, bytes);
                    if (FORM == kForward) {
                        tma_3d(a, &lanes_map, s * kDepth, t.lane0, t.e, full);
                    } else {
                        for (int i = 0; i < halves; ++i) {
                            if (FORM == kGradX)
                                tma_3d(a + i * kChunk, &lanes_map, t.lane0 + 64 * i, s * kDepth, t.e, full);
                            else
                                tma_2d(a + i * kChunk, &lanes_map, t.lane0 + 64 * i, t.row0 + s * kDepth, full);
                        }
                    }
                    for (int i = 0; i < boxes; ++i) {
                        if (FORM == kGradW)
                            tma_2d(b + i * kChunk, &cols_map, t.col0 + 64 * i, t.row0 + s * kDepth, full);
                        else
                            tma_2d(b + i * box_bytes, &cols_map, s * kDepth, t.col0 + i * box, full);
                    }
                }
                __syncwarp();
                if (++st == n_stages) st = 0, phase ^= 1u;
            }
        }
    } else if (warp == kWarpMma) {
        uint32_t st = 0, phase = 0, set = 0, dphase = 1;
        bool ok = true;
        while (ok && t.next(p)) {
            const uint32_t idesc = p.idesc | uint32_t(t.width >> 3) << 17;
            if (!(ok = warp_wait(bars + (kBarDFree + set) * 8, dphase, abort, p.wait_ns))) break;
            tc_fence_after_sync();   // behind the epilogue's loads of these accumulators
            const uint32_t acc = tmem + set * kTileN;
            for (int s = 0; s < t.steps; ++s) {
                if (!(ok = warp_wait(bars + (kBarFull + st) * 8, phase, abort, p.wait_ns))) break;
                const uint32_t a = stages0 + st * stage_bytes, b = a + kStageA;
                const int depth = s + 1 < t.steps ? kDepth : t.last;
                if (FORM == kGradW && depth % 16) {
                    // the rows behind the expert's last one, up to the next 16: zeros (a row of depth is 128 bytes in every chunk, whatever the swizzle)
                    const int extra = 16 - depth % 16, chunks = 2 + (t.width + 63) / 64;
                    for (int i = lane; i < chunks * extra * 8; i += 32) {
                        const int r = i >> 3, c = r / extra;
                        const uint32_t at = (c < 2 ? a + c * kChunk : b + (c - 2) * kChunk) + uint32_t(depth + r - c * extra) * 128 + (i & 7) * 16;
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                    }
                    fence_async_smem();   // generic-proxy writes: visible to the tensor core
                    __syncwarp();
                }
                if (elect_one()) {
                    const uint64_t da = FORM == kForward ? umma_desc_sw128(a) : umma_desc_mn(a), db = FORM == kGradW ? umma_desc_mn(b) : umma_desc_sw128(b);
                    constexpr uint64_t kStepK = 32 >> 4, kStepMn = 16 * 128 >> 4;   // 16 of depth
#pragma unroll
                    for (int k = 0; k < kDepth / 16; ++k) {
                        if (k * 16 >= depth) break;
                        umma_f16(acc, da + k * (FORM == kForward ? kStepK : kStepMn), db + k * (FORM == kGradW ? kStepMn : kStepK), idesc, s + k > 0);
                    }
                    umma_commit(bars + (kBarFree + st) * 8);
                }
                __syncwarp();
                if (++st == n_stages) st = 0, phase ^= 1u;
            }
            if (ok && elect_one()) umma_commit(bars + (kBarDFull + set) * 8);
            __syncwarp();
            set ^= 1u;
            if (set == 0) dphase ^= 1u;
        }
    } else {
        // ---------------- epilogue: a warp has a quarter of the lanes and every second 16 columns
        const int quarter = warp & 3, part = warp >> 2, m = quarter * 32 + lane;
        constexpr int size = TYPE == FRX_F32 ? 4 : 2;
        uint32_t set = 0, phase = 0;
        const bool pairs = TYPE != FRX_F32 && p.lanes % 2 == 0 && p.ldy % 2 == 0 && (FORM != kGradW || p.ldye % 2 == 0) && reinterpret_cast<uintptr_t>(p.y) % 4 == 0;
        bool lost = false;   // a wait ran out: NaN, not a wrong number, and no more waits
        while (t.next(p)) {
            lost = lost || !warp_wait(bars + (kBarDFull + set) * 8, phase, abort, p.wait_ns);
            tc_fence_after_sync();
            const uint32_t acc = tmem + (uint32_t(quarter * 32) << 16) + set * kTileN;
            const bool have = t.lane0 + m < p.lanes, empty = FORM == kGradW && t.steps == 0;
            uint8_t* y = static_cast<uint8_t*>(p.y) + ((FORM == kGradW ? t.e * p.ldye : 0) + t.col0 * p.ldy + t.lane0 + m) * size;
            for (int c = part * 16; c < t.width && !(empty && p.add); c += 32) {
                uint32_t v[2][8];
                if (lost || empty) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[0][i] = v[1][i] = lost ? 0x7fffffffu : 0u;
                } else {
                    tmem_ld16(acc + c, v);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint8_t* at = y + (c + 8 * h) * p.ldy * size;
                    if (FORM == kGradW && p.add) add8<TYPE>(v[h], at, p.ldy, t.live - c - 8 * h, have);
                    store8<TYPE>(v[h], at, p.ldy, t.live - c - 8 * h, have, pairs);
                }
            }
            if (!lost) {
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
    }
    if (warp == kWarpMma) tmem_free(tmem, 512);
}

template <int FORM, int TYPE>
int launch_typed(Product& p, const CUtensorMap& lanes_map, const CUtensorMap& cols_map, cudaStream_t stream) {
    const size_t tables = size_t(p.E) * 16;
    int rc = allow_smem<k_moe_product<FORM, TYPE>>();
    if (rc != FRX_OK) return rc;
    const int64_t lane_tiles = (p.lanes + kTileM - 1) / kTileM;
    const int64_t most = FORM == kGradW ? lane_tiles * ((p.cols + kTileN - 1) / kTileN) * p.E : lane_tiles * (int64_t(p.S) / p.width + std::min(p.E, p.S));
    if (most > 0x7fff0000 || p.S / 16 >= (1 << 24)) return fail(FRX_ERR_SHAPE, "product by expert: %lld tiles of %d rows", (long long)most, p.S);
    p.most = int(most);
    p.stages = int(std::min<size_t>(kMaxStages, (kSmemMost - kHead - tables) / size_t(p.stage_bytes)));
    static_assert((kSmemMost - kHead - 4096 * 16) / (kStageA + kTileN * kDepth * 2) >= 3, "stages beside the tables of 4096 experts");
    p.wait_ns = wait_limit_ns();
    const unsigned grid = unsigned(std::min<int64_t>(sm_count(), std::max<int64_t>(1, most)));
    FRX_LAUNCH(kKGateUp, stream, launch_pdl(k_moe_product<FORM, TYPE>, dim3(grid), dim3(kThreads), kHead + size_t(p.stages) * p.stage_bytes + tables, stream, p, lanes_map, cols_map));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}
template <int FORM>
int launch(Product& p, int type, const CUtensorMap& lanes_map, const CUtensorMap& cols_map, cudaStream_t stream) {
    switch (type) {
        case FRX_F32: return launch_typed<FORM, FRX_F32>(p, lanes_map, cols_map, stream);
        case FRX_BF16: return launch_typed<FORM, FRX_BF16>(p, lanes_map, cols_map, stream);
        default: return launch_typed<FORM, FRX_F16>(p, lanes_map, cols_map, stream);
    }
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
    p.width = 16;
    while (p.width < kTileN && p.width < 2 * average) p.width *= 2;
    p.box = p.width >= 128 ? 32 : 16;
    p.stage_bytes = kStageA + p.width * kDepth * 2;
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
    p.idesc = f16_idesc(dtype, false, false);
    CUtensorMap wm, xm;
    if ((rc = matrices_map(wm, w, ldw, lde, dtype, E, rows, n, kTileM)) != FRX_OK || (rc = rows_map(xm, x, ldx, dtype, S, n, p.box)) != FRX_OK) return rc;
    return launch<kForward>(p, out_dtype, wm, xm, stream);
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
    p.idesc = f16_idesc(dtype, true, false);
    CUtensorMap wm, gm;
    if ((rc = matrices_map(wm, w, ldw, lde, dtype, E, rows, n, kDepth)) != FRX_OK || (rc = rows_map(gm, gy, ldgy, dtype, S, rows, p.box)) != FRX_OK) return rc;
    return launch<kGradX>(p, out_dtype, wm, gm, stream);
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
    p.stage_bytes = kStageA + std::min((rows + 63) / 64, kTileN / 64) * kChunk;
    p.idesc = f16_idesc(dtype, true, true);
    CUtensorMap xm, gm;
    if ((rc = rows_map(xm, x, ldx, dtype, S, n, kDepth)) != FRX_OK || (rc = rows_map(gm, gy, ldgy, dtype, S, rows, kDepth)) != FRX_OK) return rc;
    return launch<kGradW>(p, out_dtype, xm, gm, stream);
}

}  // extern "C"
