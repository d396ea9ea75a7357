// Tokens sorted by expert and back: the plan (which row every (token, expert) slot gets), the rows carried there and
// the weighted sums carried back, with the gradients of both and of the routing weights.
//
// With S = T * K slots, slot s = t * K + k, and rows numbered expert after expert (slots of one expert in slot order):
//   xs[row_of[t][k]] = x[t]                                  gx[t]  = sum_k gxs[row_of[t][k]]
//   out[t] = sum_k w[t][k] * ys[row_of[t][k]]                gys[row_of[t][k]] = w[t][k] * gout[t]
//                                                            gw[t][k] = <gout[t], ys[row_of[t][k]]>
// Every one is a pass over the S rows that must be read or written, so bandwidth is the bound. They all walk tokens, not
// rows: a token's row is then read (or written) once and its K sorted rows are whole contiguous rows, so nothing is read
// twice and sums over k need no atomics: they are made in k order, in 32 bits, and round once. 163,840 bf16 rows of 2,048 (16,384 tokens): out 119 us (6.2 TB/s),
// back 112 (6.6), gradients of back 231 (6.1). The sorted rows of the way back are read for the last time there (load_last): 4,096 tokens 27.6 us instead of 30.9, gradients
// 61.7 instead of 65.4, since what is written next finds room in the L2.
#include <algorithm>
#include <initializer_list>
#include <mutex>
#include <type_traits>

#include "frx_rows.cuh"
#include "frx_sort.cuh"

namespace frx {
namespace {

#include "frx_scan.cuh"

// Every kernel here may start while the one in front still writes what it reads. So nothing that is read is declared as data that no one writes (const
// __restrict__, __ldg): such loads could be moved across pdl_wait(). With and without the declaration: 16,384 tokens of
// ten rows there and back 246.8 and 246.8 us, the gradients of 4,096 tokens 84.0 and 83.8.

// the expert of slot s, or -1 where it has no row; an id beyond the experts is reported
__device__ __forceinline__ int slot_expert(const int32_t* ids, int s, int S, int E, int* status) {
    if (s >= S) return -1;
    const int e = ids[s];
    if (e >= E) {
        if (status) {
            status[0] = kDevBadExpertId;
            status[2] = s;
        }
        return -1;
    }
    return e < 0 ? -1 : e;
}

// counts of every chunk's experts: cnt [chunks][E]
__global__ void __launch_bounds__(kChunkSlots) k_sort_count(const int32_t* ids, int S, int E, int* __restrict__ cnt, int* status) {
    extern __shared__ __align__(16) int hist[];
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0 && threadIdx.x == 0 && status[3] != kCookie) {   // first use of this workspace
        status[0] = kDevOk;
        status[2] = 0;
        status[3] = kCookie;
    }
    for (int e = threadIdx.x; e < E; e += kChunkSlots) hist[e] = 0;
    __syncthreads();
    const int s = blockIdx.x * kChunkSlots + threadIdx.x, e = s < S ? ids[s] : -1;
    if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < E; i += kChunkSlots) cnt[size_t(blockIdx.x) * E + i] = hist[i];
}

// cnt[c][e] to the slots of expert e in the chunks in front of c, and cnt[chunks][e] to all of them; a thread per expert
__global__ void __launch_bounds__(32) k_sort_scan(int* cnt, int chunks, int E) {
    pdl_wait();
    pdl_trigger();
    const int e = blockIdx.x * 32 + threadIdx.x;
    if (e >= E) return;
    int run = 0;
    constexpr int kBatch = 32;   // loads in flight: the running sum is a chain, the loads need not be
    for (int c0 = 0; c0 < chunks; c0 += kBatch) {
        int v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) v[i] = c0 + i < chunks ? cnt[size_t(c0 + i) * E + e] : 0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (c0 + i < chunks) cnt[size_t(c0 + i) * E + e] = run;
            run += v[i];
        }
    }
    cnt[size_t(chunks) * E + e] = run;
}

// A chunk's slots to their rows. A slot's lane finds the equal experts of its warp by one ballot for each bit of the expert's number, adds what the warps in front
// have of it, and the chunks in front. (Comparing with every slot of a part of 128 instead took 7.3 us for 1,020 slots, this 4.2.) Up to kOwnScan chunks every block
// adds up the chunk counts itself (`scanned` false: one launch less); with a single chunk there are none and the warps' counts are all.
constexpr int kSortWarps = kChunkSlots / 32;
__host__ __device__ inline int warp_counts(int E) { return (E + 15) & ~15; }   // bytes of a warp's counts
__global__ void __launch_bounds__(kChunkSlots) k_sort_place(const int32_t* ids, int S, int E, const int* cnt, int chunks, bool scanned,
                                                           int32_t* offsets, int32_t* __restrict__ slot_of, int32_t* __restrict__ row_of,
                                                           int* status) {
    extern __shared__ __align__(16) uint8_t sort_smem[];   // [warps][E] slots of the expert in the warp; [E] where an expert's rows of this chunk begin
    __shared__ int tot[32];
    uint8_t* warp_cnt = sort_smem;
    const int stride = warp_counts(E);
    int* begin = reinterpret_cast<int*>(sort_smem + kSortWarps * stride);
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, c = blockIdx.x, s = c * kChunkSlots + tid, warp = tid >> 5, lane = tid & 31;
    const int warps = min(kSortWarps, (min(S - c * kChunkSlots, kChunkSlots) + 31) >> 5);   // with slots
    if (chunks == 1 && tid == 0 && status && status[3] != kCookie) {
        status[0] = kDevOk;
        status[2] = 0;
        status[3] = kCookie;
    }
    for (int i = tid; i < warps * stride / 16; i += kChunkSlots) reinterpret_cast<uint4*>(warp_cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    const int e = slot_expert(ids, s, S, E, status), key = e < 0 ? E : e;
    int rank = 0;
    if (warp < warps) {
        unsigned same = 0xffffffffu;
        for (int b = 32 - __clz(E); b-- > 0;) {   // (E, the key of no expert, is the largest)
            const unsigned bit = (unsigned(key) >> b) & 1u, ones = __ballot_sync(0xffffffffu, bit != 0u);
            same &= bit ? ones : ~ones;
        }
        rank = __popc(same & ((1u << lane) - 1u));
        if (e >= 0 && rank == 0) warp_cnt[warp * stride + e] = uint8_t(__popc(same));
    }
    __syncthreads();
    // where every expert's rows begin, and this chunk's within them; a thread takes E / 1024 experts in a row
    const int per = (E + kChunkSlots - 1) / kChunkSlots, e0 = min(E, tid * per), e1 = min(E, e0 + per);
    int sum = 0;
    for (int i = e0; i < e1; ++i) {
        int total = 0, front = 0;
        if (chunks == 1) {
#pragma unroll 8
            for (int w = 0; w < warps; ++w) total += warp_cnt[w * stride + i];
        } else if (scanned) {
            front = cnt[size_t(c) * E + i];
            total = cnt[size_t(chunks) * E + i];
        } else {
#pragma unroll 16
            for (int j = 0; j < chunks; ++j) {
                const int v = cnt[size_t(j) * E + i];
                total += v;
                front += j < c ? v : 0;
            }
        }
        begin[i] = sum + front;
        if (c == 0) offsets[i] = sum;   // completed below
        sum += total;
    }
    int rows = 0;
    const int at = block_scan(sum, tot, rows);
    for (int i = e0; i < e1; ++i) {
        begin[i] += at;
        if (c == 0) offsets[i] += at;
    }
    if (c == 0 && tid == 0) offsets[E] = rows;
    __syncthreads();
    if (s >= S) return;
    if (slot_of && s >= rows) slot_of[s] = -1;   // rows behind the last expert's belong to no slot
    int row = -1;
    if (e >= 0) {
        row = begin[e] + rank;
#pragma unroll 8
        for (int w = 0; w < warp; ++w) row += warp_cnt[w * stride + e];
        if (slot_of) slot_of[row] = s;
    }
    row_of[s] = row;
}
constexpr int kOwnScan = 64;
constexpr int kMaxExperts = 4096;
inline size_t sort_place_smem(int E) { return size_t(kSortWarps) * warp_counts(E) + size_t(E) * 4; }

// ---- rows out and back. A block per token; the token's K rows are looked up once, in shared memory.
constexpr int kMaxK = 32;

// The rows that the token has in a buffer of `rows`, in k order, by the first warp: row[i] of the slot slot[i], and how many; a row that the
// buffer does not have is none. (Lists without gaps: what loops over them loads without asking, so that the loads are in flight together.)
struct TokenRows {
    int row[kMaxK], slot[kMaxK], count;
};
__device__ __forceinline__ void load_rows(TokenRows& list, const int32_t* row_of, size_t t, int K, int64_t rows) {
    if (threadIdx.x < 32) {
        const int r = int(threadIdx.x) < K ? __ldcg(row_of + t * K + threadIdx.x) : -1;
        const bool have = r >= 0 && r < rows;
        const unsigned all = __ballot_sync(0xffffffffu, have);
        const int at = __popc(all & ((1u << threadIdx.x) - 1u));
        if (have) {
            list.row[at] = r;
            list.slot[at] = threadIdx.x;
        }
        if (threadIdx.x == 0) list.count = __popc(all);
    }
    __syncthreads();
}

// xs[row_of[t][k]] = x[t]
template <class V>
__global__ void __launch_bounds__(256) k_rows_out(const V* x, int64_t ldx, const int32_t* row_of, int K, int nv, V* __restrict__ xs,
                                                  int64_t lds, int64_t rows) {
    __shared__ TokenRows list;
    pdl_wait();
    pdl_trigger();
    const size_t t = blockIdx.x;
    const int first = threadIdx.x;
    V v{};
    if (first < nv) v = x[t * ldx + first];
    load_rows(list, row_of, t, K, rows);
    for (int i = first; i < nv; i += blockDim.x) {
        if (i != first) v = x[t * ldx + i];
        for (int k = 0; k < list.count; ++k) xs[size_t(list.row[k]) * lds + i] = v;
    }
}

// out[t] = sum_k w * ys[row], FLIGHT rows in flight (all of them are loaded, asked or not: loads behind a condition waited for one another, 226 us instead of 127). early: the plan was complete before the kernel in front began, and is read before the wait for it.
template <class T, class O, int N, int FLIGHT>
__global__ void __launch_bounds__(256) k_rows_back(const T* ys, int64_t ldy, const float* wts, const int32_t* row_of, int K, int n,
                                                   O* __restrict__ out, int64_t ldo, int64_t rows, bool early) {
    __shared__ TokenRows list;
    if (!early) pdl_wait();
    const size_t t = blockIdx.x;
    load_rows(list, row_of, t, K, rows);
    if (early) pdl_wait();
    pdl_trigger();
    const int count = list.count;
    for (int i = (blockIdx.y * blockDim.x + threadIdx.x) * N; i < n; i += gridDim.y * blockDim.x * N) {
        float acc[N];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        for (int k0 = 0; k0 < count; k0 += FLIGHT) {
            Vec<T, N> v[FLIGHT];
            float w[FLIGHT];
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k) {   // (behind the last row the last again, with weight 0 and not added)
                const int at = min(k0 + k, count - 1);
                v[k] = load_last(reinterpret_cast<const Vec<T, N>*>(ys + size_t(list.row[at]) * ldy + i));
                w[k] = wts ? wts[t * K + list.slot[at]] : 1.0f;
            }
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k)
                if (k0 + k < count)
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] = fmaf(w[k], to_float(v[k].v[j]), acc[j]);
        }
        Vec<O, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = from_float<O>(acc[j]);
        *reinterpret_cast<Vec<O, N>*>(out + t * ldo + i) = o;
    }
}

// gys[row] = w * gout[t], gw[t][k] = <gout[t], ys[row]>: a row of ys is read once and its gradient written in the same pass
template <class T, int N, int FLIGHT>
__global__ void __launch_bounds__(256) k_rows_back_grad(const T* gout, int64_t ldg, const T* ys, int64_t ldy, const float* wts,
                                                        const int32_t* row_of, int K, int n, T* __restrict__ gys, int64_t ldgy, float* __restrict__ gw,
                                                        int64_t rows) {
    __shared__ TokenRows list;
    __shared__ float part[8][kMaxK];
    pdl_wait();
    pdl_trigger();
    const size_t t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    load_rows(list, row_of, t, K, rows);
    const int count = list.count;
    for (int k0 = 0; k0 < count; k0 += FLIGHT) {
        float dot[FLIGHT], w[FLIGHT];
        size_t at[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {
            const int l = min(k0 + k, count - 1);
            dot[k] = 0.0f;
            at[k] = size_t(list.row[l]);
            w[k] = wts[t * K + list.slot[l]];
        }
        for (int i = threadIdx.x * N; i < n; i += blockDim.x * N) {
            Vec<T, N> v[FLIGHT];
            const Vec<T, N> g = *reinterpret_cast<const Vec<T, N>*>(gout + t * ldg + i);
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k) v[k] = load_last(reinterpret_cast<const Vec<T, N>*>(ys + at[k] * ldy + i));
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k)
                if (k0 + k < count) {
                    Vec<T, N> o;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float gj = to_float(g.v[j]);
                        dot[k] = fmaf(gj, to_float(v[k].v[j]), dot[k]);
                        o.v[j] = from_float<T>(w[k] * gj);
                    }
                    *reinterpret_cast<Vec<T, N>*>(gys + at[k] * ldgy + i) = o;
                }
        }
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {
#pragma unroll
            for (int d = 16; d; d >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], d);
            if (lane == 0 && k0 + k < count) part[warp][list.slot[k0 + k]] = dot[k];
        }
    }
    __syncthreads();
    if (int(threadIdx.x) < K) {
        float sum = 0.0f;
        bool have = false;
        for (int i = 0; i < count; ++i) have = have || list.slot[i] == int(threadIdx.x);
        if (have)
            for (int p = 0; p < warps; ++p) sum += part[p][threadIdx.x];
        gw[t * K + threadIdx.x] = sum;   // 0 for a slot without a row
    }
}

// The weights of a token are the softmax over its chosen logits (frx_route_topk: p / sum of the chosen p, whose floor of 2^-14
// no sum of the largest of at most 1024 probabilities reaches), so
//   glogits[ids[k]] = w[k] * (gw[k] - sum_j w[j] gw[j]), and 0 for every other expert.
// A warp per token; the row of E zeros that has to be written is the work.
template <int V>
__global__ void __launch_bounds__(256) k_route_grad(const float* gw, const float* wts, const int32_t* ids, int T, int E, int K,
                                                    float* gl) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x * 8 + int(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= T) return;
    const size_t at = size_t(t) * K + lane;
    const int id = lane < K ? ids[at] : -1;
    const float w = lane < K ? wts[at] : 0.0f, g = lane < K ? gw[at] : 0.0f;
    float inner = w * g;
#pragma unroll
    for (int d = 16; d; d >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, d);
    const float mine = w * (g - inner);
    float* row = gl + size_t(t) * E;
    for (int e = lane * V; e < E; e += 32 * V)
        *reinterpret_cast<Vec<float, V>*>(row + e) = Vec<float, V>{};
    // an expert named twice gets the sum of its slots' terms, in slot order, from the first of them
    float sum = 0.0f;
    bool first = true;
    for (int k = 0; k < K; ++k) {
        const int other = __shfl_sync(0xffffffffu, id, k);
        const float term = __shfl_sync(0xffffffffu, mine, k);
        if (other == id) {
            sum += term;
            first = first && k >= lane;
        }
    }
    __syncwarp();   // the zeros are there
    if (lane < K && first && id >= 0 && id < E) row[id] = sum;
}

int row_args(const char* who, int T, int K, int n, int dtype) {
    if (T < 0 || n < 0) return fail(FRX_ERR_ARG, "%s: T %d, n %d", who, T, n);
    if (!dtype_size(dtype)) return fail(FRX_ERR_ARG, "%s: element type %d", who, dtype);
    if (K < 1 || K > kMaxK) return fail(FRX_ERR_SHAPE, "%s: K %d", who, K);
    if ((long long)T * K > 0x7fffffffLL) return fail(FRX_ERR_SHAPE, "%s: T * K %lld", who, (long long)T * K);
    return FRX_OK;
}
int row_buffer(const char* who, const char* what, const void* p, int64_t ld, int n, int dtype) {
    if (!p) return fail(FRX_ERR_ARG, "%s: null pointer (%s)", who, what);
    if (ld < n) return fail(FRX_ERR_ARG, "%s: rows of %s are %lld elements apart and %d long", who, what, (long long)ld, n);
    if (!rows_aligned(p, dtype_size(dtype))) return fail(FRX_ERR_ARG, "%s: misaligned pointer (%s)", who, what);
    return FRX_OK;
}
#define FRX_TRY(expr)                    \
    do {                                 \
        const int rc_ = (expr);          \
        if (rc_ != FRX_OK) return rc_;   \
    } while (0)

// How many rows a token's loop has in flight: what leaves the fewest loads behind the last of K rows, the larger of two that leave as many. (16,384 tokens of ten
// bf16 rows of 2,048: back with 8 in flight 127 us, with 10 118, with 5 111 = 6.65 TB/s.)
inline int rows_in_flight(int K, std::initializer_list<int> choices) {
    int best = 0, cost = 0;
    for (int f : choices) {   // ascending
        const int c = (K + f - 1) / f * f;
        if (!best || c <= cost) best = f, cost = c;
    }
    return best;
}

// Blocks that share a token's row: one, or with few tokens one for each 256 pieces of it (a token's loads then wait for one another once less).
inline unsigned row_parts(int T, int pieces) { return T <= 128 ? unsigned(std::max(1, std::min(8, (pieces + 255) / 256))) : 1u; }
inline unsigned row_threads(int pieces) { return unsigned(std::min(256, std::max(32, (pieces + 31) / 32 * 32))); }

}  // namespace

size_t sort_scratch_bytes(long long S, int E) { return S <= kChunkSlots ? 0 : size_t((S + kChunkSlots - 1) / kChunkSlots + 1) * size_t(E) * 4; }

int sort_slots(const int32_t* ids, int S, int E, int32_t* offsets, int32_t* slot_of, int32_t* row_of, int* status, int* scratch, cudaStream_t stream) {
    const int chunks = std::max(1, int((int64_t(S) + kChunkSlots - 1) / kChunkSlots));
    const bool scan = chunks > kOwnScan;
    if (sort_place_smem(E) > 48 * 1024) {
        // The limit belongs to the kernel, not to a call: once per device, what the most experts need. (Calls of other threads may lie between this and the launch.)
        static std::once_flag once[64];
        int dev = 0;
        FRX_CUDA(cudaGetDevice(&dev));
        cudaError_t rc = cudaSuccess;
        auto allow = [&] { rc = cudaFuncSetAttribute(k_sort_place, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sort_place_smem(kMaxExperts))); };
        dev >= 0 && dev < 64 ? std::call_once(once[dev], allow) : allow();
        FRX_CUDA(rc);
    }
    if (chunks > 1)
        FRX_LAUNCH(kKGroup, stream, launch_pdl(k_sort_count, dim3(chunks), dim3(kChunkSlots), size_t(E) * 4, stream, ids, S, E, scratch, status));
    if (scan) FRX_LAUNCH(kKGroup, stream, launch_pdl(k_sort_scan, dim3((E + 31) / 32), dim3(32), 0, stream, scratch, chunks, E));
    FRX_LAUNCH(kKGroup, stream, launch_pdl(k_sort_place, dim3(chunks), dim3(kChunkSlots), sort_place_smem(E), stream, ids, S, E, (const int*)scratch, chunks, scan, offsets,
                                           slot_of, row_of, status));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int rows_back(const void* ys, int64_t ldy, int in_dtype, const float* wts, const int32_t* row_of, int64_t rows, int T, int K, int n, void* out, int64_t ldo,
              int out_dtype, bool early, cudaStream_t stream) {
    const bool vec = rows_vec16(ys, ldy, n, dtype_size(in_dtype)) && rows_vec16(out, ldo, n, dtype_size(out_dtype)) && (in_dtype == out_dtype || n % 8 == 0);
    auto launch = [&](auto in, auto o, auto width) {
        using T_ = decltype(in);
        using O_ = decltype(o);
        constexpr int N = decltype(width)::value;
        auto with_flight = [&](auto flight) {
            FRX_LAUNCH(kKCombine, stream, launch_pdl(k_rows_back<T_, O_, N, decltype(flight)::value>, dim3(T, row_parts(T, (n + N - 1) / N)), dim3(row_threads((n + N - 1) / N)), 0, stream,
                                                     static_cast<const T_*>(ys), ldy, wts, row_of, K, n, static_cast<O_*>(out), ldo, rows, early));
        };
        switch (rows_in_flight(K, {2, 4, 5, 8})) {
            case 2: with_flight(std::integral_constant<int, 2>{}); break;
            case 4: with_flight(std::integral_constant<int, 4>{}); break;
            case 5: with_flight(std::integral_constant<int, 5>{}); break;
            default: with_flight(std::integral_constant<int, 8>{}); break;
        }
    };
    if (in_dtype == out_dtype)
        with_rows(in_dtype, vec, [&](auto v, auto width) { launch(v, v, width); });
    else if (in_dtype == FRX_F32 && out_dtype == FRX_F16)   // (the expert layer's: rows kept in 32 bits)
        vec ? launch(float{}, __half{}, std::integral_constant<int, 4>{}) : launch(float{}, __half{}, std::integral_constant<int, 1>{});
    else if (in_dtype == FRX_F32 && out_dtype == FRX_BF16)
        vec ? launch(float{}, __nv_bfloat16{}, std::integral_constant<int, 4>{}) : launch(float{}, __nv_bfloat16{}, std::integral_constant<int, 1>{});
    else
        return fail(FRX_ERR_ARG, "rows of type %d to rows of type %d", in_dtype, out_dtype);
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

}  // namespace frx

using namespace frx;

extern "C" {

size_t frx_moe_sort_workspace_bytes(int T, int K, int E) {
    if (T < 0 || K < 1 || K > kMaxK || E < 1 || E > kMaxExperts || (long long)T * K > 0x7fffffffLL) return 0;
    return kAlign + align_up(sort_scratch_bytes((long long)T * K, E));
}

int frx_moe_sort(frx_stream_t stream, const int32_t* ids, int T, int K, int E, int32_t* offsets, int32_t* slot_of, int32_t* row_of, void* ws, size_t ws_bytes) {
    const char* who = "frx_moe_sort";
    if (T < 0) return fail(FRX_ERR_ARG, "%s: T %d", who, T);
    const size_t need = frx_moe_sort_workspace_bytes(T, K, E);
    if (!need) return fail(FRX_ERR_SHAPE, "%s: unsupported shape T %d, K %d, E %d", who, T, K, E);
    if (!offsets || (!ws && (long long)T * K > kChunkSlots) || (T > 0 && (!ids || !slot_of || !row_of))) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (uintptr_t(ws) % 16) return fail(FRX_ERR_ARG, "%s: misaligned workspace", who);
    if (ws && ws_bytes < need) return fail(FRX_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, need);
    return sort_slots(ids, T * K, E, offsets, slot_of, row_of, static_cast<int*>(ws), ws ? reinterpret_cast<int*>(static_cast<uint8_t*>(ws) + kAlign) : nullptr, stream);
}

int frx_moe_sort_rows(frx_stream_t stream, const void* x, int64_t ldx, int dtype, const int32_t* row_of, int T, int K, int n, void* xs, int64_t ldxs, int64_t rows) {
    const char* who = "frx_moe_sort_rows";
    FRX_TRY(row_args(who, T, K, n, dtype));
    if (T == 0 || n == 0 || rows <= 0) return FRX_OK;
    if (!row_of) return fail(FRX_ERR_ARG, "%s: null pointer (row_of)", who);
    FRX_TRY(row_buffer(who, "x", x, ldx, n, dtype));
    FRX_TRY(row_buffer(who, "xs", xs, ldxs, n, dtype));
    const int size = dtype_size(dtype);
    auto launch = [&](auto v) {
        using V = decltype(v);
        const int per = int(sizeof(V)) / size;
        FRX_LAUNCH(kKGroup, stream, launch_pdl(k_rows_out<V>, dim3(T), dim3(row_threads(n / per)), 0, stream, static_cast<const V*>(x), ldx / per, row_of, K, n / per,
                                               static_cast<V*>(xs), ldxs / per, rows));
    };
    if (rows_vec16(x, ldx, n, size) && rows_vec16(xs, ldxs, n, size))
        launch(uint4{});
    else if (size == 4)
        launch(uint32_t{});
    else
        launch(uint16_t{});
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_moe_sort_rows_backward(frx_stream_t stream, const void* gxs, int64_t ldgxs, int64_t rows, int dtype, const int32_t* row_of, int T, int K, int n, void* gx,
                               int64_t ldgx) {
    const char* who = "frx_moe_sort_rows_backward";
    FRX_TRY(row_args(who, T, K, n, dtype));
    if (T == 0 || n == 0) return FRX_OK;
    if (!row_of) return fail(FRX_ERR_ARG, "%s: null pointer (row_of)", who);
    if (rows > 0) FRX_TRY(row_buffer(who, "gxs", gxs, ldgxs, n, dtype));
    FRX_TRY(row_buffer(who, "gx", gx, ldgx, n, dtype));
    return rows_back(gxs, ldgxs, dtype, nullptr, row_of, rows, T, K, n, gx, ldgx, dtype, false, stream);
}

int frx_moe_unsort_rows(frx_stream_t stream, const void* ys, int64_t ldys, int64_t rows, int dtype, const float* wts, const int32_t* row_of, int T, int K, int n, void* out,
                        int64_t ldo) {
    const char* who = "frx_moe_unsort_rows";
    FRX_TRY(row_args(who, T, K, n, dtype));
    if (T == 0 || n == 0) return FRX_OK;
    if (!row_of || !wts) return fail(FRX_ERR_ARG, "%s: null pointer (row_of, wts)", who);
    if (rows > 0) FRX_TRY(row_buffer(who, "ys", ys, ldys, n, dtype));
    FRX_TRY(row_buffer(who, "out", out, ldo, n, dtype));
    return rows_back(ys, ldys, dtype, wts, row_of, rows, T, K, n, out, ldo, dtype, false, stream);
}

int frx_moe_unsort_rows_backward(frx_stream_t stream, const void* gout, int64_t ldg, const void* ys, int64_t ldys, int64_t rows, int dtype, const float* wts,
                                 const int32_t* row_of, int T, int K, int n, void* gys, int64_t ldgys, float* gwts) {
    const char* who = "frx_moe_unsort_rows_backward";
    FRX_TRY(row_args(who, T, K, n, dtype));
    if (T == 0) return FRX_OK;
    if (!row_of || !wts || !gwts) return fail(FRX_ERR_ARG, "%s: null pointer (row_of, wts, gwts)", who);
    if (n > 0) {
        FRX_TRY(row_buffer(who, "gout", gout, ldg, n, dtype));
        if (rows > 0) FRX_TRY(row_buffer(who, "ys", ys, ldys, n, dtype));
        if (rows > 0) FRX_TRY(row_buffer(who, "gys", gys, ldgys, n, dtype));
    }
    const int size = dtype_size(dtype);
    const bool vec = rows_vec16(gout, ldg, n, size) && rows_vec16(ys, ldys, n, size) && rows_vec16(gys, ldgys, n, size);
    with_rows(dtype, vec, [&](auto v, auto width) {
        using T_ = decltype(v);
        constexpr int N = decltype(width)::value;
        auto with_flight = [&](auto flight) {
            FRX_LAUNCH(kKCombine, stream, launch_pdl(k_rows_back_grad<T_, N, decltype(flight)::value>, dim3(T), dim3(row_threads((n + N - 1) / N)), 0, stream,
                                                     static_cast<const T_*>(gout), ldg, static_cast<const T_*>(ys), ldys, wts, row_of, K, n, static_cast<T_*>(gys), ldgys, gwts, rows));
        };
        switch (rows_in_flight(K, {2, 4, 5})) {
            case 2: with_flight(std::integral_constant<int, 2>{}); break;
            case 4: with_flight(std::integral_constant<int, 4>{}); break;
            default: with_flight(std::integral_constant<int, 5>{}); break;
        }
    });
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

int frx_route_topk_backward(frx_stream_t stream, const float* gwts, const float* wts, const int32_t* ids, int T, int E, int k, float* glogits) {
    const char* who = "frx_route_topk_backward";
    if (T < 0) return fail(FRX_ERR_ARG, "%s: T %d", who, T);
    if (E < 1 || E > 1024 || k < 1 || k > 32 || k > E) return fail(FRX_ERR_SHAPE, "%s: unsupported shape E %d, k %d", who, E, k);
    if (T == 0) return FRX_OK;
    if (!gwts || !wts || !ids || !glogits) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    const unsigned grid = unsigned((int64_t(T) + 7) / 8);
    if (E % 4 == 0 && uintptr_t(glogits) % 16 == 0)
        FRX_LAUNCH(kKRoute, stream, launch_pdl(k_route_grad<4>, dim3(grid), dim3(256), 0, stream, gwts, wts, ids, T, E, k, glogits));
    else
        FRX_LAUNCH(kKRoute, stream, launch_pdl(k_route_grad<1>, dim3(grid), dim3(256), 0, stream, gwts, wts, ids, T, E, k, glogits));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}

}  // extern "C"
