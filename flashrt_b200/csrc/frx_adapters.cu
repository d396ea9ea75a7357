// Low-rank adapters of many requests beside a shared projection (frx_adapter_add in frx.h).
#include <algorithm>
#include <type_traits>

#include "frx_groups.cuh"

namespace frx {
namespace {

// out[t] = y[t] + scale_j B_j (A_j x[t]), j the adapter of t's request. What has to move is x, y and out, and each adapter once; the products are few. So one kernel does
// both of them and v = A_j x never leaves the SM:
//   first   v[t][k] = sum_c x[t][c] A_j[k][c]     up to 128 tokens of a request are the lanes, the rank is N
//   second  d[m][t] = sum_k B_j[m][k] v[t][k]     128 rows of B_j are the lanes (contiguous in y), 64 tokens are N
// v is kept in 32 bits: it goes into the second product as three 16-bit pieces whose sum it is (for float16, whose exponents do not reach, as multiples of a power of two of its token).
// A tile (128 tokens of a request) is the work of a cluster of up to eight blocks, as many as fit the GPU at once: they share the first product's depth, add their
// parts up through one another's shared memory (in the order of the blocks), and share the second product's rows. y is read ahead of the sums it is added to.
constexpr int kTok = 128, kHalf = 64, kRows = 128, kDepth = 64;
constexpr int kStages = 3, kBufs = 2;
constexpr int kWarpsEpi = 8, kWarpLoad = 8, kWarpMma = 9, kThreads = 32 * 10;
constexpr int kBarFull = 0, kBarFree = kBarFull + kStages, kBarBFull = kBarFree + kStages, kBarBFree = kBarBFull + kBufs, kBarDFull = kBarBFree + kBufs, kBarDFree = kBarDFull + 2,
              kBarV = kBarDFree + 2, kBarVIn = kBarV + 1, kBarPart = kBarVIn + 1, kBars = kBarPart + 1;
constexpr int kAbort = 256, kSlot = 260, kFound = 264, kSums = 320, kTokScale = 512, kTokMax = kTokScale + 4 * kTok, kHead = 2048;
static_assert(kBars * 8 <= kAbort && kSums + 8 * kThreads / 32 <= kTokScale && kTokMax + 8 * kTok <= kHead, "the block's head");
constexpr int kPiece = kTok * 128;   // bytes of 64 of the rank of a piece of v, or of 128 rows of B_j
constexpr int kColD = 128, kCols = 256;   // tensor memory: v's sums, then two sets of 64 columns; two blocks an SM

struct Adapters {
    const int32_t* offsets;   // [R + 1]
    const int32_t* which;     // [R]
    const float* scale;       // [L] or null
    const void* y;
    void* out;
    int64_t ldy, ldo;
    unsigned long long wait_ns;
    int T, R, L, n, rows, rank, rank16;   // rank16: the rank rounded up to 16
    int box, stage_bytes, ring_bytes;     // rows of a load of x; bytes of a stage; of all of them (v's pieces come to the same place)
    uint32_t idesc;
};

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
__device__ __forceinline__ float4 ld_peer(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mbar_arrive_peer(uint32_t addr) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory"); }
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
__device__ __forceinline__ void tmem_ld8(uint32_t addr, float (&v)[8]) {
    uint32_t u[8];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
}

// f's 16-bit bits, and what they leave of it (nothing of an infinity or a NaN, which the first piece carries alone)
template <int XTYPE>
__device__ __forceinline__ uint32_t take_piece(float& f) {
    float back;
    uint16_t bits;
    if (XTYPE == FRX_BF16) {
        const __nv_bfloat16 h = __float2bfloat16_rn(f);
        bits = __bfloat16_as_ushort(h);
        back = __bfloat162float(h);
    } else {
        const __half h = __float2half_rn(f);
        bits = __half_as_ushort(h);
        back = __half2float(h);
    }
    f = fabsf(back) <= 3.4e38f ? f - back : 0.0f;   // (exact)
    return bits;
}

// y's values of 16 columns (tokens) for this lane's row, read ahead of the sums they are added to. 16-bit elements of even rows apart come two rows a lane: of an even column
// to even lanes, of an odd one to odd lanes, which is also how they are written.
template <int TYPE>
struct Ahead {
    uint32_t w[16];
    __device__ __forceinline__ void load(const void* y, int64_t ldy, int live, bool have, bool pairs) {
        if (TYPE == FRX_F32) {
            const float* p = static_cast<const float*>(y);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < live && have) w[i] = __float_as_uint(p[i * ldy]);
        } else if (pairs) {
            const int odd = threadIdx.x & 1;
            const uint16_t* p = static_cast<const uint16_t*>(y) + (odd ? ldy - 1 : 0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (2 * i + odd < live && have) w[i] = *reinterpret_cast<const uint32_t*>(p + 2 * i * ldy);
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(y);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < live && have) w[i] = p[i * ldy];
        }
    }
};
template <int TYPE>
__device__ __forceinline__ float wide(uint32_t bits) {   // of the low half
    if (TYPE == FRX_BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half(uint16_t(bits)));
}
template <int TYPE>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
    if (TYPE == FRX_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// eight columns of sums added to what was read ahead, rounded once and written
template <int TYPE>
__device__ __forceinline__ void add_and_store8(const float (&v)[8], const Ahead<TYPE>& a, int h, void* out, int64_t ldo, int live, bool have, bool pairs) {
    if (TYPE == FRX_F32) {
        float* p = static_cast<float*>(out);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live && have) p[i * ldo] = v[i] + __uint_as_float(a.w[8 * h + i]);
    } else if (pairs) {
        const bool odd = threadIdx.x & 1;
        uint16_t* p = static_cast<uint16_t*>(out) + (odd ? ldo - 1 : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v[2 * i] : v[2 * i + 1], 1);
            const float lo = odd ? got : v[2 * i], hi = odd ? v[2 * i + 1] : got;
            const uint32_t old = a.w[4 * h + i];
            if (2 * i + int(odd) < live && have) *reinterpret_cast<uint32_t*>(p + 2 * i * ldo) = narrow2<TYPE>(lo + wide<TYPE>(old), hi + wide<TYPE>(old >> 16));
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(out);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < live && have) p[i * ldo] = uint16_t(narrow2<TYPE>(v[i] + wide<TYPE>(a.w[8 * h + i]), 0.0f));
    }
}

template <int XTYPE, int TYPE>
__global__ void __launch_bounds__(kThreads, 2) k_adapter(const Adapters p, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap a_map,
                                                         const __grid_constant__ CUtensorMap b_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t s0 = smem_u32(smem), ring = s0 + kHead, bbuf = ring + uint32_t(p.ring_bytes), bars = s0, abort = s0 + kAbort;
    const int chunks = p.rank16 > 64 ? 2 : 1;   // of 64 of the rank
    const uint32_t bbuf_bytes = uint32_t(chunks) * kPiece, part = bbuf + kBufs * bbuf_bytes;
    const uint32_t rank = cluster_rank(), blocks = cluster_size();
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kAbort);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSlot);
    int* found = reinterpret_cast<int*>(smem + kFound);   // first token, tokens, adapter
    float* tok_scale = reinterpret_cast<float*>(smem + kTokScale);
    float* tok_max = reinterpret_cast<float*>(smem + kTokMax);
    if (threadIdx.x == 0) {
        uint64_t* b = reinterpret_cast<uint64_t*>(smem);
        for (int i = 0; i < kBars; ++i)
            mbar_init(b + i, i >= kBarDFree && i < kBarDFree + 2 ? kWarpsEpi : i == kBarVIn ? kWarpsEpi : i == kBarPart ? kWarpsEpi * blocks : 1);
        asm volatile("prefetch.tensormap [%0];" ::"l"(&x_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&b_map) : "memory");
        *abort_flag = 0;
        found[1] = 0;
        mbar_fence_init();
    }
    if (warp == kWarpMma) tmem_alloc(tmem_slot, kCols);
    pdl_wait();
    pdl_trigger();
    {   // the cluster's tile: a thread takes a few requests in a row
        const int tile = int(blockIdx.x / blocks), per = (p.R + kThreads - 1) / kThreads, r0 = min(p.R, int(threadIdx.x) * per), r1 = min(p.R, r0 + per);
        auto range = [&](int r, int& a) {   // (what the ranges say beyond the tokens that there are is left out)
            a = min(max(__ldcg(p.offsets + r), 0), p.T);
            return min(max(__ldcg(p.offsets + r + 1), a), p.T) - a;
        };
        long long sum = 0;
        int a;
        for (int r = r0; r < r1; ++r) sum += (range(r, a) + kTok - 1) / kTok;
        long long inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        long long* sums = reinterpret_cast<long long*>(smem + kSums);
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        long long before = inc - sum;
        for (int i = 0; i < warp; ++i) before += sums[i];
        if (tile >= before && tile < before + sum) {
            for (int r = r0; r < r1; ++r) {
                const int count = range(r, a), t = int(tile - before);
                before += (count + kTok - 1) / kTok;
                if (tile < before) {
                    const int j = __ldcg(p.which + r);
                    found[0] = a + t * kTok;
                    found[1] = min(kTok, count - t * kTok);
                    found[2] = j >= p.L ? -1 : j;
                    break;
                }
            }
        }
    }
    tc_fence_before_sync();
    __syncwarp();
    if (blocks > 1)
        cluster_sync_all();   // the barriers of all blocks are there
    else
        __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int t0 = found[0], live = found[1], j = found[2];
    const bool work = live > 0 && j >= 0;
    const int row_chunks = (p.rows + kRows - 1) / kRows, halves = (live + kHalf - 1) / kHalf;
    const int depths = (p.n + kDepth - 1) / kDepth, d0 = int(int64_t(depths) * rank / blocks), d1 = int(int64_t(depths) * (rank + 1) / blocks);
    bool lost = false;

    if (!work) {
        constexpr int size = TYPE == FRX_F32 ? 4 : 2;
        using Element = std::conditional_t<size == 4, uint32_t, uint16_t>;
        if (live > 0 && p.out != p.y) {   // no adapter: y as it is
            for (int t = int(rank); t < live; t += int(blocks)) {
                const Element* from = static_cast<const Element*>(p.y) + (t0 + t) * p.ldy;
                Element* to = static_cast<Element*>(p.out) + (t0 + t) * p.ldo;
                for (int i = threadIdx.x; i < p.rows; i += kThreads) to[i] = from[i];
            }
        }
    } else if (warp == kWarpLoad) {
        // ---------------- loads: the first product's stages, and this block's rows of B_j as soon as there is room
        const int boxes = (live + p.box - 1) / p.box;
        const uint32_t bytes = uint32_t(boxes * p.box * 128 + p.rank16 * 128);
        uint32_t st = 0, phase = 1, buf = 0, bphase = 1;
        int c = int(rank);
        bool ok = true;
        auto rows_of_b = [&]() {
            if (!(ok = warp_wait(bars + (kBarBFree + buf) * 8, bphase, abort, p.wait_ns))) return;
            const uint32_t full = bars + (kBarBFull + buf) * 8, to = bbuf + buf * bbuf_bytes;
            if (lane == 0) {
                mbar_expect_tx(full, bbuf_bytes);
                for (int i = 0; i < chunks; ++i) tma_3d(to + i * kPiece, &b_map, i * 64, c * kRows, j, full);
            }
            __syncwarp();
            c += int(blocks);
            if (++buf == kBufs) buf = 0, bphase ^= 1u;
        };
        for (int s = d0; s < d1 && ok; ++s) {
            if (!(ok = warp_wait(bars + (kBarFree + st) * 8, phase, abort, p.wait_ns))) break;
            const uint32_t full = bars + (kBarFull + st) * 8, x = ring + st * uint32_t(p.stage_bytes), a = x + kTok * 128;
            if (lane == 0) {
                mbar_expect_tx(full, bytes);
                for (int i = 0; i < boxes; ++i) tma_2d(x + i * p.box * 128, &x_map, s * kDepth, t0 + i * p.box, full);
                tma_3d(a, &a_map, s * kDepth, 0, j, full);
            }
            __syncwarp();
            if (++st == kStages) st = 0, phase ^= 1u;
            if (s - d0 == kStages - 1)
                for (int i = 0; i < kBufs && c < row_chunks && ok; ++i) rows_of_b();
        }
        while (c < row_chunks && ok) rows_of_b();
    } else if (warp == kWarpMma) {
        uint32_t st = 0, phase = 0;
        bool ok = true;
        const uint32_t idesc = p.idesc | uint32_t(p.rank16 >> 3) << 17;
        for (int s = d0; s < d1; ++s) {
            if (!(ok = warp_wait(bars + (kBarFull + st) * 8, phase, abort, p.wait_ns))) break;
            const uint32_t x = ring + st * uint32_t(p.stage_bytes);
            const int depth = min(kDepth, p.n - s * kDepth);
            if (elect_one()) {
                const uint64_t da = umma_desc_sw128(x), db = umma_desc_sw128(x + kTok * 128);
#pragma unroll
                for (int k = 0; k < kDepth / 16; ++k) {
                    if (k * 16 >= depth) break;
                    umma_f16(tmem, da + k * 2, db + k * 2, idesc, s + k > d0);
                }
                umma_commit(bars + (kBarFree + st) * 8);
                if (s + 1 == d1) umma_commit(bars + kBarV * 8);
            }
            __syncwarp();
            if (++st == kStages) st = 0, phase ^= 1u;
        }
        ok = ok && warp_wait(bars + kBarVIn * 8, 0, abort, p.wait_ns);
        uint32_t buf = 0, bphase = 0, set = 0, dphase = 1;
        for (int c = int(rank); c < row_chunks && ok; c += int(blocks)) {
            if (!(ok = warp_wait(bars + (kBarBFull + buf) * 8, bphase, abort, p.wait_ns))) break;
            for (int h = 0; h < halves; ++h) {
                if (!(ok = warp_wait(bars + (kBarDFree + set) * 8, dphase, abort, p.wait_ns))) break;
                tc_fence_after_sync();
                const uint32_t width = uint32_t((min(kHalf, live - h * kHalf) + 15) & ~15), id = p.idesc | (width >> 3) << 17;
                if (elect_one()) {
                    for (int q = 0; q < 3; ++q)
                        for (int k = 0; k < p.rank16; k += 16) {
                            const uint32_t at = uint32_t(k >> 6) * kPiece, in = uint32_t(k & 63) * 2;
                            umma_f16(tmem + kColD + set * kHalf, umma_desc_sw128(bbuf + buf * bbuf_bytes + at) + (in >> 4),
                                     umma_desc_sw128(ring + q * bbuf_bytes + at + h * kHalf * 128) + (in >> 4), id, q + k > 0);
                        }
                    if (h + 1 == halves) umma_commit(bars + (kBarBFree + buf) * 8);
                    umma_commit(bars + (kBarDFull + set) * 8);
                }
                __syncwarp();
                set ^= 1u;
                if (set == 0) dphase ^= 1u;
            }
            if (++buf == kBufs) buf = 0, bphase ^= 1u;
        }
    } else {
        const int quarter = warp & 3, side = warp >> 2, token = quarter * 32 + lane;
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        // ---------------- v: a lane is a token, a warp has half of the rank
        const int half = p.rank16 / 2, k0 = side * half;
        const bool empty = d0 == d1;   // no part of the depth here
        if (!empty) {
            lost = !warp_wait(bars + kBarV * 8, 0, abort, p.wait_ns);
            tc_fence_after_sync();
        }
        const uint32_t mine = part + uint32_t(token * p.rank16) * 4;
        if (blocks > 1) {
            for (int k = k0; k < k0 + half; k += 8) {
                float v[8];
                if (empty || lost) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = lost ? __uint_as_float(0x7fffffffu) : 0.0f;
                } else {
                    tmem_ld8(tmem + lanes + k, v);
                }
                if (token < live) {
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + k * 4), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + k * 4 + 16), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
                }
            }
            __syncwarp();
            if (lane < int(blocks)) mbar_arrive_peer(peer_addr(bars + kBarPart * 8, uint32_t(lane)));
            lost = !warp_wait_cluster(bars + kBarPart * 8, 0, abort, p.wait_ns) || lost;
        }
        auto take8 = [&](int k, float (&v)[8]) {
            if (blocks > 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
                if (token < live && !lost)
                    for (uint32_t b = 0; b < blocks; ++b) {
                        const uint32_t at = peer_addr(mine + k * 4, b);
                        const float4 lo = ld_peer(at), hi = ld_peer(at + 16);
                        v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w, v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
                    }
            } else {
                tmem_ld8(tmem + lanes + k, v);   // (sums that nobody has finished, where the wait ran out: the outputs are NaN then)
            }
        };
        const float scale = p.scale ? __ldcg(p.scale + j) : 1.0f;
        float up = 1.0f;
        if (XTYPE == FRX_F16) {
            // the token's largest magnitude to [2^14, 2^15): pieces of float16 then hold every bit of the others that counts
            float most = 0.0f;
            for (int k = k0; k < k0 + half; k += 8) {
                float v[8];
                take8(k, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i] * scale));
            }
            tok_max[side * kTok + token] = most;
            named_bar_sync(1, 32 * kWarpsEpi);
            most = fmaxf(tok_max[token], tok_max[kTok + token]);
            const uint32_t e = __float_as_uint(most) >> 23;   // its exponent + 127
            // 2^(141 - e) and back, within what 32 bits hold; nothing for zeros, infinities and NaN
            const uint32_t f = e == 255u || most == 0.0f ? 127u : min(max(268u - e, 1u), 253u);
            up = __uint_as_float(f << 23);
            if (side == 0) tok_scale[token] = __uint_as_float((254u - f) << 23);
        }
        for (int k = k0; k < k0 + half; k += 8) {
            float v[8];
            take8(k, v);
            uint32_t bits[3][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float f = v[i] * scale * up;
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    const uint32_t b = take_piece<XTYPE>(f);
                    bits[q][i / 2] = i & 1 ? bits[q][i / 2] | b << 16 : b;
                }
            }
            const uint32_t at = ring + uint32_t(k >> 6) * kPiece + uint32_t(token) * 128 + uint32_t(((k & 63) >> 3) ^ (token & 7)) * 16;   // (the 128-byte swizzle)
#pragma unroll
            for (int q = 0; q < 3; ++q)
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + q * bbuf_bytes), "r"(bits[q][0]), "r"(bits[q][1]), "r"(bits[q][2]), "r"(bits[q][3]) : "memory");
        }
        fence_async_smem();   // generic-proxy writes: visible to the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kBarVIn * 8);
        if (XTYPE == FRX_F16) named_bar_sync(1, 32 * kWarpsEpi);   // tok_scale is there
        // ---------------- the second product's sums: a lane is a row of y, a warp has 32 of 64 tokens
        constexpr int size = TYPE == FRX_F32 ? 4 : 2;
        const bool pairs = TYPE != FRX_F32 && p.rows % 2 == 0 && p.ldy % 2 == 0 && p.ldo % 2 == 0 && (reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.out)) % 4 == 0;
        uint32_t set = 0, phase = 0;
        for (int c = int(rank); c < row_chunks; c += int(blocks)) {
            const int row = c * kRows + quarter * 32 + lane;
            const bool have = row < p.rows;
            for (int h = 0; h < halves; ++h) {
                const int tok = h * kHalf + side * 32, count = live - tok;   // the warp's first token, and tokens from it on
                const uint8_t* y = static_cast<const uint8_t*>(p.y) + ((t0 + tok) * p.ldy + row) * size;
                uint8_t* out = static_cast<uint8_t*>(p.out) + ((t0 + tok) * p.ldo + row) * size;
                Ahead<TYPE> old[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) old[q].load(y + q * 16 * p.ldy * size, p.ldy, count - q * 16, have, pairs);
                lost = !warp_wait(bars + (kBarDFull + set) * 8, phase, abort, p.wait_ns) || lost;
                tc_fence_after_sync();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[8];
                    if (q * 8 >= count) break;
                    if (lost) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7fffffffu);
                    } else {
                        tmem_ld8(tmem + lanes + kColD + set * kHalf + side * 32 + q * 8, v);
                    }
                    if (XTYPE == FRX_F16) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] *= tok_scale[tok + q * 8 + i];
                    }
                    add_and_store8<TYPE>(v, old[q / 2], q & 1, out + q * 8 * p.ldo * size, p.ldo, count - q * 8, have, pairs);
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0 && !lost) mbar_arrive(bars + (kBarDFree + set) * 8);
                set ^= 1u;
                if (set == 0) phase ^= 1u;
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        // A wait ran out: copies and MMAs may still be in flight. Give them time to land before tensor memory and the block's
        // shared memory are released.
        const uint64_t begin = global_ns();
        while (global_ns() - begin < 2000000ull) {
        }
        __syncthreads();
    }
    if (warp == kWarpMma) tmem_free(tmem, kCols);
    if (blocks > 1) cluster_sync_all();   // the others have read what they needed of this block's shared memory
}

template <int XTYPE, int TYPE>
int launch_typed(Adapters& p, const CUtensorMap& x_map, const CUtensorMap& a_map, const CUtensorMap& b_map, cudaStream_t stream) {
    int rc = allow_smem<k_adapter<XTYPE, TYPE>>();
    if (rc != FRX_OK) return rc;
    const int chunks = p.rank16 > 64 ? 2 : 1;
    const int64_t tiles = int64_t(p.T) / kTok + std::min(p.R, p.T);   // of any requests that do not overlap
    // as many blocks a tile as run at the same time (two an SM, one where the rank is more than 64)
    unsigned blocks = 8;
    while (blocks > 1 && tiles * blocks > int64_t(sm_count()) * (chunks == 1 ? 2 : 1)) blocks /= 2;
    if (tiles * blocks > 0x7fff0000) return fail(FRX_ERR_SHAPE, "adapters: %lld tiles", (long long)tiles);
    p.stage_bytes = kTok * 128 + p.rank16 * 128;
    p.ring_bytes = std::max(kStages * p.stage_bytes, 3 * chunks * kPiece);
    const size_t smem = size_t(kHead) + p.ring_bytes + kBufs * chunks * kPiece + (blocks > 1 ? size_t(kTok) * p.rank16 * 4 : 0);
    static_assert(kHead + 3 * 2 * kPiece + kBufs * 2 * kPiece + kTok * 128 * 4 <= kSmemMost, "the largest rank");
    static_assert(3 * (kHead + kStages * (kTok + 16) * 128 + kBufs * kPiece) > 228 * 1024, "no third block an SM, which would wait for tensor memory");
    p.wait_ns = wait_limit_ns();
    FRX_LAUNCH(kKGateUp, stream, launch_pdl_cluster(k_adapter<XTYPE, TYPE>, dim3(unsigned(tiles) * blocks), dim3(kThreads), smem, stream, blocks, p, x_map, a_map, b_map));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}
template <int XTYPE>
int launch(Adapters& p, int type, const CUtensorMap& x_map, const CUtensorMap& a_map, const CUtensorMap& b_map, cudaStream_t stream) {
    switch (type) {
        case FRX_F32: return launch_typed<XTYPE, FRX_F32>(p, x_map, a_map, b_map, stream);
        case FRX_BF16: return launch_typed<XTYPE, FRX_BF16>(p, x_map, a_map, b_map, stream);
        default: return launch_typed<XTYPE, FRX_F16>(p, x_map, a_map, b_map, stream);
    }
}

}  // namespace
}  // namespace frx

using namespace frx;

extern "C" int frx_adapter_add(frx_stream_t stream, const void* x, int64_t ldx, const void* a, int64_t lda, int64_t stride_a, const void* b, int64_t ldb, int64_t stride_b, int dtype,
                               int L, int rank, int n, int rows, const int32_t* offsets, const int32_t* which, int R, const float* scale, int T, const void* y, int64_t ldy, void* out,
                               int64_t ldo, int y_dtype) {
    const char* who = "frx_adapter_add";
    if (T < 0 || R < 0) return fail(FRX_ERR_ARG, "%s: %d tokens of %d requests", who, T, R);
    if (dtype != FRX_BF16 && dtype != FRX_F16) return fail(FRX_ERR_ARG, "%s: element type %d (bfloat16 or float16)", who, dtype);
    if (!dtype_size(y_dtype)) return fail(FRX_ERR_ARG, "%s: element type %d", who, y_dtype);
    if (L < 1 || rank < 1 || rank > 128 || n < 1 || rows < 1 || n > (1 << 20) || rows > (1 << 20))
        return fail(FRX_ERR_SHAPE, "%s: unsupported shape: %d adapters of rank %d, n %d, rows %d", who, L, rank, n, rows);
    if (T == 0 || R == 0) return FRX_OK;
    if (!offsets || !which || !y || !out) return fail(FRX_ERR_ARG, "%s: null pointer", who);
    if (ldy < rows || ldo < rows) return fail(FRX_ERR_ARG, "%s: rows of y and out are %lld and %lld elements apart and %d long", who, (long long)ldy, (long long)ldo, rows);
    if (!rows_aligned(y, dtype_size(y_dtype)) || !rows_aligned(out, dtype_size(y_dtype))) return fail(FRX_ERR_ARG, "%s: misaligned pointer", who);
    int rc;
    if ((rc = operand(who, "x", x, ldx, T, n)) != FRX_OK || (rc = operand(who, "a", a, lda, rank, n)) != FRX_OK || (rc = operand(who, "b", b, ldb, rows, rank)) != FRX_OK ||
        (rc = operand(who, "a (its matrices)", a, stride_a, L, (rank - 1) * lda + n)) != FRX_OK ||
        (rc = operand(who, "b (its matrices)", b, stride_b, L, (rows - 1) * ldb + rank)) != FRX_OK)
        return rc;
    Adapters p{};
    p.offsets = offsets;
    p.which = which;
    p.scale = scale;
    p.y = y;
    p.out = out;
    p.ldy = ldy;
    p.ldo = ldo;
    p.T = T;
    p.R = R;
    p.L = L;
    p.n = n;
    p.rows = rows;
    p.rank = rank;
    p.rank16 = (rank + 15) & ~15;
    p.box = T / R >= 64 ? 64 : 16;   // rows of a load: few where most requests have a token or two
    p.idesc = f16_idesc(dtype, false, false);
    CUtensorMap xm, am, bm;
    if ((rc = rows_map(xm, x, ldx, dtype, T, n, p.box)) != FRX_OK || (rc = matrices_map(am, a, lda, stride_a, dtype, L, rank, n, p.rank16)) != FRX_OK ||
        (rc = matrices_map(bm, b, ldb, stride_b, dtype, L, rows, rank, kRows)) != FRX_OK)
        return rc;
    return dtype == FRX_BF16 ? launch<FRX_BF16>(p, y_dtype, xm, am, bm, stream) : launch<FRX_F16>(p, y_dtype, xm, am, bm, stream);
}
