// Low-rank adapters of many requests beside a shared projection (frx_adapter_add in frx.h).
#include <algorithm>
#include <type_traits>

#include "frx_groups.cuh"

namespace frx {
namespace {

// out[t] = y[t] + scale_j B_j (A_j x[t]), j the adapter of t's request. What has to move is x, y and out, and each adapter once; the products are few. So one kernel does
// both of them and v = A_j x never leaves the SM:
//   first   v[t][k] = sum_c x[t][c] A_j[k][c]     up to 64 tokens of a request are the lanes (of 128), the rank is N
//   second  d[t][m] = sum_k v[t][k] B_j[m][k]     the tokens are the lanes, twice (so that all warps have some), 128 rows of B_j are N
// v is kept in 32 bits: it goes into the second product as three 16-bit pieces whose sum it is (for float16, whose exponents do not reach, as multiples of a power of two of its token).
// A tile (64 tokens of a request) is the work of a cluster of up to eight blocks, as many as fit the GPU at once: they share the first product's depth, add their
// parts up through one another's shared memory (in the order of the blocks), and share the second product's rows. y is read two steps (32 bits: one) ahead of the sums it is added
// to, from before the first product on.
constexpr int kTok = 64, kRows = 128, kDepth = 64, kFewRank = 16;
constexpr int kMaxStages = 10, kMinStages = 3, kBufs = 2;
constexpr int kWarpsEpi = 8, kWarpLoad = 8, kWarpMma = 9, kThreads = 32 * 10;
constexpr int kBarFull = 0, kBarFree = kBarFull + kMaxStages, kBarBFull = kBarFree + kMaxStages, kBarBFree = kBarBFull + kBufs, kBarDFull = kBarBFree + kBufs, kBarDFree = kBarDFull + 2,
              kBarV = kBarDFree + 2, kBarVIn = kBarV + 1, kBarPart = kBarVIn + 1, kBars = kBarPart + 1;
constexpr int kAbort = 256, kSlot = 260, kFound = 264, kSums = 320, kTokScale = 512, kTokMax = kTokScale + 4 * kTok, kHead = 2048;
static_assert(kBars * 8 <= kAbort && kSums + 8 * kThreads / 32 <= kTokScale && kTokMax + 8 * kTok <= kHead, "the block's head");
constexpr int kPieceV = 2 * kTok * 128, kPieceB = kRows * 128;   // bytes of 64 of the rank: of a piece of v, of 128 rows of B_j
constexpr int kCols = 256;   // tensor memory: two sets of 128 columns, the first of them also for v's sums; two blocks an SM
constexpr int kSmemTwo = 228 * 512 - 1024;   // shared memory of a block of which an SM holds two

// y and out move in accesses of 32 bytes a lane, four lanes 128 bytes of a row, where rows allow it (copies of 16,384 rows of 4 KB: 5.3 TB/s in pieces of 256 bytes a row, 4.1 with a row a
// lane). The sums come out of tensor memory in the form of 16 lanes x 8 columns, in which a thread has columns 2 i, 2 i + 1 (i = lane % 4) of every eight: so the rows of B_j go into shared memory in
// the order that makes these consecutive. Of G = 16 (32-bit y: 8) rows an access, column 8 k + 2 i + b of 4 G columns is row G i + 2 k + b: three dimensions of the tensor map.
//
// What bounds it. 16,384 tokens, rank 32, 2,048 by 2,048: 47 to 50 us for 204 MB (a copy takes 31): the two halves of the kernel, x in (15 us) and y through (25), each near the rate of memory, follow
// one another, and 3 us of start and end. 1,000 tokens of 41 users, rank 64, 32-bit y: 27 us, a chain of 16 KB stages, three in flight, the exchange between four blocks, and five steps over rows of y.
// 64 users, rank 16: 8.6 us, one: 5.9 (8.5 for the call from Python).
// Where y and out do not allow accesses of 32 bytes (rows, distances or addresses that are not multiples of 32 bytes) a lane adds element by element, each behind the store of the last: ten
// times as long for 16,384 tokens (2,040 rows instead of 2,048: 496 us instead of 48), seven for the 1,000 with 16-bit y (128 instead of 18.5), nothing for tiles of single tokens up to a rank of 64.
// Every block looks through all requests: 64 tokens at a time of thousands of them are bound by that (1,024 single tokens of rank 16 50 us, 4,096 229, 16,384 2.8 ms).
struct Adapters {
    const int32_t* offsets;   // [R + 1]
    const int32_t* which;     // [R]
    const float* scale;       // [L] or null
    const void *x, *a, *b, *y;
    void* out;
    int64_t ldx, lda, stride_a, ldb, stride_b, ldy, ldo;
    unsigned long long wait_ns;
    int T, R, L, n, rows, rank, rank16;   // rank16: the rank rounded up to 16
    int box, ring_bytes;                        // rows of a load of x; bytes of the first product's stages (v's pieces come to the same place)
    uint32_t idesc;
    int whole;                                  // y and out allow accesses of 32 bytes
};

__device__ __forceinline__ float ld_peer1(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int u, int v, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(v),
                 "r"(bar)
                 : "memory");
}
// 64 columns of 16 lanes (two rows of eight columns a lane and step: v[k][0], [1] of row lane / 4, [2], [3] of row lane / 4 + 8, columns 8 k + 2 (lane % 4) and the next), complete on return
__device__ __forceinline__ void tmem_ld_16x256(uint32_t addr, uint32_t (&v)[8][4]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0][0]), "=r"(v[0][1]), "=r"(v[0][2]), "=r"(v[0][3]), "=r"(v[1][0]), "=r"(v[1][1]), "=r"(v[1][2]), "=r"(v[1][3]), "=r"(v[2][0]), "=r"(v[2][1]), "=r"(v[2][2]),
          "=r"(v[2][3]), "=r"(v[3][0]), "=r"(v[3][1]), "=r"(v[3][2]), "=r"(v[3][3]), "=r"(v[4][0]), "=r"(v[4][1]), "=r"(v[4][2]), "=r"(v[4][3]), "=r"(v[5][0]), "=r"(v[5][1]),
          "=r"(v[5][2]), "=r"(v[5][3]), "=r"(v[6][0]), "=r"(v[6][1]), "=r"(v[6][2]), "=r"(v[6][3]), "=r"(v[7][0]), "=r"(v[7][1]), "=r"(v[7][2]), "=r"(v[7][3])
        : "r"(addr)
        : "memory");
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

// 32 bytes of y, of which nothing is waited for here (as a conditional assignment the load became a branch that was: one load after the other)
__device__ __forceinline__ void load_if(uint32_t* w, const void* p, bool on) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.u32 q, %9, 0;\n\t"
        "@q ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t}"
        : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3]), "+r"(w[4]), "+r"(w[5]), "+r"(w[6]), "+r"(w[7])
        : "l"(p), "r"(uint32_t(on)));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
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
// 32 bytes of y with as many sums added, rounded once and written
template <int TYPE>
__device__ __forceinline__ void add_and_store(const float* f, const uint32_t* y, void* out) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = TYPE == FRX_F32 ? __float_as_uint(f[i] + __uint_as_float(y[i])) : narrow2<TYPE>(f[2 * i] + wide<TYPE>(y[i]), f[2 * i + 1] + wide<TYPE>(y[i] >> 16));
    store32(out, w);
}
// the same of 16 elements one by one, as far as there are so many
template <int TYPE>
__device__ __forceinline__ void add_and_store_each(const float (&f)[16], const void* y, void* out, int live) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < live) {
            if (TYPE == FRX_F32)
                static_cast<float*>(out)[i] = f[i] + static_cast<const float*>(y)[i];
            else
                static_cast<uint16_t*>(out)[i] = uint16_t(narrow2<TYPE>(f[i] + wide<TYPE>(static_cast<const uint16_t*>(y)[i]), 0.0f));
        }
}

// rows t0 .. t0 + live - 1 of `size`-byte elements to another place, a row a warp: 16 bytes a lane where both sides allow it, eight accesses in flight
template <class Access>
__device__ __forceinline__ void copy_row(const Access* from, Access* to, int count) {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < count; i += 8 * 32) {
        Access v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + 32 * k < count) v[k] = from[i + 32 * k];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + 32 * k < count) to[i + 32 * k] = v[k];
    }
}
template <int SIZE>
__device__ __forceinline__ void copy_rows(const void* from, int64_t ld_from, void* to, int64_t ld_to, int t0, int live, int n, int warp, int warps) {
    using Element = std::conditional_t<SIZE == 4, uint32_t, uint16_t>;
    const bool wide = ((reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(to) | uintptr_t(ld_from * SIZE) | uintptr_t(ld_to * SIZE) | uintptr_t(n * SIZE)) & 15) == 0;
    for (int t = warp; t < live; t += warps) {
        const Element* a = static_cast<const Element*>(from) + (t0 + t) * ld_from;
        Element* b = static_cast<Element*>(to) + (t0 + t) * ld_to;
        if (wide)
            copy_row(reinterpret_cast<const uint4*>(a), reinterpret_cast<uint4*>(b), n * SIZE / 16);
        else
            copy_row(a, b, n);
    }
}

// eight 16-bit elements from p on, `count` of which are there (the others 0); p on a 16-byte boundary
struct Eight {
    uint4 v;
    __device__ __forceinline__ void load(const uint16_t* p, int count, bool tails) {   // tails: whether there are counts between 0 and 8 at all
        v = make_uint4(0u, 0u, 0u, 0u);
        asm volatile(
            "{\n\t.reg .pred q;\n\t"
            "setp.ge.s32 q, %5, 8;\n\t"
            "@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
            : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
            : "l"(p), "r"(count));
        if (tails && count > 0 && count < 8) {
            uint32_t w[4] = {};
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < count) w[i / 2] |= uint32_t(p[i]) << (i % 2 * 16);
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    template <int XTYPE>
    __device__ __forceinline__ void wide8(float (&f)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = wide<XTYPE>(w[i]);
            f[2 * i + 1] = wide<XTYPE>(w[i] >> 16);
        }
    }
};

// A tile of one token and a rank of up to 16 by fused multiply-adds: the steps between are fewer than by way of the tensor cores, whose instructions take 128 lanes and 16 columns
// whatever there is (64 users 12.9 -> 8.6 us, 256 31 -> 15; more of the rank is more of these than memory waits for). First product: a warp has two rows of A_j, the lanes the columns
// of this block's part of the depth. Second: two lanes have a row of B_j, eight of the rank each; its rows and y's elements are read four steps ahead, the
// first before v is there.
template <int XTYPE, int TYPE>
__device__ __forceinline__ void one_token(const Adapters& p, uint32_t bars, uint32_t abort, float* part, uint32_t part_addr, float* v, int t0, int j, int c0, int c1, uint32_t rank, uint32_t blocks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kWarps = kThreads / 32, kAhead = 4, size = TYPE == FRX_F32 ? 4 : 2;
    const uint16_t* x = static_cast<const uint16_t*>(p.x) + int64_t(t0) * p.ldx;
    const uint16_t* a = static_cast<const uint16_t*>(p.a) + int64_t(j) * p.stride_a;
    const uint16_t* b = static_cast<const uint16_t*>(p.b) + int64_t(j) * p.stride_b;
    static_assert(2 * kWarps >= kFewRank, "two rows a warp");
    {
        float acc[2] = {};
        const bool first = warp < p.rank, second = warp + kWarps < p.rank, tails = p.n % 8 != 0;
#pragma unroll 4
        for (int c = c0 + lane * 8; c < c1; c += 256) {
            const int count = min(8, c1 - c);
            Eight av[2], xv;
            av[0].load(a + int64_t(warp) * p.lda + c, first ? count : 0, tails);
            av[1].load(a + int64_t(warp + kWarps) * p.lda + c, second ? count : 0, tails);
            xv.load(x + c, count, tails);
            float af[2][8], xf[8];
            av[0].wide8<XTYPE>(af[0]);
            av[1].wide8<XTYPE>(af[1]);
            xv.wide8<XTYPE>(xf);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[0] = fmaf(xf[i], af[0][i], acc[0]);
                acc[1] = fmaf(xf[i], af[1][i], acc[1]);
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int o = 16; o; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
            if (lane == 0 && (m ? second : first)) part[warp + m * kWarps] = acc[m];
        }
    }
    constexpr int kPer = 16, kSteps = kRows / kPer;   // rows a warp's step; steps of a chunk of rows
    const int q = lane & 1;
    const int row_chunks = (p.rows + kRows - 1) / kRows, count = int(rank) < row_chunks ? ((row_chunks - 1 - int(rank)) / int(blocks) + 1) * kSteps : 0;   // steps of this block
    auto row_of = [&](int i) { return (int(rank) + i / kSteps * int(blocks)) * kRows + i % kSteps * kPer + lane / 2; };
    Eight bv[kAhead];
    uint32_t yv[kAhead] = {};
    auto read = [&](int m, int i) {
        const int row = row_of(i);
        const bool have = i < count && row < p.rows;
        bv[m].load(b + int64_t(row) * p.ldb + q * 8, have ? min(8, p.rank - q * 8) : 0, p.rank % 8 != 0);
        load_one_if<TYPE>(yv[m], static_cast<const uint8_t*>(p.y) + (t0 * p.ldy + row) * size, have && q == 0);
    };
#pragma unroll
    for (int m = 0; m < kAhead; ++m) read(m, warp + m * kWarps);
    __syncthreads();
    bool ok = true;
    if (blocks > 1) {
        if (warp < kWarpsEpi && lane < int(blocks)) mbar_arrive_peer(peer_addr(bars + kBarPart * 8, uint32_t(lane)));
        ok = warp_wait_cluster(bars + kBarPart * 8, 0, abort, p.wait_ns);
    }
    if (threadIdx.x < kFewRank) {
        const int k = threadIdx.x;
        float sum = 0.0f;
        if (k < p.rank) {
            if (blocks > 1) {
                float of[8];
#pragma unroll
                for (uint32_t m = 0; m < 8; ++m) of[m] = m < blocks ? ld_peer1(peer_addr(part_addr + uint32_t(k) * 4, m)) : 0.0f;
#pragma unroll
                for (int m = 0; m < 8; ++m) sum += of[m];
            } else {
                sum = part[k];
            }
            sum *= p.scale ? __ldcg(p.scale + j) : 1.0f;
        }
        v[k] = sum;
    }
    __syncthreads();
    ok = ok && lds32(abort) == 0;   // (whoever's wait ran out, its sums are everybody's)
    float vf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) vf[i] = v[q * 8 + i];
    for (int i0 = warp; i0 < count; i0 += kAhead * kWarps) {
#pragma unroll
        for (int m = 0; m < kAhead; ++m) {
            const int i = i0 + m * kWarps, row = row_of(i);
            float bf[8], sum = 0.0f;
            bv[m].wide8<XTYPE>(bf);
            const uint32_t old = yv[m];
            read(m, i + kAhead * kWarps);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = q * 8 + e < p.rank ? fmaf(bf[e], vf[e], sum) : sum;   // (nothing beyond the rank, were v infinite)
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            if (!ok) sum = __uint_as_float(0x7fffffffu);   // a wait ran out
            if (i < count && row < p.rows && q == 0) {
                uint8_t* to = static_cast<uint8_t*>(p.out) + (t0 * p.ldo + row) * size;
                if (TYPE == FRX_F32)
                    *reinterpret_cast<float*>(to) = sum + __uint_as_float(old);
                else
                    *reinterpret_cast<uint16_t*>(to) = uint16_t(narrow2<TYPE>(sum + wide<TYPE>(old), 0.0f));
            }
        }
    }
}

// Eight 16-bit elements from p on (on a 16-byte boundary), `count` of which are there and the others 0, to this lane's place in shared memory, on their own
__device__ __forceinline__ void fetch8(uint32_t dst, const uint16_t* p, int count) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p), "r"(2 * min(max(count, 0), 8)) : "memory");
}
__device__ __forceinline__ void fetch_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>   // until all but the last N groups are there
__device__ __forceinline__ void fetch_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds8(uint32_t addr, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}
// D (16 x 8, 32 bits) += A (16 x 16) B (16 x 8) of one warp
template <int XTYPE>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (XTYPE == FRX_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The power of two that brings v's largest magnitude to [2^14, 2^15), and its inverse (`down`), within what 32 bits hold; 1 for zeros, infinities and NaN
__device__ __forceinline__ float power_up(float most, float& down) {
    const uint32_t e = __float_as_uint(most) >> 23;   // its exponent + 127
    const uint32_t f = e == 255u || most == 0.0f ? 127u : min(max(268u - e, 1u), 253u);   // 2^(141 - e)
    down = __uint_as_float((254u - f) << 23);
    return __uint_as_float(f << 23);
}

// The same of a rank of 17 to 64, by warps' own matrix instructions (16 rows of a matrix by 8 tokens, of which there is one): a lane's eight elements of a row come in one asynchronous copy to a
// place of the lane's own, kSlots of which it has, so that nothing is waited for but its own copies and none take registers. (The order of the depth inside an instruction is free as long as
// both operands have the same.) First product: a warp has 16 rows of A_j and every so many-th 32 of this block's depth, summed over 128 from zero and added up rounded to nearest. Second: a warp has 16
// rows of B_j a step, y read four steps ahead. NB: the rank in 32s. 256 users, rank 32: 20 us (36 as tiles of 64 tokens), rank 64: 31 (46); 64 users 11 and 14.
constexpr int kSlots = 15, kSlotBytes = kThreads * 16;
template <int XTYPE, int TYPE, int NB>
__device__ __forceinline__ void one_token_of_rank(const Adapters& p, uint32_t bars, uint32_t abort, uint32_t slots, float* own, float* part, uint32_t part_addr, float* v, int t0, int j, int c0, int c1, uint32_t rank,
                                                  uint32_t blocks) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    constexpr int kWarps = kThreads / 32, kDeep = kSlots / 3, kRowsDeep = kSlots / (2 * NB), kAhead = 4, size = TYPE == FRX_F32 ? 4 : 2;
    const uint16_t* x = static_cast<const uint16_t*>(p.x) + int64_t(t0) * p.ldx;
    const uint16_t* a = static_cast<const uint16_t*>(p.a) + int64_t(j) * p.stride_a;
    const uint16_t* b = static_cast<const uint16_t*>(p.b) + int64_t(j) * p.stride_b;
    const uint32_t mine = slots + threadIdx.x * 16;
    const int tiles = p.rank16 / 16, phases = kWarps / tiles, r0 = warp % tiles * 16, phase = warp / tiles;   // (of a rank of 64 four tiles of rows and two warps each)
    float sum[4] = {};
    if (phase < phases) {
        const int first = c0 + phase * 32, step = 32 * phases, steps = max(0, (c1 - first + step - 1) / step);
        const uint16_t *pa = a + int64_t(r0 + g) * p.lda + first + q * 8, *px = x + first + q * 8;   // of the next fetch
        const int64_t eight = int64_t(8) * p.lda;
        const bool on = r0 + g < p.rank, on8 = r0 + g + 8 < p.rank, onx = g == 0;
        int left = c1 - first - q * 8;   // elements from there on
        auto fetch = [&](uint32_t at) {
            fetch8(at, on && left > 0 ? pa : a, on ? left : 0);
            fetch8(at + kSlotBytes, on8 && left > 0 ? pa + eight : a, on8 ? left : 0);
            fetch8(at + 2 * kSlotBytes, onx && left > 0 ? px : x, onx ? left : 0);
            fetch_group();
            pa += step;
            px += step;
            left -= step;
        };
        for (int i = 0; i < kDeep; ++i) fetch(mine + i * 3 * kSlotBytes);
        float d[4] = {};
        uint32_t at = mine;
        for (int i = 0; i < steps; ++i) {
            fetch_wait<kDeep - 1>();
            uint32_t lo[4], hi[4], xv[4];
            lds8(at, lo);
            lds8(at + kSlotBytes, hi);
            lds8(at + 2 * kSlotBytes, xv);
#pragma unroll
            for (int h = 0; h < 4; h += 2) mma_16x8x16<XTYPE>(d, lo[h], hi[h], lo[h + 1], hi[h + 1], xv[h], xv[h + 1]);
            fetch(at);
            at = at + 3 * kSlotBytes == mine + kDeep * 3 * kSlotBytes ? mine : at + 3 * kSlotBytes;
            if ((i & 3) == 3 || i + 1 == steps) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += d[e], d[e] = 0.0f;
            }
        }
        fetch_wait<0>();   // (those from behind the depth write zeros to the places of the next: copies have no order among themselves)
    }
    // the second product's first rows are on their way while the parts are added up
    const int all16 = (p.rows + 15) / 16, from16 = int(int64_t(all16) * rank / blocks), count = int(int64_t(all16) * (rank + 1) / blocks) - from16;   // this block's rows, 16 a step
    const int row0 = (from16 + warp) * 16 + g;   // the lane's first row, and eight further its second; those of the next step 16 kWarps further
    const uint16_t* pb = b + int64_t(row0) * p.ldb + q * 8;   // of the next fetch
    const int64_t eight = int64_t(8) * p.ldb, step_b = int64_t(16 * kWarps) * p.ldb;
    int row_b = row0, ahead = warp;
    auto fetch = [&](uint32_t at) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int have = ahead < count ? p.rank - k * 32 - q * 8 : 0;
            const bool lo = have > 0 && row_b < p.rows, hi = have > 0 && row_b + 8 < p.rows;
            fetch8(at + 2 * k * kSlotBytes, lo ? pb + k * 32 : b, lo ? have : 0);
            fetch8(at + (2 * k + 1) * kSlotBytes, hi ? pb + eight + k * 32 : b, hi ? have : 0);
        }
        fetch_group();
        ahead += kWarps;
        row_b += 16 * kWarps;
        pb += step_b;
    };
    const uint8_t* py = static_cast<const uint8_t*>(p.y) + (t0 * p.ldy + row0) * size;
    uint8_t* po = static_cast<uint8_t*>(p.out) + (t0 * p.ldo + row0) * size;
    uint32_t yv[kAhead][2] = {};
    int row_y = row0, step_y = warp;
    auto read_y = [&](int m) {
#pragma unroll
        for (int h = 0; h < 2; ++h) load_one_if<TYPE>(yv[m][h], py + h * 8 * size, q == 0 && step_y < count && row_y + h * 8 < p.rows);
        py += 16 * kWarps * size;
        row_y += 16 * kWarps;
        step_y += kWarps;
    };
    for (int i = 0; i < kRowsDeep; ++i) fetch(mine + i * 2 * NB * kSlotBytes);
#pragma unroll
    for (int m = 0; m < kAhead; ++m) read_y(m);
    // v: the sums of the warps, then of the blocks
    if (phase < phases && q == 0) {
        own[phase * 64 + r0 + g] = sum[0];
        own[phase * 64 + r0 + g + 8] = sum[2];
    }
    __syncthreads();
    const int k = threadIdx.x;
    float all = 0.0f;
    if (k < p.rank16)
        for (int m = 0; m < phases; ++m) all += own[m * 64 + k];
    bool ok = true;
    if (blocks > 1) {
        if (k < p.rank16) part[k] = all;
        __syncthreads();
        if (warp < kWarpsEpi && lane < int(blocks)) mbar_arrive_peer(peer_addr(bars + kBarPart * 8, uint32_t(lane)));
        ok = warp_wait_cluster(bars + kBarPart * 8, 0, abort, p.wait_ns);
        all = 0.0f;
        if (k < p.rank16) {
            float of[8];
#pragma unroll
            for (uint32_t m = 0; m < 8; ++m) of[m] = m < blocks ? ld_peer1(peer_addr(part_addr + uint32_t(k) * 4, m)) : 0.0f;
#pragma unroll
            for (int m = 0; m < 8; ++m) all += of[m];
        }
    }
    if (k < 64) v[k] = k < p.rank ? all * (p.scale ? __ldcg(p.scale + j) : 1.0f) : 0.0f;
    __syncthreads();
    ok = ok && lds32(abort) == 0;   // (whoever's wait ran out, its sums are everybody's)
    // its three 16-bit pieces, in the lanes of the one token
    float f[NB][8], most = 0.0f, up = 1.0f, down = 1.0f;
#pragma unroll
    for (int i = 0; i < NB * 8; ++i) {
        f[i / 8][i % 8] = v[i / 8 * 32 + q * 8 + i % 8];
        most = fmaxf(most, fabsf(f[i / 8][i % 8]));
    }
    if (XTYPE == FRX_F16) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        up = power_up(most, down);
    }
    uint32_t bits[3][NB][4];
#pragma unroll
    for (int i = 0; i < NB * 8; ++i) {
        float rest = g == 0 ? f[i / 8][i % 8] * up : 0.0f;
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            const uint32_t piece = take_piece<XTYPE>(rest);
            uint32_t& w = bits[s][i / 8][i % 8 / 2];
            w = i & 1 ? w | piece << 16 : piece;
        }
    }
    uint32_t at = mine;
    int row = row0;
    for (int i0 = warp; i0 < count; i0 += kAhead * kWarps) {
#pragma unroll
        for (int m = 0; m < kAhead; ++m) {
            if (i0 + m * kWarps >= count) continue;
            fetch_wait<kRowsDeep - 1>();
            float d[4] = {};
            uint32_t lo[NB][4], hi[NB][4];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                lds8(at + 2 * n * kSlotBytes, lo[n]);
                lds8(at + (2 * n + 1) * kSlotBytes, hi[n]);
            }
#pragma unroll
            for (int s = 2; s >= 0; --s)   // (the smallest first)
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int h = 0; h < 4; h += 2) mma_16x8x16<XTYPE>(d, lo[n][h], hi[n][h], lo[n][h + 1], hi[n][h + 1], bits[s][n][h], bits[s][n][h + 1]);
            fetch(at);
            at = at + 2 * NB * kSlotBytes == mine + kRowsDeep * 2 * NB * kSlotBytes ? mine : at + 2 * NB * kSlotBytes;
            const uint32_t old[2] = {yv[m][0], yv[m][1]};
            read_y(m);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float add = ok ? d[2 * h] * down : __uint_as_float(0x7fffffffu);   // (NaN: a wait ran out)
                if (q == 0 && row + h * 8 < p.rows) {
                    uint8_t* to = po + h * 8 * size;
                    if (TYPE == FRX_F32)
                        *reinterpret_cast<float*>(to) = add + __uint_as_float(old[h]);
                    else
                        *reinterpret_cast<uint16_t*>(to) = uint16_t(narrow2<TYPE>(add + wide<TYPE>(old[h]), 0.0f));
                }
            }
            po += 16 * kWarps * size;
            row += 16 * kWarps;
        }
    }
    fetch_wait<0>();
}

// SINGLES: most tiles are of one token, of a rank of 17 to 64 (a kernel of its own: in one with the others it took registers from them, 3 to 7 %)
template <int XTYPE, int TYPE, bool SINGLES>
__global__ void __launch_bounds__(kThreads, 2) k_adapter(const Adapters p, const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap a_map,
                                                         const __grid_constant__ CUtensorMap b_map) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t s0 = smem_u32(smem), ring = s0 + kHead, bbuf = ring + uint32_t(p.ring_bytes), bars = s0, abort = s0 + kAbort;
    const int chunks = p.rank16 > 64 ? 2 : 1;   // of 64 of the rank
    const uint32_t bbuf_bytes = uint32_t(chunks) * kPieceB, v_bytes = uint32_t(chunks) * kPieceV, part = bbuf + kBufs * bbuf_bytes;
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
            const int from = __ldcg(p.offsets + r), to = __ldcg(p.offsets + r + 1);
            a = min(max(from, 0), p.T);
            return min(max(to, a), p.T) - a;
        };
        // (of few requests a thread has one: its adapter is read along with its range)
        int a = 0, count = 0, j = 0;
        if (r0 < r1) {
            j = __ldcg(p.which + r0);
            count = range(r0, a);
        }
        long long sum = (count + kTok - 1) / kTok;
        for (int r = r0 + 1; r < r1; ++r) {
            int unused;
            sum += (range(r, unused) + kTok - 1) / kTok;
        }
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
            int t = int(tile - before);   // of the thread's requests
            for (int r = r0; t >= (count + kTok - 1) / kTok && ++r < r1;) {
                t -= (count + kTok - 1) / kTok;
                j = __ldcg(p.which + r);
                count = range(r, a);
            }
            found[0] = a + t * kTok;
            found[1] = min(kTok, count - t * kTok);
            found[2] = j >= p.L ? -1 : j;
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
    const int row_chunks = (p.rows + kRows - 1) / kRows;
    const int depths = (p.n + kDepth - 1) / kDepth, d0 = int(int64_t(depths) * rank / blocks), d1 = int(int64_t(depths) * (rank + 1) / blocks);
    const int turn = int((blockIdx.x / blocks) % unsigned(row_chunks));
    auto chunk = [&](int c) { return c + turn < row_chunks ? c + turn : c + turn - row_chunks; };
    // A stage is the tokens' rows of x, as many as the loads bring, and A_j's: of one token 4 KB instead of 10 at a rank of 16, so that most of its depth is in flight at once.
    const int boxes = (live + p.box - 1) / p.box;
    const uint32_t x_bytes = uint32_t(boxes * p.box) * 128, stage_bytes = x_bytes + uint32_t(p.rank16) * 128, stages = min(uint32_t(kMaxStages), uint32_t(p.ring_bytes) / max(stage_bytes, 1u));
    // The tensor cores add to their sums by cutting off (half a step of 2^-23 each time on average, towards zero): the first product's depth goes into several sums, some 256 of it each as far as
    // tensor memory has room (eight sums up to a rank of 32, four of 64, two of 128: 1,024 each of a depth of 2,048 in one block), which are added up rounded to nearest; of the second product's
    // pieces the smallest come first. 32-bit results of 1,000 tokens, rank 64, y among them, are off by 2.2e-7 in the root mean square (plain products in 32 bits: 1.5e-7).
    const int room = kCols / p.rank16, part_depths = max(4, (d1 - d0 + min(room, 8) - 1) / min(room, 8)), parts = (d1 - d0 + part_depths - 1) / part_depths;
    bool lost = false;

    if (!work) {
        // no adapter: y as it is
        if (live > 0 && p.out != p.y) copy_rows<TYPE == FRX_F32 ? 4 : 2>(p.y, p.ldy, p.out, p.ldo, t0, live, p.rows, int(rank) * (kThreads / 32) + warp, int(blocks) * (kThreads / 32));
    } else if (live == 1 && (SINGLES || p.rank16 == 16)) {
        // (the room of the stages and of B_j's rows: the lanes' places, the warps' sums, v)
        float *own = reinterpret_cast<float*>(smem + kHead + kSlots * kSlotBytes), *v = own + 10 * 64, *sums = reinterpret_cast<float*>(smem + (blocks > 1 ? part : smem_u32(own)) - s0);
        const int c0 = d0 * kDepth, c1 = min(p.n, d1 * kDepth);
        if constexpr (!SINGLES)
            one_token<XTYPE, TYPE>(p, bars, abort, sums, part, v, t0, j, c0, c1, rank, blocks);
        else if (p.rank16 == 32)
            one_token_of_rank<XTYPE, TYPE, 1>(p, bars, abort, ring, own, sums, part, v, t0, j, c0, c1, rank, blocks);
        else
            one_token_of_rank<XTYPE, TYPE, 2>(p, bars, abort, ring, own, sums, part, v, t0, j, c0, c1, rank, blocks);
    } else if (warp == kWarpLoad) {
        // ---------------- loads: the first product's stages, and this block's rows of B_j as soon as there is room
        uint32_t st = 0, phase = 1, buf = 0, bphase = 1;
        int c = int(rank);
        bool ok = true;
        auto rows_of_b = [&]() {
            if (!(ok = warp_wait(bars + (kBarBFree + buf) * 8, bphase, abort, p.wait_ns))) return;
            const uint32_t full = bars + (kBarBFull + buf) * 8, to = bbuf + buf * bbuf_bytes;
            if (lane == 0) {
                mbar_expect_tx(full, bbuf_bytes);
                for (int i = 0; i < chunks; ++i) {
                    if (p.whole) {
                        constexpr int kGroup = TYPE == FRX_F32 ? 8 : 16;
                        for (int m = 0; m < kRows; m += 4 * kGroup) tma_5d(to + i * kPieceB + m * 128, &b_map, i * 64, 0, (chunk(c) * kRows + m) / kGroup, 0, j, full);
                    } else {
                        tma_3d(to + i * kPieceB, &b_map, i * 64, chunk(c) * kRows, j, full);
                    }
                }
            }
            __syncwarp();
            c += int(blocks);
            if (++buf == kBufs) buf = 0, bphase ^= 1u;
        };
        for (int s = d0; s < d1 && ok; ++s) {
            if (!(ok = warp_wait(bars + (kBarFree + st) * 8, phase, abort, p.wait_ns))) break;
            const uint32_t full = bars + (kBarFull + st) * 8, x = ring + st * stage_bytes, a = x + x_bytes;
            if (lane == 0) {
                mbar_expect_tx(full, stage_bytes);
                for (int i = 0; i < boxes; ++i) tma_2d(x + i * p.box * 128, &x_map, s * kDepth, t0 + i * p.box, full);
                tma_3d(a, &a_map, s * kDepth, 0, j, full);
            }
            __syncwarp();
            if (++st == stages) st = 0, phase ^= 1u;
            if (s - d0 == int(stages) - 1)
                for (int i = 0; i < kBufs && c < row_chunks && ok; ++i) rows_of_b();
        }
        while (c < row_chunks && ok) rows_of_b();
    } else if (warp == kWarpMma) {
        uint32_t st = 0, phase = 0;
        bool ok = true;
        const uint32_t idesc = p.idesc | uint32_t(p.rank16 >> 3) << 17;
        for (int s = d0; s < d1; ++s) {
            if (!(ok = warp_wait(bars + (kBarFull + st) * 8, phase, abort, p.wait_ns))) break;
            const uint32_t x = ring + st * stage_bytes;   // (lanes without a token are whatever lies behind)
            const int depth = min(kDepth, p.n - s * kDepth), in_part = (s - d0) % part_depths;
            const uint32_t acc = tmem + uint32_t((s - d0) / part_depths * p.rank16);
            if (elect_one()) {
                const uint64_t da = umma_desc_sw128(x), db = umma_desc_sw128(x + x_bytes);
#pragma unroll
                for (int k = 0; k < kDepth / 16; ++k) {
                    if (k * 16 >= depth) break;
                    umma_f16(acc, da + k * 2, db + k * 2, idesc, in_part + k > 0);
                }
                umma_commit(bars + (kBarFree + st) * 8);
                if (s + 1 == d1) umma_commit(bars + kBarV * 8);
            }
            __syncwarp();
            if (++st == stages) st = 0, phase ^= 1u;
        }
        ok = ok && warp_wait(bars + kBarVIn * 8, 0, abort, p.wait_ns);
        uint32_t buf = 0, bphase = 0, set = 0, dphase = 1;
        const uint32_t id = p.idesc | uint32_t(kRows >> 3) << 17;
        for (int c = int(rank); c < row_chunks && ok; c += int(blocks)) {
            if (!(ok = warp_wait(bars + (kBarBFull + buf) * 8, bphase, abort, p.wait_ns))) break;
            if (!(ok = warp_wait(bars + (kBarDFree + set) * 8, dphase, abort, p.wait_ns))) break;
            tc_fence_after_sync();
            if (elect_one()) {
                for (int q = 2; q >= 0; --q)
                    for (int k = 0; k < p.rank16; k += 16) {
                        const uint32_t in = uint32_t(k & 63) * 2;
                        umma_f16(tmem + set * kRows, umma_desc_sw128(ring + q * v_bytes + uint32_t(k >> 6) * kPieceV) + (in >> 4),
                                 umma_desc_sw128(bbuf + buf * bbuf_bytes + uint32_t(k >> 6) * kPieceB) + (in >> 4), id, q < 2 || k > 0);
                    }
                umma_commit(bars + (kBarBFree + buf) * 8);
                umma_commit(bars + (kBarDFull + set) * 8);
            }
            __syncwarp();
            set ^= 1u;
            if (set == 0) dphase ^= 1u;
            if (++buf == kBufs) buf = 0, bphase ^= 1u;
        }
    } else {
        const int quarter = warp & 3, side = warp >> 2, token = quarter * 32 + lane;
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        // In the second product a warp has 16 of the tokens (of which there are two of 64 lanes) and 64 of the 128 columns, a lane two of these tokens, eight apart, and 16 columns
        // of each; where y and out do not allow that, a lane is a token and a warp has 32 of them and 32 columns.
        constexpr int size = TYPE == FRX_F32 ? 4 : 2, kAhead = TYPE == FRX_F32 ? 1 : 2, kPer = 32 / size, kAccesses = 16 / kPer;   // values of an access, accesses of 16 values
        const int t = p.whole ? (quarter & 1) * 32 + side * 16 + lane / 4 : (quarter & 1) * 32 + lane;
        const int col = p.whole ? (quarter >> 1) * 64 + (lane & 3) * kPer : (quarter >> 1) * 64 + side * 32;
        const uint8_t* y = static_cast<const uint8_t*>(p.y) + ((t0 + t) * p.ldy + col) * size;
        uint8_t* out = static_cast<uint8_t*>(p.out) + ((t0 + t) * p.ldo + col) * size;
        uint32_t old[kAhead][2][8 * kAccesses] = {};
        auto read_ahead = [&](uint32_t (&w)[2][8 * kAccesses], int c) {
            if (c >= row_chunks || !p.whole) return;
            const int first = chunk(c) * kRows;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int q = 0; q < kAccesses; ++q) load_if(w[r] + 8 * q, y + (8 * r * p.ldy + first + 4 * q * kPer) * size, t + 8 * r < live && first + col + 4 * q * kPer < p.rows);
        };
#pragma unroll
        for (int d = 0; d < kAhead; ++d) read_ahead(old[d], int(rank) + d * int(blocks));
        // ---------------- v: a lane is a token, a warp has every second eight of the rank (every fourth of a sum over blocks, which any warp can read)
        const int k0 = side * 8;
        const bool empty = d0 == d1;   // no part of the depth here
        if (!empty) {
            lost = !warp_wait(bars + kBarV * 8, 0, abort, p.wait_ns);
            tc_fence_after_sync();
        }
        const uint32_t mine = part + uint32_t(token) * 4;   // token after token: a warp's read of another block's shared memory is 128 bytes (as 16 bytes a lane it was 32 requests: 3 us for eight of the rank)
        auto sum_parts = [&](int k, float (&v)[8]) {
            tmem_ld8(tmem + lanes + k, v);
            for (int g = 1; g < parts; ++g) {
                float more[8];
                tmem_ld8(tmem + lanes + g * p.rank16 + k, more);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += more[i];
            }
        };
        if (blocks > 1) {
            float most = 0.0f;
            for (int k = k0; k < p.rank16; k += 16) {
                float v[8];
                if (empty || lost) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = lost ? __uint_as_float(0x7fffffffu) : 0.0f;
                } else {
                    sum_parts(k, v);
                }
                if (XTYPE == FRX_F16) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
                }
                if (token < live) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + uint32_t(k + i) * kTok * 4), "f"(v[i]) : "memory");
                }
            }
            if (XTYPE == FRX_F16 && token < kTok) tok_max[side * kTok + token] = most;
            __syncwarp();
            if (lane < int(blocks)) mbar_arrive_peer(peer_addr(bars + kBarPart * 8, uint32_t(lane)));
            lost = !warp_wait_cluster(bars + kBarPart * 8, 0, abort, p.wait_ns) || lost;
        }
        const int taken = blocks > 1 ? (quarter & 1) * 32 + lane : token, first_k = blocks > 1 ? k0 + (quarter >> 1) * 16 : k0, step_k = blocks > 1 ? 32 : 16;   // the lane's token, and its warp's part of the rank
        auto take8 = [&](int k, float (&v)[8]) {
            if (blocks > 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
                if (taken < live)
                    for (uint32_t b = 0; b < blocks; b += 4) {   // (2, 4 or 8 blocks) the loads of four at once: each takes half a microsecond
                        float of[4][8];
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            const uint32_t at = peer_addr(part + uint32_t(k * kTok + taken) * 4, min(b + i, blocks - 1));
#pragma unroll
                            for (int c = 0; c < 8; ++c) of[i][c] = b + i < blocks ? ld_peer1(at + c * kTok * 4) : 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int c = 0; c < 8; ++c) v[c] += of[i][c];
                    }
            } else {
                sum_parts(k, v);
            }
        };
        const float scale = p.scale ? __ldcg(p.scale + j) : 1.0f;
        float up = 1.0f;
        if (XTYPE == FRX_F16) {
            // the token's largest magnitude (or, of a sum over blocks, that of the parts) to [2^14, 2^15): pieces of float16 then hold every bit of the others that counts
            float most = 0.0f;
            if (blocks > 1) {
                if (taken < live && !lost)
                    for (uint32_t b = 0; b < blocks; ++b)
                        most += fmaxf(ld_peer1(peer_addr(s0 + kTokMax + taken * 4, b)), ld_peer1(peer_addr(s0 + kTokMax + (kTok + taken) * 4, b)));
            } else {
                for (int k = first_k; k < p.rank16 && !lost; k += step_k) {
                    float v[8];
                    take8(k, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
                }
                if (token < kTok) tok_max[side * kTok + token] = most;
                named_bar_sync(1, 32 * kWarpsEpi);
                if (token < kTok) most = fmaxf(tok_max[token], tok_max[kTok + token]);
            }
            most *= fabsf(scale);
            float down;
            up = power_up(most, down);
            if (side == 0 && token < kTok) tok_scale[taken] = down;
        }
        // Where a wait ran out nothing is written, since the first product may still use its stages, and the arrival is left out: other warps, whose outputs need this warp's part of v, may
        // have been in time. There is no second product then, and all waits for its sums run out.
        for (int k = first_k; k < p.rank16 && !lost; k += step_k) {
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
            const uint32_t at = ring + uint32_t(k >> 6) * kPieceV + uint32_t(taken) * 128 + uint32_t(((k & 63) >> 3) ^ (taken & 7)) * 16;   // (the 128-byte swizzle)
#pragma unroll
            for (int q = 0; q < 6 && taken < kTok; ++q)
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + (q % 3) * v_bytes + (q / 3) * kTok * 128), "r"(bits[q % 3][0]), "r"(bits[q % 3][1]), "r"(bits[q % 3][2]),
                             "r"(bits[q % 3][3])
                             : "memory");
        }
        fence_async_smem();       // generic-proxy writes: visible to the tensor core
        tc_fence_before_sync();   // behind the loads of the first product's sums, whose columns the second product's take
        __syncwarp();
        if (lane == 0 && !lost) mbar_arrive(bars + kBarVIn * 8);
        float down = 1.0f, down8 = 1.0f;   // of the lane's tokens
        if (XTYPE == FRX_F16) {
            named_bar_sync(1, 32 * kWarpsEpi);
            down = tok_scale[t];
            down8 = tok_scale[min(t + 8, kTok - 1)];
        }
        // ---------------- the second product's sums
        uint32_t set = 0, phase = 0;
        for (int c0 = int(rank); c0 < row_chunks; c0 += kAhead * int(blocks)) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                const int c = c0 + d * int(blocks);
                if (c >= row_chunks) continue;
                const int first = chunk(c) * kRows;
                lost = lost || !warp_wait(bars + (kBarDFull + set) * 8, phase, abort, p.wait_ns);
                tc_fence_after_sync();
                const uint32_t sums = tmem + lanes + set * kRows;
                if (p.whole) {
                    uint32_t v[8][4];
                    if (lost) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i / 4][i % 4] = 0x7fffffffu;
                    } else {
                        tmem_ld_16x256(sums + (uint32_t(side * 16) << 16) + (quarter >> 1) * 64, v);
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int q = 0; q < kAccesses; ++q) {
                            float f[kPer];
#pragma unroll
                            for (int i = 0; i < kPer; ++i) f[i] = __uint_as_float(v[q * kPer / 2 + i / 2][2 * r + i % 2]) * (r ? down8 : down);   // (exact; by 1 for bfloat16)
                            if (t + 8 * r < live && first + col + 4 * q * kPer < p.rows)
                                add_and_store<TYPE>(f, old[d][r] + 8 * q, out + (8 * r * p.ldo + first + 4 * q * kPer) * size);
                        }
                    read_ahead(old[d], c + kAhead * int(blocks));
                } else {
                    for (int h = 0; h < 32; h += 16) {
                        uint32_t v[2][8];
                        float f[16];
                        if (lost) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = 0x7fffffffu;
                        } else {
                            tmem_ld16(sums + col + h, v);
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(v[i / 8][i % 8]) * down;
                        if (t < live) add_and_store_each<TYPE>(f, y + (first + h) * size, out + (first + h) * size, p.rows - first - col - h);
                    }
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

// b for the second product: 128 rows a load, or, with a group, four groups of so many rows, in the order in which a thread finds its columns side by side
int second_map(CUtensorMap& map, const void* b, int64_t ldb, int64_t stride_b, int dtype, int L, int rows, int rank, int group) {
    if (!group) return matrices_map(map, b, ldb, stride_b, dtype, L, rows, rank, kRows);
    const cuuint64_t dims[5] = {cuuint64_t(rank), 2, cuuint64_t(rows / group), cuuint64_t(group / 2), cuuint64_t(L)};
    const cuuint64_t strides[4] = {cuuint64_t(ldb) * 2, cuuint64_t(ldb) * 2 * group, cuuint64_t(ldb) * 4, cuuint64_t(stride_b) * 2};
    const cuuint32_t boxes[5] = {64, 2, 4, cuuint32_t(group / 2), 1};
    return encode_16(map, dtype, 5, b, dims, strides, boxes);
}

template <int XTYPE, int TYPE, bool SINGLES>
int launch_as(Adapters& p, const CUtensorMap& x_map, const CUtensorMap& a_map, const CUtensorMap& b_map, cudaStream_t stream) {
    int rc = allow_smem<k_adapter<XTYPE, TYPE, SINGLES>>();
    if (rc != FRX_OK) return rc;
    const int chunks = p.rank16 > 64 ? 2 : 1;
    const int64_t requests = std::min(p.R, p.T), tiles = (p.T - requests) / kTok + requests;   // of any requests that do not overlap
    // As many blocks a tile as run at the same time (two an SM, one where the rank is more than 64), and the stages have the room that is left.
    unsigned blocks = 8;
    while (blocks > 1 && tiles * blocks > int64_t(sm_count()) * (chunks == 1 ? 2 : 1)) blocks /= 2;
    if (tiles * blocks > 0x7fff0000) return fail(FRX_ERR_SHAPE, "adapters: %lld tiles", (long long)tiles);
    const int rest = kHead + kBufs * chunks * kPieceB + (blocks > 1 ? kTok * p.rank16 * 4 : 0);
    static_assert(kHead + kBufs * kPieceB + kTok * 64 * 4 + std::max(kMinStages * (kTok + 64) * 128, 3 * kPieceV) <= kSmemTwo, "two blocks an SM up to a rank of 64");
    static_assert(kSlots * kSlotBytes + 11 * 64 * 4 <= (kSmemTwo - kHead - kBufs * kPieceB - kTok * 64 * 4) / 1024 * 1024 + kBufs * kPieceB, "the room of a tile of one token");
    static_assert(kHead + kBufs * 2 * kPieceB + kTok * 128 * 4 + std::max(kMinStages * (kTok + 128) * 128, 3 * 2 * kPieceV) <= int(kSmemMost), "the largest rank");
    p.ring_bytes = std::max(((chunks == 1 ? kSmemTwo : int(kSmemMost)) - rest) / 1024 * 1024, 3 * chunks * kPieceV);
    const size_t smem = size_t(rest + p.ring_bytes);   // (about half of an SM's, or all of it: a third block would wait for tensor memory)
    p.wait_ns = wait_limit_ns();
    FRX_LAUNCH(kKAdapter, stream, launch_pdl_cluster(k_adapter<XTYPE, TYPE, SINGLES>, dim3(unsigned(tiles) * blocks), dim3(kThreads), smem, stream, blocks, p, x_map, a_map, b_map));
    FRX_CUDA(cudaGetLastError());
    return FRX_OK;
}
template <int XTYPE, int TYPE>
int launch_typed(Adapters& p, const CUtensorMap& x_map, const CUtensorMap& a_map, const CUtensorMap& b_map, cudaStream_t stream) {
    // where most requests are of one token (among large tiles their many loads take longer: 1,000 tokens of 41 users 27 -> 29 us)
    return p.rank16 > 16 && p.rank16 <= 64 && p.T < 2 * int64_t(p.R) ? launch_as<XTYPE, TYPE, true>(p, x_map, a_map, b_map, stream) : launch_as<XTYPE, TYPE, false>(p, x_map, a_map, b_map, stream);
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
    if (out == y && ldo != ldy && T > 1) return fail(FRX_ERR_ARG, "%s: out is y, with rows %lld instead of %lld elements apart", who, (long long)ldo, (long long)ldy);
    int rc;
    if ((rc = operand(who, "x", x, ldx, T, n)) != FRX_OK || (rc = operand(who, "a", a, lda, rank, n)) != FRX_OK || (rc = operand(who, "b", b, ldb, rows, rank)) != FRX_OK ||
        (rc = operand(who, "a (its matrices)", a, stride_a, L, (rank - 1) * lda + n)) != FRX_OK ||
        (rc = operand(who, "b (its matrices)", b, stride_b, L, (rows - 1) * ldb + rank)) != FRX_OK)
        return rc;
    Adapters p{};
    p.offsets = offsets;
    p.which = which;
    p.scale = scale;
    p.x = x;
    p.a = a;
    p.b = b;
    p.ldx = ldx;
    p.lda = lda;
    p.stride_a = stride_a;
    p.ldb = ldb;
    p.stride_b = stride_b;
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
    const int64_t size = dtype_size(y_dtype);
    p.whole = rows * size % 32 == 0 && aligned(y, 32) && aligned(out, 32) && ldy * size % 32 == 0 && ldo * size % 32 == 0;
    CUtensorMap xm, am, bm;
    if ((rc = rows_map(xm, x, ldx, dtype, T, n, p.box)) != FRX_OK || (rc = matrices_map(am, a, lda, stride_a, dtype, L, rank, n, p.rank16)) != FRX_OK ||
        (rc = second_map(bm, b, ldb, stride_b, dtype, L, rows, rank, p.whole ? 32 / dtype_size(y_dtype) : 0)) != FRX_OK)
        return rc;
    return dtype == FRX_BF16 ? launch<FRX_BF16>(p, y_dtype, xm, am, bm, stream) : launch<FRX_F16>(p, y_dtype, xm, am, bm, stream);
}
