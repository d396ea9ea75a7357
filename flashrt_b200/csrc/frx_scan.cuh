// What the two groupings by expert share (frx_group.cuh, frx_sort.cu). Include inside namespace frx { namespace { ... } }.
#pragma once

constexpr int kCookie = 0x46525831;   // marks a workspace whose status words have been initialised
constexpr int kChunkSlots = 1024;     // slots of a chunk, which one block counts and places

// Sum of v over the threads in front of this one, and over all of them (`total`), for a block of 1024; tot: scratch.
__device__ __forceinline__ int block_scan(int v, int* tot, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    __syncthreads();   // (tot may still be read from the scan before)
    if (lane == 31) tot[warp] = inc;
    __syncthreads();
    int w = tot[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    return inc - v + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0);
}
