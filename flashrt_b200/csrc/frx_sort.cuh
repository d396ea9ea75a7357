// Host side of the sort by expert, for the entry points that use it.
#pragma once

#include "frx_common.cuh"

namespace frx {
// Bytes that sort_slots needs beside its outputs (chunk counts), for S slots and E experts.
size_t sort_scratch_bytes(long long S, int E);
// offsets [E + 1], slot_of [S] (may be null), row_of [S] of the S ids; status: the four status words of a workspace.
int sort_slots(const int32_t* ids, int S, int E, int32_t* offsets, int32_t* slot_of, int32_t* row_of, int* status, int* scratch, cudaStream_t stream);
// out[t] = sum over k of wts[t][k] * ys[row_of[t][k]] (weights 1 where wts is null), in_dtype rows to out_dtype rows.
// early: row_of was complete before the kernel in front in the stream began.
int rows_back(const void* ys, int64_t ldy, int in_dtype, const float* wts, const int32_t* row_of, int64_t rows, int T, int K, int n, void* out, int64_t ldo,
              int out_dtype, bool early, cudaStream_t stream);
}  // namespace frx
