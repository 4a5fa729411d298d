// Row statistics of hidden @ weight^T for the losses over the output projection.
#pragma once

#include "common.cuh"

namespace mt {

// Splits of the vocabulary that logit_stats works with for N rows.
int logit_stats_splits(int64_t N, int64_t V);

// Per row and split s: part_m[row * splits + s] = max of z * zscale over the
// split's vocabulary entries (-inf if it has none) and part_s[...] = the sum of
// 2^(z * zscale - part_m), z = the row's logits (tcgen05 product, logits only in
// TMEM).  hidden [N, K], weight [V, K] bf16 or fp16, contiguous, 16-byte
// aligned, K % 8 == 0, N > 0 (checked by the caller).
int logit_stats(const void* hidden, const void* weight, int dtype, int64_t N, int64_t V, int64_t K, float zscale,
                int splits, float* part_m, float* part_s, uint32_t* status, cudaStream_t stream);

}  // namespace mt
