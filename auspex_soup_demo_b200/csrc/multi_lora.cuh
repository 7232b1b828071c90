// The base product of a projection with several adapters (defined with the tcgen05
// GEMM's launchers in ce_linear.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace soup {

// out [m, n] (bf16) = a [m, k] op(b) + a2 [m, r] op(b2) + bias, where the second
// product takes, for a 256-row tile of a, the 64-wide blocks of r that the tile's word
// of k2_mask names (device memory, r <= 4096; the blocks it names must be written for
// all rows of the tile). op(b) = b^T for b [n, k], or b for b [k, n] (b_mn), b2 alike.
// No scratch is shared between launches.
int gemm_bf16_masked_k2(const void* a, int64_t lda, const void* b, int64_t ldb, bool b_mn, const void* a2,
                        int64_t lda2, const void* b2, int64_t ldb2, int64_t r, const uint64_t* k2_mask,
                        const void* bias, void* out, int64_t ldo, int64_t m, int64_t n, int64_t k,
                        cudaStream_t stream);

}  // namespace soup
