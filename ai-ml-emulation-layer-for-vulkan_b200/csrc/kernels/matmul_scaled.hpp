// The scaled int8 product (matmul_scaled.cu) as its kernels take it.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mlel {

struct ScaledProblem {
    const int8_t *a, *b;
    const float *aScales, *bScales, *biases; // biases may be null
    char *out;
    int64_t aStride, bStride, outStride; // bytes between rows
    int32_t M, N, K;
};

// Both want rows of a and b on 16-byte boundaries.
// matmul_scaled_pair.cu: false where it does not take the problem
bool matmulScaledOnPairs(const ScaledProblem &p, int32_t dtype, cudaStream_t s, int *rc);
// matmul_scaled_tiles.cu
int matmulScaledOnTiles(const ScaledProblem &p, int32_t dtype, cudaStream_t s);
int scaledPairErrorWord();
int scaledTilesErrorWord();

} // namespace mlel
