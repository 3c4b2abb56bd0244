// The scaled int8 product (matmul_scaled.cu) as its kernels take it.
#pragma once

#include <cstdint>

namespace mlel {

struct ScaledProblem {
    const int8_t *a, *b;
    const float *aScales, *bScales, *biases; // biases may be null
    char *out;
    int64_t aStride, bStride, outStride; // bytes between rows
    int32_t M, N, K;
};

} // namespace mlel
