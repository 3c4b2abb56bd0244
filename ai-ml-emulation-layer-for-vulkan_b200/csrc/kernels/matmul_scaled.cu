// Product in 8-bit integers with a scale for each token and channel:
//   out[m][n] = (sum_k a[m][k] b[n][k]) * aScale[m] * bScale[n] + bias[n]
// with the sum exact in 32-bit integers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../graph_pipeline.hpp"
#include "launch_overlapped.cuh"
#include "matmul_scaled.hpp"
#include "serving.hpp"
#include "serving_device.cuh"

namespace mlel {
namespace {

// Rows at any address: tiles of 64 x 64 outputs, both operands' K slices of 64 bytes put into shared memory byte by byte,
// four-way dot products.
constexpr int kTile = 64, kSlice = 16; // outputs a side; words of K per slice

__device__ __forceinline__ uint32_t wordAt(const int8_t *row, int k, int length) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w |= k + j < length ? uint32_t(uint8_t(row[k + j])) << (8 * j) : 0u;
    }
    return w;
}

template <class T>
__global__ void __launch_bounds__(256) matmulScaledAnyRows(const ScaledProblem p) {
    __shared__ uint32_t tileA[kTile][kSlice + 1], tileB[kTile][kSlice + 1];
    dependencySync();
    const int m0 = int(blockIdx.y) * kTile, n0 = int(blockIdx.x) * kTile;
    const int tx = int(threadIdx.x) & 15, ty = int(threadIdx.x) >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 4 * kSlice) {
        for (int i = int(threadIdx.x); i < kTile * kSlice; i += 256) {
            const int r = i / kSlice, w = i % kSlice, k = k0 + 4 * w;
            tileA[r][w] = m0 + r < p.M ? wordAt(p.a + int64_t(m0 + r) * p.aStride, k, p.K) : 0u;
            tileB[r][w] = n0 + r < p.N ? wordAt(p.b + int64_t(n0 + r) * p.bStride, k, p.K) : 0u;
        }
        __syncthreads();
#pragma unroll 4
        for (int w = 0; w < kSlice; ++w) {
            uint32_t x[4], y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = tileA[ty + 16 * j][w], y[j] = tileB[tx + 16 * j][w];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] = __dp4a(int(x[i]), int(y[j]), acc[i][j]);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty + 16 * i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx + 16 * j;
            if (m < p.M && n < p.N) {
                const float y = float(acc[i][j]) * p.aScales[m] * p.bScales[n] + (p.biases != nullptr ? p.biases[n] : 0.f);
                *reinterpret_cast<T *>(p.out + int64_t(m) * p.outStride + int64_t(n) * int64_t(sizeof(T))) = fromFloat<T>(y);
            }
        }
    }
}

template <class T> cudaError_t launchAnyRows(const ScaledProblem &p, cudaStream_t s) {
    return launchOverlapped(matmulScaledAnyRows<T>, dim3(unsigned((p.N + kTile - 1) / kTile), unsigned((p.M + kTile - 1) / kTile)), 256,
                            0, s, p);
}

// The operands of a product, checked; where there is work, on the current device.
ScaledProblem scaledProblemOf(const std::string &call, const mlel_tensor *a, const mlel_tensor *aScales, const mlel_tensor *b,
                              const mlel_tensor *bScales, const mlel_tensor *biases, const mlel_tensor *output) {
    const Operand oa = operandOf(call, "a", a, 2), sa = operandOf(call, "a_scales", aScales, 1), ob = operandOf(call, "b", b, 2),
                  sb = operandOf(call, "b_scales", bScales, 1), out = writtenOperandOf(call, "output", output, 2);
    Operand bias{};
    wantType(call, "a", oa, MLEL_I8, "int8");
    wantType(call, "b", ob, MLEL_I8, "int8");
    wantType(call, "a_scales", sa, MLEL_F32, "f32");
    wantType(call, "b_scales", sb, MLEL_F32, "f32");
    if (biases != nullptr) {
        bias = operandOf(call, "biases", biases, 1);
        wantType(call, "biases", bias, MLEL_F32, "f32");
    }
    if (!isFloat(out.dtype)) {
        throw UnsupportedError(call + ": output has to be f32, f16 or bf16");
    }
    const int64_t M = oa.dims[0], K = oa.dims[1], N = ob.dims[0];
    if (ob.dims[1] != K || sa.dims[0] != M || sb.dims[0] != N || out.dims[0] != M || out.dims[1] != N ||
        (biases != nullptr && bias.dims[0] != N)) {
        refuse(call, "the shapes of the operands do not fit together");
    }
    if (K < 1 || K > 131071) {
        refuse(call, "K has to be 1 to 131071: longer sums of products do not fit 32-bit integers");
    }
    if (M > 65535 * int64_t(kTile)) {
        refuse(call, "more than 4194240 tokens");
    }
    if (M > 0 && N > 0) {
        wantCurrentDevice(call, "output", out.ptr);
    }
    ScaledProblem p{};
    p.a = reinterpret_cast<const int8_t *>(oa.ptr), p.b = reinterpret_cast<const int8_t *>(ob.ptr);
    p.aScales = reinterpret_cast<const float *>(sa.ptr), p.bScales = reinterpret_cast<const float *>(sb.ptr);
    p.biases = reinterpret_cast<const float *>(bias.ptr), p.out = out.ptr;
    p.aStride = oa.strides[0], p.bStride = ob.strides[0], p.outStride = out.strides[0];
    p.M = int32_t(M), p.N = int32_t(N), p.K = int32_t(K);
    // strides of an axis that is not walked: any would do
    if (M == 1) {
        p.aStride = (K + 15) / 16 * 16, p.outStride = (N * elemSize(out.dtype) + 15) / 16 * 16;
    }
    if (N == 1) {
        p.bStride = (K + 15) / 16 * 16;
    }
    return p;
}

// Tensor maps describe rows on 16-byte boundaries that do not overlap; others go the way of any rows.
int launchScaled(const std::string &call, const ScaledProblem &p, int32_t dtype, cudaStream_t s) {
    if (p.aStride >= p.K && p.bStride >= p.K && aligned(p.a, 16) && p.aStride % 16 == 0 && aligned(p.b, 16) && p.bStride % 16 == 0) {
        int rc = MLEL_SUCCESS;
        return matmulScaledOnPairs(p, dtype, s, &rc) ? rc : matmulScaledOnTiles(p, dtype, s);
    }
    return launchStatus(call.c_str(), dtype == MLEL_F32   ? launchAnyRows<float>(p, s)
                                      : dtype == MLEL_F16 ? launchAnyRows<__half>(p, s)
                                                          : launchAnyRows<__nv_bfloat16>(p, s));
}

} // namespace

int matmulScaled(const mlel_tensor *a, const mlel_tensor *aScales, const mlel_tensor *b, const mlel_tensor *bScales,
                 const mlel_tensor *biases, const mlel_tensor *output, cudaStream_t s) {
    const std::string call = "mlel_cuda_matmul_scaled";
    const ScaledProblem p = scaledProblemOf(call, a, aScales, b, bScales, biases, output);
    return p.M == 0 || p.N == 0 ? int(MLEL_SUCCESS) : launchScaled(call, p, output->desc.dtype, s);
}

int quantizedLinear(const mlel_tensor *input, const mlel_tensor *b, const mlel_tensor *bScales, const mlel_tensor *biases,
                    const mlel_tensor *output, void *workspace, uint64_t workspaceBytes, cudaStream_t s) {
    const std::string call = "mlel_cuda_quantized_linear";
    const Operand x = operandOf(call, "input", input, 2);
    const int64_t M = x.dims[0], K = x.dims[1], padded = (K + 15) / 16 * 16;
    if (M > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspaceBytes < uint64_t(M * padded + 4 * M))) {
        refuse(call, "the workspace is null, off a 16-byte boundary or smaller than the quantised rows and their scales");
    }
    mlel_tensor q{}, scales{};
    q.data = workspace, scales.data = M > 0 ? static_cast<char *>(workspace) + M * padded : nullptr;
    q.desc.dtype = MLEL_I8, q.desc.rank = 2;
    q.desc.dims[0] = M, q.desc.dims[1] = K, q.desc.strides[0] = padded, q.desc.strides[1] = 1;
    scales.desc.dtype = MLEL_F32, scales.desc.rank = 1, scales.desc.dims[0] = M;
    // the product's operands are in order before anything is enqueued
    const ScaledProblem p = scaledProblemOf(call, &q, &scales, b, bScales, biases, output);
    const int rc = quantizeRows(input, &q, &scales, s);
    return rc != MLEL_SUCCESS || p.M == 0 || p.N == 0 ? rc : launchScaled(call, p, output->desc.dtype, s);
}

} // namespace mlel
