// Attention over a paged int8 cache with a scale for each page and head.
//
//   o = sum_j softmax(s)_j v_j,  s_j = scale * q . k_j, capped by softcap * tanh(s_j / softcap), over the tokens that the masks leave
//
// One warp per token and query head, one pass over the keys with the running maximum and sum.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "launch_overlapped.cuh"
#include "paged_cache.cuh"
#include "serving_device.cuh"

namespace mlel {
namespace {

struct AttendParams {
    PagedCache cache;
    PagedBatch batch;
    const char *queries;
    char *out;
    int64_t queryStride[2], outStride[2]; // bytes: token, head
    float scale, softcap;
    int32_t causal, window, queryHeads, group;
};

template <class T>
__global__ void __launch_bounds__(256) pagedAttentionSimple(const AttendParams p) {
    dependencySync();
    const int index = int(blockIdx.x), lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
    const Sequence q = sequenceOf(p.batch, index);
    if (!q.sound) {
        if (threadIdx.x == 0 && blockIdx.y == 0) {
            atomicCAS(&g_pagedError, 0, kBadSequence);
        }
        return;
    }
    const int D = p.cache.headDim, page = p.cache.page;
    for (int64_t item = int64_t(blockIdx.y) * 8 + warp; item < int64_t(q.fresh) * p.queryHeads; item += int64_t(gridDim.y) * 8) {
        const int token = int(item / p.queryHeads), head = int(item % p.queryHeads), position = q.length - q.fresh + token;
        const T *query = reinterpret_cast<const T *>(p.queries + int64_t(q.first + token) * p.queryStride[0] + head * p.queryStride[1]);
        float x[8], o[8] = {}, most = -INFINITY, sum = 0.f;
        for (int j = 0; j < 8; ++j) {
            x[j] = lane + 32 * j < D ? toFloat(query[lane + 32 * j]) : 0.f;
        }
        const int end = p.causal ? position + 1 : q.length, begin = p.window > 0 ? max(0, position - p.window + 1) : 0;
        for (int key = begin; key < end; ++key) {
            const int slot = p.batch.table[index * p.batch.tableStride + key / page];
            if (slot < 0 || slot >= p.cache.pages) {
                atomicCAS(&g_pagedError, 0, kBadPage);
                continue;
            }
            const int64_t row = int64_t(slot) * p.cache.heads + head / p.group;
            const int8_t *k = p.cache.keys + (row * page + key % page) * D, *v = p.cache.values + (row * page + key % page) * D;
            float dot = 0.f;
            for (int j = 0; j < 8 && lane + 32 * j < D; ++j) {
                dot += x[j] * float(k[lane + 32 * j]);
            }
            for (int step = 16; step > 0; step >>= 1) {
                dot += __shfl_xor_sync(0xffffffffu, dot, step);
            }
            float score = dot * p.cache.keyScales[row] * p.scale;
            if (p.softcap > 0.f) {
                score = p.softcap * tanhf(score / p.softcap);
            }
            const float top = fmaxf(most, score), keep = most == -INFINITY ? 0.f : expf(most - top),
                        weight = score == -INFINITY ? 0.f : expf(score - top);
            most = top;
            sum = sum * keep + weight;
            const float w = weight * p.cache.valueScales[row];
            for (int j = 0; j < 8 && lane + 32 * j < D; ++j) {
                o[j] = o[j] * keep + w * float(v[lane + 32 * j]);
            }
        }
        T *out = reinterpret_cast<T *>(p.out + int64_t(q.first + token) * p.outStride[0] + head * p.outStride[1]);
        for (int j = 0; j < 8 && lane + 32 * j < D; ++j) {
            out[lane + 32 * j] = fromFloat<T>(sum == 0.f ? 0.f : o[j] / sum);
        }
    }
}

AttendParams paramsOf(const std::string &call, const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *queries) {
    AttendParams p{};
    p.cache = cacheOf(call, cache, false);
    const Operand q = operandOf(call, "queries", queries, 3);
    if (q.dtype != MLEL_F16 && q.dtype != MLEL_BF16) {
        throw UnsupportedError(call + ": queries have to be f16 or bf16");
    }
    if (q.dims[2] != p.cache.headDim || q.dims[1] < 1 || q.dims[1] % p.cache.heads != 0) {
        refuse(call, "queries have to have the cache's head_dim and a multiple of its heads");
    }
    p.batch = batchOf(call, batch, p.cache, q.dims[0]);
    p.queries = q.ptr, p.queryStride[0] = q.strides[0], p.queryStride[1] = q.strides[1];
    p.queryHeads = int32_t(q.dims[1]), p.group = p.queryHeads / p.cache.heads;
    return p;
}

} // namespace

uint64_t pagedAttentionWorkspace(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *queries) {
    paramsOf("mlel_paged_attention_workspace", cache, batch, queries);
    return 0;
}

int pagedAttention(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *queries,
                   const mlel_tensor *output, float scale, int causal, int window, float softcap, void *workspace,
                   uint64_t workspaceBytes, cudaStream_t s) {
    const std::string call = "mlel_cuda_paged_attention";
    AttendParams p = paramsOf(call, cache, batch, queries);
    const Operand out = writtenOperandOf(call, "output", output, 3);
    if (out.dtype != queries->desc.dtype) {
        throw UnsupportedError(call + ": output has to be of the queries' type");
    }
    if (out.dims[0] != p.batch.tokens || out.dims[1] != p.queryHeads || out.dims[2] != p.cache.headDim) {
        refuse(call, "output has to have the shape of queries");
    }
    if (!std::isfinite(scale) || !std::isfinite(softcap) || softcap < 0.f || window < 0) {
        refuse(call, "scale has to be finite, softcap and window finite and not negative");
    }
    p.out = out.ptr, p.outStride[0] = out.strides[0], p.outStride[1] = out.strides[1];
    p.scale = scale, p.softcap = softcap, p.causal = causal != 0, p.window = window;
    (void)workspace;
    (void)workspaceBytes;
    if (p.batch.tokens == 0 || p.batch.sequences == 0) {
        return MLEL_SUCCESS;
    }
    wantCurrentDevice(call, "output", p.out);
    int64_t blocks = (int64_t(p.batch.maxNew) * p.queryHeads + 7) / 8;
    blocks = blocks < 1 ? 1 : blocks > 65535 ? 65535 : blocks;
    const auto kernel = queries->desc.dtype == MLEL_F16 ? pagedAttentionSimple<__half> : pagedAttentionSimple<__nv_bfloat16>;
    return launchStatus(call.c_str(),
                        launchOverlapped(kernel, dim3(unsigned(p.batch.sequences), unsigned(blocks)), 256, 0, s, p));
}

int takePagedErrorAttention() { return takePagedError(); }

} // namespace mlel
