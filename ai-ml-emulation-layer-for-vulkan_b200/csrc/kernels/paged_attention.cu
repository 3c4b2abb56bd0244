// Attention over a paged int8 cache with a scale for each page and head: the checks of a call, and which kernel takes it.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "matmul_scaled.hpp"
#include "paged_attention.hpp"

namespace mlel {
namespace {

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
    if (int64_t(p.batch.maxNew) * p.group > 0x7fffffff - kMostRowsOfBlock) { // the kernels number a sequence's rows in 32 bits
        refuse(call, "a sequence may have more than 2^31 rows of queries per cache head");
    }
    p.halves = q.dtype == MLEL_F16;
    p.wideQueries = aligned(q.ptr, 16) && q.strides[0] % 16 == 0 && q.strides[1] % 16 == 0;
    p.pageDiv = makeFastDiv(p.cache.page), p.groupDiv = makeFastDiv(p.group);
    return p;
}

} // namespace

uint64_t pagedAttentionWorkspace(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *queries) {
    const AttendParams p = paramsOf("mlel_paged_attention_workspace", cache, batch, queries);
    return p.batch.tokens == 0 || p.batch.sequences == 0 || pagedAttentionManyApplies(p) ? 0 : pagedAttentionFewPlan(p).workspace;
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
    p.wideOut = aligned(out.ptr, 16) && out.strides[0] % 16 == 0 && out.strides[1] % 16 == 0;
    p.scale = scale, p.softcap = softcap, p.perCap = std::min(1.f / softcap, std::numeric_limits<float>::max() / 4.f), p.causal = causal != 0, p.window = window;
    if (p.batch.tokens == 0 || p.batch.sequences == 0) {
        return MLEL_SUCCESS;
    }
    wantCurrentDevice(call, "output", p.out);
    if (pagedAttentionManyApplies(p)) {
        return pagedAttentionMany(p, s);
    }
    const FewPlan plan = pagedAttentionFewPlan(p);
    if (plan.workspace > 0 && (workspace == nullptr || workspaceBytes < plan.workspace || !aligned(workspace, 16))) {
        refuse(call, "the workspace is null, off a 16-byte boundary or smaller than mlel_paged_attention_workspace() says");
    }
    p.partials = static_cast<float *>(workspace);
    return pagedAttentionFew(p, plan, s);
}

cudaError_t takePagedErrorAttention(int &code) {
    const cudaError_t err = takePagedErrorFew(code);
    return err != cudaSuccess ? err : takePagedErrorMany(code);
}
int servingErrorWord() {
    for (const auto word : {fewAttentionErrorWord, manyAttentionErrorWord, scaledTilesErrorWord, scaledPairErrorWord}) {
        if (const int code = word()) {
            return code;
        }
    }
    return 0;
}

} // namespace mlel
