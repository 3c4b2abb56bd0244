// Attention over the paged int8 cache as its kernels take it (paged_attention.cu chooses among them).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "gemm_i8_tcgen05.hpp"
#include "paged_cache.cuh"

namespace mlel {

constexpr int kMostRowsOfBlock = 256; // the rows of a sequence are handed out in blocks of at most so many

struct AttendParams {
    PagedCache cache;
    PagedBatch batch;
    const char *queries;
    char *out;
    int64_t queryStride[2], outStride[2]; // bytes: token, head
    float scale, softcap, perCap;         // softcap 0: none; perCap: 1 / softcap, and finite
    int32_t causal, window, queryHeads, group;
    int32_t halves;      // queries and output are f16 (else bf16)
    int32_t wideQueries; // every head of the queries starts on a 16-byte boundary; the same for the output
    int32_t wideOut;
    float *partials; // split calls: see paged_attention_few.cu
    FastDiv pageDiv, groupDiv;
};

// paged_attention_few.cu: few rows per cache head (single tokens, or a handful), keys split over the whole device
struct FewPlan {
    int split;          // blocks of the cluster that shares a tile's keys; 0: all blocks share all keys
    int blocks;
    uint64_t workspace; // where parts of a tile may lie with blocks that are no cluster: a second kernel joins them
};
FewPlan pagedAttentionFewPlan(const AttendParams &p);
int pagedAttentionFew(const AttendParams &p, const FewPlan &plan, cudaStream_t s);
cudaError_t takePagedErrorFew(int &code);
int fewAttentionErrorWord();

// paged_attention_many.cu: many rows per cache head (prompts)
bool pagedAttentionManyApplies(const AttendParams &p);
int pagedAttentionMany(const AttendParams &p, cudaStream_t s);
cudaError_t takePagedErrorMany(int &code);
int manyAttentionErrorWord();

} // namespace mlel
