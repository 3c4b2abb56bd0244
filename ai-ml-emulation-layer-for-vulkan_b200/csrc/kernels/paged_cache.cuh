// The paged int8 cache and its batches as kernels take them, and the checks of a call's operands.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../graph_pipeline.hpp"
#include "serving.hpp"

namespace mlel {

// What the kernels of the including translation unit left out (mlel_paged_error).
static __device__ int g_pagedError = 0;
enum : int { kBadSequence = 1, kBadPage = 2 };

static inline cudaError_t takePagedError(int &code) {
    const int zero = 0;
    int v = 0;
    cudaError_t err = cudaMemcpyFromSymbol(&v, g_pagedError, sizeof(int));
    if (err == cudaSuccess && v != 0) {
        err = cudaMemcpyToSymbol(g_pagedError, &zero, sizeof(int));
        code = code != 0 ? code : v;
    }
    return err;
}

struct PagedCache {
    int8_t *keys, *values;
    float *keyScales, *valueScales;
    int32_t pages, heads, page, headDim;
};

struct PagedBatch {
    const int32_t *starts, *lengths, *table;
    int64_t tableStride; // entries between rows
    int32_t sequences, maxNew, maxLength;
    int32_t tokens; // rows of the token axis
};

// One sequence of a batch: its new tokens are rows first .. first + fresh - 1 and the last of `length`.
struct Sequence {
    int32_t first, fresh, length;
    bool sound;
};
__device__ __forceinline__ Sequence sequenceOf(const PagedBatch &b, int index) {
    Sequence q;
    const int32_t end = b.starts[index + 1];
    q.first = b.starts[index], q.length = b.lengths[index];
    q.sound = q.first >= 0 && end >= q.first && end <= b.tokens && q.length >= 0 && q.length <= b.maxLength;
    q.fresh = q.sound ? end - q.first : 0;
    q.sound = q.sound && q.fresh <= b.maxNew && q.fresh <= q.length;
    return q;
}

inline PagedCache cacheOf(const std::string &call, const mlel_paged_cache *cache, bool written) {
    if (cache == nullptr) {
        refuse(call, "cache is missing");
    }
    const auto view = [&](const char *name, const mlel_tensor *t, int rank) {
        const Operand o = written ? writtenOperandOf(call, name, t, rank) : operandOf(call, name, t, rank);
        wantPacked(call, name, o);
        return o;
    };
    const Operand k = view("keys of the cache", &cache->keys, 4), v = view("values of the cache", &cache->values, 4),
                  ks = view("key_scales", &cache->key_scales, 2), vs = view("value_scales", &cache->value_scales, 2);
    wantType(call, "keys of the cache", k, MLEL_I8, "int8");
    wantType(call, "values of the cache", v, MLEL_I8, "int8");
    wantType(call, "key_scales", ks, MLEL_F32, "f32");
    wantType(call, "value_scales", vs, MLEL_F32, "f32");
    for (int i = 0; i < 4; ++i) {
        if (k.dims[i] != v.dims[i] || (i < 2 && (ks.dims[i] != k.dims[i] || vs.dims[i] != k.dims[i])) || k.dims[i] < 1) {
            refuse(call, "the shapes of the cache's parts do not fit together, or one is empty");
        }
    }
    if (k.dims[2] % 16 != 0 || k.dims[2] > 256) {
        throw UnsupportedError(call + ": pages have to hold a multiple of 16 tokens, at most 256");
    }
    if (k.dims[3] % 16 != 0 || k.dims[3] > 256) {
        throw UnsupportedError(call + ": head_dim has to be a multiple of 16, at most 256");
    }
    if (k.dims[0] * k.dims[1] > 0x7fffffff / k.dims[2]) {
        refuse(call, "the cache has too many rows");
    }
    if (!aligned(k.ptr, 16) || !aligned(v.ptr, 16)) {
        refuse(call, "the cache has to start on 16-byte boundaries");
    }
    PagedCache c{};
    c.keys = reinterpret_cast<int8_t *>(k.ptr), c.values = reinterpret_cast<int8_t *>(v.ptr);
    c.keyScales = reinterpret_cast<float *>(ks.ptr), c.valueScales = reinterpret_cast<float *>(vs.ptr);
    c.pages = int32_t(k.dims[0]), c.heads = int32_t(k.dims[1]), c.page = int32_t(k.dims[2]), c.headDim = int32_t(k.dims[3]);
    return c;
}

inline PagedBatch batchOf(const std::string &call, const mlel_paged_batch *batch, const PagedCache &cache, int64_t tokens) {
    if (batch == nullptr) {
        refuse(call, "batch is missing");
    }
    const Operand starts = operandOf(call, "starts", &batch->starts, 1), lengths = operandOf(call, "lengths", &batch->lengths, 1),
                  table = operandOf(call, "page_table", &batch->page_table, 2);
    wantType(call, "starts", starts, MLEL_I32, "i32");
    wantType(call, "lengths", lengths, MLEL_I32, "i32");
    wantType(call, "page_table", table, MLEL_I32, "i32");
    wantPacked(call, "starts", starts);
    wantPacked(call, "lengths", lengths);
    if (starts.dims[0] != lengths.dims[0] + 1 || table.dims[0] != lengths.dims[0]) {
        refuse(call, "starts, lengths and page_table are not of as many sequences");
    }
    if (batch->max_new < 0 || batch->max_new > batch->max_length || batch->max_length > (1 << 30)) {
        refuse(call, "max_new and max_length have to be 0 <= max_new <= max_length <= 2^30");
    }
    if ((int64_t(batch->max_length) + cache.page - 1) / cache.page > table.dims[1]) {
        refuse(call, "page_table has fewer columns than max_length tokens need");
    }
    PagedBatch b{};
    b.starts = reinterpret_cast<const int32_t *>(starts.ptr), b.lengths = reinterpret_cast<const int32_t *>(lengths.ptr);
    b.table = reinterpret_cast<const int32_t *>(table.ptr);
    b.tableStride = table.strides[0] / 4;
    // no sequence has more new tokens than the token axis: a loose bound costs nothing
    b.sequences = int32_t(lengths.dims[0]), b.maxNew = int32_t(std::min<int64_t>(batch->max_new, tokens)), b.maxLength = batch->max_length;
    b.tokens = int32_t(tokens);
    return b;
}

} // namespace mlel
