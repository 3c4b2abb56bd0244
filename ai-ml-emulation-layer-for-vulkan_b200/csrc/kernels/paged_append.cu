// New keys and values into a paged int8 cache, the keys rotated by their positions, with the queries' rotation in the same
// launch.
//
// A unit of work is one page of one sequence and one head that receives tokens: the largest magnitude of its new keys
// (values) decides the page's scale; older integers of the page are rescaled where it grows; the new tokens are rounded
// with it.  One block does the keys and the values of a unit, a half of its warps each, reading the tokens twice (the second
// time from the cache that the first brought them into).  The queries take blocks of their own behind the units.
//
// Rounded keys are decided in 64 bits: the product of an f16 or bf16 element and an f32 cosine has 35 bits, and the rotated
// element is the sum of two, so a result of 32 bits would be off by half a unit in its last place before it is
// compared with the middle between two integers.  Queries are rounded to 16 bits and rotated in 32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "launch_overlapped.cuh"
#include "paged_cache.cuh"
#include "serving_device.cuh"

namespace mlel {
namespace {

constexpr int kSideThreads = 128; // threads for the keys of a unit, and as many for its values

struct AppendParams {
    PagedCache cache;
    PagedBatch batch;
    const char *keys, *values, *queries;
    char *rotated;
    const float *cosines, *sines;
    int64_t keyStride[2], valueStride[2], queryStride[2], rotatedStride[2]; // bytes: token, head
    int64_t angleStride;                                                    // elements between positions
    int32_t half;                                                           // rotated pairs of a head; 0: none
    int32_t interleaved, queryHeads;
    FastDiv units, heads; // pages that a sequence may touch; cache heads
    int64_t unitBlocks;
};

// Element d of a head after rotation, exact to 64 bits.
template <class T> __device__ __forceinline__ double rotatedElement(const T *head, const float *cosines, const float *sines, int d, int half, int interleaved) {
    const double x = double(toFloat(head[d]));
    if (d >= 2 * half) {
        return x;
    }
    const int pair = interleaved ? d >> 1 : (d < half ? d : d - half);
    const bool second = interleaved ? (d & 1) != 0 : d >= half;
    const int other = interleaved ? d ^ 1 : (second ? d - half : d + half);
    const double y = double(toFloat(head[other])), c = double(cosines[pair]), s = double(sines[pair]);
    return second ? fma(x, c, y * s) : fma(x, c, -(y * s));
}

template <class T> __device__ __forceinline__ void appendUnit(const AppendParams &p, int64_t unit, unsigned long long *partial) {
    const uint32_t overHeads = fastDiv(uint32_t(unit), p.heads), index = fastDiv(overHeads, p.units);
    const int head = int(uint32_t(unit) - overHeads * p.heads.d), ordinal = int(overHeads - index * p.units.d);
    const Sequence q = sequenceOf(p.batch, int(index));
    const bool reporter = threadIdx.x == 0 && head == 0;
    if (!q.sound) {
        if (reporter && ordinal == 0) {
            atomicCAS(&g_pagedError, 0, kBadSequence);
        }
        return;
    }
    const int D = p.cache.headDim, page = p.cache.page;
    const int old = q.length - q.fresh, pageIndex = old / page + ordinal;
    const int lo = max(old, pageIndex * page), hi = min(q.length, (pageIndex + 1) * page);
    if (lo >= hi) {
        return;
    }
    const int slot = p.batch.table[index * p.batch.tableStride + pageIndex];
    if (slot < 0 || slot >= p.cache.pages) {
        if (reporter) {
            atomicCAS(&g_pagedError, 0, kBadPage);
        }
        return;
    }
    const bool values = threadIdx.x >= kSideThreads;
    const int at = int(threadIdx.x) % kSideThreads;
    const int64_t row = int64_t(slot) * p.cache.heads + head;
    int8_t *store = (values ? p.cache.values : p.cache.keys) + row * page * D;
    float *scaleAt = (values ? p.cache.valueScales : p.cache.keyScales) + row;
    const char *from = (values ? p.values + head * p.valueStride[1] : p.keys + head * p.keyStride[1]) +
                       int64_t(q.first + lo - old) * (values ? p.valueStride[0] : p.keyStride[0]);
    const int64_t tokenStride = values ? p.valueStride[0] : p.keyStride[0];
    const int half = values ? 0 : p.half, fresh = hi - lo, before = lo - pageIndex * page;
    const auto element = [&](int token, int d) {
        const int64_t angle = int64_t(lo + token) * p.angleStride;
        return rotatedElement(reinterpret_cast<const T *>(from + token * tokenStride), p.cosines + angle, p.sines + angle, d, half, p.interleaved);
    };
    unsigned long long most = 0;
    for (int i = at; i < fresh * D; i += kSideThreads) {
        const int token = i / D;
        most = max(most, (unsigned long long)(__double_as_longlong(element(token, i - token * D))) & 0x7fffffffffffffffull);
    }
    for (int step = 16; step > 0; step >>= 1) {
        most = max(most, __shfl_xor_sync(0xffffffffu, most, step));
    }
    if ((threadIdx.x & 31) == 0) {
        partial[threadIdx.x >> 5] = most;
    }
    __syncthreads();
    most = 0;
#pragma unroll
    for (int w = 0; w < kSideThreads / 32; ++w) {
        most = max(most, partial[(values ? kSideThreads / 32 : 0) + w]);
    }
    // magnitudes are compared as bits here too: what is not finite stays the largest
    const float fresh32 = float(__longlong_as_double((long long)most) / 127.0);
    const uint32_t oldBits = before > 0 ? __float_as_uint(*scaleAt) & 0x7fffffffu : 0u;
    const uint32_t nowBits = max(oldBits, __float_as_uint(fresh32) & 0x7fffffffu);
    const float now = __uint_as_float(nowBits), was = __uint_as_float(oldBits);
    const bool finite = nowBits < 0x7f800000u;
    __syncthreads(); // every thread has read the old scale
    if (at == 0) {
        *scaleAt = now;
    }
    if (finite && nowBits > oldBits && oldBits != 0u) {
        for (int i = at; i < before * D; i += kSideThreads) {
            store[i] = int8_t(int(rint(double(store[i]) * double(was) / double(now))));
        }
    }
    const double inverse = finite && nowBits != 0u ? 1.0 / double(now) : 0.0;
    for (int i = at; i < fresh * D; i += kSideThreads) {
        const int token = i / D;
        double q8 = 0.0;
        if (inverse != 0.0) {
            const double x = element(token, i - token * D), y = x * inverse;
            q8 = rint(y);
            if (fabs(y - q8) > 0.4999999) {
                q8 = rint(x / double(now)); // a quotient in the middle between two integers is formed exactly
            }
            q8 = fmin(fmax(q8, -127.0), 127.0);
        }
        store[before * D + i] = int8_t(int(q8));
    }
}

// The sequence that row `token` belongs to, or -1; all lanes of a warp together.
__device__ __forceinline__ int sequenceOfToken(const PagedBatch &b, int token) {
    int lo = 0, hi = b.sequences; // the answer, if any, is the last index in [lo, hi) whose start is not behind the token
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, probe = lo + int(threadIdx.x & 31) * step;
        const uint32_t below = __ballot_sync(0xffffffffu, probe < hi && b.starts[probe] <= token);
        if (below == 0u) {
            return -1;
        }
        const int last = 31 - __clz(int(below));
        lo += last * step;
        hi = min(hi, lo + step);
    }
    return b.starts[lo] <= token && token < b.starts[lo + 1] ? lo : -1;
}

template <class T> __device__ __forceinline__ void rotateQueries(const AppendParams &p, int token) {
    if (p.batch.sequences == 0) {
        return;
    }
    const int index = sequenceOfToken(p.batch, token);
    if (index < 0) {
        return; // a row of no sequence
    }
    const Sequence q = sequenceOf(p.batch, index);
    if (!q.sound) {
        return; // recorded by the sequence's first unit
    }
    const int D = p.cache.headDim, half = p.half;
    const int64_t angle = int64_t(q.length - q.fresh + token - q.first) * p.angleStride;
    const float *cosines = p.cosines + angle, *sines = p.sines + angle;
    const char *from = p.queries + int64_t(token) * p.queryStride[0];
    char *to = p.rotated + int64_t(token) * p.rotatedStride[0];
    const int pairs = D / 2;
    for (int i = int(threadIdx.x); i < p.queryHeads * pairs; i += int(blockDim.x)) {
        const int head = i / pairs, pair = i - head * pairs;
        const T *x = reinterpret_cast<const T *>(from + head * p.queryStride[1]);
        T *y = reinterpret_cast<T *>(to + head * p.rotatedStride[1]);
        if (pair < half) {
            const int one = p.interleaved ? 2 * pair : pair, two = p.interleaved ? 2 * pair + 1 : pair + half;
            const float a = toFloat(x[one]), b = toFloat(x[two]), c = cosines[pair], s = sines[pair];
            y[one] = fromFloat<T>(fmaf(a, c, -(b * s)));
            y[two] = fromFloat<T>(fmaf(b, c, a * s));
        } else {
            y[2 * pair] = x[2 * pair];
            y[2 * pair + 1] = x[2 * pair + 1];
        }
    }
}

template <class T>
__global__ void __launch_bounds__(2 * kSideThreads) pagedAppendKernel(const AppendParams p) {
    __shared__ unsigned long long partial[2 * kSideThreads / 32];
    dependencySync();
    if (int64_t(blockIdx.x) < p.unitBlocks) {
        appendUnit<T>(p, blockIdx.x, partial);
    } else {
        rotateQueries<T>(p, int(int64_t(blockIdx.x) - p.unitBlocks));
    }
}

} // namespace

int pagedAppend(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *keys, const mlel_tensor *values,
                const mlel_tensor *cosines, const mlel_tensor *sines, const mlel_tensor *queries, const mlel_tensor *rotated,
                int interleaved, cudaStream_t s) {
    const std::string call = "mlel_cuda_paged_append";
    AppendParams p{};
    p.cache = cacheOf(call, cache, true);
    const Operand k = operandOf(call, "keys", keys, 3), v = operandOf(call, "values", values, 3);
    if (k.dtype != MLEL_F16 && k.dtype != MLEL_BF16) {
        throw UnsupportedError(call + ": keys have to be f16 or bf16");
    }
    if (v.dtype != k.dtype) {
        throw UnsupportedError(call + ": values have to be of the keys' type");
    }
    const int64_t tokens = k.dims[0];
    for (int i = 0; i < 3; ++i) {
        if (k.dims[i] != v.dims[i] || (i == 1 && k.dims[i] != p.cache.heads) || (i == 2 && k.dims[i] != p.cache.headDim)) {
            refuse(call, "the shapes of keys and values do not fit the cache or one another");
        }
    }
    p.batch = batchOf(call, batch, p.cache, tokens);
    if ((cosines == nullptr) != (sines == nullptr)) {
        refuse(call, "cosines and sines come together");
    }
    if (cosines != nullptr) {
        const Operand c = operandOf(call, "cosines", cosines, 2), n = operandOf(call, "sines", sines, 2);
        wantType(call, "cosines", c, MLEL_F32, "f32");
        wantType(call, "sines", n, MLEL_F32, "f32");
        if (c.dims[0] != n.dims[0] || c.dims[1] != n.dims[1] || (c.dims[0] > 1 && c.strides[0] != n.strides[0])) {
            refuse(call, "cosines and sines have to be of one shape and layout");
        }
        if (c.dims[0] < p.batch.maxLength || 2 * c.dims[1] > p.cache.headDim) {
            refuse(call, "cosines and sines have fewer rows than max_length or more pairs than head_dim / 2");
        }
        p.cosines = reinterpret_cast<const float *>(c.ptr), p.sines = reinterpret_cast<const float *>(n.ptr);
        p.angleStride = c.strides[0] / 4, p.half = int32_t(c.dims[1]), p.interleaved = interleaved != 0;
    }
    if ((queries == nullptr) != (rotated == nullptr)) {
        refuse(call, "queries and rotated_queries come together");
    }
    if (queries != nullptr) {
        const Operand q = operandOf(call, "queries", queries, 3), r = writtenOperandOf(call, "rotated_queries", rotated, 3);
        if (q.dtype != k.dtype || r.dtype != k.dtype) {
            throw UnsupportedError(call + ": queries have to be of the keys' type");
        }
        if (q.dims[0] != tokens || r.dims[0] != tokens || q.dims[1] != r.dims[1] || q.dims[2] != p.cache.headDim ||
            r.dims[2] != p.cache.headDim) {
            refuse(call, "the shapes of queries and rotated_queries do not fit the keys or one another");
        }
        if (q.ptr == r.ptr && q.count() > 0 && (q.strides[0] != r.strides[0] || q.strides[1] != r.strides[1])) {
            refuse(call, "queries rotated in place need one layout");
        }
        p.queries = q.ptr, p.rotated = r.ptr, p.queryHeads = int32_t(q.dims[1]);
        p.queryStride[0] = q.strides[0], p.queryStride[1] = q.strides[1];
        p.rotatedStride[0] = r.strides[0], p.rotatedStride[1] = r.strides[1];
    }
    if (tokens == 0 || p.batch.sequences == 0) {
        return MLEL_SUCCESS;
    }
    p.keys = k.ptr, p.values = v.ptr;
    p.keyStride[0] = k.strides[0], p.keyStride[1] = k.strides[1];
    p.valueStride[0] = v.strides[0], p.valueStride[1] = v.strides[1];
    // n tokens touch at most (n - 2) / page + 2 pages, those that a first token starts included
    const int64_t units = (int64_t(p.batch.maxNew) + p.cache.page - 2) / p.cache.page + 1;
    p.unitBlocks = units * p.batch.sequences * p.cache.heads;
    const int64_t blocks = p.unitBlocks + (p.queryHeads > 0 ? tokens : 0);
    if (blocks > 0x7fffffff) {
        refuse(call, "too many pages and tokens for one call");
    }
    p.units = makeFastDiv(units), p.heads = makeFastDiv(p.cache.heads);
    wantCurrentDevice(call, "the cache", p.cache.keys);
    const auto kernel = k.dtype == MLEL_F16 ? pagedAppendKernel<__half> : pagedAppendKernel<__nv_bfloat16>;
    return launchStatus(call.c_str(), launchOverlapped(kernel, dim3(unsigned(blocks)), 2 * kSideThreads, 0, s, p));
}

int takePagedErrorAppend() { return takePagedError(); }

} // namespace mlel
