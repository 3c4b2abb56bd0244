// New keys and values into a paged int8 cache, the keys rotated by their positions, with the queries' rotation in the same
// launch.
//
// A unit of work is one page of one sequence and one head that receives tokens: the largest magnitude of its new keys
// (values) decides the page's scale; older integers of the page are rescaled where it grows; the new tokens are rounded
// with it.  One block does the keys and the values of a unit, a half of its warps each.  The queries have blocks of their own.
//
// What bounds it: memory, the queries' above all (they are four to eight times as many as the keys).  So a thread moves 16-byte
// vectors: 8 elements and the 8 they turn with (their neighbours where pairs lie side by side).
//
// Integers are those of exact arithmetic.  A rotated key u c - w s in 32 bits is off by at most 2^-24 (|w s| + the result): the
// largest magnitude is formed again in 64 bits from the elements within twice that of the largest found, and a quotient
// that lies as near to the middle between two integers is decided in 64 bits.  (All of it in 64 bits, in two passes over the
// tokens: 87 us for 8270 tokens with 8 heads of keys and 32 of queries, 128 elements each, so 63: some 25 of them the queries', at
// 5.4 TB/s.)  A unit of up to 512 vector
// pairs stays in registers between the two; larger ones, and magnitudes beyond 32 bits, take two passes in 64 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "device_common.cuh"
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
    FastDiv vectors;      // pairs of vectors in a head: head_dim / 16
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

// Vector pair v of a head: 8 elements from `one` and 8 from `two` on; pair j of them is (one + j, two + j), or with `interleaved`
// the j-th of the eight neighbours (two == one + 8); turned by the angles from `angle` on, or not at all.
struct VectorPair {
    int one, two, angle;
    bool turned;
};
__device__ __forceinline__ VectorPair vectorPair(const AppendParams &p, int v) {
    if (p.interleaved || 8 * v >= p.half) {
        const int first = p.interleaved ? 16 * v : 2 * p.half + 16 * (v - p.half / 8);
        return {first, first + 8, 8 * v, first < 2 * p.half};
    }
    return {8 * v, p.half + 8 * v, 8 * v, true};
}
// The 16 elements as the first and second members of eight pairs, and back.
__device__ __forceinline__ void pairUp(bool interleaved, float (&x)[8], float (&y)[8]) {
    if (interleaved) {
        float a[8], b[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = x[2 * j], b[j] = x[2 * j + 1], a[4 + j] = y[2 * j], b[4 + j] = y[2 * j + 1];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = a[j], y[j] = b[j];
        }
    }
}
template <class V> __device__ __forceinline__ void pairDown(bool interleaved, V (&x)[8], V (&y)[8]) {
    if (interleaved) {
        V a[8], b[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[2 * j] = x[j], a[2 * j + 1] = y[j], b[2 * j] = x[4 + j], b[2 * j + 1] = y[4 + j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = a[j], y[j] = b[j];
        }
    }
}
// Four bytes from the low bytes of four words.
__device__ __forceinline__ uint32_t lowBytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// x / scale to the nearest integer within [-127, 127], as a word whose low byte it is; `inverse` is 1 / scale.  `careful`: the
// scale is so small that it is itself rounded coarsely, and quotients may exceed 127.
__device__ __forceinline__ uint32_t roundedExactly(double x, double inverse, double scale, bool careful) {
    constexpr double kMagic = 6755399441055744.0; // 1.5 * 2^52
    const double y = x * inverse, t = y + kMagic;
    if (__builtin_expect(careful || !(fabs(y - (t - kMagic)) <= 0.4999999), 0)) {
        return uint32_t(max(-127, min(127, int(rint(x / scale))))); // a quotient in the middle between two integers is formed exactly
    }
    return uint32_t(__double2loint(t));
}

// What the warps of a block tell one another; a side's warps stand together.
struct AppendExchange {
    unsigned long long most[2 * kSideThreads / 32];
    uint32_t magnitude[2 * kSideThreads / 32], product[2 * kSideThreads / 32];
};

constexpr int kHeldPairs = 4;     // vector pairs that a thread keeps
constexpr int kShortUnit = 512;  // elements of a unit that are taken one by one

template <class T, bool WIDE> __device__ __forceinline__ void appendUnit(const AppendParams &p, int64_t unit, AppendExchange &exchange) {
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
    const int slot = p.batch.table[index * p.batch.tableStride + pageIndex]; // (looked at when the tokens have been)
    const bool values = threadIdx.x >= kSideThreads;
    const int at = int(threadIdx.x) % kSideThreads;
    const int64_t tokenStride = values ? p.valueStride[0] : p.keyStride[0];
    const char *from = (values ? p.values + head * p.valueStride[1] : p.keys + head * p.keyStride[1]) + int64_t(q.first + lo - old) * tokenStride;
    const int half = values ? 0 : p.half, fresh = hi - lo, before = lo - pageIndex * page, vectors = int(p.vectors.d);
    const bool rotates = !values && p.half > 0;
    // one element, and 16 of them in pairs
    const auto element = [&](int token, int d) {
        const int64_t angle = int64_t(lo + token) * p.angleStride;
        return rotatedElement(reinterpret_cast<const T *>(from + token * tokenStride), p.cosines + angle, p.sines + angle, d, half, p.interleaved);
    };
    [[maybe_unused]] const auto vectorOf = [&](int token, const VectorPair &v, float (&x)[8], float (&y)[8]) {
        const T *head = reinterpret_cast<const T *>(from + token * tokenStride);
        loadWide(head + v.one, x);
        loadWide(head + v.two, y);
    };
    const auto turn = [&](int token, const VectorPair &v, float (&x)[8], float (&y)[8], double (&a)[8], double (&b)[8]) {
        float c[8], s[8];
        const int64_t angle = int64_t(lo + token) * p.angleStride + v.angle;
        loadWide(p.cosines + angle, c);
        loadWide(p.sines + angle, s);
        pairUp(p.interleaved != 0, x, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double u = double(x[j]), w = double(y[j]), cosine = double(c[j]), sine = double(s[j]);
            a[j] = fma(u, cosine, -(w * sine)), b[j] = fma(w, cosine, u * sine);
        }
    };
    const int warp = int(threadIdx.x) >> 5, sideWarp = values ? kSideThreads / 32 : 0;
    bool held = WIDE && fresh * vectors <= kHeldPairs * kSideThreads; // (the same for the whole block)
    uint4 one[kHeldPairs], two[kHeldPairs];                           // as they lie in memory
    float slack = 0.f;                                                // twice what a rotated element may be off by in 32 bits
    // the largest magnitude, as the bits of a 64-bit float
    unsigned long long most = 0;
    // pair h of this thread, rotated in 32 bits: first members of eight pairs, then the second ones
    const auto heldPair = [&](int h, VectorPair &v, int &token, float (&x)[8], float (&y)[8], uint32_t &product) {
        const int i = at + h * kSideThreads;
        token = int(fastDiv(uint32_t(i), p.vectors));
        v = vectorPair(p, i - token * vectors);
        unpackEight(one[h], x, T());
        unpackEight(two[h], y, T());
        if (rotates && v.turned) {
            float c[8], s[8];
            const int64_t angle = int64_t(lo + token) * p.angleStride + v.angle;
            loadWide(p.cosines + angle, c);
            loadWide(p.sines + angle, s);
            pairUp(p.interleaved != 0, x, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = x[j], w = y[j], ws = w * s[j], us = u * s[j];
                x[j] = fmaf(u, c[j], -ws), y[j] = fmaf(w, c[j], us);
                product = max(product, max(__float_as_uint(ws) & 0x7fffffffu, __float_as_uint(us) & 0x7fffffffu));
            }
        }
    };
    // which element of the head member j of those sixteen is
    const auto elementOf = [&](const VectorPair &v, int j) {
        return rotates && v.turned && p.interleaved ? v.one + 2 * (j & 7) + (j >> 3) : (j < 8 ? v.one + j : v.two + j - 8);
    };
    if (held) {
        uint32_t magnitude = 0, product = 0;
#pragma unroll
        for (int h = 0; h < kHeldPairs; ++h) {
            const int i = at + h * kSideThreads;
            one[h] = two[h] = {0u, 0u, 0u, 0u};
            if (i < fresh * vectors) {
                const int token = int(fastDiv(uint32_t(i), p.vectors));
                const VectorPair v = vectorPair(p, i - token * vectors);
                const T *head = reinterpret_cast<const T *>(from + token * tokenStride);
                one[h] = *reinterpret_cast<const uint4 *>(head + v.one), two[h] = *reinterpret_cast<const uint4 *>(head + v.two);
            }
        }
#pragma unroll
        for (int h = 0; h < kHeldPairs; ++h) {
            const int i = at + h * kSideThreads;
            if (i < fresh * vectors) {
                if (rotates && vectorPair(p, i - int(fastDiv(uint32_t(i), p.vectors)) * vectors).turned) {
                    VectorPair v;
                    int token;
                    float x[8], y[8];
                    heldPair(h, v, token, x, y, product);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        magnitude = max(magnitude, max(__float_as_uint(x[j]) & 0x7fffffffu, __float_as_uint(y[j]) & 0x7fffffffu));
                    }
                } else { // magnitudes of 16 bits are ordered like their bits
                    constexpr uint32_t kSigns = 0x7fff7fffu;
                    const uint4 a = one[h], b = two[h];
                    const uint32_t m = maxHalves(maxHalves(maxHalves(a.x & kSigns, a.y & kSigns), maxHalves(a.z & kSigns, a.w & kSigns)),
                                                 maxHalves(maxHalves(b.x & kSigns, b.y & kSigns), maxHalves(b.z & kSigns, b.w & kSigns)));
                    magnitude = max(magnitude, __float_as_uint(unpackTwo(max(m & 0xffffu, m >> 16), T()).x));
                }
            }
        }
        if (p.half > 0) { // (without rotation the elements are exact)
            const float own = __uint_as_float(magnitude);
            magnitude = __reduce_max_sync(0xffffffffu, magnitude), product = __reduce_max_sync(0xffffffffu, product);
            if ((threadIdx.x & 31) == 0) {
                exchange.magnitude[warp] = magnitude, exchange.product[warp] = product;
            }
            __syncthreads();
            bool finite = true;
            magnitude = product = 0;
#pragma unroll
            for (int w = 0; w < 2 * kSideThreads / 32; ++w) {
                finite = finite && exchange.magnitude[w] < 0x7f800000u && exchange.product[w] < 0x7f800000u;
                if (w >= sideWarp && w < sideWarp + kSideThreads / 32) {
                    magnitude = max(magnitude, exchange.magnitude[w]), product = max(product, exchange.product[w]);
                }
            }
            held = finite; // what 32 bits cannot hold may yet be a number: 64 bits tell
            if (held) {
                const float top = __uint_as_float(magnitude);
                slack = rotates ? (__uint_as_float(product) + top) * (1.f / 8388608.f) : 0.f;
                if (own >= top - slack) { // few threads
#pragma unroll
                    for (int h = 0; h < kHeldPairs; ++h) {
                        if (at + h * kSideThreads < fresh * vectors) {
                            VectorPair v;
                            int token;
                            float x[8], y[8];
                            heldPair(h, v, token, x, y, product);
                            uint32_t near = 0;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                near |= fabsf(x[j]) >= top - slack ? 1u << j : 0u;
                                near |= fabsf(y[j]) >= top - slack ? 256u << j : 0u;
                            }
#pragma unroll 1
                            while (near != 0u) {
                                const int d = elementOf(v, __ffs(int(near)) - 1);
                                near &= near - 1u;
                                most = max(most, (unsigned long long)(__double_as_longlong(element(token, d))) & 0x7fffffffffffffffull);
                            }
                        }
                    }
                }
            }
        } else {
            most = (unsigned long long)(__double_as_longlong(double(__uint_as_float(magnitude)))) & 0x7fffffffffffffffull;
        }
    }
    if (held) {
        // done
    } else if (!WIDE) {
        for (int i = at; i < fresh * D; i += kSideThreads) {
            const int token = i / D;
            most = max(most, (unsigned long long)(__double_as_longlong(element(token, i - token * D))) & 0x7fffffffffffffffull);
        }
    } else {
        uint32_t most32 = 0;
#pragma unroll 2
        for (int i = at; i < fresh * vectors; i += kSideThreads) {
            const int token = int(fastDiv(uint32_t(i), p.vectors));
            const VectorPair v = vectorPair(p, i - token * vectors);
            float x[8], y[8];
            vectorOf(token, v, x, y);
            if (rotates && v.turned) {
                double a[8], b[8];
                turn(token, v, x, y, a, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    most = max(most, (unsigned long long)(__double_as_longlong(a[j])) & 0x7fffffffffffffffull);
                    most = max(most, (unsigned long long)(__double_as_longlong(b[j])) & 0x7fffffffffffffffull);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    most32 = max(most32, max(__float_as_uint(x[j]) & 0x7fffffffu, __float_as_uint(y[j]) & 0x7fffffffu));
                }
            }
        }
        most = max(most, (unsigned long long)(__double_as_longlong(double(__uint_as_float(most32)))) & 0x7fffffffffffffffull);
    }
    if (slot < 0 || slot >= p.cache.pages) { // (the whole block)
        if (reporter) {
            atomicCAS(&g_pagedError, 0, kBadPage);
        }
        return;
    }
    const int64_t row = int64_t(slot) * p.cache.heads + head;
    int8_t *store = (values ? p.cache.values : p.cache.keys) + row * page * D;
    float *scaleAt = (values ? p.cache.valueScales : p.cache.keyScales) + row;
    const uint32_t oldBits = before > 0 ? __float_as_uint(*scaleAt) & 0x7fffffffu : 0u;
    for (int step = 16; step > 0; step >>= 1) {
        most = max(most, __shfl_xor_sync(0xffffffffu, most, step));
    }
    if ((threadIdx.x & 31) == 0) {
        exchange.most[warp] = most;
    }
    __syncthreads();
    most = 0;
#pragma unroll
    for (int w = 0; w < kSideThreads / 32; ++w) {
        most = max(most, exchange.most[sideWarp + w]);
    }
    // magnitudes are compared as bits here too: what is not finite stays the largest
    const float fresh32 = float(__longlong_as_double((long long)most) / 127.0);
    const uint32_t nowBits = max(oldBits, __float_as_uint(fresh32) & 0x7fffffffu);
    const float now = __uint_as_float(nowBits), was = __uint_as_float(oldBits);
    const bool finite = nowBits < 0x7f800000u;
    if (at == 0) { // (every thread had read the old scale before the barrier)
        *scaleAt = now;
    }
    if (finite && nowBits > oldBits && oldBits != 0u) {
        // 16 older integers at a time; a product of 32 bits is off by at most 2^-23 of 127
        const float ratio = __fdiv_rn(was, now);
        for (int i = at * 16; i < before * D; i += kSideThreads * 16) {
            union {
                uint4 vector;
                int8_t q[16];
            } o;
            o.vector = *reinterpret_cast<const uint4 *>(store + i);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float y = float(o.q[j]) * ratio;
                float whole = rintf(y);
                if (!(fabsf(y - whole) <= 0.4999f) || now < 1e-36f) {
                    whole = float(rint(double(o.q[j]) * double(was) / double(now)));
                }
                o.q[j] = int8_t(int(whole));
            }
            *reinterpret_cast<uint4 *>(store + i) = o.vector;
        }
    }
    const bool some = finite && nowBits != 0u, careful = some && now < 1e-36f;
    const double inverse = some ? 1.0 / double(now) : 0.0;
    int8_t *to = store + before * D;
    if (held) {
        const float inverse32 = some && !careful ? __fdiv_rn(1.f, now) : 0.f;
        // 2^-23 of a quotient for the inverse and the product, and what the element may be off by
        const float middle = careful ? -1.f : 0.49998f - slack * inverse32;
#pragma unroll
        for (int h = 0; h < kHeldPairs; ++h) {
            if (at + h * kSideThreads < fresh * vectors) {
                VectorPair v;
                int token;
                float x[8], y[8];
                uint32_t product = 0;
                heldPair(h, v, token, x, y, product);
                // (as quantizeEight: the nearest whole number by one fused multiply-add, how far the product lies from it by another)
                constexpr float kMagic = 12582912.f;
                uint32_t a[8], b[8];
                float farthest = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float t0 = fmaf(x[j], inverse32, kMagic), t1 = fmaf(y[j], inverse32, kMagic);
                    farthest = fmaxf(farthest, fmaxf(fabsf(fmaf(x[j], inverse32, kMagic - t0)), fabsf(fmaf(y[j], inverse32, kMagic - t1))));
                    a[j] = __float_as_uint(t0), b[j] = __float_as_uint(t1);
                }
                if (rotates && v.turned) {
                    pairDown(p.interleaved != 0, a, b);
                }
                const uint2 low = {lowBytes(a[0], a[1], a[2], a[3]), lowBytes(a[4], a[5], a[6], a[7])},
                            high = {lowBytes(b[0], b[1], b[2], b[3]), lowBytes(b[4], b[5], b[6], b[7])};
                *reinterpret_cast<uint2 *>(to + token * D + v.one) = some ? low : uint2{0u, 0u};
                *reinterpret_cast<uint2 *>(to + token * D + v.two) = some ? high : uint2{0u, 0u};
                if (__builtin_expect(some && !(farthest <= middle), 0)) {
                    uint32_t doubtful = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float t0 = fmaf(x[j], inverse32, kMagic), t1 = fmaf(y[j], inverse32, kMagic);
                        doubtful |= !(fabsf(fmaf(x[j], inverse32, kMagic - t0)) <= middle) ? 1u << j : 0u;
                        doubtful |= !(fabsf(fmaf(y[j], inverse32, kMagic - t1)) <= middle) ? 256u << j : 0u;
                    }
#pragma unroll 1
                    while (doubtful != 0u) {
                        const int d = elementOf(v, __ffs(int(doubtful)) - 1);
                        doubtful &= doubtful - 1u;
                        to[token * D + d] = int8_t(roundedExactly(element(token, d), inverse, double(now), careful));
                    }
                }
            }
        }
    } else if (!WIDE) {
        for (int i = at; i < fresh * D; i += kSideThreads) {
            const int token = i / D;
            to[i] = some ? int8_t(roundedExactly(element(token, i - token * D), inverse, double(now), careful)) : int8_t(0);
        }
    } else {
        RowScale scale;
        scale.value = now, scale.careful = careful, scale.inverse = some && !careful ? __fdiv_rn(1.f, now) : 0.f;
#pragma unroll 2
        for (int i = at; i < fresh * vectors; i += kSideThreads) {
            const int token = int(fastDiv(uint32_t(i), p.vectors));
            const VectorPair v = vectorPair(p, i - token * vectors);
            float x[8], y[8];
            uint2 low = {0u, 0u}, high = {0u, 0u};
            if (some) {
                vectorOf(token, v, x, y);
                if (rotates && v.turned) {
                    double a[8], b[8];
                    uint32_t r[8], s[8];
                    turn(token, v, x, y, a, b);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        r[j] = roundedExactly(a[j], inverse, double(now), careful), s[j] = roundedExactly(b[j], inverse, double(now), careful);
                    }
                    pairDown(p.interleaved != 0, r, s);
                    low = {lowBytes(r[0], r[1], r[2], r[3]), lowBytes(r[4], r[5], r[6], r[7])};
                    high = {lowBytes(s[0], s[1], s[2], s[3]), lowBytes(s[4], s[5], s[6], s[7])};
                } else {
                    low = quantizeEight(x, scale), high = quantizeEight(y, scale);
                }
            }
            *reinterpret_cast<uint2 *>(to + token * D + v.one) = low;
            *reinterpret_cast<uint2 *>(to + token * D + v.two) = high;
        }
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

// The queries of one token by `count` threads, of which this is number `thread`.
template <class T, bool WIDE> __device__ __forceinline__ void rotateQueries(const AppendParams &p, int token, int thread, int count) {
    const int index = p.batch.sequences > 0 ? sequenceOfToken(p.batch, token) : -1;
    if (index < 0) {
        return; // a row of no sequence
    }
    const Sequence q = sequenceOf(p.batch, index);
    if (!q.sound) {
        return; // recorded by the sequence's first unit
    }
    const int D = p.cache.headDim, half = p.half, pairs = D / 2, vectors = int(p.vectors.d);
    const int64_t angle = int64_t(q.length - q.fresh + token - q.first) * p.angleStride;
    const float *cosines = p.cosines + angle, *sines = p.sines + angle;
    const char *from = p.queries + int64_t(token) * p.queryStride[0];
    char *to = p.rotated + int64_t(token) * p.rotatedStride[0];
    if constexpr (WIDE) {
#pragma unroll 4
        for (int i = thread; i < p.queryHeads * vectors; i += count) {
            const int head = int(fastDiv(uint32_t(i), p.vectors));
            const VectorPair v = vectorPair(p, i - head * vectors);
            const T *x = reinterpret_cast<const T *>(from + head * p.queryStride[1]);
            T *y = reinterpret_cast<T *>(to + head * p.rotatedStride[1]);
            const uint4 one = *reinterpret_cast<const uint4 *>(x + v.one), two = *reinterpret_cast<const uint4 *>(x + v.two);
            if (half > 0 && v.turned) {
                float a[8], b[8], c[8], s[8];
                unpackEight(one, a, T());
                unpackEight(two, b, T());
                loadWide(cosines + v.angle, c);
                loadWide(sines + v.angle, s);
                pairUp(p.interleaved != 0, a, b);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float u = a[j], w = b[j];
                    a[j] = fmaf(u, c[j], -(w * s[j])), b[j] = fmaf(w, c[j], u * s[j]);
                }
                pairDown(p.interleaved != 0, a, b);
                *reinterpret_cast<uint4 *>(y + v.one) = packEight(a, T());
                *reinterpret_cast<uint4 *>(y + v.two) = packEight(b, T());
            } else {
                *reinterpret_cast<uint4 *>(y + v.one) = one;
                *reinterpret_cast<uint4 *>(y + v.two) = two;
            }
        }
    } else {
        for (int i = thread; i < p.queryHeads * pairs; i += count) {
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
}

// Units, and behind them the queries, a token a block.
template <class T, bool WIDE_UNITS, bool WIDE>
__global__ void __launch_bounds__(2 * kSideThreads) pagedAppendKernel(const AppendParams p) {
    __shared__ AppendExchange exchange;
    dependencySync();
    if (int64_t(blockIdx.x) < p.unitBlocks) {
        appendUnit<T, WIDE_UNITS>(p, blockIdx.x, exchange);
    } else {
        rotateQueries<T, WIDE>(p, int(int64_t(blockIdx.x) - p.unitBlocks), int(threadIdx.x), 2 * kSideThreads);
    }
}

// The queries of many tokens, a token a warp, in a kernel of few registers.
constexpr int kQueryWarps = 4;
template <class T, bool WIDE>
__global__ void __launch_bounds__(kQueryWarps * 32) rotateQueriesKernel(const AppendParams p) {
    dependencySync();
    const int64_t token = int64_t(blockIdx.x) * kQueryWarps + (threadIdx.x >> 5);
    if (token < p.batch.tokens) {
        rotateQueries<T, WIDE>(p, int(token), int(threadIdx.x) & 31, 32);
    }
}

template <class T, bool WIDE> cudaError_t launchAppend(const AppendParams &p, cudaStream_t s) {
    const unsigned tokens = p.queryHeads > 0 ? unsigned(p.batch.tokens) : 0u;
    // Units of a few tokens element by element: the short way through little code (64 units of one token and 128 elements 5.8 us, by
    // vectors 9.3).
    const bool wideUnits = WIDE && int64_t(p.batch.maxNew) * p.cache.headDim > kShortUnit;
    const auto kernel = wideUnits ? pagedAppendKernel<T, WIDE, WIDE> : pagedAppendKernel<T, false, WIDE>;
    // Up to eight blocks an SM one launch for both (64 tokens: 5.8 us; as two launches 8.0).  Above, the queries, which have most of
    // the bytes, in a kernel whose registers let four times as many threads wait for memory (8270 tokens, with units in 64 bits: 107 and 87 us).
    if (p.unitBlocks + tokens <= 8 * kNumSMs || tokens == 0) {
        return launchOverlapped(kernel, dim3(unsigned(p.unitBlocks) + tokens), 2 * kSideThreads, 0, s, p);
    }
    const cudaError_t err = launchOverlapped(kernel, dim3(unsigned(p.unitBlocks)), 2 * kSideThreads, 0, s, p);
    return err != cudaSuccess ? err
                              : launchOverlapped(rotateQueriesKernel<T, WIDE>, dim3((tokens + kQueryWarps - 1) / kQueryWarps), kQueryWarps * 32,
                                                 0, s, p);
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
    if (p.unitBlocks + tokens > 0x7fffffff) {
        refuse(call, "too many pages and tokens for one call");
    }
    p.units = makeFastDiv(units), p.heads = makeFastDiv(p.cache.heads), p.vectors = makeFastDiv(p.cache.headDim / 16);
    wantCurrentDevice(call, "the cache", p.cache.keys);
    const auto vectorRows = [](const char *ptr, const int64_t (&strides)[2]) {
        return ptr == nullptr || (aligned(ptr, 16) && strides[0] % 16 == 0 && strides[1] % 16 == 0);
    };
    const bool wide = vectorRows(p.keys, p.keyStride) && vectorRows(p.values, p.valueStride) && vectorRows(p.queries, p.queryStride) &&
                      vectorRows(p.rotated, p.rotatedStride) && p.half % 8 == 0 && aligned(p.cosines, 16) && aligned(p.sines, 16) &&
                      p.angleStride % 4 == 0;
    return launchStatus(call.c_str(), k.dtype == MLEL_F16 ? (wide ? launchAppend<__half, true>(p, s) : launchAppend<__half, false>(p, s))
                                      : wide              ? launchAppend<__nv_bfloat16, true>(p, s)
                                                          : launchAppend<__nv_bfloat16, false>(p, s));
}

cudaError_t takePagedErrorAppend(int &code) { return takePagedError(code); }

} // namespace mlel
