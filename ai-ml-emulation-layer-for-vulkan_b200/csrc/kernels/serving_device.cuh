// Device helpers of the 8-bit decoder layer's kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace mlel {

__device__ __forceinline__ float toFloat(float x) { return x; }
__device__ __forceinline__ float toFloat(__half x) { return __half2float(x); }
__device__ __forceinline__ float toFloat(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T> __device__ __forceinline__ T fromFloat(float x);
template <> __device__ __forceinline__ float fromFloat<float>(float x) { return x; }
template <> __device__ __forceinline__ __half fromFloat<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two values as one word, the first in its low half.
__device__ __forceinline__ uint32_t packTwo(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t packTwo(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpackTwo(uint32_t w, __half) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ float2 unpackTwo(uint32_t w, __nv_bfloat16) {
    return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}

template <class T> __device__ __forceinline__ void unpackEight(const uint4 &v, float (&x)[8], T) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = unpackTwo(w[j], T());
        x[2 * j] = f.x, x[2 * j + 1] = f.y;
    }
}
template <class T> __device__ __forceinline__ uint4 packEight(const float (&x)[8], T) {
    return {packTwo(x[0], x[1], T()), packTwo(x[2], x[3], T()), packTwo(x[4], x[5], T()), packTwo(x[6], x[7], T())};
}
// Eight elements at a 16-byte boundary.
template <class T> __device__ __forceinline__ void loadWide(const T *from, float (&x)[8]) {
    unpackEight(*reinterpret_cast<const uint4 *>(from), x, T());
}
__device__ __forceinline__ void loadWide(const float *from, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(from)[0], b = reinterpret_cast<const float4 *>(from)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

__device__ __forceinline__ bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Four elements from `at` on; zeros from `length` on.
__device__ __forceinline__ float4 fourOf(const float *from, int at, int length) {
    return {at < length ? from[at] : 0.f, at + 1 < length ? from[at + 1] : 0.f, at + 2 < length ? from[at + 2] : 0.f,
            at + 3 < length ? from[at + 3] : 0.f};
}

// A row's scale, from the bits of its largest magnitude.
struct RowScale {
    float value;   // what is stored
    float inverse; // 0: every element becomes 0 (an empty row, or one without a finite scale)
    bool careful;  // the scale is too small for `inverse` to mean anything
};
__device__ __forceinline__ RowScale rowScale(uint32_t mostBits) {
    RowScale r;
    const float most = __uint_as_float(mostBits);
    const bool finite = mostBits < 0x7f800000u;
    r.value = finite ? __fdiv_rn(most, 127.f) : most;
    r.careful = finite && r.value > 0.f && r.value < 1e-36f;
    r.inverse = finite && r.value > 0.f && !r.careful ? __fdiv_rn(1.f, r.value) : 0.f;
    return r;
}

// x / scale to the nearest whole number, as a float plus 1.5 * 2^23, whose low byte is then that number.  x * inverse is
// off by at most 2^-23 of itself, under 2e-5: only where it lies closer than 1e-4 to the middle between two whole
// numbers the quotient is formed in 64 bits, in which no quotient of two 32-bit floats is rounded onto such a middle.
__device__ __forceinline__ uint32_t roundedQuotient(float x, const RowScale &s) {
    constexpr float kMagic = 12582912.f;
    const float y = x * s.inverse, t = y + kMagic;
    if (__builtin_expect(s.careful || !(fabsf(y - (t - kMagic)) <= 0.4999f), 0)) {
        if (s.inverse == 0.f && !s.careful) {
            return 0u; // an infinity or a NaN in a row that has no finite scale
        }
        const int q = int(rint(double(x) / double(s.value)));
        return uint32_t(q > 127 ? 127 : q < -127 ? -127 : q);
    }
    return __float_as_uint(t);
}
// Eight at a time: the nearest whole number by one fused multiply-add, how far the product lies from it by another.  Only the
// scale's inverse is rounded there, so the distance is off by at most 2^-24 of 127.
__device__ __forceinline__ uint2 quantizeEight(const float (&x)[8], const RowScale &s) {
    if (s.inverse == 0.f && !s.careful) { // an empty row, or one without a finite scale
        return {0u, 0u};
    }
    constexpr float kMagic = 12582912.f;
    uint32_t q[8];
    float farthest = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = fmaf(x[j], s.inverse, kMagic);
        farthest = fmaxf(farthest, fabsf(fmaf(x[j], s.inverse, kMagic - t)));
        q[j] = __float_as_uint(t);
    }
    if (__builtin_expect(s.careful || farthest > 0.4999f, 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q[j] = roundedQuotient(x[j], s);
        }
    }
    uint2 r;
    r.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
    return r;
}

// The larger of two pairs of 16-bit magnitudes, by halves.
__device__ __forceinline__ uint32_t maxHalves(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

} // namespace mlel
