// Device helpers of the kernels that attend to the paged int8 cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "paged_attention.hpp"
#include "serving_device.cuh"

namespace mlel {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2Fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap * tanh(x / cap), `perCap` being 1 / cap.  As cap * (1 - 2 / (e^(2 x / cap) + 1)) it is off by a few units in cap's last place:
// enough up to kWideCap, where that is 5e-5 of a score's logarithm and weights are rounded to f16.  For larger caps below a half of
// them, where the difference cancels, by the continued fraction of tanh z cut off after 9, z (945 + 105 z^2 + z^4) / (945 + 420 z^2 +
// 15 z^4), which is off by 1e-10 of itself.  (That for all caps: chunks at 256 elements a head 71 us for 55, prompts 213 for 159.)
constexpr float kWideCap = 128.f;
template <bool WIDE> __device__ __forceinline__ float softCapped(float x, float cap, float perCap) {
    const float e = exp2Fast(x * (2.f * kLog2e * perCap));
    if (!WIDE) {
        return cap * (1.f - __fdividef(2.f, e + 1.f));
    }
    const float z = x * perCap, square = z * z;
    const bool small = fabsf(z) < 0.5f;
    const float over = small ? x * fmaf(square, fmaf(square, 1.f / 945.f, 1.f / 9.f), 1.f) : 2.f;
    const float under = small ? fmaf(square, fmaf(square, 1.f / 63.f, 4.f / 9.f), 1.f) : e + 1.f;
    const float q = __fdividef(over, under);
    return small ? q : fmaf(-cap, q, cap);
}
// The larger magnitude; infinities and NaNs are above all numbers.
__device__ __forceinline__ float maxBits(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}
// The power of two that brings a row whose largest magnitude is `most` to [2^14, 2^15), as far as it is a normal number; 1 for
// rows that are not finite.
__device__ __forceinline__ float halfUnit(float most) {
    const int e = int(__float_as_uint(most) >> 23);
    return e == 255 ? 1.f : __uint_as_float(uint32_t(max(e - 14, 1)) << 23);
}
// The smallest power of two that is not below a positive finite x (2^127 above that).
__device__ __forceinline__ float powerAbove(float x) {
    const uint32_t bits = __float_as_uint(x), e = (bits >> 23) + ((bits & 0x7fffffu) != 0u ? 1u : 0u);
    return __uint_as_float((e < 1u ? 1u : e > 254u ? 254u : e) << 23);
}

// Four signed bytes as f16: u = x + 128 in the low mantissa bits of 1024, minus 1152.
__device__ __forceinline__ uint32_t minus1152(uint32_t two) {
    const uint32_t bias = 0x64806480u; // 1152, 1152
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&two), *reinterpret_cast<const __half2 *>(&bias));
    return *reinterpret_cast<const uint32_t *>(&y);
}
__device__ __forceinline__ void bytesToHalves(uint32_t word, uint32_t &low, uint32_t &high) {
    const uint32_t u = word ^ 0x80808080u;
    low = minus1152(__byte_perm(u, 0x64646464u, 0x4140));
    high = minus1152(__byte_perm(u, 0x64646464u, 0x4342));
}
// Four signed bytes x as the subnormal halves (x + 128) 2^-24.
__device__ __forceinline__ void bytesToSubnormals(uint32_t word, uint32_t &low, uint32_t &high) {
    const uint32_t u = word ^ 0x80808080u;
    low = __byte_perm(u, 0u, 0x4140), high = __byte_perm(u, 0u, 0x4342);
}
// 8 x 8 halves, lane (g, t) holding row g, columns 2 t and 2 t + 1: the same of the transposed matrix.
__device__ __forceinline__ uint32_t transposeHalves(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float4 loadCluster(uint32_t clusterAddr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(clusterAddr) : "memory");
    return v;
}
// Byte d of `a` and of `b` side by side as f16, d = 0 .. 3.
__device__ __forceinline__ void transposeToHalves(uint32_t a, uint32_t b, uint32_t (&out)[4]) {
    bytesToHalves(__byte_perm(a, b, 0x5140), out[0], out[1]);
    bytesToHalves(__byte_perm(a, b, 0x7362), out[2], out[3]);
}

__device__ __forceinline__ void mmaF16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ldsVector(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 ldsPair(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
// Address of the 16 bytes `chunk` of row `row` of 16 rows of DP bytes, as the swizzled boxes of a bulk copy lay them down.
template <int DP> __device__ __forceinline__ uint32_t panelAddr(uint32_t base, int row, int chunk) {
    if (DP < 128) {
        return base + uint32_t(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
    }
    return base + uint32_t((chunk >> 3) * 2048 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// Elements first .. first + 15 of a query, two to a word; zeros from `length` (a multiple of 16) on.
template <class T>
__device__ __forceinline__ void loadQuerySixteen(const T *q, int first, int length, bool wide, uint32_t (&words)[8]) {
    if (first >= length) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            words[j] = 0u;
        }
    } else if (wide) {
        const uint4 a = reinterpret_cast<const uint4 *>(q + first)[0], b = reinterpret_cast<const uint4 *>(q + first)[1];
        words[0] = a.x, words[1] = a.y, words[2] = a.z, words[3] = a.w, words[4] = b.x, words[5] = b.y, words[6] = b.z, words[7] = b.w;
    } else {
        const uint16_t *e = reinterpret_cast<const uint16_t *>(q + first);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            words[j] = uint32_t(e[2 * j]) | uint32_t(e[2 * j + 1]) << 16;
        }
    }
}

// What turns units of 2^from into units of 2^to, both maxima of one row and from <= to.
__device__ __forceinline__ float unitsOf(float from, float to) { return from == to ? 1.f : exp2Fast(from - to); }
// Logarithm of a value scale: that of the smallest number for 0, NaN for what is not finite.
__device__ __forceinline__ float logOfScale(float scale) {
    const float y = log2f(scale);
    return y < -150.f ? -150.f : y;
}
// Four elements of one row of the answer: y / sum * 2^exponent, or zeros for a row that nothing was added to.
template <class T>
__device__ __forceinline__ void writeOut(const AttendParams &p, int firstToken, int row, int head, int d, float4 y, float sum, float exponent) {
    if (d >= p.cache.headDim) {
        return;
    }
    const int token = row / p.group, queryHead = head * p.group + row - token * p.group;
    T *to = reinterpret_cast<T *>(p.out + int64_t(firstToken + token) * p.outStride[0] + queryHead * p.outStride[1]) + d;
    // (in two halves: the power of two may be outside the normal numbers where the result is not)
    const float unit = sum == 0.f ? 0.f : exp2Fast(0.5f * exponent), f = sum == 0.f ? 0.f : unit / sum;
    const uint2 packed = {packTwo(y.x * f * unit, y.y * f * unit, T()), packTwo(y.z * f * unit, y.w * f * unit, T())};
    if (p.wideOut) {
        *reinterpret_cast<uint2 *>(to) = packed;
    } else {
        uint16_t *e = reinterpret_cast<uint16_t *>(to);
        e[0] = uint16_t(packed.x), e[1] = uint16_t(packed.x >> 16), e[2] = uint16_t(packed.y), e[3] = uint16_t(packed.y >> 16);
    }
}

} // namespace mlel
