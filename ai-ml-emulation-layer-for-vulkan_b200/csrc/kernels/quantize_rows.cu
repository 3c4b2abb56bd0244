// Rows in 8 bits with a scale found at run time: scale = max |x| / 127, q = x / scale to the nearest whole number, ties to
// the even one, decided as exact arithmetic would (see roundedQuotient).
//
// What bounds it: memory.  A row is read once: its 16-byte vectors stay in registers between the maximum and the
// rounding, four to a thread, as they lie in memory (16-bit magnitudes are compared two at a time), and as many threads share a
// row as that takes (32 to 1024; longer rows are read again).  8192 rows of 8192 f16 elements: 41 us, 4.9 TB/s; 24 rows of 5120 bf16: 3.1.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../graph_pipeline.hpp"
#include "launch_overlapped.cuh"
#include "serving.hpp"
#include "serving_device.cuh"

namespace mlel {
namespace {

constexpr int kHeld = 4; // vectors of a row that a thread keeps

struct QuantizeParams {
    const char *in;
    int8_t *out;
    float *scales;
    int64_t inStride, outStride; // bytes between rows
    int32_t rows, length;
};

// Eight elements as they lie in memory, and their largest magnitude as the bits of a float.
template <class T> struct Eight {
    uint4 w;
    __device__ void clear() { w = {0u, 0u, 0u, 0u}; }
    __device__ void load(const T *from) { w = *reinterpret_cast<const uint4 *>(from); }
    __device__ void set(int j, T x) { reinterpret_cast<T *>(&w)[j] = x; }
    __device__ void values(float (&x)[8]) const { unpackEight(w, x, T()); }
    __device__ uint32_t most() const { // (magnitudes of 16 bits are ordered like their bits, as those of floats are)
        const uint32_t m = maxHalves(maxHalves(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), maxHalves(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
        const uint32_t top = max(m & 0xffffu, m >> 16);
        const float2 f = unpackTwo(top, T());
        return __float_as_uint(f.x);
    }
};
template <> struct Eight<float> {
    float v[8];
    __device__ void clear() {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = 0.f;
        }
    }
    __device__ void load(const float *from) { loadWide(from, v); }
    __device__ void set(int j, float x) { v[j] = x; }
    __device__ void values(float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = v[j];
        }
    }
    __device__ uint32_t most() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        }
        return m;
    }
};

// Where thread `at` of a team finds the elements of its vector v: eight neighbours from (v TEAM + at) 8 on, or, for rows at any
// address, every TEAM-th from v 8 TEAM + at on, so that neighbouring threads read neighbouring elements.
template <class T, int TEAM, bool WIDE> __device__ __forceinline__ void loadEight(const T *row, int v, int at, int length, Eight<T> &x) {
    if (WIDE) {
        const int first = (v * TEAM + at) * 8;
        if (first + 8 <= length) {
            x.load(row + first);
        } else {
            x.clear();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (first + j < length) {
                    x.set(j, row[first + j]);
                }
            }
        }
    } else {
        x.clear();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = (v * 8 + j) * TEAM + at;
            if (i < length) {
                x.set(j, row[i]);
            }
        }
    }
}
template <int TEAM, bool WIDE> __device__ __forceinline__ void storeEight(int8_t *out, int v, int at, int length, uint2 packed) {
    const int first = (v * TEAM + at) * 8;
    if (WIDE && first + 8 <= length) {
        *reinterpret_cast<uint2 *>(out + first) = packed;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int i = WIDE ? first + j : (v * 8 + j) * TEAM + at;
        if (i < length) {
            out[i] = int8_t((j < 4 ? packed.x >> (8 * j) : packed.y >> (8 * (j - 4))) & 0xffu);
        }
    }
}

template <class T, int TEAM, bool WIDE>
__global__ void __launch_bounds__(TEAM < 256 ? 256 : TEAM) quantizeRowsKernel(const QuantizeParams p) {
    constexpr int kTeams = TEAM < 256 ? 256 / TEAM : 1;
    __shared__ uint32_t partial[32];
    dependencySync();
    const int team = int(threadIdx.x) / TEAM, at = int(threadIdx.x) % TEAM;
    const int64_t rowIndex = int64_t(blockIdx.x) * kTeams + team;
    const bool live = rowIndex < p.rows;
    const T *row = reinterpret_cast<const T *>(p.in + (live ? rowIndex : 0) * p.inStride);
    const int length = live ? p.length : 0, vectors = (length + 8 * TEAM - 1) / (8 * TEAM);
    Eight<T> x[kHeld];
    uint32_t most = 0; // magnitudes as bits: an infinity is above every number and a NaN above that
#pragma unroll
    for (int v = 0; v < kHeld; ++v) {
        loadEight<T, TEAM, WIDE>(row, v, at, length, x[v]);
    }
#pragma unroll
    for (int v = 0; v < kHeld; ++v) {
        most = max(most, x[v].most());
    }
    for (int v = kHeld; v < vectors; ++v) {
        Eight<T> y;
        loadEight<T, TEAM, WIDE>(row, v, at, length, y);
        most = max(most, y.most());
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (TEAM > 32) {
        const int warp = int(threadIdx.x) >> 5, firstWarp = team * (TEAM / 32);
        if ((threadIdx.x & 31) == 0) {
            partial[warp] = most;
        }
        __syncthreads();
        most = 0;
#pragma unroll
        for (int w = 0; w < TEAM / 32; ++w) {
            most = max(most, partial[firstWarp + w]);
        }
    }
    if (!live) {
        return;
    }
    const RowScale scale = rowScale(most);
    if (at == 0) {
        p.scales[rowIndex] = scale.value;
    }
    int8_t *out = p.out + rowIndex * p.outStride;
    float y[8];
#pragma unroll
    for (int v = 0; v < kHeld; ++v) {
        x[v].values(y);
        storeEight<TEAM, WIDE>(out, v, at, length, quantizeEight(y, scale));
    }
    for (int v = kHeld; v < vectors; ++v) {
        Eight<T> z;
        loadEight<T, TEAM, WIDE>(row, v, at, length, z);
        z.values(y);
        storeEight<TEAM, WIDE>(out, v, at, length, quantizeEight(y, scale));
    }
}

template <class T, int TEAM> cudaError_t launchTeam(const QuantizeParams &p, bool wide, cudaStream_t s) {
    constexpr int kTeams = TEAM < 256 ? 256 / TEAM : 1;
    const dim3 grid(unsigned((int64_t(p.rows) + kTeams - 1) / kTeams));
    constexpr unsigned threads = TEAM < 256 ? 256 : TEAM;
    return wide ? launchOverlapped(quantizeRowsKernel<T, TEAM, true>, grid, threads, 0, s, p)
                : launchOverlapped(quantizeRowsKernel<T, TEAM, false>, grid, threads, 0, s, p);
}

template <class T> cudaError_t launchType(const QuantizeParams &p, bool wide, cudaStream_t s) {
    const int vectors = (p.length + 7) / 8;
    if (vectors <= 32 * kHeld) {
        return launchTeam<T, 32>(p, wide, s);
    }
    if (vectors <= 128 * kHeld) {
        return launchTeam<T, 128>(p, wide, s);
    }
    return vectors <= 256 * kHeld ? launchTeam<T, 256>(p, wide, s) : launchTeam<T, 1024>(p, wide, s);
}

} // namespace

int quantizeRows(const mlel_tensor *input, const mlel_tensor *output, const mlel_tensor *scales, cudaStream_t s) {
    const std::string call = "mlel_cuda_quantize_rows";
    const Operand in = operandOf(call, "input", input, 2), out = writtenOperandOf(call, "output", output, 2),
                  sc = writtenOperandOf(call, "scales", scales, 1);
    if (!isFloat(in.dtype)) {
        throw UnsupportedError(call + ": input has to be f32, f16 or bf16");
    }
    wantType(call, "output", out, MLEL_I8, "int8");
    wantType(call, "scales", sc, MLEL_F32, "f32");
    if (out.dims[0] != in.dims[0] || out.dims[1] != in.dims[1] || sc.dims[0] != in.dims[0]) {
        refuse(call, "the shapes of input, output and scales do not fit together");
    }
    if (in.dims[0] == 0) {
        return MLEL_SUCCESS;
    }
    if (in.dims[1] == 0) {
        refuse(call, "rows without elements have no scale");
    }
    if (in.dims[1] > (1 << 30)) {
        refuse(call, "rows of more than 2^30 elements");
    }
    wantCurrentDevice(call, "output", out.ptr);
    const QuantizeParams p{in.ptr, reinterpret_cast<int8_t *>(out.ptr), reinterpret_cast<float *>(sc.ptr), in.strides[0], out.strides[0],
                           int32_t(in.dims[0]), int32_t(in.dims[1])};
    const bool wide = aligned(in.ptr, 16) && (in.strides[0] % 16 == 0 || p.rows == 1) && aligned(out.ptr, 8) &&
                      (out.strides[0] % 8 == 0 || p.rows == 1);
    return launchStatus(call.c_str(), in.dtype == MLEL_F32   ? launchType<float>(p, wide, s)
                                      : in.dtype == MLEL_F16 ? launchType<__half>(p, wide, s)
                                                             : launchType<__nv_bfloat16>(p, wide, s));
}

} // namespace mlel
