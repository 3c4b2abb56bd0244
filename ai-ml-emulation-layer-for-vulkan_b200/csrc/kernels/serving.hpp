// Operators of an 8-bit decoder layer behind the direct entry points mlel_cuda_quantize_rows, mlel_cuda_matmul_scaled,
// mlel_cuda_quantized_linear, mlel_cuda_paged_append and mlel_cuda_paged_attention: their launchers, and the checks of operands that they share.
// Launchers return an mlel_status, or throw what the C boundary turns into one.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "kernels.hpp"

namespace mlel {

int quantizeRows(const mlel_tensor *input, const mlel_tensor *output, const mlel_tensor *scales, cudaStream_t s);
int matmulScaled(const mlel_tensor *a, const mlel_tensor *aScales, const mlel_tensor *b, const mlel_tensor *bScales,
                 const mlel_tensor *biases, const mlel_tensor *output, cudaStream_t s);
int quantizedLinear(const mlel_tensor *input, const mlel_tensor *b, const mlel_tensor *bScales, const mlel_tensor *biases,
                    const mlel_tensor *output, void *workspace, uint64_t workspaceBytes, cudaStream_t s);
int pagedAppend(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *keys, const mlel_tensor *values,
                const mlel_tensor *cosines, const mlel_tensor *sines, const mlel_tensor *queries, const mlel_tensor *rotated,
                int interleaved, cudaStream_t s);
int pagedAttention(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *queries,
                   const mlel_tensor *output, float scale, int causal, int window, float softcap, void *workspace,
                   uint64_t workspaceBytes, cudaStream_t s);
uint64_t pagedAttentionWorkspace(const mlel_paged_cache *cache, const mlel_paged_batch *batch, const mlel_tensor *queries);

// The words in which the kernels of the paged cache record what they left out, read into `code` where that is still 0 and cleared.
cudaError_t takePagedErrorAppend(int &code);
cudaError_t takePagedErrorAttention(int &code);

// An operand of a direct call with its strides filled in.
struct Operand {
    char *ptr;
    int32_t dtype, rank;
    int64_t dims[kMaxRank], strides[kMaxRank]; // strides in bytes
    int64_t count() const {
        int64_t n = 1;
        for (int i = 0; i < rank; ++i) {
            n *= dims[i];
        }
        return n;
    }
};

[[noreturn]] inline void refuse(const std::string &call, const std::string &what) { throw std::runtime_error(call + ": " + what); }

// Checks what every operand has to be: a described tensor of `rank` axes, elements of the last axis side by side, the
// other axes at whole elements from one another, on a boundary of its type.
inline Operand operandOf(const std::string &call, const char *name, const mlel_tensor *t, int rank) {
    if (t == nullptr) {
        refuse(call, std::string(name) + " is missing");
    }
    Operand o{};
    o.ptr = static_cast<char *>(t->data), o.dtype = t->desc.dtype, o.rank = t->desc.rank;
    if (o.rank != rank) {
        refuse(call, std::string(name) + " has " + std::to_string(o.rank) + " axes, not " + std::to_string(rank));
    }
    const int size = elemSize(o.dtype);
    if (size <= 0) {
        refuse(call, std::string(name) + " has no known element type");
    }
    int64_t packed = size, most = (int64_t(1) << 46);
    for (int i = rank - 1; i >= 0; --i) {
        o.dims[i] = t->desc.dims[i];
        if (o.dims[i] < 0 || o.dims[i] > 0x7fffffff) {
            refuse(call, std::string(name) + " has an axis of " + std::to_string(o.dims[i]));
        }
        o.strides[i] = t->desc.strides[0] == 0 ? packed : t->desc.strides[i];
        if (o.dims[i] > 0 && packed > most / o.dims[i]) {
            refuse(call, std::string(name) + " is too large");
        }
        packed *= o.dims[i] > 0 ? o.dims[i] : 1;
    }
    if (o.count() == 0) {
        return o;
    }
    if (o.ptr == nullptr || reinterpret_cast<uintptr_t>(o.ptr) % uintptr_t(size) != 0) {
        refuse(call, std::string(name) + " is null or not on a boundary of its element type");
    }
    for (int i = 0; i < rank; ++i) {
        const bool last = i == rank - 1;
        if (o.dims[i] > 1 && (last ? o.strides[i] != size : o.strides[i] <= 0 || o.strides[i] % size != 0 || o.strides[i] > most)) {
            refuse(call, std::string(name) + (last ? ": the elements of the last axis have to lie side by side"
                                                   : ": strides have to be positive whole elements"));
        }
        if (o.dims[i] == 1) { // never taken: any value would do
            o.strides[i] = last ? size : packed;
        }
    }
    return o;
}

// The same for an operand that is written: no two of its elements may share an address.
inline Operand writtenOperandOf(const std::string &call, const char *name, const mlel_tensor *t, int rank) {
    const Operand o = operandOf(call, name, t, rank);
    int64_t extent = elemSize(o.dtype);
    bool done[kMaxRank] = {};
    for (int n = 0; n < rank && o.count() > 0; ++n) { // axes by growing stride, each beyond the extent of those before it
        int next = -1;
        for (int i = 0; i < rank; ++i) {
            if (!done[i] && (next < 0 || o.strides[i] < o.strides[next])) {
                next = i;
            }
        }
        done[next] = true;
        if (o.dims[next] > 1) {
            if (o.strides[next] < extent) {
                refuse(call, std::string(name) + " is written, but parts of it overlap");
            }
            extent = o.strides[next] * (o.dims[next] - 1) + extent;
        }
    }
    return o;
}

inline void wantPacked(const std::string &call, const char *name, const Operand &o) {
    int64_t below = elemSize(o.dtype);
    for (int i = o.rank - 1; i >= 0 && o.count() > 0; --i) {
        if (o.dims[i] > 1 && o.strides[i] != below) {
            refuse(call, std::string(name) + " has to be packed");
        }
        below *= o.dims[i];
    }
}

inline void wantType(const std::string &call, const char *name, const Operand &o, int32_t dtype, const char *typeName) {
    if (o.dtype != dtype) {
        refuse(call, std::string(name) + " has to be " + typeName);
    }
}
inline bool isFloat(int32_t dtype) { return dtype == MLEL_F16 || dtype == MLEL_BF16 || dtype == MLEL_F32; }

inline bool aligned(const void *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % uintptr_t(bytes) == 0; }

// Work goes to the device that is current: refuses memory of another device (an address that the driver does not know
// is refused too).  Called when the arguments are otherwise in order.
inline void wantCurrentDevice(const std::string &call, const char *name, const void *p) {
    int device = 0;
    cudaPointerAttributes at{};
    if (cudaGetDevice(&device) != cudaSuccess || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        refuse(call, "no CUDA device");
    }
    if ((at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) || (at.type == cudaMemoryTypeDevice && at.device != device)) {
        refuse(call, std::string(name) + " is not in the memory of the current device");
    }
}

inline int launchStatus(const char *call, cudaError_t err) {
    if (err != cudaSuccess) {
        setLastError(std::string(call) + ": launch failed: " + cudaGetErrorString(err));
        return MLEL_ERROR_DEVICE;
    }
    return MLEL_SUCCESS;
}

} // namespace mlel
