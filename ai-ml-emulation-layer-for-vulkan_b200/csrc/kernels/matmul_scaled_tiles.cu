// The scaled int8 product on single CTAs' tcgen05 tiles of 128 output channels by 16 to 128 tokens:
//
//   D[n, m] = sum_k b[n, k] * a[m, k]          A operand: weights (128 rows), B operand: tokens
//
// and for few tokens the sum over k split over the CTAs of a cluster, which add up their 32-bit integers through distributed
// shared memory (whole numbers: the order does not matter).  With few tokens the weights' bytes bound the product: splitting puts
// every SM to reading them, and two or three CTAs an SM (96 to 108 KB each) keep one reading while another starts or ends.
// A lane of the epilogue has one channel, its scale and its bias; a warp stores 32 neighbouring channels of a token,
// which takes any alignment of the output.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "matmul_scaled.hpp"
#include "serving.hpp"
#include "serving_device.cuh"
#include "tcgen05_common.cuh"
#include "tcgen05_pair.cuh"

namespace mlel {
namespace {

using namespace tc;

constexpr int kChannels = 128; // of a tile
constexpr int kRoles = 2;      // warps in front of the epilogue's four: copies, products

template <int TN> struct TileShape {
    static constexpr int kStageBytes = (kChannels + TN) * BK;
    static constexpr int kStages = TN == 16 ? 6 : TN == 32 ? 5 : TN == 64 ? 4 : 3;
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + 1024;
    static constexpr uint32_t kTmemCols = TN < 32 ? 32 : TN;
    static_assert(kStages * kStageBytes >= TN * kChannels * 4, "the partial sums fit the stages");
};

__device__ __forceinline__ int loadShared(uint32_t clusterAddr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(clusterAddr) : "memory");
    return v;
}

template <int TN, class T>
__global__ void __launch_bounds__((kRoles + 4) * 32)
matmulScaledTiles(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const ScaledProblem p, const int split) {
    using Shape = TileShape<TN>;
    constexpr int NST = Shape::kStages;
    extern __shared__ uint8_t rawSmem[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rawSmem) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[NST], empty[NST], accFull;
    __shared__ uint32_t tmemSlot;
    const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31;
    const int rank = split > 1 ? int(clusterCtaRank()) : 0;
    const int c0 = int(blockIdx.x) / split * kChannels, m0 = int(blockIdx.y) * TN;
    const int allKb = (p.K + BK - 1) / BK, kb0 = int(int64_t(allKb) * rank / split), kb1 = int(int64_t(allKb) * (rank + 1) / split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbarInit(&full[s], 1u);
            mbarInit(&empty[s], 1u);
        }
        mbarInit(&accFull, 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&tmemSlot)), "r"(Shape::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmemSlot;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbarWait(&empty[s], phase ^ 1u, 71)) {
                    break;
                }
                uint8_t *to = smem + s * Shape::kStageBytes;
                mbarArriveExpectTx(&full[s], uint32_t(Shape::kStageBytes));
                tmaLoad3d(&mapW, to, &full[s], kb * BK, c0, 0);
                tmaLoad3d(&mapX, to + kChannels * BK, &full[s], kb * BK, m0, 0);
                s = s + 1 == NST ? 0 : s + 1;
                phase ^= s == 0 ? 1u : 0u;
            }
        }
    } else if (warp == 1) {
        // (the whole warp: see ummaBlockPeek)
        constexpr uint32_t idesc = instrDesc(TN, false);
        const DescWords w0 = descWords(smemDesc(smemAddr(smem), 16, 1024)), x0 = descWords(smemDesc(smemAddr(smem) + kChannels * BK, 16, 1024));
        uint32_t s = 0, phase = 0, ready = 0;
        bool failed = false;
        int left = p.K - kb0 * BK;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (ready == 0) {
                failed = failed || !mbarWait(&full[s], phase, 72);
            }
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t next = s + 1 == uint32_t(NST) ? 0u : s + 1, nextPhase = next == 0 ? phase ^ 1u : phase;
            const uint32_t step = s * uint32_t(Shape::kStageBytes >> 4);
            ready = ummaBlockPeek(tmem, {w0.low + step, w0.high}, UMMA_K >> 4, {x0.low + step, x0.high}, UMMA_K >> 4, idesc,
                                  kb != kb0 ? 1u : 0u, ummaCountFor(left), &empty[s], &full[next], nextPhase);
            left -= BK;
            s = next, phase = nextPhase;
        }
        ummaCommit(&accFull);
    } else {
        const int quarter = warp & 3, channel = c0 + quarter * 32 + lane;
        const bool live = channel < p.N;
        const float scale = live ? p.bScales[channel] : 0.f, bias = live && p.biases != nullptr ? p.biases[channel] : 0.f;
        const bool done = mbarWaitWarp(&accFull, 0u, 73);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        int *part = reinterpret_cast<int *>(smem);
        char *out = p.out + int64_t(channel) * int64_t(sizeof(T));
#pragma unroll 1
        for (int col = 0; col < TN && done; col += 16) {
            uint32_t r[16];
            tmemLoad16(tmem + (uint32_t(quarter * 32) << 16) + uint32_t(col), r);
            tmemWait16(r);
            if (split > 1) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    part[(col + j) * kChannels + quarter * 32 + lane] = int(r[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int m = m0 + col + j;
                    if (m < p.M && live) {
                        *reinterpret_cast<T *>(out + int64_t(m) * p.outStride) = fromFloat<T>(float(int(r[j])) * p.aScales[m] * scale + bias);
                    }
                }
            }
        }
    }
    if (split > 1) { // every CTA adds up the tokens rank, rank + split, ...
        __syncwarp();
        clusterSync();
        if (warp >= kRoles) {
            const int quarter = warp & 3, channel = c0 + quarter * 32 + lane;
            if (channel < p.N) {
                const float scale = p.bScales[channel], bias = p.biases != nullptr ? p.biases[channel] : 0.f;
                const uint32_t at = smemAddr(smem) + uint32_t(quarter * 32 + lane) * 4u;
                for (int m = rank; m < TN && m0 + m < p.M; m += split) {
                    int sum = 0;
                    for (int r = 0; r < split; ++r) {
                        sum += loadShared(mapToCta(at + uint32_t(m * kChannels * 4), uint32_t(r)));
                    }
                    *reinterpret_cast<T *>(p.out + int64_t(m0 + m) * p.outStride + int64_t(channel) * int64_t(sizeof(T))) =
                        fromFloat<T>(float(sum) * p.aScales[m0 + m] * scale + bias);
                }
            }
        }
        __syncwarp();
        clusterSync(); // nobody leaves while its sums are being read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kTmemCols) : "memory");
    }
}

template <int TN, class T> int launchTiles(const ScaledProblem &p, int split, cudaStream_t s) {
    using Shape = TileShape<TN>;
    CUtensorMap w, x;
    if (!makeMap(&w, p.b, uint64_t(p.K), uint64_t(p.N), 1, uint64_t(p.bStride), uint64_t(p.bStride) * p.N, BK, kChannels) ||
        !makeMap(&x, p.a, uint64_t(p.K), uint64_t(p.M), 1, uint64_t(p.aStride), uint64_t(p.aStride) * p.M, BK, TN)) {
        return MLEL_ERROR_DEVICE;
    }
    const auto kernel = matmulScaledTiles<TN, T>;
    if (!allowDynamicSmem(reinterpret_cast<const void *>(kernel), Shape::kSmem)) {
        return MLEL_ERROR_DEVICE;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned((p.N + kChannels - 1) / kChannels * split), unsigned((p.M + TN - 1) / TN));
    cfg.blockDim = dim3((kRoles + 4) * 32);
    cfg.dynamicSmemBytes = Shape::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2]{};
    int count = 0;
    if (dependentLaunches()) {
        attrs[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[count++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (split > 1) {
        attrs[count].id = cudaLaunchAttributeClusterDimension;
        attrs[count].val.clusterDim.x = unsigned(split), attrs[count].val.clusterDim.y = 1, attrs[count++].val.clusterDim.z = 1;
    }
    cfg.attrs = attrs;
    cfg.numAttrs = unsigned(count);
    return launchStatus("mlel_cuda_matmul_scaled", cudaLaunchKernelEx(&cfg, kernel, w, x, p, split));
}

template <int TN> int launchTilesType(const ScaledProblem &p, int32_t dtype, int split, cudaStream_t s) {
    return dtype == MLEL_F32   ? launchTiles<TN, float>(p, split, s)
           : dtype == MLEL_F16 ? launchTiles<TN, __half>(p, split, s)
                               : launchTiles<TN, __nv_bfloat16>(p, split, s);
}

} // namespace

int matmulScaledOnTiles(const ScaledProblem &p, int32_t dtype, cudaStream_t s) {
    const int width = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
    const int64_t tiles = int64_t((p.N + kChannels - 1) / kChannels) * ((p.M + width - 1) / width);
    const int allKb = (p.K + BK - 1) / BK;
    // the sum is split while that gives CTAs that the SMs have room for, and leaves each four K blocks
    int split = 1;
    while (split < 8 && tiles * split * 2 <= int64_t(smCount()) * 2 && allKb >= split * 8) {
        split *= 2;
    }
    switch (width) {
    case 16:
        return launchTilesType<16>(p, dtype, split, s);
    case 32:
        return launchTilesType<32>(p, dtype, split, s);
    case 64:
        return launchTilesType<64>(p, dtype, split, s);
    default:
        return launchTilesType<128>(p, dtype, split, s);
    }
}

int scaledTilesErrorWord() { return tc::readErrorWord(); }

} // namespace mlel
