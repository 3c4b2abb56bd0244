// The scaled int8 product on single CTAs' tcgen05 tiles of 128 output channels by 16 to 128 tokens:
//
//   D[n, m] = sum_k b[n, k] * a[m, k]          A operand: weights (128 rows), B operand: tokens
//
// and for few tokens the sum over k split over the CTAs of a cluster, which add up their 32-bit integers through distributed
// shared memory (whole numbers: the order does not matter).  With few tokens the weights' bytes bound the product: splitting puts
// every SM to reading them.  What an SM reads at a time decides how fast that is: its CTAs, one to three, share some 200 KB of
// stages (96 KB to a lone CTA of 512 x 4096 x 4096: 24 us, a K block every 1100 cycles).
// A lane of the epilogue puts its channel's sums into shared memory, token by token; then a warp takes a token at a time, four
// neighbouring channels a lane, from every CTA of the cluster, which takes any alignment of the output.  (One channel a lane and
// a 32-bit read per token and CTA: 256 x 4096 x 4096 36 us with its quantisation.)
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "matmul_scaled.hpp"
#include "serving.hpp"
#include "serving_device.cuh"
#include "serving_wait.cuh"
#include "tcgen05_common.cuh"
#include "tcgen05_pair.cuh"

namespace mlel {
namespace {

using namespace tc;

constexpr int kChannels = 128; // of a tile
constexpr int kRoles = 2;      // warps in front of the epilogue's four: copies, products

constexpr int kMostStages = 8;

template <int TN> struct TileShape {
    static constexpr int kStageBytes = (kChannels + TN) * BK;
    static constexpr int kLeastStages = (TN * kChannels * 4 + kStageBytes - 1) / kStageBytes; // hold the partial sums at the end
    static constexpr uint32_t kTmemCols = TN < 32 ? 32 : TN;
};

// Barrier among the epilogue's four warps (named barrier 1).
__device__ __forceinline__ void epilogueBarrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ int4 loadShared(uint32_t clusterAddr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(clusterAddr) : "memory");
    return v;
}
// Four neighbouring values of the output.
__device__ __forceinline__ uint4 packFour(const float4 &y, float) {
    return {__float_as_uint(y.x), __float_as_uint(y.y), __float_as_uint(y.z), __float_as_uint(y.w)};
}
template <class T> __device__ __forceinline__ uint2 packFour(const float4 &y, T) { return {packTwo(y.x, y.y, T()), packTwo(y.z, y.w, T())}; }

template <int TN, class T>
__global__ void __launch_bounds__((kRoles + 4) * 32)
matmulScaledTiles(const __grid_constant__ CUtensorMap mapW, const __grid_constant__ CUtensorMap mapX, const ScaledProblem p, const int split,
                  const int stages) {
    using Shape = TileShape<TN>;
    extern __shared__ uint8_t rawSmem[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rawSmem) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[kMostStages], empty[kMostStages], accFull;
    __shared__ uint32_t tmemSlot;
    __shared__ float tokenScales[TN];
    const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31;
    const int rank = split > 1 ? int(clusterCtaRank()) : 0;
    const int c0 = int(blockIdx.x) / split * kChannels, m0 = int(blockIdx.y) * TN;
    const int allKb = (p.K + BK - 1) / BK, kb0 = int(int64_t(allKb) * rank / split), kb1 = int(int64_t(allKb) * (rank + 1) / split);
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
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
                if (!mbarPoll(&empty[s], phase ^ 1u, 71)) {
                    break;
                }
                uint8_t *to = smem + s * Shape::kStageBytes;
                mbarArriveExpectTx(&full[s], uint32_t(Shape::kStageBytes));
                tmaLoad3d(&mapW, to, &full[s], kb * BK, c0, 0);
                tmaLoad3d(&mapX, to + kChannels * BK, &full[s], kb * BK, m0, 0);
                s = s + 1 == stages ? 0 : s + 1;
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
                failed = failed || !mbarPoll(&full[s], phase, 72);
            }
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t next = s + 1 == uint32_t(stages) ? 0u : s + 1, nextPhase = next == 0 ? phase ^ 1u : phase;
            const uint32_t step = s * uint32_t(Shape::kStageBytes >> 4);
            ready = ummaBlockPeek(tmem, {w0.low + step, w0.high}, UMMA_K >> 4, {x0.low + step, x0.high}, UMMA_K >> 4, idesc,
                                  kb != kb0 ? 1u : 0u, ummaCountFor(left), &empty[s], &full[next], nextPhase);
            left -= BK;
            s = next, phase = nextPhase;
        }
        ummaCommit(&accFull);
    } else {
        for (int m = int(threadIdx.x) - kRoles * 32; m < TN; m += 128) {
            tokenScales[m] = m0 + m < p.M ? p.aScales[m0 + m] : 0.f;
        }
        const int quarter = warp & 3;
        const bool done = mbarPollWarp(&accFull, 0u, 73);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        int *part = reinterpret_cast<int *>(smem) + quarter * 32 + lane;
#pragma unroll 2
        for (int col = 0; col < TN && done; col += 16) {
            uint32_t r[16];
            tmemLoad16(tmem + (uint32_t(quarter * 32) << 16) + uint32_t(col), r);
            tmemWait16(r);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                part[(col + j) * kChannels] = int(r[j]);
            }
        }
        epilogueBarrier();
    }
    __syncwarp();
    if (split > 1) {
        clusterSync();
    }
    if (warp >= kRoles) { // tokens rank, rank + split, ... of the tile, a warp each in turn
        const int channel = c0 + 4 * lane;
        const float4 scale = fourOf(p.bScales, channel, p.N);
        const float4 bias = p.biases != nullptr ? fourOf(p.biases, channel, p.N) : float4{};
        const bool wide = channel + 4 <= p.N && (reinterpret_cast<uintptr_t>(p.out) | uintptr_t(p.outStride)) % (4 * sizeof(T)) == 0;
        const uint32_t at = smemAddr(smem) + uint32_t(lane) * 16u;
#pragma unroll 4
        for (int m = rank + split * (warp - kRoles); m < TN; m += split * 4) {
            if (m0 + m < p.M) {
                int4 sum = {0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r < split) {
                        const uint32_t from = at + uint32_t(m * kChannels * 4);
                        const int4 v = loadShared(split > 1 ? mapToCta(from, uint32_t(r)) : from);
                        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                    }
                }
                const float token = tokenScales[m];
                const float4 y = {float(sum.x) * token * scale.x + bias.x, float(sum.y) * token * scale.y + bias.y,
                                  float(sum.z) * token * scale.z + bias.z, float(sum.w) * token * scale.w + bias.w};
                T *out = reinterpret_cast<T *>(p.out + int64_t(m0 + m) * p.outStride) + channel;
                if (wide) {
                    *reinterpret_cast<decltype(packFour(y, T())) *>(out) = packFour(y, T());
                } else {
                    const float v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (channel + j < p.N) {
                            out[j] = fromFloat<T>(v[j]);
                        }
                    }
                }
            }
        }
    }
    if (split > 1) {
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
    // CTAs that an SM gets, and the stages that each has room for
    const int64_t ctas = int64_t((p.N + kChannels - 1) / kChannels) * split * ((p.M + TN - 1) / TN);
    const int perSm = ctas <= smCount() ? 1 : ctas <= 2 * int64_t(smCount()) || TN == 128 ? 2 : 3;
    const int ownKb = ((p.K + BK - 1) / BK + split - 1) / split;
    const int stages = std::max(Shape::kLeastStages, std::min({kMostStages, 200 * 1024 / perSm / Shape::kStageBytes, std::max(2, ownKb)}));
    const size_t smemBytes = size_t(stages) * Shape::kStageBytes + 1024;
    if (!allowDynamicSmem(reinterpret_cast<const void *>(kernel), size_t(std::min(kMostStages, 200 * 1024 / Shape::kStageBytes)) * Shape::kStageBytes + 1024)) {
        return MLEL_ERROR_DEVICE;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned((p.N + kChannels - 1) / kChannels * split), unsigned((p.M + TN - 1) / TN));
    cfg.blockDim = dim3((kRoles + 4) * 32);
    cfg.dynamicSmemBytes = smemBytes;
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
    return launchStatus("mlel_cuda_matmul_scaled", cudaLaunchKernelEx(&cfg, kernel, w, x, p, split, stages));
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
    // What a tile's sum is split into: as the SM with the most CTAs sees it, each CTA costs its K blocks and as much as three more
    // for its start and end.  (56 x 8192 x 10240, 80 tiles of 64 K blocks: 28 us in 2 parts, 20 in 5.)
    const int64_t sms = smCount(), resident = (width == 128 ? 2 : 3) * sms;
    int split = 1;
    int64_t best = 0;
    for (int parts = 1; parts <= 8 && (parts == 1 || (parts * 4 <= allKb && tiles * parts <= resident)); ++parts) {
        const int64_t cost = (tiles * parts + sms - 1) / sms * ((allKb + parts - 1) / parts + 3);
        if (parts == 1 || cost < best) {
            split = parts, best = cost;
        }
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
