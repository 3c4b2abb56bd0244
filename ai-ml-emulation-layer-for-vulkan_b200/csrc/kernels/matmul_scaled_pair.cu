// The scaled int8 product on pairs of CTAs (tcgen05.mma.cta_group::2): a tile is 256 tokens by BN output channels,
//
//   D[m, n] = sum_k a[m, k] * b[n, k]          A operand: tokens, 128 rows from each CTA; B operand: weights, BN / 2 rows from each
//
// with the protocol of the pair in gemm_i8_pair.cu's head (barriers full, empty, accFull, accEmpty), persistent over the tiles, two
// accumulators, so that the epilogue of a tile runs under the products of the next.
//
// What bounds it: the tensor pipe.  A K block of 128 takes a pair 512 cycles at BN = 256 and brings each CTA 32 KB.  8192 x 8192 x 8192:
// 369 us, 2.98 POP/s.
//
// Epilogue: a lane has one token, its columns are neighbouring channels: integer to float, times the two scales, plus the bias, packed
// and put into a 128-byte swizzled box of 32 rows of the warp's own, which a bulk tensor store takes to the output.  No
// barrier between the warps.
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

constexpr int kEpiWarps = 8, kFirstEpi = 4; // warps 0 products, 1 copies, 2 and 3 idle
constexpr int kBoxBytes = 32 * 128;

template <int BN> struct PairShape {
    static constexpr int kTileA = 128 * BK, kTileB = BN / 2 * BK, kStageBytes = kTileA + kTileB;
    static constexpr int kStages = BN == 256 ? 5 : 6;
    static constexpr size_t kSmem = size_t(kStages) * kStageBytes + 2 * kEpiWarps * kBoxBytes + 1024;
    static constexpr uint32_t kTmemCols = 2 * BN;
};

struct PairBarriers {
    uint64_t full[6], empty[6], accFull[2], accEmpty[2];
    uint32_t tmemBase;
};

__device__ __forceinline__ void tmemLoad32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
                   "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
                   "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmemWait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                   "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// 16 bytes of the output at a time: four f32, or eight of 16 bits.
__device__ __forceinline__ uint4 packVector(const float *y, float) {
    return {__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
}
template <class T> __device__ __forceinline__ uint4 packVector(const float *y, T) {
    return {packTwo(y[0], y[1], T()), packTwo(y[2], y[3], T()), packTwo(y[4], y[5], T()), packTwo(y[6], y[7], T())};
}

template <int BN, class T>
__global__ void __launch_bounds__((kFirstEpi + kEpiWarps) * 32, 1)
matmulScaledPair(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                 const __grid_constant__ CUtensorMap mapOut, const ScaledProblem p, const FastDiv tilesM) {
    using Shape = PairShape<BN>;
    constexpr int NST = Shape::kStages;
    extern __shared__ uint8_t rawSmem[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rawSmem) + 1023) & ~uintptr_t(1023));
    uint8_t *tilesA = smem, *tilesB = smem + NST * Shape::kTileA, *boxes = smem + NST * Shape::kStageBytes;
    __shared__ PairBarriers bars;
    const int warp = int(threadIdx.x) >> 5, lane = int(threadIdx.x) & 31;
    const uint32_t rank = clusterCtaRank();
    const int first = int(blockIdx.x >> 1), pairs = int(gridDim.x >> 1);
    const int numKb = (p.K + BK - 1) / BK, tiles = int(tilesM.d) * ((p.N + BN - 1) / BN);
    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbarInit(&bars.full[s], 1u);
            mbarInit(&bars.empty[s], 1u);
        }
        for (int b = 0; b < 2; ++b) {
            mbarInit(&bars.accFull[b], 1u);
            mbarInit(&bars.accEmpty[b], uint32_t(2 * kEpiWarps));
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddr(&bars.tmemBase)),
                     "r"(Shape::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    clusterSync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmemBase = bars.tmemBase;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 1) {
        if (lane == 0) {
            const uint32_t fullLeader = mapToCta(smemAddr(&bars.full[0]), 0u);
            uint32_t ready = 0, phase = 0;
            int s = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += pairs) {
                const int column = int(fastDiv(uint32_t(t), tilesM)), m0 = (t - column * int(tilesM.d)) * 256 + int(rank) * 128,
                          n0 = column * BN + int(rank) * (BN / 2);
                for (int kb = 0; kb < numKb; ++kb) {
                    if (ready == 0) {
                        ok = mbarPoll(&bars.empty[s], phase ^ 1u, 81);
                        if (!ok) {
                            break;
                        }
                    }
                    const int next = s + 1 == NST ? 0 : s + 1;
                    const uint32_t nextPhase = next == 0 ? phase ^ 1u : phase;
                    ready = tmaStagePeekTiledPair(&bars.full[s], rank == 0 ? uint32_t(2 * Shape::kStageBytes) : 0u,
                                                  fullLeader + uint32_t(s) * 8u, &mapA, tilesA + s * Shape::kTileA, kb * BK, m0, 0, &mapB,
                                                  tilesB + s * Shape::kTileB, kb * BK, n0, 0, &bars.empty[next], nextPhase ^ 1u);
                    s = next, phase = nextPhase;
                }
            }
        }
    } else if (warp == 0) {
        if (rank == 0) { // (the whole warp: see ummaBlockPeek)
            constexpr uint32_t idesc = instrDescPair(BN, false);
            const DescWords a0 = descWords(smemDesc(smemAddr(tilesA), 16, 1024)), b0 = descWords(smemDesc(smemAddr(tilesB), 16, 1024));
            const uint32_t emptyOwn = smemAddr(&bars.empty[0]), emptyPeer = mapToCta(emptyOwn, 1u);
            const uint32_t accFullOwn = smemAddr(&bars.accFull[0]), accFullPeer = mapToCta(accFullOwn, 1u);
            uint32_t s = 0, phase = 0, count = 0, ready = 0;
            bool failed = false;
            for (int t = first; t < tiles; t += pairs, ++count) {
                const uint32_t buf = count & 1u;
                failed = failed || !mbarPoll(&bars.accEmpty[buf], ((count >> 1) & 1u) ^ 1u, 82);
                __syncwarp();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                int left = p.K;
                for (int kb = 0; kb < numKb; ++kb) {
                    if (ready == 0) {
                        failed = failed || !mbarPoll(&bars.full[s], phase, 83);
                    }
                    __syncwarp();
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t next = s + 1 == uint32_t(NST) ? 0u : s + 1, nextPhase = next == 0 ? phase ^ 1u : phase;
                    ready = ummaBlockPeekPair(tmemBase + buf * uint32_t(BN), {a0.low + s * uint32_t(Shape::kTileA >> 4), a0.high}, UMMA_K >> 4,
                                              {b0.low + s * uint32_t(Shape::kTileB >> 4), b0.high}, UMMA_K >> 4, idesc, kb != 0 ? 1u : 0u,
                                              ummaCountFor(left), emptyOwn + s * 8u, emptyPeer + s * 8u, &bars.full[next], nextPhase);
                    left -= BK;
                    s = next, phase = nextPhase;
                }
                ummaCommitPair(accFullOwn + buf * 8u);
                ummaCommitPair(accFullPeer + buf * 8u);
            }
        }
    } else if (warp >= kFirstEpi) {
        constexpr int kColumns = 128 / int(sizeof(T)), kVector = 16 / int(sizeof(T)); // of a box, of 16 bytes
        const int own = warp - kFirstEpi, quarter = warp & 3, half = own >> 2;
        uint8_t *box = boxes + own * 2 * kBoxBytes;
        const uint32_t accEmpty = mapToCta(smemAddr(&bars.accEmpty[0]), 0u);
        const bool wideScales = aligned16(p.bScales) && (p.biases == nullptr || aligned16(p.biases));
        uint32_t count = 0, boxCount = 0;
        for (int t = first; t < tiles; t += pairs, ++count) {
            const uint32_t buf = count & 1u;
            const int column = int(fastDiv(uint32_t(t), tilesM));
            const int row0 = (t - column * int(tilesM.d)) * 256 + int(rank) * 128 + quarter * 32, n0 = column * BN + half * (BN / 2);
            const float rowScale = row0 + lane < p.M ? p.aScales[row0 + lane] : 0.f;
            if (!mbarPollWarp(&bars.accFull[buf], (count >> 1) & 1u, 84)) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t from = tmemBase + buf * uint32_t(BN) + (uint32_t(quarter * 32) << 16) + uint32_t(half * (BN / 2));
#pragma unroll 1
            for (int col = 0; col < BN / 2; col += kColumns, ++boxCount) {
                uint8_t *to = box + (boxCount & 1u) * kBoxBytes;
                if (lane == 0) { // the store before the last has read this box
                    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                }
                __syncwarp();
#pragma unroll
                for (int part = 0; part < kColumns; part += 32) {
                    uint32_t r[32];
                    tmemLoad32(from + uint32_t(col + part), r);
                    tmemWait32(r);
                    const int n = n0 + col + part;
#pragma unroll
                    for (int v = 0; v < 32; v += kVector) {
                        float y[kVector];
#pragma unroll
                        for (int j = 0; j < kVector; j += 4) {
                            const int at = n + v + j;
                            float4 scale = {}, bias = {};
                            if (wideScales && at + 4 <= p.N) {
                                scale = *reinterpret_cast<const float4 *>(p.bScales + at);
                                if (p.biases != nullptr) {
                                    bias = *reinterpret_cast<const float4 *>(p.biases + at);
                                }
                            } else {
                                scale = fourOf(p.bScales, at, p.N);
                                if (p.biases != nullptr) {
                                    bias = fourOf(p.biases, at, p.N);
                                }
                            }
                            y[j] = float(int(r[v + j])) * rowScale * scale.x + bias.x;
                            y[j + 1] = float(int(r[v + j + 1])) * rowScale * scale.y + bias.y;
                            y[j + 2] = float(int(r[v + j + 2])) * rowScale * scale.z + bias.z;
                            y[j + 3] = float(int(r[v + j + 3])) * rowScale * scale.w + bias.w;
                        }
                        const int chunk = (part + v) / kVector;
                        *reinterpret_cast<uint4 *>(to + lane * 128 + ((chunk ^ (lane & 7)) << 4)) = packVector(y, T());
                    }
                }
                if (col + kColumns == BN / 2) { // the accumulator has been read
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(accEmpty + buf * 8u) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (row0 < p.M && n0 + col < p.N) {
                        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                                         reinterpret_cast<uint64_t>(&mapOut)),
                                     "r"(smemAddr(to)), "r"(n0 + col), "r"(row0), "r"(0)
                                     : "memory");
                    }
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        }
        if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
        __syncwarp();
    }
    // neither CTA leaves, or releases tensor memory, while the other's products, commits or arrivals can still reach it
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncwarp();
    clusterSync();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmemBase), "r"(Shape::kTmemCols) : "memory");
    }
}

// The output as boxes of 128 bytes by 32 rows, 128-byte swizzle.
bool makeOutMap(CUtensorMap *map, const ScaledProblem &p, int32_t dtype) {
    EncodeTiledFn fn = encodeTiled();
    if (fn == nullptr) {
        setLastError("cuTensorMapEncodeTiled is not available from the driver");
        return false;
    }
    const int size = dtype == MLEL_F32 ? 4 : 2;
    const cuuint64_t dims[3] = {cuuint64_t(p.N), cuuint64_t(p.M), 1}, strides[2] = {cuuint64_t(p.outStride), cuuint64_t(p.outStride) * p.M};
    const cuuint32_t box[3] = {cuuint32_t(128 / size), 32, 1}, elemStrides[3] = {1, 1, 1};
    const MapKey key{{7, reinterpret_cast<uint64_t>(p.out), dims[0], dims[1], strides[0], uint64_t(size)}};
    return rememberedMap(map, key, [&](CUtensorMap *m) {
        const CUresult rc = fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, p.out, dims, strides, box,
                               elemStrides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (rc != CUDA_SUCCESS) {
            setLastError("cuTensorMapEncodeTiled failed with code " + std::to_string(int(rc)));
        }
        return rc == CUDA_SUCCESS;
    });
}

template <int BN, class T> int launchPair(const ScaledProblem &p, int32_t dtype, cudaStream_t s) {
    using Shape = PairShape<BN>;
    CUtensorMap a, b, out;
    if (!makeMap(&a, p.a, uint64_t(p.K), uint64_t(p.M), 1, uint64_t(p.aStride), uint64_t(p.aStride) * p.M, BK, 128) ||
        !makeMap(&b, p.b, uint64_t(p.K), uint64_t(p.N), 1, uint64_t(p.bStride), uint64_t(p.bStride) * p.N, BK, BN / 2) ||
        !makeOutMap(&out, p, dtype)) {
        return MLEL_ERROR_DEVICE;
    }
    const auto kernel = matmulScaledPair<BN, T>;
    if (!allowDynamicSmem(reinterpret_cast<const void *>(kernel), Shape::kSmem)) {
        return MLEL_ERROR_DEVICE;
    }
    const int64_t tilesM = (int64_t(p.M) + 255) / 256, tiles = tilesM * ((p.N + BN - 1) / BN);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(2 * std::min<int64_t>(tiles, smCount() / 2)));
    cfg.blockDim = dim3((kFirstEpi + kEpiWarps) * 32);
    cfg.dynamicSmemBytes = Shape::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = 2, attrs[0].val.clusterDim.y = 1, attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = dependentLaunches() ? 2 : 1;
    return launchStatus("mlel_cuda_matmul_scaled", cudaLaunchKernelEx(&cfg, kernel, a, b, out, p, makeFastDiv(tilesM)));
}

template <int BN> int launchPairType(const ScaledProblem &p, int32_t dtype, cudaStream_t s) {
    return dtype == MLEL_F32   ? launchPair<BN, float>(p, dtype, s)
           : dtype == MLEL_F16 ? launchPair<BN, __half>(p, dtype, s)
                               : launchPair<BN, __nv_bfloat16>(p, dtype, s);
}

} // namespace

bool matmulScaledOnPairs(const ScaledProblem &p, int32_t dtype, cudaStream_t s, int *rc) {
    // the bulk stores want rows of the output on 16-byte boundaries
    if (!aligned(p.out, 16) || p.outStride % 16 != 0) {
        return false;
    }
    // Tiles of 256 or 128 channels, whichever ends sooner: rounds over the pairs, each K block 512 cycles or, bound by the bytes that
    // arrive, some 300, an epilogue as much as two of them.
    const int64_t pairs = smCount() / 2, rows = (int64_t(p.M) + 255) / 256, numKb = (p.K + BK - 1) / BK;
    const int64_t wide = rows * ((p.N + 255) / 256), narrow = rows * ((p.N + 127) / 128);
    // Under a third of the pairs at work, or with rows for one CTA of each only, the tiles of single CTAs and parts of the sum are quicker.
    if (p.M <= 128 || 3 * narrow < pairs || narrow > 0x7fffffff / 2) {
        return false;
    }
    const int64_t wideCost = (wide + pairs - 1) / pairs * (numKb + 2) * 512, narrowCost = (narrow + pairs - 1) / pairs * (numKb + 2) * 300;
    *rc = wideCost <= narrowCost ? launchPairType<256>(p, dtype, s) : launchPairType<128>(p, dtype, s);
    return true;
}

int scaledPairErrorWord() { return tc::readErrorWord(); }

} // namespace mlel
