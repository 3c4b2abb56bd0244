// Device helpers of the kernels that run tcgen05.mma.cta_group::2 on pairs of CTAs.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "tcgen05_common.cuh"

namespace mlel {
namespace tc {

__device__ __forceinline__ uint32_t clusterCtaRank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// shared::cluster address of the same shared-memory location in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t mapToCta(uint32_t ctaAddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(ctaAddr), "r"(rank));
    return r;
}

__device__ __forceinline__ void clusterSync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Tiled bulk tensor load of one CTA of a pair: lands in this CTA's shared memory, completes on `barAddr`, a
// shared::cluster address that may name a barrier of the peer CTA.
__device__ __forceinline__ void tmaLoad3dPair(const CUtensorMap *map, void *dst, uint32_t barAddr, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smemAddr(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(barAddr), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

// The same in im2col mode (see tmaLoadIm2col4d).
__device__ __forceinline__ void tmaLoadIm2col4dPair(const CUtensorMap *map, void *dst, uint32_t barAddr, int c, int w, int h,
                                                    int n, uint16_t offW, uint16_t offH) {
    asm volatile("cp.async.bulk.tensor.4d.im2col.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5, %6}], [%2], {%7, %8};" ::"r"(smemAddr(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(barAddr), "r"(c), "r"(w), "r"(h), "r"(n), "h"(offW), "h"(offH)
                 : "memory");
}

// kind::i8 instruction descriptor of the pair's MMA (see instrDesc): M = 256, A optionally MN-major.
__host__ __device__ constexpr uint32_t instrDescPair(int n, bool aMnMajor) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(aMnMajor) << 15) | (uint32_t(n >> 3) << 17) |
           (uint32_t(256 >> 4) << 24);
}

__device__ __forceinline__ void ummaPair(uint32_t tmemD, uint64_t descA, uint64_t descB, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
                 ::"r"(tmemD), "l"(descA), "l"(descB), "r"(idesc), "r"(accumulate), "r"(0u)
                 : "memory");
}

// Makes the barrier at `barAddr` (shared::cluster address, this CTA's or the peer's) complete one arrival when
// all MMAs issued so far by this warp have finished.
__device__ __forceinline__ void ummaCommitPair(uint32_t barAddr) {
    asm volatile("{\n\t.reg .pred l;\n\telect.sync _|l, 0xffffffff;\n\t"
                 "@l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(barAddr) : "memory");
}

// One K block of the pair: the four MMAs, the two commits that hand the stage back to both CTAs and, issued ahead
// of them, a non-blocking test of the barrier the next K block waits for (see ummaBlockPeek).
__device__ __forceinline__ uint32_t ummaBlockPeekPair(uint32_t tmemD, DescWords a, uint32_t stepA, DescWords b, uint32_t stepB,
                                                      uint32_t idesc, uint32_t accumulateFirst, int count, uint32_t commitOwn,
                                                      uint32_t commitPeer, uint64_t *peekBar, uint32_t peekParity) {
    uint32_t ready;
    asm volatile("{\n\t.reg .pred q, l, a0, a1, g1, g2, g3;\n\t"
                 ".reg .b32 la, lb;\n\t.reg .b64 da, db;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 q, [%1], %2;\n\t"
                 "elect.sync _|l, 0xffffffff;\n\t"
                 "setp.ne.b32 a0, %9, 0;\n\t"
                 "setp.eq.b32 a1, %10, 0;\n\t"
                 "setp.gt.and.s32 g1, %11, 1, l;\n\t"
                 "setp.gt.and.s32 g2, %11, 2, l;\n\t"
                 "setp.gt.and.s32 g3, %11, 3, l;\n\t"
                 "mov.b64 da, {%4, %5};\n\tmov.b64 db, {%6, %7};\n\t"
                 "@l tcgen05.mma.cta_group::2.kind::i8 [%3], da, db, %8, {%10, %10, %10, %10, %10, %10, %10, %10}, a0;\n\t"
                 "add.u32 la, %4, %14;\n\tadd.u32 lb, %6, %15;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %7};\n\t"
                 "@g1 tcgen05.mma.cta_group::2.kind::i8 [%3], da, db, %8, {%10, %10, %10, %10, %10, %10, %10, %10}, a1;\n\t"
                 "add.u32 la, la, %14;\n\tadd.u32 lb, lb, %15;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %7};\n\t"
                 "@g2 tcgen05.mma.cta_group::2.kind::i8 [%3], da, db, %8, {%10, %10, %10, %10, %10, %10, %10, %10}, a1;\n\t"
                 "add.u32 la, la, %14;\n\tadd.u32 lb, lb, %15;\n\tmov.b64 da, {la, %5};\n\tmov.b64 db, {lb, %7};\n\t"
                 "@g3 tcgen05.mma.cta_group::2.kind::i8 [%3], da, db, %8, {%10, %10, %10, %10, %10, %10, %10, %10}, a1;\n\t"
                 "@l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%12];\n\t"
                 "@l tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%13];\n\t"
                 "selp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(ready)
                 : "r"(smemAddr(peekBar)), "r"(peekParity), "r"(tmemD), "r"(a.low), "r"(a.high), "r"(b.low), "r"(b.high), "r"(idesc),
                   "r"(accumulateFirst), "r"(0u), "r"(count), "r"(commitOwn), "r"(commitPeer), "r"(stepA), "r"(stepB)
                 : "memory");
    return ready;
}

// The producer's counterpart (see tmaStagePeekTiled): the stage's two loads of this CTA, completing on the leader's
// barrier `fullAddr`; `expectBytes` != 0 (the leader only) announces the bytes of both CTAs on `fullOwn` first.
__device__ __forceinline__ uint32_t tmaStagePeekTiledPair(uint64_t *fullOwn, uint32_t expectBytes, uint32_t fullAddr,
                                                          const CUtensorMap *mapW, void *dstW, int w0, int w1, int w2,
                                                          const CUtensorMap *mapX, void *dstX, int x0, int x1, int x2,
                                                          uint64_t *peekBar, uint32_t peekParity) {
    uint32_t ready;
    asm volatile("{\n\t.reg .pred q, e;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 q, [%1], %2;\n\t"
                 "setp.ne.b32 e, %4, 0;\n\t"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%3], %4;\n\t"
                 "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%5], [%6, {%7, %8, %9}], [%15];\n\t"
                 "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%10], [%11, {%12, %13, %14}], [%15];\n\t"
                 "selp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(ready)
                 : "r"(smemAddr(peekBar)), "r"(peekParity), "r"(smemAddr(fullOwn)), "r"(expectBytes), "r"(smemAddr(dstW)),
                   "l"(reinterpret_cast<uint64_t>(mapW)), "r"(w0), "r"(w1), "r"(w2), "r"(smemAddr(dstX)),
                   "l"(reinterpret_cast<uint64_t>(mapX)), "r"(x0), "r"(x1), "r"(x2), "r"(fullAddr)
                 : "memory");
    return ready;
}
__device__ __forceinline__ uint32_t tmaStagePeekIm2colPair(uint64_t *fullOwn, uint32_t expectBytes, uint32_t fullAddr,
                                                           const CUtensorMap *mapW, void *dstW, int w0, int w1, int w2,
                                                           const CUtensorMap *mapX, void *dstX, int c, int w, int h, int n,
                                                           uint16_t offW, uint16_t offH, uint64_t *peekBar,
                                                           uint32_t peekParity) {
    uint32_t ready;
    asm volatile("{\n\t.reg .pred q, e;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 q, [%1], %2;\n\t"
                 "setp.ne.b32 e, %4, 0;\n\t"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%3], %4;\n\t"
                 "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%5], [%6, {%7, %8, %9}], [%18];\n\t"
                 "cp.async.bulk.tensor.4d.im2col.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
                 "[%10], [%11, {%12, %13, %14, %15}], [%18], {%16, %17};\n\t"
                 "selp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(ready)
                 : "r"(smemAddr(peekBar)), "r"(peekParity), "r"(smemAddr(fullOwn)), "r"(expectBytes), "r"(smemAddr(dstW)),
                   "l"(reinterpret_cast<uint64_t>(mapW)), "r"(w0), "r"(w1), "r"(w2), "r"(smemAddr(dstX)),
                   "l"(reinterpret_cast<uint64_t>(mapX)), "r"(c), "r"(w), "r"(h), "r"(n), "h"(offW), "h"(offH), "r"(fullAddr)
                 : "memory");
    return ready;
}

} // namespace tc
} // namespace mlel
