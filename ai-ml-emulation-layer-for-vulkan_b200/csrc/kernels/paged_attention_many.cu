// Attention over a paged int8 cache for many rows per cache head: prompts and chunks of them, on tcgen05.
//
//   o = sum_j softmax(s)_j v_j,  s_j = scale * q . k_j (capped or not), over the tokens that the masks leave
//
// A block takes 256 rows of one sequence and cache head (a row is one token's query head; the heads that share a cache head are
// neighbouring rows) as two tiles of 128, and walks the keys they see in tiles of 128:
//   one warp       copies, integers into staging buffers: a page at a time, or the part of it that falls into a tile
//   four warps     integers -> f16 (exact), in the 128-byte swizzled layout that both products read: keys are rows of a
//                  K-major operand, values rows of an MN-major one, the same bytes either way
//   one warp       products: S = Q K^T into tensor memory, O += P V with P read from tensor memory
//   two x eight    softmax, a lane half a row: S out of tensor memory, weights as f16 back over it
// The tiles take turns: while one's products run the other's softmax does.  Tensor memory is full (two times S and O), so a tile's
// next scores wait for its weights to be used up; what counts is how long a tile's softmax takes, hence two warps to a
// scheduler for it (with one, whose lanes had a row each: 5200 cycles per 128 keys, of which 2700 the softmax).
//
// What bounds it: per 256 x 128 scores the products take 2048 cycles at 128 elements a head, and 32768 exponentials the
// same at 16 a cycle; everything else (a multiply-add, half a maximum, half a sum, half a conversion per score, and the
// keys' and values' conversion) shares the four schedulers with them: some 4500 cycles.  Four prompts of 6000 tokens, 32 heads of 128
// elements over 8: 818 us, 777 TFLOP/s.
//
// Softmax in one pass where it can: scores are weighed with the maximum known from the tiles before, and only if one exceeds
// it by more than 2^8, or at a row's first tile and where the values' reference grows, the maximum is taken first and sums
// and result are rescaled.  A row keeps two maxima: m of its scores x, in whose units the sum of the softmax is, and e of
// x + log2(value scale), in whose units the result is.  The scale of 16 values is part of the exponent: w = 2^(x + log2(scale) - e + 7),
// so a weight is at most 2^15, and f16's steps end 2^-31 below what counts most in the row's own result: values that a row does not see,
// or gives next to no weight, take no bits from the others, however large they are.  (e is kept against r, a running power of two
// above the scales, so that log2(scale / r) and its power belong to a tile and not to a row.)
// The sum is over the weights as they are rounded, so that what rounding does to the key that has most of a row cancels (a seventh off
// the error against 64 bits).
// Tiles that a mask cuts, or with scales far below r, go a second way, which asks for each key, passes over groups that no row sees and
// forms by the row what the first way takes from the tile.  The two are apart, rather than a group at a time, so that the weights of 64
// keys and all else fit 80 registers: what does not comes back from L2, shared memory having all of the L1 cache (both ways in one
// loop: 860 us).  (With eight scores at a time instead of sixteen in the second way these prompts take 800 us, but 2000 new tokens with a
// window of 100, all of whose tiles are cut, 70 for 64.)  The queries' loads are issued one after another before any is used: the compiler
// would save registers and wait for each in turn (3.6 us a block).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "paged_attention.hpp"
#include "paged_attention_device.cuh"
#include "paged_attention_map.hpp"
#include "serving_device.cuh"
#include "serving_wait.cuh"
#include "tcgen05_common.cuh"
#include "tcgen05_pair.cuh"

namespace mlel {
namespace {

using namespace tc;

constexpr int kRows = 128, kGroup = 16, kMostGroups = 8;
constexpr int kConvertWarps = 4;
constexpr int kParamRing = 5, kStaging = 4, kSlots = 3; // of a tile's keys or values: integers on their way, and f16
constexpr float kGrowth = 8.f;                          // in powers of two
constexpr float kWeightBits = 7.f;
constexpr float kEvenBits = -6.f;   // of a value scale against the reference: no weight that matters is a subnormal number
constexpr float kSlack = 60.f;      // by which scores may exceed m where the scales do not bound it: it only is the sum's unit

// Heads of 256 elements: one tile of rows (its result alone has 256 columns of tensor memory), and 64 keys at a time, whose f16 form is
// as large as that of 128 keys of 128 elements.
template <int DP> struct ManyShape {
    static constexpr int kTilesOfRows = DP > 128 ? 1 : 2, kKeys = DP > 128 ? 64 : 128, kGroups = kKeys / kGroup, kHalfGroups = kGroups / 2;
    static constexpr int kTileWarps = 8, kSoftmaxWarps = kTilesOfRows * kTileWarps; // two for 32 rows
    static constexpr int kCopyWarp = kSoftmaxWarps + kConvertWarps, kProductWarp = kCopyWarp + 1, kThreads = (kProductWarp + 1) * 32;
    static constexpr int kPanels = DP / 64;
    static constexpr int kQueryBytes = kRows * DP * 2; // of one tile: panels of 64 elements
    static constexpr int kSlotBytes = kKeys * DP * 2;
    static constexpr int kStagingBytes = kKeys * DP;
    static constexpr size_t kTiles = kTilesOfRows * size_t(kQueryBytes) + kSlots * size_t(kSlotBytes) + kStaging * size_t(kStagingBytes);
    // tensor-memory columns of the tiles
    static constexpr __device__ uint32_t scores(int which) { return uint32_t(128 * which); }
    static constexpr __device__ uint32_t result(int which) { return uint32_t(256 + DP * which); }
};

// What the softmax needs to know of a tile of keys.
struct TileParams {
    float keyScale[kMostGroups];  // 0 where there is nothing
    float shift[kMostGroups];     // log2(value scale) - reference + kWeightBits
    float perWeight[kMostGroups]; // 2^-shift
    int reference;           // a power of two
    uint32_t there;          // groups that exist
    uint32_t uneven;         // those whose value scale is too far below the reference for a sum of rounded weights
};

struct ManyBarriers {
    uint64_t queries, params[kParamRing], stagingFull[kStaging], stagingEmpty[kStaging], full[kSlots], empty[kSlots];
    uint64_t scores[2], weights[2], result[2], added;
    uint32_t tmemBase;
};

// What lies behind the tiles in shared memory.
struct ManyState {
    ManyBarriers bars;
    TileParams params[kParamRing];
    float exchange[2][kRows][2]; // between the two lanes of a row
};

// kind::f16: f32 results, f16 operands, M = 128
constexpr uint32_t instrF16(int n, bool bMnMajor) {
    return (1u << 4) | (uint32_t(bMnMajor) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
}
// Four products of 16 elements of k each in one statement (see ummaBlock): both operands in shared memory, K-major, 32 bytes of
// a swizzled row apart ...
__device__ __forceinline__ void mmaSharedFour(uint32_t d, DescWords a, DescWords b, uint32_t idesc, uint32_t accumulateFirst) {
    asm volatile("{\n\t.reg .pred l, p;\n\t.reg .b32 x, y;\n\t.reg .b64 a, b;\n\t"
                 "elect.sync _|l, 0xffffffff;\n\t"
                 "setp.ne.b32 p, %6, 0;\n\t"
                 "mov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
                 "setp.eq.b32 p, %5, %5;\n\t"
                 "add.u32 x, %1, 2;\n\tadd.u32 y, %3, 2;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
                 "add.u32 x, %1, 4;\n\tadd.u32 y, %3, 4;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
                 "add.u32 x, %1, 6;\n\tadd.u32 y, %3, 6;\n\tmov.b64 a, {x, %2};\n\tmov.b64 b, {y, %4};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d),
                 "r"(a.low), "r"(a.high), "r"(b.low), "r"(b.high), "r"(idesc), "r"(accumulateFirst)
                 : "memory");
}
// ... and the first one in tensor memory, eight columns apart, the second MN-major in shared memory, 16 rows of 128 bytes apart.
__device__ __forceinline__ void mmaTensorFour(uint32_t d, uint32_t a, DescWords b, uint32_t idesc, uint32_t accumulateFirst) {
    asm volatile("{\n\t.reg .pred l, p;\n\t.reg .b32 x, y;\n\t.reg .b64 b;\n\t"
                 "elect.sync _|l, 0xffffffff;\n\t"
                 "setp.ne.b32 p, %5, 0;\n\t"
                 "mov.b64 b, {%2, %3};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t"
                 "setp.eq.b32 p, %4, %4;\n\t"
                 "add.u32 x, %1, 8;\n\tadd.u32 y, %2, 128;\n\tmov.b64 b, {y, %3};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, p;\n\t"
                 "add.u32 x, %1, 16;\n\tadd.u32 y, %2, 256;\n\tmov.b64 b, {y, %3};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, p;\n\t"
                 "add.u32 x, %1, 24;\n\tadd.u32 y, %2, 384;\n\tmov.b64 b, {y, %3};\n\t"
                 "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %4, p;\n\t}" ::"r"(d),
                 "r"(a), "r"(b.low), "r"(b.high), "r"(idesc), "r"(accumulateFirst)
                 : "memory");
}
__device__ __forceinline__ void tmemStore32(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
                 "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
                 "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tmemStore16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
template <int N> __device__ __forceinline__ void tmemStoreWeights(uint32_t taddr, const uint32_t (&r)[N]) {
    if constexpr (N == 32) {
        tmemStore32(taddr, r);
    } else {
        tmemStore16(taddr, r);
    }
}
// Two 32-bit floats at a time.
__device__ __forceinline__ float2 fmaTwo(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 addTwo(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float maxThree(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Barrier of two warps that tells whether the predicate holds for any of their lanes.
__device__ __forceinline__ uint32_t pairVote(int barrier, bool predicate) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any)
                 : "r"(barrier), "r"(predicate ? 1u : 0u)
                 : "memory");
    return any;
}
// 1 / unit for a power of two from 2^-126 to 2^126.
__device__ __forceinline__ float inverseOfPower(float unit) { return __uint_as_float(0x7f000000u - __float_as_uint(unit)); }
// 16 bytes from a 16-byte boundary where `there`, zeros elsewhere.  (In order with one another: a row of these is on its way at once,
// where the compiler would rather save registers and wait for each in turn.)
__device__ __forceinline__ uint4 loadIf(const char *from, bool there) {
    uint4 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
                 "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
                 : "l"(from), "r"(there ? 1u : 0u)
                 : "memory");
    return v;
}
// exp2Fast, not to be moved ahead of others (whose results would wait in registers).
__device__ __forceinline__ float exp2InOrder(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tmemStoreWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

enum Cap : int { kNoCap, kCap, kLargeCap }; // see softCapped

template <int DP, bool HALF, int CAP>
__global__ void __launch_bounds__(ManyShape<DP>::kThreads, 1)
pagedAttentionManyKernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const AttendParams p,
                         const FastDiv heads, const int levels, const int boxRows, const int split) {
    using Shape = ManyShape<DP>;
    constexpr int kKeys = Shape::kKeys, kGroups = Shape::kGroups, kHalfGroups = Shape::kHalfGroups, kTileWarps = Shape::kTileWarps,
                  kSoftmaxWarps = Shape::kSoftmaxWarps, kCopyWarp = Shape::kCopyWarp, kProductWarp = Shape::kProductWarp,
                  kBlockRows = Shape::kTilesOfRows * kRows;
    constexpr int kPitch = DP + 4; // floats between the rows of a part
    static_assert(kBlockRows <= kMostRowsOfBlock, "row numbers of the last block fit 32 bits");
    static_assert(size_t(kBlockRows) * kPitch * 4 <= Shape::kTilesOfRows * size_t(Shape::kQueryBytes) + kSlots * size_t(Shape::kSlotBytes),
                  "the parts of the rows fit the queries' and keys' memory");
    using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
    extern __shared__ __align__(1024) uint8_t rawSmem[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rawSmem) + 1023) & ~uintptr_t(1023));
    uint8_t *queries = smem, *slots = smem + Shape::kTilesOfRows * Shape::kQueryBytes, *staging = slots + kSlots * Shape::kSlotBytes;
    ManyState &state = *reinterpret_cast<ManyState *>(smem + Shape::kTiles);
    ManyBarriers &bars = state.bars;
    TileParams(&params)[kParamRing] = state.params;
    float(&exchange)[2][kRows][2] = state.exchange;
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) >> 5, 0), lane = int(threadIdx.x) & 31;
    // There is no room to spare for rounding the address up; without static shared memory it is a multiple of 1024 already.
    if (smem != rawSmem) {
        if (threadIdx.x == 0) {
            atomicCAS(&g_tcgen05Error, 0, 89);
        }
        return;
    }
    dependencySync();

    // blocks: the tiles that see the most keys first
    const uint32_t item = split > 1 ? blockIdx.x / uint32_t(split) : blockIdx.x, overHeads = fastDiv(item, heads);
    const int head = int(item - overHeads * heads.d), level = int(overHeads / uint32_t(p.batch.sequences)),
              index = int(overHeads - uint32_t(level) * uint32_t(p.batch.sequences));
    const Sequence q = sequenceOf(p.batch, index);
    const int rank = split > 1 ? int(clusterCtaRank()) : 0;
    if (!q.sound && level == 0 && head == 0 && rank == 0 && threadIdx.x == 0) {
        atomicCAS(&g_pagedError, 0, kBadSequence);
    }
    const int allRows = q.sound ? q.fresh * p.group : 0, firstRow = (levels - 1 - level) * kBlockRows;
    if (firstRow >= allRows) {
        return;
    }
    const int rows = min(kBlockRows, allRows - firstRow), old = q.length - q.fresh;
    const int firstToken = int(fastDiv(uint32_t(firstRow), p.groupDiv)), lastToken = int(fastDiv(uint32_t(firstRow + rows - 1), p.groupDiv));
    // the keys that any row sees, and of those this block's part: whole tiles
    const int allLo = (p.window > 0 ? max(0, old + firstToken - p.window + 1) : 0) / boxRows * boxRows;
    const int allHi = p.causal ? old + lastToken + 1 : q.length, allTiles = (allHi - allLo + kKeys - 1) / kKeys;
    const int firstTile = split > 1 ? int(int64_t(allTiles) * rank / split) : 0, endTile = split > 1 ? int(int64_t(allTiles) * (rank + 1) / split) : allTiles;
    const int keyLo = allLo + firstTile * kKeys, keyHi = min(allHi, allLo + endTile * kKeys), tiles = endTile - firstTile;
    const int32_t *table = p.batch.table + index * p.batch.tableStride;
    const int active = rows > kRows ? 2 : 1; // tiles with rows
    // One tile alone has both places for scores in turn: the next ones are formed before the softmax wants them.  Keys then come
    // before the values of the tile in front of them.  (Three sequences of 300 new tokens, 16 heads of 256 elements over 8, window 1024,
    // capped: 61 us with one place, so 51; 16 sequences of 4000 tokens, 32 rows a head of 128: 76 and 64.)
    const bool ahead = active == 1;

    if (threadIdx.x == 0) {
        mbarInit(&bars.queries, uint32_t(active * kTileWarps));
        for (int i = 0; i < kParamRing; ++i) {
            mbarInit(&bars.params[i], 1u);
        }
        for (int i = 0; i < kStaging; ++i) {
            mbarInit(&bars.stagingFull[i], 1u);
            mbarInit(&bars.stagingEmpty[i], kConvertWarps);
        }
        for (int i = 0; i < kSlots; ++i) {
            mbarInit(&bars.full[i], kConvertWarps);
            mbarInit(&bars.empty[i], 1u);
        }
        for (int i = 0; i < 2; ++i) {
            mbarInit(&bars.scores[i], 1u);
            mbarInit(&bars.weights[i], uint32_t(kTileWarps));
            mbarInit(&bars.result[i], 1u);
        }
        mbarInit(&bars.added, 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kProductWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smemAddr(&bars.tmemBase)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bars.tmemBase;

    if (warp == kCopyWarp) {
        // ---------------- copies, and what the softmax needs to know of their pages ----------------
        const int groups = (keyHi - keyLo + kGroup - 1) / kGroup, groupsOfBox = boxRows / kGroup;
        const auto slotOf = [&](int tile) { // lane 0 .. 7: the page of a group of the tile; -1: there is none
            const int n = tile * kGroups + lane;
            return lane < kGroups && n < groups ? table[fastDiv(uint32_t(keyLo + n * kGroup), p.pageDiv)] : -1;
        };
        const auto checked = [&](int tile, int slot) { // a tile later, when the entry has arrived
            if (uint32_t(slot) >= uint32_t(p.cache.pages)) {
                if (lane < kGroups && tile * kGroups + lane < groups) {
                    atomicCAS(&g_pagedError, 0, kBadPage);
                }
                return -1;
            }
            return slot;
        };
        // (a scale that is not finite is no number, whatever it would be multiplied with)
        const auto scaleOf = [&](const float *scales, int slot) {
            const float scale = slot >= 0 ? scales[int64_t(slot) * p.cache.heads + head] : 0.f;
            return scale < INFINITY ? scale : NAN;
        };
        int nextNextSlot = slotOf(1), nextSlot = checked(0, slotOf(0)), reference = -126;
        float nextKeyScale = scaleOf(p.cache.keyScales, nextSlot), nextValueScale = scaleOf(p.cache.valueScales, nextSlot);
        uint32_t unit = 0; // keys and values of the tiles in turn
        const auto copy = [&](const CUtensorMap &map, int row, int count) {
            const uint32_t buffer = unit % kStaging;
            if (!mbarPollWarp(&bars.stagingEmpty[buffer], ((unit / kStaging) & 1u) ^ 1u, 91)) {
                return false;
            }
            if (lane == 0) { // the last box may reach behind the sequence, not behind its page
                mbarArriveExpectTx(&bars.stagingFull[buffer], uint32_t((count + groupsOfBox - 1) / groupsOfBox * boxRows * DP));
            }
            __syncwarp();
            if (lane < kGroups && lane % groupsOfBox == 0 && lane < count) {
                tmaLoad3d(&map, staging + buffer * Shape::kStagingBytes + lane * kGroup * DP, &bars.stagingFull[buffer], 0, row, 0);
            }
            ++unit;
            return true;
        };
        int lastRow = 0, lastCount = 0;
        bool ok = true;
        for (int tile = 0; tile < tiles && ok; ++tile) {
            const int slot = nextSlot, afterSlot = nextNextSlot;
            const float keyScale = nextKeyScale, valueScale = nextValueScale;
            nextNextSlot = slotOf(tile + 2);
            // the copies first: what they need has long been here
            const int key = keyLo + (tile * kGroups + lane) * kGroup, count = min(kGroups, groups - tile * kGroups);
            const int row = (max(slot, 0) * p.cache.heads + head) * p.cache.page + key - int(fastDiv(uint32_t(key), p.pageDiv)) * p.cache.page;
            ok = copy(mapK, row, count);
            if (!ok) {
                break;
            }
            {
                // Parameters of the tile.  Here the converters are done with the keys of tile - 2, for which the values of tile - 4
                // (tile - 5, where keys come before values) had been used up by both tiles: the softmax is past tile - 5,
                // whose place this is.
                TileParams &to = params[tile % kParamRing];
                const float magnitude = fabsf(valueScale);
                int exponent = magnitude > 0.f && magnitude < INFINITY ? int(__float_as_uint(powerAbove(magnitude)) >> 23) - 127 : -126;
                exponent = __reduce_max_sync(0xffffffffu, exponent);
                reference = max(reference, exponent);
                const float bits = logOfScale(valueScale) - float(reference); // (no number for a scale that is not finite)
                if (lane < kGroups) {
                    to.keyScale[lane] = keyScale, to.shift[lane] = bits + kWeightBits, to.perWeight[lane] = exp2f(-kWeightBits - bits);
                }
                const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0);
                const uint32_t uneven = __ballot_sync(0xffffffffu, slot >= 0 && !(bits >= kEvenBits));
                if (lane == 0) {
                    to.reference = reference, to.there = there, to.uneven = uneven;
                }
                __syncwarp();
                if (lane == 0) {
                    mbarArrive(&bars.params[tile % kParamRing]);
                }
            }
            if (!ahead) {
                ok = copy(mapV, row, count);
            } else if (tile > 0) {
                ok = copy(mapV, lastRow, kGroups);
            }
            lastRow = row, lastCount = count;
            nextSlot = checked(tile + 1, afterSlot);
            nextKeyScale = scaleOf(p.cache.keyScales, nextSlot), nextValueScale = scaleOf(p.cache.valueScales, nextSlot);
        }
        if (ahead && ok && tiles > 0) {
            copy(mapV, lastRow, lastCount);
        }
        __syncwarp();
    } else if (warp == kProductWarp) {
        // ---------------- products (the whole warp: see ummaBlockPeek) ----------------
        constexpr uint32_t kScoreDesc = instrF16(kKeys, false), kResultDesc = instrF16(DP, true);
        constexpr uint32_t kQueryPanel = kRows * 128, kPanel = kKeys * 128, kPlace = uint32_t(Shape::kSlotBytes) >> 4; // bytes of 64 elements; units of 16
        const DescWords queryDesc = descWords(smemDesc(smemAddr(queries), 16, 1024)), keyDesc = descWords(smemDesc(smemAddr(slots), 16, 1024)),
                        valueDesc = descWords(smemDesc(smemAddr(slots), kPanel, 1024));
        bool failed = !mbarPoll(&bars.queries, 0u, 92);
        const auto scoreProduct = [&](int tile, int which) {
            const uint32_t unit = ahead ? uint32_t(max(0, 2 * tile - 1)) : uint32_t(2 * tile), place = unit % kSlots;
            const int buffer = ahead ? tile & 1 : which;
            if (which == 0) {
                failed = failed || !mbarPoll(&bars.full[place], (unit / kSlots) & 1u, 93);
            }
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int panel = 0; panel < Shape::kPanels; ++panel) {
                mmaSharedFour(tmem + Shape::scores(buffer),
                              {queryDesc.low + uint32_t(which * (Shape::kQueryBytes >> 4)) + uint32_t(panel) * (kQueryPanel >> 4), queryDesc.high},
                              {keyDesc.low + place * kPlace + uint32_t(panel) * (kPanel >> 4), keyDesc.high}, kScoreDesc, panel != 0 ? 1u : 0u);
            }
            ummaCommit(&bars.scores[buffer]);
            if (which == active - 1) {
                ummaCommit(&bars.empty[place]);
            }
        };
        const auto resultProduct = [&](int tile, int which) {
            const uint32_t unit = uint32_t(ahead ? min(2 * tile + 2, 2 * tiles - 1) : 2 * tile + 1), place = unit % kSlots;
            const int buffer = ahead ? tile & 1 : which;
            if (which == 0) {
                failed = failed || !mbarPoll(&bars.full[place], (unit / kSlots) & 1u, 94);
            }
            failed = failed || !mbarPoll(&bars.weights[buffer], uint32_t(ahead ? tile >> 1 : tile) & 1u, 95);
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int k = 0; k < kGroups; k += 4) { // the weights of 16 keys lie in eight columns
                mmaTensorFour(tmem + Shape::result(which), tmem + Shape::scores(buffer) + uint32_t(k * 8),
                              {valueDesc.low + place * kPlace + uint32_t(k) * 128u, valueDesc.high}, kResultDesc, tile != 0 || k != 0 ? 1u : 0u);
            }
            if (ahead) {
                ummaCommit(&bars.added);
            }
            if (tile == tiles - 1) {
                ummaCommit(&bars.result[which]);
            }
            if (which == active - 1) {
                ummaCommit(&bars.empty[place]);
            }
        };
        for (int which = 0; which < active && tiles > 0; ++which) {
            scoreProduct(0, which);
        }
        for (int tile = 0; tile < tiles; ++tile) {
            if (ahead && tile + 1 < tiles) {
                scoreProduct(tile + 1, 0);
            }
            for (int which = 0; which < active; ++which) {
                resultProduct(tile, which);
                if (!ahead && tile + 1 < tiles) {
                    scoreProduct(tile + 1, which);
                }
            }
        }
    } else if (warp >= kSoftmaxWarps) {
        // ---------------- integers -> f16 ----------------
        // A lane takes 16 bytes of a row: bytes 16 (lane % 4) on of a panel of 64.  Eight neighbouring lanes write four chunks of two
        // rows, which the swizzle keeps in different banks.
        constexpr int kPanels = Shape::kPanels, kRowsOfWarp = 8 / kPanels, kRowsAtOnce = kConvertWarps * kRowsOfWarp;
        const int own = warp - kSoftmaxWarps, panel = (lane >> 2) / kRowsOfWarp, part = lane & 3;
        const int row0 = own * kRowsOfWarp + (lane >> 2) % kRowsOfWarp; // its low three bits are those of all its rows
        static_assert(kRowsAtOnce % 8 == 0, "rows of a lane share their swizzle");
        const uint32_t fromLane = smemAddr(staging) + uint32_t(row0 * DP + panel * 64 + part * 16);
        const uint32_t toLane = smemAddr(slots) + uint32_t(panel * (kKeys * 128) + row0 * 128);
        const uint32_t low = toLane + uint32_t(((2 * part) ^ (row0 & 7)) << 4), high = toLane + uint32_t(((2 * part + 1) ^ (row0 & 7)) << 4);
        for (uint32_t unit = 0; unit < uint32_t(2 * tiles); ++unit) {
            const uint32_t buffer = unit % kStaging, place = unit % kSlots;
            if (!mbarPollWarp(&bars.stagingFull[buffer], (unit / kStaging) & 1u, 96) ||
                !mbarPollWarp(&bars.empty[place], ((unit / kSlots) & 1u) ^ 1u, 97)) {
                break;
            }
            const uint32_t from = fromLane + buffer * uint32_t(Shape::kStagingBytes), to = place * uint32_t(Shape::kSlotBytes);
#pragma unroll 8
            for (int step = 0; step < kKeys / kRowsAtOnce; ++step) {
                const uint4 v = ldsVector(from + uint32_t(step * kRowsAtOnce * DP));
                uint4 a, b;
                bytesToHalves(v.x, a.x, a.y);
                bytesToHalves(v.y, a.z, a.w);
                bytesToHalves(v.z, b.x, b.y);
                bytesToHalves(v.w, b.z, b.w);
                const uint32_t line = to + uint32_t(step * kRowsAtOnce * 128);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(low + line), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w) : "memory");
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(high + line), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbarArrive(&bars.full[place]);
                mbarArrive(&bars.stagingEmpty[buffer]);
            }
        }
        __syncwarp();
    } else if (warp < active * kTileWarps) {
        // ---------------- softmax: a lane half a row ----------------
        const int which = warp / kTileWarps, half = (warp >> 2) & 1, quarter = warp & 3, tileRow = quarter * 32 + lane,
                  row = firstRow + which * kRows + tileRow;
        const int pairBarrier = 1 + which * 4 + quarter; // of the two warps that share 32 rows
        const bool live = which * kRows + tileRow < rows;
        const int token = live ? int(fastDiv(uint32_t(row), p.groupDiv)) : lastToken;
        float rowScale;
        {
            // The warp's half of its 32 rows, as runs of DP bytes: kLanes lanes a row, kRowsAtOnce rows at a time, all on their way at once.
            constexpr int kLanes = DP / 16, kRowsAtOnce = 32 / kLanes, kSteps = 32 / kRowsAtOnce;
            const int chunk = lane % kLanes, element = half * (DP / 2) + chunk * 8;
            const auto queryOf = [&](int r) { // where the lane's eight elements of a row of the tile lie
                const int global = firstRow + which * kRows + r, itsToken = int(fastDiv(uint32_t(global), p.groupDiv));
                return p.queries + int64_t(q.first + itsToken) * p.queryStride[0] + (head * p.group + global - itsToken * p.group) * p.queryStride[1] +
                       element * 2;
            };
            uint4 words[kSteps];
            if (p.wideQueries) {
#pragma unroll
                for (int step = 0; step < kSteps; ++step) {
                    const int r = quarter * 32 + step * kRowsAtOnce + lane / kLanes;
                    const bool there = which * kRows + r < rows && element < p.cache.headDim;
                    words[step] = loadIf(queryOf(there ? r : 0), there);
                }
            } else {
#pragma unroll
                for (int step = 0; step < kSteps; ++step) {
                    const int r = quarter * 32 + step * kRowsAtOnce + lane / kLanes;
                    words[step] = {0u, 0u, 0u, 0u};
                    if (which * kRows + r < rows && element < p.cache.headDim) {
                        const uint16_t *e = reinterpret_cast<const uint16_t *>(queryOf(r));
                        words[step] = {uint32_t(e[0]) | uint32_t(e[1]) << 16, uint32_t(e[2]) | uint32_t(e[3]) << 16,
                                       uint32_t(e[4]) | uint32_t(e[5]) << 16, uint32_t(e[6]) | uint32_t(e[7]) << 16};
                    }
                }
            }
            float unit = 1.f;
            if (!HALF) {
#pragma unroll
                for (int step = 0; step < kSteps; ++step) { // magnitudes of 16 bits are ordered like their bits
                    constexpr uint32_t kSigns = 0x7fff7fffu;
                    uint32_t m = maxHalves(maxHalves(words[step].x & kSigns, words[step].y & kSigns), maxHalves(words[step].z & kSigns, words[step].w & kSigns));
#pragma unroll
                    for (int other = 1; other < kLanes; other <<= 1) {
                        m = maxHalves(m, __shfl_xor_sync(0xffffffffu, m, other));
                    }
                    if (chunk == 0) {
                        exchange[which][quarter * 32 + step * kRowsAtOnce + lane / kLanes][half] = __uint_as_float(max(m & 0xffffu, m >> 16) << 16);
                    }
                }
                asm volatile("bar.sync %0, 64;" ::"r"(pairBarrier) : "memory");
                unit = halfUnit(maxBits(exchange[which][tileRow][0], exchange[which][tileRow][1]));
#pragma unroll
                for (int step = 0; step < kSteps; ++step) {
                    const int r = quarter * 32 + step * kRowsAtOnce + lane / kLanes;
                    const float inverse = inverseOfPower(halfUnit(maxBits(exchange[which][r][0], exchange[which][r][1])));
                    float x[8];
                    unpackEight(words[step], x, T());
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] *= inverse;
                    }
                    words[step] = packEight(x, __half());
                }
                asm volatile("bar.sync %0, 64;" ::"r"(pairBarrier) : "memory"); // `exchange` is used again
            }
            rowScale = unit * fabsf(p.scale) * (CAP != kNoCap ? 1.f : kLog2e);
            const uint32_t sign = p.scale < 0.f ? 0x80008000u : 0u; // keeps the order of scores that of the products
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                const int r = quarter * 32 + step * kRowsAtOnce + lane / kLanes;
                const uint32_t to = smemAddr(queries) + uint32_t(which * Shape::kQueryBytes + (element / 64) * (kRows * 128) + r * 128) +
                                    uint32_t((((element % 64) / 8) ^ (r & 7)) << 4);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(words[step].x ^ sign), "r"(words[step].y ^ sign),
                             "r"(words[step].z ^ sign), "r"(words[step].w ^ sign)
                             : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbarArrive(&bars.queries);
            }
        }
        // The keys that the lane's row sees, and its place among the rows: formed where they are wanted, from a lane number that is read
        // again, so that they are not held in registers meanwhile.
        const auto rowAgain = [&] {
            int own;
            asm volatile("mov.u32 %0, %%laneid;" : "=r"(own));
            return quarter * 32 + own;
        };
        const auto limits = [&](int &lo, int &hi) {
            const int own = which * kRows + rowAgain(), position = old + int(fastDiv(uint32_t(firstRow + min(own, rows - 1)), p.groupDiv));
            hi = own >= rows ? 0 : p.causal ? position + 1 : q.length, lo = p.window > 0 ? max(0, position - p.window + 1) : 0;
        };
        // keys that every row of this tile sees
        const int tileFirst = firstRow + which * kRows, tileLast = min(tileFirst + kRows, firstRow + rows) - 1;
        const int openHi = p.causal ? old + int(fastDiv(uint32_t(tileFirst), p.groupDiv)) + 1 : q.length;
        const int openLo = p.window > 0 ? max(0, old + int(fastDiv(uint32_t(tileLast), p.groupDiv)) - p.window + 1) : 0;
        const uint32_t laneBase = tmem + (uint32_t(quarter * 32) << 16);
        const uint32_t resultAt = laneBase + Shape::result(which) + uint32_t(half * (DP / 2));

        bool ok = true, late = false;
        // e against the reference, and m (of this lane's half of the keys; at least e); the sums since e was last taken up, in units of
        // 2^loudest, and all others, in units of 2^most
        float loudest = -INFINITY, most = -INFINITY, sum = 0.f, others = 0.f;
        int reference = -126;
        const auto scoreOf = [&](uint32_t s, float factor) { // in powers of two
            const float x = __uint_as_float(s) * factor;
            return CAP != kNoCap ? softCapped<CAP == kLargeCap>(x, p.softcap, p.perCap) * kLog2e : x;
        };
        for (int tile = 0; tile < tiles && ok; ++tile) {
            const int buffer = ahead ? tile & 1 : which;
            const uint32_t scoresAt = laneBase + Shape::scores(buffer) + uint32_t(half * (kKeys / 2)),
                           weightsAt = laneBase + Shape::scores(buffer) + uint32_t(half * (kKeys / 4));
            ok = mbarPollWarp(&bars.params[tile % kParamRing], uint32_t(tile / kParamRing) & 1u, 98) &&
                 mbarPollWarp(&bars.scores[buffer], uint32_t(ahead ? tile >> 1 : tile) & 1u, 99);
            ok = pairVote(pairBarrier, !ok || late) == 0u; // a wait that ran out ends it for both warps of the rows
            if (!ok) {
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const TileParams &tp = params[tile % kParamRing];
            const int key0 = keyLo + tile * kKeys + half * (kKeys / 2);
            const bool masked = keyLo + (tile + 1) * kKeys > openHi || keyLo + tile * kKeys < openLo || tp.there != (1u << kGroups) - 1u;
            // keys of group g that this row sees, a bit each
            const auto seen = [&](int g, int rowLo, int rowHi) {
                const int first = key0 + g * kGroup, hi = max(0, min(kGroup, rowHi - first)), lo = max(0, min(kGroup, rowLo - first));
                return ((tp.there >> (half * kHalfGroups + g)) & 1u) != 0u ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
            };
            bool pending = ahead && tile > 0; // whether the products of the tile before may still be adding to the result
            const auto addedBefore = [&] {
                if (pending) {
                    late = !mbarPollWarp(&bars.added, uint32_t(tile - 1) & 1u, 88) || late;
                    pending = false;
                }
            };
            uint32_t weights[kKeys / 4];
            bool maximumFirst = tile == 0 || tp.reference != reference;
            float added, apart; // to the sum: in units of 2^loudest, and of 2^most
            while (true) {
                if (maximumFirst) {
                    float top = -INFINITY, topScore = -INFINITY;
                    int rowLo, rowHi;
                    limits(rowLo, rowHi);
#pragma unroll 1
                    for (int g = 0; g < kHalfGroups; ++g) {
                        const uint32_t bits = masked ? seen(g, rowLo, rowHi) : 0xffffu;
                        uint32_t s[16];
                        tmemLoad16(scoresAt + uint32_t(g * 16), s);
                        tmemWait16(s);
                        const float factor = rowScale * tp.keyScale[half * kHalfGroups + g];
                        float topOfGroup = -INFINITY;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            topOfGroup = ((bits >> j) & 1u) != 0u ? fmaxf(topOfGroup, scoreOf(s[j], factor)) : topOfGroup;
                        }
                        top = fmaxf(top, topOfGroup + (tp.shift[half * kHalfGroups + g] - kWeightBits)), topScore = fmaxf(topScore, topOfGroup);
                    }
                    const int own = rowAgain();
                    exchange[which][own][half] = top;
                    asm volatile("bar.sync %0, 64;" ::"r"(pairBarrier) : "memory");
                    // results are in units of 2^(loudest + reference): a reference that grows lowers the maximum
                    const float same = loudest - float(tp.reference - reference);
                    top = fmaxf(fmaxf(top, exchange[which][own][half ^ 1]), same);
                    const float keep = unitsOf(same, top);
                    topScore = fmaxf(fmaxf(topScore, top), most);
                    others = others * unitsOf(most, topScore) + sum * unitsOf(loudest, topScore);
                    most = topScore, sum = 0.f;
                    if (tile > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
                        addedBefore();
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (int d = 0; d < DP / 2; d += 16) {
                            uint32_t o[16];
                            tmemLoad16(resultAt + uint32_t(d), o);
                            tmemWait16(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                            }
                            tmemStore16(resultAt + uint32_t(d), o);
                        }
                        tmemStoreWait();
                    }
                    loudest = top, reference = tp.reference;
                }
                bool grows = false;
                const float base = loudest == -INFINITY ? 0.f : loudest;
                added = apart = 0.f;
                if (!masked && tp.uneven == 0u) {
#pragma unroll
                    for (int g = 0; g < kHalfGroups; ++g) {
                        uint32_t s[16];
                        tmemLoad16(scoresAt + uint32_t(g * 16), s);
                        const float factor = rowScale * tp.keyScale[half * kHalfGroups + g], bitsOfScale = tp.shift[half * kHalfGroups + g],
                                    shift = bitsOfScale - base;
                        const float2 factors = {factor, factor}, shifts = {shift, shift};
                        float2 parts = {0.f, 0.f};
                        float top = -INFINITY;
                        tmemWait16(s);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float2 x = {__uint_as_float(s[j]), __uint_as_float(s[j + 1])};
                            if (CAP != kNoCap) {
                                x.x = scoreOf(s[j], factor), x.y = scoreOf(s[j + 1], factor);
                            }
                            top = maxThree(top, x.x, x.y);
                            x = CAP != kNoCap ? addTwo(x, shifts) : fmaTwo(x, factors, shifts);
                            const float2 w = {exp2Fast(x.x), exp2Fast(x.y)};
                            weights[g * 8 + j / 2] = packTwo(w.x, w.y, __half());
                            parts = addTwo(parts, unpackTwo(weights[g * 8 + j / 2], __half()));
                        }
                        grows = grows || (CAP != kNoCap ? top + bitsOfScale : fmaf(top, factor, bitsOfScale)) > loudest + (kWeightBits + kGrowth);
                        added = fmaf(parts.x + parts.y, tp.perWeight[half * kHalfGroups + g], added);
                    }
                } else {
                    // What the mask hides stays out, whatever its page's scales are.  Scales count as 2^-60 of e's at least, so that their
                    // weights reach the sum.
                    const float least = kWeightBits - 60.f - (most - base);
                    int rowLo, rowHi;
                    limits(rowLo, rowHi);
#pragma unroll
                    for (int g = 0; g < kHalfGroups; ++g) {
                        const uint32_t bits = masked ? seen(g, rowLo, rowHi) : 0xffffu;
                        if (!__any_sync(0xffffffffu, bits != 0u)) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                weights[8 * g + j] = 0u;
                            }
                            continue;
                        }
                        uint32_t s[16];
                        tmemLoad16(scoresAt + uint32_t(g * 16), s);
                        const float factor = rowScale * tp.keyScale[half * kHalfGroups + g], bitsOfScale = tp.shift[half * kHalfGroups + g];
                        const float shift = (bitsOfScale < least ? least : bitsOfScale) - base; // (a NaN stays one)
                        const bool rounded = shift + most >= 1.f;
                        float top = -INFINITY, part = 0.f;
                        tmemWait16(s);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            const float x = scoreOf(s[j], factor), y = scoreOf(s[j + 1], factor);
                            const bool one = ((bits >> j) & 1u) != 0u, two = ((bits >> (j + 1)) & 1u) != 0u;
                            const float e0 = exp2InOrder(x + shift), e1 = exp2InOrder(y + shift), w0 = one ? e0 : 0.f, w1 = two ? e1 : 0.f;
                            top = one ? fmaxf(top, x) : top, top = two ? fmaxf(top, y) : top;
                            weights[g * 8 + j / 2] = packTwo(w0, w1, __half());
                            const float2 w = unpackTwo(weights[g * 8 + j / 2], __half());
                            part += rounded ? w.x + w.y : w0 + w1;
                        }
                        grows = grows || top + bitsOfScale > loudest + (kWeightBits + kGrowth) || top > most + kSlack;
                        apart = part == 0.f ? apart : fmaf(part, exp2Fast(-shift - most), apart);
                    }
                }
                // Both warps of the rows have read their scores, and agree whether a maximum has to be taken up.
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                const uint32_t again = pairVote(pairBarrier, grows && !maximumFirst);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (again == 0u) {
                    break;
                }
                maximumFirst = true;
            }
            sum += added, others += apart;
            addedBefore(); // (waited for at every tile: no phase is passed over)
            tmemStoreWeights<kKeys / 4>(weightsAt, weights);
            tmemStoreWait();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbarArrive(&bars.weights[buffer]);
            }
        }
        ok = (tiles == 0 || mbarPollWarp(&bars.result[which], 0u, 90)) && ok;
        // the two halves' sums in units of the larger m
        exchange[which][tileRow][half] = most;
        asm volatile("bar.sync %0, 64;" ::"r"(pairBarrier) : "memory");
        const float mostOfBoth = fmaxf(most, exchange[which][tileRow][half ^ 1]);
        sum = others * unitsOf(most, mostOfBoth) + sum * unitsOf(loudest, mostOfBoth), most = mostOfBoth;
        asm volatile("bar.sync %0, 64;" ::"r"(pairBarrier) : "memory");
        exchange[which][tileRow][half] = sum;
        asm volatile("bar.sync %0, 64;" ::"r"(pairBarrier) : "memory");
        sum += exchange[which][tileRow][half ^ 1];
        const float exponent = loudest + float(reference) - kWeightBits; // of the results' units
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (split > 1) {
            // ---- parts of the rows, over the queries and keys, which no product of either tile reads any more ----
            asm volatile("bar.sync 9, %0;" ::"r"(active * kTileWarps * 32) : "memory");
            float *part = reinterpret_cast<float *>(smem) + (which * kRows + tileRow) * kPitch;
#pragma unroll 1
            for (int d = 0; d < DP / 2; d += 16) {
                uint32_t o[16] = {};
                if (tiles > 0) {
                    tmemLoad16(resultAt + uint32_t(d), o);
                    tmemWait16(o);
                }
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    *reinterpret_cast<float4 *>(part + half * (DP / 2) + d + j) = {__uint_as_float(o[j]), __uint_as_float(o[j + 1]),
                                                                                   __uint_as_float(o[j + 2]), __uint_as_float(o[j + 3])};
                }
            }
            if (half == 0) {
                *reinterpret_cast<float4 *>(part + DP) = {exponent, sum, most, 0.f};
            }
        } else if (ok) { // ---- the rows, by way of the queries' memory, which no product reads any more ----
            // (in two halves: the power of two may be outside the normal numbers where the result is not)
            const float unit = exp2Fast(0.5f * (exponent - most)), f = unit / sum;
            uint8_t *mine = queries + which * Shape::kQueryBytes + (quarter * 2 + half) * (32 * DP);
            constexpr int kChunks = DP / 16, kLinesAtOnce = 32 / kChunks; // 16-byte chunks of half a row
#pragma unroll 1
            for (int d = 0; d < DP / 2; d += 16) {
                uint32_t o[16];
                tmemLoad16(resultAt + uint32_t(d), o);
                tmemWait16(o);
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = sum == 0.f ? 0.f : __uint_as_float(o[2 * j]) * f * unit,
                                y = sum == 0.f ? 0.f : __uint_as_float(o[2 * j + 1]) * f * unit;
                    w[j] = packTwo(x, y, T());
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) { // each lane's chunks turned by its number
                    *reinterpret_cast<uint4 *>(mine + lane * DP + (((d / 8 + h) ^ (lane & (kChunks - 1))) << 4)) = {w[4 * h], w[4 * h + 1],
                                                                                                                w[4 * h + 2], w[4 * h + 3]};
                }
            }
            __syncwarp();
            const int chunk = lane % kChunks, element = half * (DP / 2) + chunk * 8;
#pragma unroll 1
            for (int r = lane / kChunks; r < 32; r += kLinesAtOnce) {
                const int outRow = firstRow + which * kRows + quarter * 32 + r;
                if (which * kRows + quarter * 32 + r < rows && element < p.cache.headDim) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(mine + r * DP + ((chunk ^ (r & (kChunks - 1))) << 4));
                    const int outToken = int(fastDiv(uint32_t(outRow), p.groupDiv)), outHead = head * p.group + outRow - outToken * p.group;
                    char *to = p.out + int64_t(q.first + outToken) * p.outStride[0] + outHead * p.outStride[1] + element * 2;
                    if (p.wideOut) {
                        *reinterpret_cast<uint4 *>(to) = v;
                    } else {
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            reinterpret_cast<uint16_t *>(to)[2 * j] = uint16_t(w[j]), reinterpret_cast<uint16_t *>(to)[2 * j + 1] = uint16_t(w[j] >> 16);
                        }
                    }
                }
            }
        }
    }
    if (split > 1) { // the cluster's parts as one, four elements of a row a thread
        __syncwarp();
        clusterSync();
        const uint32_t from = smemAddr(smem);
        for (int i = int(threadIdx.x) + rank * Shape::kThreads; i < rows * (DP / 4); i += split * Shape::kThreads) {
            const int r = i / (DP / 4), d = (i - r * (DP / 4)) * 4;
            float top = -INFINITY, loud = -INFINITY, weights = 0.f;
            float4 y = {};
            for (int other = 0; other < split; ++other) { // one pass with running maxima, as over keys
                const float4 stats = loadCluster(mapToCta(from + uint32_t((r * kPitch + DP) * 4), uint32_t(other)));
                const float4 a = loadCluster(mapToCta(from + uint32_t((r * kPitch + d) * 4), uint32_t(other)));
                const float nowTop = fmaxf(top, stats.z), nowLoud = fmaxf(loud, stats.x);
                weights = weights * unitsOf(top, nowTop) + stats.y * unitsOf(stats.z, nowTop);
                const float keep = unitsOf(loud, nowLoud), factor = unitsOf(stats.x, nowLoud);
                y.x = y.x * keep + a.x * factor, y.y = y.y * keep + a.y * factor, y.z = y.z * keep + a.z * factor, y.w = y.w * keep + a.w * factor;
                top = nowTop, loud = nowLoud;
            }
            writeOut<T>(p, q.first, firstRow + r, head, d, y, weights, loud - top);
        }
        __syncwarp();
        clusterSync(); // nobody leaves while its parts are being read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kProductWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int DP, bool HALF, int CAP> int launchMany(const AttendParams &p, cudaStream_t s) {
    using Shape = ManyShape<DP>;
    constexpr size_t smemBytes = Shape::kTiles + sizeof(ManyState);
    static_assert(smemBytes <= 232448, "shared memory per block");
    // rows of a copy: the largest power of two of them, up to a tile, that pages are made of
    int boxRows = Shape::kKeys;
    while (p.cache.page % boxRows != 0) {
        boxRows /= 2;
    }
    CUtensorMap k, v;
    if (!makeCacheMap(&k, p.cache.keys, p.cache, DP, boxRows, false) || !makeCacheMap(&v, p.cache.values, p.cache, DP, boxRows, false)) {
        return MLEL_ERROR_DEVICE;
    }
    const auto kernel = pagedAttentionManyKernel<DP, HALF, CAP>;
    if (!allowDynamicSmem(reinterpret_cast<const void *>(kernel), smemBytes)) {
        return MLEL_ERROR_DEVICE;
    }
    const int64_t levels = (int64_t(p.batch.maxNew) * p.group + Shape::kTilesOfRows * kRows - 1) / (Shape::kTilesOfRows * kRows);
    const int64_t blocks = levels * p.cache.heads * p.batch.sequences;
    if (blocks > 0x7fffffff) {
        refuse("mlel_cuda_paged_attention", "too many tokens and sequences for one call");
    }
    // Few blocks with many keys each share them in clusters (one sequence, 128 new tokens of 16000, 16 blocks: 323 us, in parts of
    // eight 117), as long as a part keeps four tiles or so of the longest sequence.
    const int64_t keys = p.window > 0 ? std::min<int64_t>(p.batch.maxLength, int64_t(p.window) + p.batch.maxNew) : p.batch.maxLength;
    int split = 1;
    while (split < 8 && blocks * split * 2 <= smCount() && keys >= int64_t(split) * 2 * 4 * Shape::kKeys) {
        split *= 2;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(blocks * split));
    cfg.blockDim = dim3(Shape::kThreads);
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
    return launchStatus("mlel_cuda_paged_attention",
                        cudaLaunchKernelEx(&cfg, kernel, k, v, p, makeFastDiv(p.cache.heads), int(levels), boxRows, split));
}

template <int DP> int launchManyType(const AttendParams &p, cudaStream_t s) {
    if (p.softcap > kWideCap) {
        return p.halves ? launchMany<DP, true, kLargeCap>(p, s) : launchMany<DP, false, kLargeCap>(p, s);
    }
    if (p.softcap > 0.f) {
        return p.halves ? launchMany<DP, true, kCap>(p, s) : launchMany<DP, false, kCap>(p, s);
    }
    return p.halves ? launchMany<DP, true, kNoCap>(p, s) : launchMany<DP, false, kNoCap>(p, s);
}

} // namespace

// More than 32 rows per cache head, or 16 of more than 128 elements.  (The kernel for few of them, whose tiles have 8 rows, and this
// one: 16 sequences of up to 4000 tokens, 8 heads of 128 elements, 32 rows 56 and 64 us, 48 rows 77 and 64; 4 heads of 256, 12 rows 39
// and 56, 24 rows 60 and 57.)
bool pagedAttentionManyApplies(const AttendParams &p) { return int64_t(p.batch.maxNew) * p.group > (p.cache.headDim <= 128 ? 32 : 16); }
int pagedAttentionMany(const AttendParams &p, cudaStream_t s) {
    return p.cache.headDim <= 64 ? launchManyType<64>(p, s) : p.cache.headDim <= 128 ? launchManyType<128>(p, s) : launchManyType<256>(p, s);
}

cudaError_t takePagedErrorMany(int &code) { return takePagedError(code); }
int manyAttentionErrorWord() { return tc::readErrorWord(); }

} // namespace mlel
