// Attention over a paged int8 cache for few rows per cache head: single tokens, or a handful that a draft proposed.
//
//   o = sum_j softmax(s)_j v_j,  s_j = scale * q . k_j (capped or not), over the tokens that the masks leave
//
// What bounds it: the bytes of the cache, and close behind them the instructions that turn them into operands.  Every key and
// value is read once per tile of 8 rows (a row is one token's query head; the heads that share a cache head are rows of
// one tile), by the second and further tiles of a cache head out of L2.  (Tiles of 16 rows for 9 to 16, 16 sequences of up to 4000
// tokens, 8 heads of 128 elements, 16 rows: 41 us, of 8 rows 33; 4 heads of 256, 12 rows: 71 and 39.)  At 6.5 TB/s an SM gets some
// 23 bytes a cycle, 16 keys and values of 128 elements every 180 cycles.  32 sequences of up to 16000 tokens, 8 heads of 128: 106 us,
// 5.8 TB/s; 8 of up to 700: 9.2 us.
//
// Work.  All tiles' keys, in steps of 128, form one line that is cut into as many equal pieces as there are blocks, whatever the
// lengths of the sequences: a block works through the ends of the tiles that its piece touches.  Tiles that lie in
// one piece are written straight away; of the others the blocks leave (maximum, sum, unscaled result) in the workspace,
// and a second kernel joins them.  A block has four warps; two to three blocks fit an SM, so that one's start and end of a tile
// run under the others' reads.  Where the line is short, a cluster of up to eight blocks takes a tile instead, each an equal part of
// its keys, and joins the parts through distributed shared memory: no search, no workspace and no second kernel.
//
// A warp has a ring of its own, 32 keys and values a stage, filled by its own lanes with bulk tensor copies of 16 rows (128-byte
// or 64-byte swizzle; pages hold a multiple of 16 tokens, so 16 keys lie in one page, with one scale), and no barrier with
// the other warps before the end of a tile.
//
// Products on m16n8k16 in f16 with f32 sums, transposed: S^T = K Q^T and O^T = V^T P^T, so that 16 keys (16 elements of the
// result) are the rows and 8 queries the columns: half the products and half the scores per lane of the untransposed form, which
// pads to 16.  P^T changes from result to operand by a transposition of 8 x 8.
// Which element of a head is which k of the first product is free as long as both operands agree, so a lane takes 16
// consecutive bytes of a key; which key is which row is free as long as weights and values agree, so a lane's keys are t,
// t + 4, t + 8, t + 12 and its values 16 consecutive bytes of each.  All these reads are free of bank conflicts.
//
// Integers of 8 bits are exact in f16.  Keys: x + 128 as the low byte of a half is the subnormal number (x + 128) 2^-24, one byte
// permutation per two; the product's accumulator starts at -128 sum(q) 2^-24 and the scale takes the 2^24.  (Sums are then some four
// times as large as they need be, and still 2^-22 exact.)  Values: x + 128 in the low bits of 1024, minus 1152: an offset in the
// result would have to be subtracted from sums that may be a thousand times smaller than it.
//
// bf16 queries become f16 after a row-wise power of two that puts the largest at 2^14; elements down to 2^-29 of that stay
// exact.  A row keeps two maxima: m of its scores x, in whose units the sum of the softmax is, and e of x + log2(value scale), in
// whose units the result is.  The scale of 16 values is part of the exponent: weights are rounded to f16 as 2^(x + log2(scale) - e + 14), so
// that what is lost lies 2^-38 below what counts most in the row's own result: values that a row does not see, or gives next to no
// weight, take no bits from the others, however large they are.  (A scale below 2^-60 of e's counts as 2^-60 of it, so that its
// weights reach the sum.)  The sum is over the weights as they are rounded, so that what rounding does to the key that has most of
// a row cancels.  The result stays in registers; it is rescaled only when a maximum grows, which one vote per 32 keys finds out.
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

constexpr int kWarps = 4, kTileRows = 8;
constexpr int kGroup = 16; // keys that share a page and a scale for certain
constexpr int kStageGroups = 2;
constexpr int kStepGroups = kWarps * kStageGroups;
constexpr float kWeightBits = 14.f; // a row's largest weight is 2^14
constexpr float kNothing = -3e38f;  // both maxima of a row that has seen no key: differences with it are numbers
constexpr float kSlack = 30.f;      // by which scores may exceed m, in powers of two, before it is taken up: it only is the sum's unit
constexpr int kClusterSteps = 3; // steps by which a cluster's blocks may outlast the line's

template <int DP> struct FewShape {
    static constexpr int kGroupBytes = kGroup * DP; // of keys, or of values
    static constexpr int kStageBytes = 2 * kStageGroups * kGroupBytes;
    static constexpr int kPanel = DP < 128 ? DP : 128; // bytes of a row of a swizzled box
    static constexpr int kPanels = DP / kPanel;
    static constexpr int kStages = DP == 64 ? 3 : 2;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kPitch = DP + 4; // floats between the rows of results
};

// Keys that any row of a sequence sees, in groups of 16, and the tiles that need them.
struct FewWork {
    Sequence q;
    int firstGroup, groups, steps, tiles, work;
};
__device__ __forceinline__ FewWork fewWorkOf(const AttendParams &p, int index) {
    FewWork w{};
    w.q = sequenceOf(p.batch, index);
    if (w.q.sound && w.q.fresh > 0) {
        const int lo = p.window > 0 ? max(0, w.q.length - w.q.fresh - p.window + 1) : 0;
        w.firstGroup = lo / kGroup;
        w.groups = (w.q.length + kGroup - 1) / kGroup - w.firstGroup;
        w.steps = (w.groups + kStepGroups - 1) / kStepGroups;
        w.tiles = (w.q.fresh * p.group + kTileRows - 1) / kTileRows * p.cache.heads;
        w.work = w.steps * w.tiles; // (the plan has seen to it that the whole line has fewer than 2^31 steps)
    }
    return w;
}

// The line of `total` steps in pieces: the first `longer` have one step more than the others.
struct Pieces {
    int base, longer;
    __device__ Pieces(int total, int pieces) : base(total / pieces), longer(total - total / pieces * pieces) {}
    __device__ int start(int c) const { return c * base + min(c, longer); }
    __device__ int of(int x) const { // the piece that step x lies in
        const int edge = longer * (base + 1);
        return x < edge ? x / (base + 1) : longer + (x - edge) / base;
    }
};

struct FewScan {
    int sums[kWarps];
    int total, before, sequence; // steps of all, and in front of the sequence found
    FewWork work;
};

// All threads: how many steps the batch has, and the sequence that this block's piece starts in.
__device__ void locate(const AttendParams &p, FewScan &scan, int piece, int pieces, bool report) {
    const int B = p.batch.sequences, each = (B + kWarps * 32 - 1) / (kWarps * 32);
    const int lo = min(B, int(threadIdx.x) * each), hi = min(B, lo + each);
    const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
    int own = 0;
    FewWork w{};
    for (int b = lo; b < hi; ++b) {
        w = fewWorkOf(p, b);
        own += w.work;
        if (report && !w.q.sound) {
            atomicCAS(&g_pagedError, 0, kBadSequence);
        }
    }
    int upTo = own;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upTo, step);
        upTo += lane >= step ? other : 0;
    }
    if (lane == 31) {
        scan.sums[warp] = upTo;
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
        upTo += v < warp ? scan.sums[v] : 0;
        total += scan.sums[v];
    }
    const int at = Pieces(total, pieces).start(piece);
    int before = upTo - own;
    if (at >= before && at < upTo) {
        int b = lo;
        if (each > 1) {
            for (;; ++b) {
                w = fewWorkOf(p, b);
                if (at < before + w.work) {
                    break;
                }
                before += w.work;
            }
        }
        scan.before = before, scan.sequence = b, scan.work = w;
    }
    if (threadIdx.x == 0) {
        scan.total = total;
    }
    __syncthreads();
}

// One row of a partial result: e, sum, m and nothing, then DP elements.
template <int DP> __device__ __forceinline__ float *partialRow(const AttendParams &p, int piece, int which, int row) {
    return p.partials + ((int64_t(piece) * 2 + which) * kTileRows + row) * (DP + 4);
}

template <int DP, bool HALF, bool LARGE_CAP> // (see softCapped)
__global__ void __launch_bounds__(kWarps * 32, DP <= 128 ? 3 : 2)
pagedAttentionFewKernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const AttendParams p,
                        const int split) { // blocks of the cluster that shares a tile; 0: pieces of the line
    using Shape = FewShape<DP>;
    constexpr int SEGS = DP / 64, MT = DP / 16, STAGES = Shape::kStages;
    constexpr int AT = DP <= 128 ? 2 : 1; // groups taken at once: as many as the registers hold
    using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
    extern __shared__ uint8_t rawSmem[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rawSmem) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[kWarps][STAGES];
    __shared__ FewScan scan;
    __shared__ float joinMost[kWarps][kTileRows], joinLoudest[kWarps][kTileRows], joinSum[kWarps][kTileRows];
    const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; ++w) {
            for (int s = 0; s < STAGES; ++s) {
                mbarInit(&full[w][s], 1u);
            }
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int index, before = 0, begin, end, rank = 0;
    FewWork w;
    if (split > 0) {
        rank = int(clusterCtaRank());
        const int cluster = int(blockIdx.x) / split, perSequence = int(gridDim.x) / (split * p.batch.sequences);
        index = cluster / perSequence;
        w = fewWorkOf(p, index);
        const int tile = cluster - index * perSequence;
        if (!w.q.sound && tile == 0 && rank == 0 && threadIdx.x == 0) {
            atomicCAS(&g_pagedError, 0, kBadSequence);
        }
        if (tile >= w.tiles) { // (the whole cluster)
            return;
        }
        begin = tile * w.steps + w.steps * rank / split, end = tile * w.steps + w.steps * (rank + 1) / split;
        __syncthreads();
    } else {
        locate(p, scan, int(blockIdx.x), int(gridDim.x), blockIdx.x == 0); // (its barriers cover mbarInit too)
        const Pieces pieces(scan.total, int(gridDim.x));
        begin = pieces.start(int(blockIdx.x)), end = pieces.start(int(blockIdx.x) + 1);
        if (begin >= end) {
            return; // (what has ended lets the next kernel in)
        }
        index = scan.sequence, before = scan.before, w = scan.work;
    }
    uint8_t *own = ring + warp * (STAGES * Shape::kStageBytes);
    int stage = 0;      // next to be read
    uint32_t phase = 0; // of that stage
    bool broken = false;

    int at = begin;
    do { // (a block of a cluster whose part is empty still takes part in joining)
        while (split == 0 && at >= before + w.work) {
            before += w.work;
            w = fewWorkOf(p, ++index); // (there is one: `at` lies on the line)
        }
        const int tileIndex = split > 0 ? int(blockIdx.x) / split % (int(gridDim.x) / (split * p.batch.sequences)) : (at - before) / w.steps;
        const int firstStep = at - before - tileIndex * w.steps, lastStep = min(w.steps, firstStep + (end - at));
        const int head = tileIndex % p.cache.heads, firstRow = tileIndex / p.cache.heads * kTileRows;
        const int rows = min(kTileRows, w.q.fresh * p.group - firstRow), old = w.q.length - w.q.fresh;
        // this warp's stages: two groups each, every fourth pair of the piece
        const int firstGroup = w.firstGroup + firstStep * kStepGroups + warp * kStageGroups,
                  groupEnd = min(w.firstGroup + w.groups, w.firstGroup + lastStep * kStepGroups);
        const int count = firstGroup < groupEnd ? (groupEnd - firstGroup + kStepGroups - 1) / kStepGroups : 0;
        const int32_t *table = p.batch.table + index * p.batch.tableStride;

        // The pages and scales of 16 stages at a time, a lane a group: scales are fetched a batch, pages two batches ahead.
        const auto groupOf = [&](int n) { return firstGroup + (n >> 1) * kStepGroups + (n & 1); }; // n: groups of this warp
        const auto slotOf = [&](int n) {
            const int group = groupOf(n);
            int slot = -1;
            if (group < groupEnd) {
                slot = table[fastDiv(uint32_t(group * kGroup), p.pageDiv)];
                if (uint32_t(slot) >= uint32_t(p.cache.pages)) {
                    atomicCAS(&g_pagedError, 0, kBadPage);
                    slot = -1;
                }
            }
            return slot;
        };
        // A key scale of -1 stands for a group that is not there; no number, whatever it would be multiplied with, for one whose scales are
        // not both finite.
        const auto scalesOf = [&](int slot, float &key, float &valueLog) {
            const int64_t at = int64_t(max(slot, 0)) * p.cache.heads + head;
            const float value = slot >= 0 ? p.cache.valueScales[at] : 0.f;
            key = slot < 0 ? -1.f : p.cache.keyScales[at];
            key = key < INFINITY && value < INFINITY ? key : NAN, valueLog = logOfScale(value);
        };
        int slots = slotOf(lane), nextSlots = slotOf(32 + lane);
        float keyScales, valueLogs;
        scalesOf(slots, keyScales, valueLogs);
        int issued = 0, writeStage = stage, issueSlots = slots;
        // lanes that issue a copy: keys or values, which of the two groups, which panel
        const int side = lane & 1, sub = (lane >> 1) & 1, panel = lane >> 2;
        const auto fill = [&] { // the next stage of the ring, all lanes together
            if (issued > 0 && (issued & 15) == 0) {
                issueSlots = nextSlots;
            }
            const int slot = max(0, __shfl_sync(0xffffffffu, issueSlots, (2 * issued + sub) & 31));
            const int group = groupOf(2 * issued + sub), key = group * kGroup;
            const int row = (slot * p.cache.heads + head) * p.cache.page + key - int(fastDiv(uint32_t(key), p.pageDiv)) * p.cache.page;
            uint64_t *bar = &full[warp][writeStage];
            const int groups = min(kStageGroups, groupEnd - groupOf(2 * issued));
            if (lane == 0) {
                mbarArriveExpectTx(bar, uint32_t(groups * 2 * Shape::kGroupBytes));
            }
            __syncwarp();
            if (lane < 4 * Shape::kPanels && sub < groups) {
                tmaLoad3d(side == 0 ? &mapK : &mapV,
                          own + writeStage * Shape::kStageBytes + (2 * side + sub) * Shape::kGroupBytes + panel * (kGroup * Shape::kPanel), bar,
                          panel * 128, row, 0);
            }
            ++issued;
            writeStage = writeStage + 1 == STAGES ? 0 : writeStage + 1;
        };

        // queries, the second operand of S^T: lane (g, t) holds row g, elements 64 seg + 16 t .. + 15
        uint32_t qf[SEGS][4][2];
        float rowScale[2], offset[2]; // of rows 2 t and 2 t + 1, whose scores the lane gets
        int rowLo[2], rowHi[2];
        const int row = firstRow + g;
        const bool live = g < rows;
        const int token = live ? int(fastDiv(uint32_t(row), p.groupDiv)) : 0, queryHead = head * p.group + (live ? row - token * p.group : 0);
        const T *q = reinterpret_cast<const T *>(p.queries + int64_t(w.q.first + token) * p.queryStride[0] + queryHead * p.queryStride[1]);
        uint32_t words[SEGS][8]; // two elements each, as they lie in memory
#pragma unroll
        for (int seg = 0; seg < SEGS; ++seg) {
            loadQuerySixteen(q, seg * 64 + t * 16, live ? p.cache.headDim : 0, p.wideQueries != 0, words[seg]);
        }
        // the first copies go out while the queries are on their way
        for (int n = 0; n < min(count, STAGES) && !broken; ++n) {
            fill();
        }
        float unit = 1.f, total = 0.f;
        if (!HALF) {
            float most = 0.f;
#pragma unroll
            for (int seg = 0; seg < SEGS; ++seg) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 f = unpackTwo(words[seg][j], T());
                    most = maxBits(most, maxBits(f.x, f.y));
                }
            }
            most = maxBits(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = maxBits(most, __shfl_xor_sync(0xffffffffu, most, 2));
            unit = halfUnit(most);
            const float inverse = 1.f / unit; // powers of two
#pragma unroll
            for (int seg = 0; seg < SEGS; ++seg) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 f = unpackTwo(words[seg][j], T());
                    words[seg][j] = packTwo(f.x * inverse, f.y * inverse, __half());
                }
            }
        }
#pragma unroll
        for (int seg = 0; seg < SEGS; ++seg) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                qf[seg][u][0] = words[seg][2 * u], qf[seg][u][1] = words[seg][2 * u + 1];
                const float2 a = unpackTwo(words[seg][2 * u], __half()), b = unpackTwo(words[seg][2 * u + 1], __half());
                total += (a.x + a.y) + (b.x + b.y);
            }
        }
        total += __shfl_xor_sync(0xffffffffu, total, 1);
        total += __shfl_xor_sync(0xffffffffu, total, 2);
        const int position = old + token;
        const int hi = !live ? 0 : p.causal ? position + 1 : w.q.length, lo = p.window > 0 ? max(0, position - p.window + 1) : 0;
#pragma unroll
        for (int x = 0; x < 2; ++x) { // from the lanes that hold rows 2 t and 2 t + 1
            const int from = (2 * t + x) * 4;
            rowScale[x] = __shfl_sync(0xffffffffu, unit, from) * 16777216.f * p.scale * (p.softcap > 0.f ? 1.f : kLog2e);
            offset[x] = __shfl_sync(0xffffffffu, total, from) * (-128.f / 16777216.f);
            rowLo[x] = __shfl_sync(0xffffffffu, lo, from), rowHi[x] = __shfl_sync(0xffffffffu, hi, from);
        }
        // keys below `openLo` or from `openHi` on are hidden from some row
        const int lastToken = int(fastDiv(uint32_t(firstRow + rows - 1), p.groupDiv)), firstToken = int(fastDiv(uint32_t(firstRow), p.groupDiv));
        const int openHi = p.causal ? old + firstToken + 1 : w.q.length, openLo = p.window > 0 ? max(0, old + lastToken - p.window + 1) : 0;

        float o[MT][4] = {}, most[2], loudest[2], sum[2] = {}; // m and e of two rows
        most[0] = most[1] = loudest[0] = loudest[1] = kNothing;
        for (int n = 0; n < count; ++n) {
            if (n > 0 && (n & 15) == 0) {
                slots = nextSlots;
                scalesOf(slots, keyScales, valueLogs);
                nextSlots = slotOf(2 * n + 32 + lane);
            }
            if (n < issued) {
                broken = !mbarPollWarp(&full[warp][stage], phase, 61) || broken;
            }
#pragma unroll 1
            for (int h0 = 0; h0 < kStageGroups && !broken; h0 += AT) {
                float keyScale[AT], valueLog[AT];
                bool absent = false;
#pragma unroll
                for (int h = 0; h < AT; ++h) {
                    keyScale[h] = __shfl_sync(0xffffffffu, keyScales, (2 * n + h0 + h) & 31);
                    valueLog[h] = __shfl_sync(0xffffffffu, valueLogs, (2 * n + h0 + h) & 31);
                    absent = absent || keyScale[h] == -1.f;
                }
                const int key0 = groupOf(2 * n + h0) * kGroup;
                const uint32_t keys = smemAddr(own + stage * Shape::kStageBytes) + uint32_t(h0 * Shape::kGroupBytes),
                               values = keys + kStageGroups * Shape::kGroupBytes;
                float s[AT][4]; // [group][..]: keys g and g + 8 in the lanes' order, rows 2 t and 2 t + 1
#pragma unroll
                for (int h = 0; h < AT; ++h) {
                    s[h][0] = s[h][2] = offset[0], s[h][1] = s[h][3] = offset[1];
#pragma unroll
                    for (int seg = 0; seg < SEGS; ++seg) {
                        const uint32_t group = keys + uint32_t(h * Shape::kGroupBytes);
                        const uint4 k0 = ldsVector(panelAddr<DP>(group, (g >> 1) + 4 * (g & 1), seg * 4 + t));
                        const uint4 k1 = ldsVector(panelAddr<DP>(group, 8 + (g >> 1) + 4 * (g & 1), seg * 4 + t));
                        const uint32_t low[4] = {k0.x, k0.y, k0.z, k0.w}, high[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint32_t a[4];
                            bytesToSubnormals(low[u], a[0], a[2]);
                            bytesToSubnormals(high[u], a[1], a[3]);
                            mmaF16(s[h], a, qf[seg][u][0], qf[seg][u][1]);
                        }
                    }
                }
                const bool masked = key0 + AT * kGroup > openHi || key0 < openLo || absent;
                bool grows = false;
#pragma unroll
                for (int h = 0; h < AT; ++h) {
                    // what a score may be before one of the maxima grows
                    const float limit[2] = {fminf(loudest[0] - valueLog[h], most[0] + kSlack), fminf(loudest[1] - valueLog[h], most[1] + kSlack)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = s[h][e] * (rowScale[e & 1] * keyScale[h]);
                        if (p.softcap > 0.f) {
                            x = softCapped<LARGE_CAP>(x, p.softcap, p.perCap) * kLog2e;
                        }
                        if (masked) { // row g (or g + 8) of the product is key (g >> 1) + 4 (g & 1) (+ 8) of the group
                            const int key = key0 + h * kGroup + (g >> 1) + 4 * (g & 1) + 8 * (e >> 1);
                            x = key < rowHi[e & 1] && key >= rowLo[e & 1] && keyScale[h] != -1.f ? x : -INFINITY;
                        }
                        s[h][e] = x;
                        grows = grows || x > limit[e & 1];
                    }
                }
                if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float top = most[x], loud = loudest[x];
#pragma unroll
                        for (int h = 0; h < AT; ++h) { // (a maximum passes over what is no number)
                            const float score = fmaxf(s[h][x], s[h][2 + x]);
                            top = fmaxf(top, score), loud = fmaxf(loud, score + valueLog[h]);
                        }
#pragma unroll
                        for (int step = 4; step < 32; step <<= 1) {
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
                            loud = fmaxf(loud, __shfl_xor_sync(0xffffffffu, loud, step));
                        }
                        sum[x] *= unitsOf(most[x], top);
                        const float factor = unitsOf(loudest[x], loud);
                        most[x] = top, loudest[x] = loud;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            o[mt][x] *= factor, o[mt][2 + x] *= factor;
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < AT; ++h) {
                    uint32_t wf[2]; // P^T: keys in pairs by t, row g
                    // what weights have in excess of their scores, and of their scores against m
                    float shift[2], excess[2], part[2] = {0.f, 0.f};
                    bool rounded[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        shift[x] = fmaxf(kWeightBits - (loudest[x] - valueLog[h]), kWeightBits - 60.f - most[x]);
                        excess[x] = shift[x] + most[x], rounded[x] = excess[x] >= 8.f; // no weight that matters is a subnormal number
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) { // what the mask hides stays out, whatever its page's scale is
                        const float x0 = s[h][2 * half], x1 = s[h][2 * half + 1];
                        const float w0 = masked && x0 == -INFINITY ? 0.f : exp2Fast(x0 + shift[0]);
                        const float w1 = masked && x1 == -INFINITY ? 0.f : exp2Fast(x1 + shift[1]);
                        const uint32_t two = packTwo(w0, w1, __half());
                        wf[half] = transposeHalves(two);
                        const float2 w = unpackTwo(two, __half());
                        part[0] += rounded[0] ? w.x : w0, part[1] += rounded[1] ? w.y : w1;
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        sum[x] = fmaf(part[x], exp2Fast(-excess[x]), sum[x]);
                    }
                    constexpr int CHUNKS = DP < 128 ? 1 : DP / 128, WORDS = DP < 128 ? 2 : 4; // 16 (or, below 128, 8) bytes of a value row per lane each
                    const uint32_t group = values + uint32_t(h * Shape::kGroupBytes);
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        uint32_t v[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (DP < 128) {
                                const uint2 x = ldsPair(panelAddr<DP>(group, t + 4 * i, g >> 1) + 8u * uint32_t(g & 1));
                                v[i][0] = x.x, v[i][1] = x.y;
                            } else {
                                const uint4 x = ldsVector(panelAddr<DP>(group, t + 4 * i, 8 * c + (g >> 1) + 4 * (g & 1)));
                                v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
                            }
                        }
#pragma unroll
                        for (int word = 0; word < WORDS; ++word) {
                            uint32_t low[4], high[4]; // elements 4 word + .. of keys t, t + 4 and of keys t + 8, t + 12
                            transposeToHalves(v[0][word], v[1][word], low);
                            transposeToHalves(v[2][word], v[3][word], high);
#pragma unroll
                            for (int d = 0; d < 2; ++d) {
                                const uint32_t a[4] = {low[2 * d], low[2 * d + 1], high[2 * d], high[2 * d + 1]};
                                mmaF16(o[c * 8 + word * 2 + d], a, wf[0], wf[1]);
                            }
                        }
                    }
                }
            }
            if (n < issued) {
                stage = stage + 1 == STAGES ? 0 : stage + 1;
                phase ^= stage == 0 ? 1u : 0u;
            }
            __syncwarp(); // the stage has been read
            if (issued < count && !broken) {
                fill();
            }
        }

        // ---- the four warps' results as one ----
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 4);
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 8);
            sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 16);
            if (g == 0) {
                joinMost[warp][2 * t + x] = most[x], joinLoudest[warp][2 * t + x] = loudest[x], joinSum[warp][2 * t + x] = sum[x];
            }
        }
        __syncthreads(); // every warp's copies have been read: the ring holds results from here on
        constexpr int kPitch = Shape::kPitch;
        float *results = reinterpret_cast<float *>(ring), *joined = results + kWarps * kTileRows * kPitch;
        static_assert((kWarps + 1) * kTileRows * kPitch * 4 <= Shape::kRing, "the results fit the ring");
        const bool whole = split <= 1 && firstStep == 0 && lastStep == w.steps;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int itsRow = 2 * t + x;
            if (itsRow < rows) {
                float loud = kNothing;
                for (int v = 0; v < kWarps; ++v) {
                    loud = fmaxf(loud, joinLoudest[v][itsRow]);
                }
                const float factor = unitsOf(loudest[x], loud);
                float *to = results + (warp * kTileRows + itsRow) * kPitch;
                // tile mt holds elements 2 (mt % 8) and the next of the lane's 16 (or 8) of each chunk
#pragma unroll
                for (int mt = 0; mt < MT; mt += 2) {
                    float4 four;
                    four.x = o[mt][x] * factor, four.y = o[mt][2 + x] * factor;
                    four.z = o[mt + 1][x] * factor, four.w = o[mt + 1][2 + x] * factor;
                    const int element = DP < 128 ? g * 8 + 2 * mt : (mt >> 3) * 128 + ((g >> 1) + 4 * (g & 1)) * 16 + 2 * (mt & 7);
                    *reinterpret_cast<float4 *>(to + element) = four;
                }
            }
        }
        __syncthreads();
        for (int i = int(threadIdx.x); i < rows * (DP / 4); i += kWarps * 32) {
            const int itsRow = i / (DP / 4), d = (i - itsRow * (DP / 4)) * 4;
            float4 y = {};
            float top = kNothing, loud = kNothing, weights = 0.f;
#pragma unroll
            for (int v = 0; v < kWarps; ++v) {
                top = fmaxf(top, joinMost[v][itsRow]), loud = fmaxf(loud, joinLoudest[v][itsRow]);
                const float4 a = *reinterpret_cast<const float4 *>(results + (v * kTileRows + itsRow) * kPitch + d);
                y.x += a.x, y.y += a.y, y.z += a.z, y.w += a.w;
            }
#pragma unroll
            for (int v = 0; v < kWarps; ++v) {
                weights += joinSum[v][itsRow] * unitsOf(joinMost[v][itsRow], top);
            }
            if (whole) {
                writeOut<T>(p, w.q.first, firstRow + itsRow, head, d, y, weights, loud - top - kWeightBits);
            } else {
                float *to = split > 0 ? joined + itsRow * kPitch : partialRow<DP>(p, blockIdx.x, at == begin ? 0 : 1, itsRow);
                *reinterpret_cast<float4 *>(to + 4 + d - (split > 0 ? 4 : 0)) = y;
                if (d == 0) {
                    *reinterpret_cast<float4 *>(to + (split > 0 ? DP : 0)) = {loud, weights, top, 0.f};
                }
            }
        }
        __syncthreads();
        if (split > 1) { // the cluster's parts as one: elements in turn
            clusterSync();
            const uint32_t from = smemAddr(joined);
            for (int i = int(threadIdx.x) + rank * (kWarps * 32); i < rows * (DP / 4); i += split * (kWarps * 32)) {
                const int itsRow = i / (DP / 4), d = (i - itsRow * (DP / 4)) * 4;
                float top = kNothing, loud = kNothing, weights = 0.f;
                float4 y = {};
                for (int r = 0; r < split; ++r) {
                    const float4 stats = loadCluster(mapToCta(from + uint32_t((itsRow * kPitch + DP) * 4), uint32_t(r)));
                    loud = fmaxf(loud, stats.x), top = fmaxf(top, stats.z);
                }
                for (int r = 0; r < split; ++r) {
                    const float4 stats = loadCluster(mapToCta(from + uint32_t((itsRow * kPitch + DP) * 4), uint32_t(r)));
                    const float4 a = loadCluster(mapToCta(from + uint32_t((itsRow * kPitch + d) * 4), uint32_t(r)));
                    const float factor = unitsOf(stats.x, loud);
                    y.x += a.x * factor, y.y += a.y * factor, y.z += a.z * factor, y.w += a.w * factor;
                    weights += stats.y * unitsOf(stats.z, top);
                }
                writeOut<T>(p, w.q.first, firstRow + itsRow, head, d, y, weights, loud - top - kWeightBits);
            }
            __syncwarp();
            clusterSync(); // nobody leaves while its part is being read
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the ring is filled by copies again
        __syncthreads();
        at += lastStep - firstStep;
    } while (split == 0 && at < end);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Joins the pieces of one row of one tile (blockIdx.y: the row).  First all pieces' maxima and sums, a thread each, then the
// results, pieces in turn over the warps, so that a row in hundreds of pieces (one long sequence) waits for a few reads only.
constexpr int kMostPieces = 1024;

template <int DP, bool HALF>
__global__ void __launch_bounds__(kWarps * 32) pagedAttentionFewJoin(const AttendParams p, const int count) {
    constexpr int THREADS = kWarps * 32;
    using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
    __shared__ int parts[2][kWarps];
    __shared__ float factors[kMostPieces], stats[3][kWarps];
    __shared__ float4 sums[THREADS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // the tiles of all sequences in a row, those of a sequence without work included: ceil(max_new * group / kTileRows) * heads each
    const int perSequence = int(gridDim.x) / p.batch.sequences, lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
    const int index = int(blockIdx.x) / perSequence, tile = int(blockIdx.x) - index * perSequence;
    // the steps of all sequences, and of those in front of this one
    int all = 0, front = 0;
    for (int b = int(threadIdx.x); b < p.batch.sequences; b += THREADS) {
        const int work = fewWorkOf(p, b).work;
        all += work;
        front += b < index ? work : 0;
    }
    const FewWork w = fewWorkOf(p, index);
    const int row = int(blockIdx.y), head = tile % p.cache.heads, firstRow = tile / p.cache.heads * kTileRows;
    if (tile >= w.tiles || row >= w.q.fresh * p.group - firstRow || w.steps < 2) { // (the whole block)
        return;
    }
    all = __reduce_add_sync(0xffffffffu, all), front = __reduce_add_sync(0xffffffffu, front);
    if (lane == 0) {
        parts[0][warp] = all, parts[1][warp] = front;
    }
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
        total += parts[0][v], before += parts[1][v];
    }
    const Pieces pieces(total, count);
    const int x0 = before + tile * w.steps, c0 = pieces.of(x0), n = pieces.of(x0 + w.steps - 1) - c0 + 1;
    if (n == 1) {
        return; // written by that piece
    }
    const int first = x0 == pieces.start(c0) ? 0 : 1; // where piece c0 left it: as its first tile, or as its last
    const auto part = [&](int c) { return partialRow<DP>(p, c0 + c, c == 0 ? first : 0, row); };
    float top = kNothing, loud = kNothing;
    for (int c = int(threadIdx.x); c < n; c += THREADS) {
        const float4 s = *reinterpret_cast<const float4 *>(part(c));
        loud = fmaxf(loud, s.x), top = fmaxf(top, s.z);
    }
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, step));
        loud = fmaxf(loud, __shfl_xor_sync(0xffffffffu, loud, step));
    }
    if (lane == 0) {
        stats[0][warp] = top, stats[2][warp] = loud;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
        top = fmaxf(top, stats[0][v]), loud = fmaxf(loud, stats[2][v]);
    }
    float weights = 0.f;
    for (int c = int(threadIdx.x); c < n; c += THREADS) {
        const float4 s = *reinterpret_cast<const float4 *>(part(c));
        factors[c] = unitsOf(s.x, loud);
        weights += s.y * unitsOf(s.z, top);
    }
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
        weights += __shfl_xor_sync(0xffffffffu, weights, step);
    }
    if (lane == 0) {
        stats[1][warp] = weights;
    }
    __syncthreads();
    weights = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
        weights += stats[1][v];
    }
    constexpr int kLanes = DP / 4, kTeams = THREADS / kLanes; // threads of a row, rows at once
    const int team = int(threadIdx.x) / kLanes, d = int(threadIdx.x) % kLanes * 4;
    float4 y = {};
#pragma unroll 4
    for (int c = team; c < n; c += kTeams) {
        const float4 a = *reinterpret_cast<const float4 *>(part(c) + 4 + d);
        const float factor = factors[c];
        y.x += a.x * factor, y.y += a.y * factor, y.z += a.z * factor, y.w += a.w * factor;
    }
    sums[threadIdx.x] = y;
    __syncthreads();
    if (team == 0) {
#pragma unroll
        for (int v = 1; v < kTeams; ++v) {
            const float4 a = sums[v * kLanes + int(threadIdx.x)];
            y.x += a.x, y.y += a.y, y.z += a.z, y.w += a.w;
        }
        writeOut<T>(p, w.q.first, firstRow + row, head, d, y, weights, loud - top - kWeightBits);
    }
}

int paddedHead(int headDim) { return headDim <= 64 ? 64 : headDim <= 128 ? 128 : 256; }

template <int DP, bool HALF> int launchFew(const AttendParams &p, const FewPlan &plan, cudaStream_t s) {
    using Shape = FewShape<DP>;
    CUtensorMap k, v;
    if (!makeCacheMap(&k, p.cache.keys, p.cache, Shape::kPanel, kGroup, true) ||
        !makeCacheMap(&v, p.cache.values, p.cache, Shape::kPanel, kGroup, true)) {
        return MLEL_ERROR_DEVICE;
    }
    constexpr size_t smemBytes = Shape::kRing + 1024;
    const auto kernel = p.softcap > kWideCap ? pagedAttentionFewKernel<DP, HALF, true> : pagedAttentionFewKernel<DP, HALF, false>;
    if (!allowDynamicSmem(reinterpret_cast<const void *>(kernel), smemBytes)) {
        return MLEL_ERROR_DEVICE;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(plan.blocks));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attrs[2]{};
    int count = 0;
    if (dependentLaunches()) {
        attrs[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attrs[count++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (plan.split > 1) {
        attrs[count].id = cudaLaunchAttributeClusterDimension;
        attrs[count].val.clusterDim.x = unsigned(plan.split), attrs[count].val.clusterDim.y = 1, attrs[count++].val.clusterDim.z = 1;
    }
    cfg.attrs = attrs;
    cfg.numAttrs = unsigned(count);
    cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, k, v, p, plan.split);
    if (err == cudaSuccess && plan.workspace > 0) {
        const int64_t rows = std::max<int64_t>(1, int64_t(p.batch.maxNew) * p.group), tiles = (rows + kTileRows - 1) / kTileRows * p.cache.heads;
        err = launchOverlapped(pagedAttentionFewJoin<DP, HALF>,
                               dim3(unsigned(tiles * p.batch.sequences), unsigned(std::min<int64_t>(rows, kTileRows))), kWarps * 32, 0, s, p, plan.blocks);
    }
    return launchStatus("mlel_cuda_paged_attention", err);
}

} // namespace

FewPlan pagedAttentionFewPlan(const AttendParams &p) {
    FewPlan plan{};
    const int dp = paddedHead(p.cache.headDim);
    const int64_t rows = std::max<int64_t>(1, int64_t(p.batch.maxNew) * p.group); // (without new tokens the sequences are looked at all the same)
    // the most tiles and steps that the batch can have
    const int64_t steps = std::max<int64_t>(1, (int64_t(p.batch.maxLength) + kGroup * kStepGroups - 1) / (kGroup * kStepGroups));
    const int64_t tiles = (rows + kTileRows - 1) / kTileRows * p.cache.heads * p.batch.sequences, work = steps * tiles;
    if (work > 0x7fffffff) {
        refuse("mlel_cuda_paged_attention", "sequences, tokens and lengths give too much work for one call");
    }
    const int64_t resident = int64_t(dp <= 128 ? 3 : 2) * smCount();
    int split = 1;
    while (split < 8 && split < steps && tiles * split * 2 <= resident) {
        split *= 2;
    }
    const int64_t inClusters = (tiles * split + resident - 1) / resident * ((steps + split - 1) / split);
    if (inClusters <= (work + resident - 1) / resident + kClusterSteps) {
        plan.split = split, plan.blocks = int(tiles * split);
        return plan;
    }
    plan.blocks = int(std::max<int64_t>(1, std::min<int64_t>({work, resident, kMostPieces})));
    plan.workspace = steps > 1 && plan.blocks > 1 ? uint64_t(plan.blocks) * 2 * kTileRows * uint64_t(dp + 4) * 4 : 0;
    return plan;
}

int pagedAttentionFew(const AttendParams &p, const FewPlan &plan, cudaStream_t s) {
    const int dp = paddedHead(p.cache.headDim);
    if (p.halves) {
        return dp == 256 ? launchFew<256, true>(p, plan, s) : dp == 128 ? launchFew<128, true>(p, plan, s) : launchFew<64, true>(p, plan, s);
    }
    return dp == 256 ? launchFew<256, false>(p, plan, s) : dp == 128 ? launchFew<128, false>(p, plan, s) : launchFew<64, false>(p, plan, s);
}

cudaError_t takePagedErrorFew(int &code) { return takePagedError(code); }
int fewAttentionErrorWord() { return tc::readErrorWord(); }

} // namespace mlel
