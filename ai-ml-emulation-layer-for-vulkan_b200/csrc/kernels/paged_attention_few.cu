// Attention over a paged int8 cache for few rows per cache head: single tokens, or a handful that a draft proposed.
//
//   o = sum_j softmax(s)_j v_j,  s_j = scale * q . k_j (capped or not), over the tokens that the masks leave
//
// What bounds it: the bytes of the cache.  Every key and value is read once per tile of 16 or 32 rows (a row is one token's query
// head; the heads that share a cache head are rows of one tile), so a tile does 2 x 16 multiply-adds per byte and the
// arithmetic has to stay out of the way of 6.5 TB/s, some 23 bytes per cycle and SM.
//
// Work.  All tiles' keys, in steps of 64, form one line that is cut into as many equal pieces as there are blocks, whatever the
// lengths of the sequences: a block works through the ends of the tiles that its piece touches.  Tiles that lie in
// one piece are written straight away; of the others the blocks leave (maximum, sum, unscaled result) in the workspace,
// and a second kernel joins them.  A block has four warps; three blocks fit an SM, so that one's start and end of a tile run
// under the others' reads.
//
// A warp has a ring of its own, 16 keys and values a stage, filled by its own lane 0 with bulk tensor copies (128-byte or 64-byte
// swizzle), and no barrier with the other warps before the end of a tile.  Pages hold a multiple of 16 tokens, so 16
// keys lie in one page, with one scale.
//
// Products on m16n8k16 in f16 with f32 sums: an integer of 8 bits is exact in f16, made by placing it (plus 128) in the low
// mantissa bits of 1024 and subtracting 1152.  Which element of a head is which k of the product is free as long as both
// operands agree, so a lane takes 16 consecutive bytes of a key; which key is which column is free as long as the weights
// and the values agree, so a lane's four keys are t, t + 4, t + 8, t + 12 and its values 16 consecutive bytes of each, which
// four byte transpositions turn into operands.  All these reads are free of bank conflicts.
//
// bf16 queries become f16 after a row-wise power of two that puts the largest at 2^14; elements down to 2^-29 of that stay
// exact.  Weights are rounded to f16: p * (v scale / reference) * 2^14, the reference a running power of two, so that
// what is lost lies 2^-38 below the largest.  The result stays in registers in units of that reference; it is
// rescaled only when a maximum or the reference grows, which one vote per 16 keys finds out.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "paged_attention.hpp"
#include "paged_attention_device.cuh"
#include "paged_attention_map.hpp"
#include "serving_device.cuh"
#include "tcgen05_common.cuh"

namespace mlel {
namespace {

using namespace tc;

constexpr int kWarps = 4;
constexpr int kGroup = 16; // keys of a stage
constexpr float kWeightScale = 16384.f;

template <int DP> struct FewShape {
    static constexpr int kStageBytes = 2 * kGroup * DP; // keys and values
    static constexpr int kPanel = DP < 128 ? DP : 128;  // bytes of a row of a swizzled box
    static constexpr int kPanels = DP / kPanel;
    static constexpr int kStages = DP == 256 ? 3 : DP == 128 ? 4 : 6;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
};

// Keys that any row of a sequence sees, in groups of 16, and the tiles that need them.
struct FewWork {
    Sequence q;
    int firstGroup, groups, steps, tiles, work;
};
template <int ROWS> __device__ __forceinline__ FewWork fewWorkOf(const AttendParams &p, int index) {
    FewWork w{};
    w.q = sequenceOf(p.batch, index);
    if (w.q.sound && w.q.fresh > 0) {
        const int lo = p.window > 0 ? max(0, w.q.length - w.q.fresh - p.window + 1) : 0;
        w.firstGroup = lo / kGroup;
        w.groups = (w.q.length + kGroup - 1) / kGroup - w.firstGroup;
        w.steps = (w.groups + kWarps - 1) / kWarps;
        w.tiles = (w.q.fresh * p.group + ROWS - 1) / ROWS * p.cache.heads;
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
template <int ROWS> __device__ void locate(const AttendParams &p, FewScan &scan, int piece, int pieces, bool report) {
    const int B = p.batch.sequences, each = (B + kWarps * 32 - 1) / (kWarps * 32);
    const int lo = min(B, int(threadIdx.x) * each), hi = min(B, lo + each);
    const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5;
    int own = 0;
    FewWork w{};
    for (int b = lo; b < hi; ++b) {
        w = fewWorkOf<ROWS>(p, b);
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
                w = fewWorkOf<ROWS>(p, b);
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

// One row of a partial result: maximum, sum, then DP elements.
template <int DP> __device__ __forceinline__ float *partialRow(const AttendParams &p, int piece, int which, int row, int rows) {
    return p.partials + ((int64_t(piece) * 2 + which) * rows + row) * (DP + 4);
}

template <int DP, int MT, bool HALF>
__global__ void __launch_bounds__(kWarps * 32, DP == 256 || MT == 2 ? 2 : 3)
pagedAttentionFewKernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV, const AttendParams p) {
    using Shape = FewShape<DP>;
    constexpr int ROWS = 16 * MT, SEGS = DP / 64, NT = DP / 8;
    using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
    extern __shared__ uint8_t rawSmem[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(rawSmem) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[kWarps][Shape::kStages];
    __shared__ FewScan scan;
    __shared__ float joinMax[kWarps][ROWS], joinSum[kWarps][ROWS];
    const int lane = int(threadIdx.x) & 31, warp = int(threadIdx.x) >> 5, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWarps; ++w) {
            for (int s = 0; s < Shape::kStages; ++s) {
                mbarInit(&full[w][s], 1u);
            }
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    dependencySync();
    locate<ROWS>(p, scan, int(blockIdx.x), int(gridDim.x), blockIdx.x == 0); // (its barriers cover mbarInit too)
    const Pieces pieces(scan.total, int(gridDim.x));
    const int begin = pieces.start(int(blockIdx.x)), end = pieces.start(int(blockIdx.x) + 1);
    int at = begin;
    if (at >= end) {
        return;
    }
    int index = scan.sequence, before = scan.before;
    FewWork w = scan.work;
    uint8_t *own = ring + warp * (Shape::kStages * Shape::kStageBytes);
    int stage = 0;      // next to be read
    uint32_t phase = 0; // of that stage
    bool broken = false;

    while (at < end) {
        while (at >= before + w.work) {
            before += w.work;
            w = fewWorkOf<ROWS>(p, ++index); // (there is one: `at` lies on the line)
        }
        const int tileIndex = (at - before) / w.steps, firstStep = at - before - tileIndex * w.steps;
        const int lastStep = min(w.steps, firstStep + (end - at));
        const int head = tileIndex % p.cache.heads, firstRow = tileIndex / p.cache.heads * ROWS;
        const int rows = min(ROWS, w.q.fresh * p.group - firstRow), old = w.q.length - w.q.fresh;
        // this warp's groups: every fourth of the piece
        const int firstGroup = w.firstGroup + firstStep * kWarps + warp,
                  groupEnd = min(w.firstGroup + w.groups, w.firstGroup + lastStep * kWarps);
        const int count = firstGroup < groupEnd ? (groupEnd - firstGroup + kWarps - 1) / kWarps : 0;
        const int32_t *table = p.batch.table + index * p.batch.tableStride;

        // The slots and scales of 32 groups at a time, a lane each: scales are fetched a batch, slots two batches ahead.
        const auto slotOf = [&](int n) {
            const int slot = n < count ? table[fastDiv(uint32_t(firstGroup + n * kWarps) * kGroup, p.pageDiv)] : -1;
            if (n < count && uint32_t(slot) >= uint32_t(p.cache.pages)) {
                atomicCAS(&g_pagedError, 0, kBadPage);
            }
            return uint32_t(slot) < uint32_t(p.cache.pages) ? slot : -1;
        };
        const auto scaleOf = [&](const float *scales, int slot) { return slot >= 0 ? scales[int64_t(slot) * p.cache.heads + head] : 0.f; };
        int slots = slotOf(lane), nextSlots = slotOf(32 + lane);
        float keyScales = scaleOf(p.cache.keyScales, slots), valueScales = scaleOf(p.cache.valueScales, slots);
        int issued = 0, writeStage = stage, issueSlots = slots;
        const auto fill = [&] { // the next group into the ring, all lanes together
            if (issued > 0 && (issued & 31) == 0) {
                issueSlots = nextSlots;
            }
            const int slot = max(0, __shfl_sync(0xffffffffu, issueSlots, issued & 31));
            if (lane == 0) {
                const int key = (firstGroup + issued * kWarps) * kGroup;
                const int inPage = key - int(fastDiv(uint32_t(key), p.pageDiv)) * p.cache.page;
                const int row = (slot * p.cache.heads + head) * p.cache.page + inPage;
                uint64_t *bar = &full[warp][writeStage];
                uint8_t *to = own + writeStage * Shape::kStageBytes;
                mbarArriveExpectTx(bar, uint32_t(Shape::kStageBytes));
#pragma unroll
                for (int panel = 0; panel < Shape::kPanels; ++panel) {
                    tmaLoad3d(&mapK, to + panel * (kGroup * Shape::kPanel), bar, panel * 128, row, 0);
                    tmaLoad3d(&mapV, to + kGroup * DP + panel * (kGroup * Shape::kPanel), bar, panel * 128, row, 0);
                }
            }
            ++issued;
            writeStage = writeStage + 1 == Shape::kStages ? 0 : writeStage + 1;
        };
        // queries: lane (g, t) holds rows g and g + 8 of each 16, elements 64 seg + 16 t .. + 15
        uint32_t qf[MT][SEGS][4][4];
        float rowScale[MT][2]; // scores in powers of two, up to the key's scale
        int rowLo[MT][2], rowHi[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = firstRow + 16 * mt + 8 * r + g;
                const bool live = 16 * mt + 8 * r + g < rows;
                const int token = live ? int(fastDiv(uint32_t(row), p.groupDiv)) : 0, queryHead = head * p.group + (live ? row - token * p.group : 0);
                const T *q = reinterpret_cast<const T *>(p.queries + int64_t(w.q.first + token) * p.queryStride[0] +
                                                         queryHead * p.queryStride[1]);
                const int position = old + token;
                rowHi[mt][r] = !live ? 0 : p.causal ? position + 1 : w.q.length;
                rowLo[mt][r] = p.window > 0 ? max(0, position - p.window + 1) : 0;
                uint32_t words[SEGS][8]; // two elements each, as they lie in memory
                float most = 0.f;
#pragma unroll
                for (int seg = 0; seg < SEGS; ++seg) {
                    loadQuerySixteen(q, seg * 64 + t * 16, live ? p.cache.headDim : 0, p.wideQueries != 0, words[seg]);
                }
                if (mt == 0 && r == 0) { // the first copies go out while the queries are on their way
                    for (int n = 0; n < min(count, Shape::kStages) && !broken; ++n) {
                        fill();
                    }
                }
#pragma unroll
                for (int seg = 0; seg < SEGS; ++seg) {
                    if (!HALF) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 f = unpackTwo(words[seg][j], T());
                            most = maxBits(most, maxBits(f.x, f.y));
                        }
                    }
                }
                float unit = 1.f;
                if (!HALF) {
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
                rowScale[mt][r] = unit * p.scale * (p.softcap > 0.f ? 1.f : kLog2e);
#pragma unroll
                for (int seg = 0; seg < SEGS; ++seg) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        qf[mt][seg][u][r] = words[seg][2 * u], qf[mt][seg][u][2 + r] = words[seg][2 * u + 1];
                    }
                }
            }
        }
        // keys below `openLo` or from `openHi` on are hidden from some row
        const int lastToken = (firstRow + rows - 1) / p.group, firstToken = firstRow / p.group;
        const int openHi = p.causal ? old + firstToken + 1 : w.q.length, openLo = p.window > 0 ? max(0, old + lastToken - p.window + 1) : 0;

        float o[MT][NT][4] = {}, most[MT][2], sum[MT][2] = {};
        float reference = 0.f, perReference = 1.f; // unit of `o`, a power of two, and kWeightScale over it
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            most[mt][0] = most[mt][1] = -INFINITY;
        }
        for (int n = 0; n < count; ++n) {
            if (n > 0 && (n & 31) == 0) {
                slots = nextSlots;
                keyScales = scaleOf(p.cache.keyScales, slots), valueScales = scaleOf(p.cache.valueScales, slots);
                nextSlots = slotOf(n + 32 + lane);
            }
            const bool there = __shfl_sync(0xffffffffu, slots, n & 31) >= 0;
            const float keyScale = __shfl_sync(0xffffffffu, keyScales, n & 31), valueScale = __shfl_sync(0xffffffffu, valueScales, n & 31);
            const int key0 = (firstGroup + n * kWarps) * kGroup;
            if (n < issued) {
                broken = !mbarWaitWarp(&full[warp][stage], phase, 61) || broken;
            }
            const uint32_t keys = smemAddr(own + stage * Shape::kStageBytes), values = keys + kGroup * DP;
            if (there && !broken) {
                float s[MT][2][4] = {};
#pragma unroll
                for (int seg = 0; seg < SEGS; ++seg) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint4 k = ldsVector(panelAddr<DP>(keys, 8 * j + (g >> 1) + 4 * (g & 1), seg * 4 + t));
                        const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint32_t b0, b1;
                            bytesToHalves(kw[u], b0, b1);
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                mmaF16(s[mt][j], qf[mt][seg][u], b0, b1);
                            }
                        }
                    }
                }
                const bool masked = key0 + kGroup > openHi || key0 < openLo;
                bool grows = false;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float x = s[mt][j][e] * (rowScale[mt][e >> 1] * keyScale);
                            if (p.softcap > 0.f) {
                                x = softCapped(x, p.softcap) * kLog2e;
                            }
                            if (masked) { // column 2 t + (e & 1) is key 8 j + t + 4 (e & 1)
                                const int key = key0 + 8 * j + t + 4 * (e & 1);
                                x = key < rowHi[mt][e >> 1] && key >= rowLo[mt][e >> 1] ? x : -INFINITY;
                            }
                            s[mt][j][e] = x;
                            grows = grows || x > most[mt][e >> 1];
                        }
                    }
                }
                // the weights' factor; a scale that is not finite reaches the rows that see it through their weights
                const float magnitude = fabsf(valueScale);
                const bool raise = magnitude > reference && magnitude < INFINITY;
                if (__any_sync(0xffffffffu, grows) || raise) {
                    const float unit = raise ? powerAbove(magnitude) : reference;
                    const float shrink = raise ? (reference > 0.f ? reference / unit : 0.f) : 1.f;
                    reference = unit;
                    perReference = unit > 0.f ? kWeightScale / unit : 1.f;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            float top = fmaxf(fmaxf(s[mt][0][2 * r], s[mt][0][2 * r + 1]), fmaxf(s[mt][1][2 * r], s[mt][1][2 * r + 1]));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                            top = fmaxf(top, most[mt][r]);
                            const float keep = top == -INFINITY ? 1.f : exp2Fast(most[mt][r] - top);
                            most[mt][r] = top;
                            sum[mt][r] *= keep;
                            const float factor = keep * shrink;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                o[mt][nt][2 * r] *= factor, o[mt][nt][2 * r + 1] *= factor;
                            }
                        }
                    }
                }
                const float weightUnit = valueScale * perReference;
                uint32_t wf[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float shift = most[mt][r] == -INFINITY ? 0.f : most[mt][r];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float x0 = s[mt][j][2 * r], x1 = s[mt][j][2 * r + 1];
                            const float p0 = exp2Fast(x0 - shift), p1 = exp2Fast(x1 - shift);
                            sum[mt][r] += p0 + p1;
                            // what the mask hides stays out, whatever its page's scale is
                            const float w0 = masked && x0 == -INFINITY ? 0.f : p0 * weightUnit;
                            const float w1 = masked && x1 == -INFINITY ? 0.f : p1 * weightUnit;
                            wf[mt][2 * j + r] = packTwo(w0, w1, __half());
                        }
                    }
                }
                constexpr int CHUNKS = DP < 128 ? 1 : DP / 128; // 16 (or, below 128, 8) bytes of a value row per lane each
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    uint32_t v[4][DP < 128 ? 2 : 4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (DP < 128) {
                            const uint2 x = ldsPair(panelAddr<DP>(values, t + 4 * i, g >> 1) + 8u * uint32_t(g & 1));
                            v[i][0] = x.x, v[i][1] = x.y;
                        } else {
                            const uint4 x = ldsVector(panelAddr<DP>(values, t + 4 * i, 8 * c + (g >> 1) + 4 * (g & 1)));
                            v[i][0] = x.x, v[i][1] = x.y, v[i][DP < 128 ? 0 : 2] = x.z, v[i][DP < 128 ? 1 : 3] = x.w;
                        }
                    }
#pragma unroll
                    for (int word = 0; word < (DP < 128 ? 2 : 4); ++word) {
                        uint32_t b0[4], b1[4];
                        transposeToHalves(v[0][word], v[1][word], b0);
                        transposeToHalves(v[2][word], v[3][word], b1);
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                mmaF16(o[mt][c * 16 + word * 4 + d], wf[mt], b0[d], b1[d]);
                            }
                        }
                    }
                }
            }
            if (n < issued) {
                stage = stage + 1 == Shape::kStages ? 0 : stage + 1;
                phase ^= stage == 0 ? 1u : 0u;
            }
            __syncwarp(); // the stage has been read
            if (issued < count && !broken) {
                fill();
            }
        }

        // ---- the four warps' results as one ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[mt][r] += __shfl_xor_sync(0xffffffffu, sum[mt][r], 1);
                sum[mt][r] += __shfl_xor_sync(0xffffffffu, sum[mt][r], 2);
                if (t == 0) {
                    joinMax[warp][16 * mt + 8 * r + g] = most[mt][r], joinSum[warp][16 * mt + 8 * r + g] = sum[mt][r];
                }
            }
        }
        __syncthreads(); // every warp's copies have been read: the ring holds results from here on
        constexpr int kPitch = DP + 4;
        float *results = reinterpret_cast<float *>(ring);
        static_assert(kWarps * 16 * kPitch * 4 <= Shape::kRing, "the results of 16 rows fit the ring");
        const bool whole = firstStep == 0 && lastStep == w.steps;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = 16 * mt + 8 * r + g;
                if (row < rows) {
                    float top = -INFINITY;
                    for (int v = 0; v < kWarps; ++v) {
                        top = fmaxf(top, joinMax[v][row]);
                    }
                    const float factor = (top == -INFINITY ? 1.f : exp2Fast(most[mt][r] - top)) * (reference * (1.f / kWeightScale));
                    float *to = results + (warp * 16 + 8 * r + g) * kPitch;
                    // column 2 t + x of tile nt is element elementOf(nt, 2 t + x)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
#pragma unroll
                        for (int nt = 0; nt < NT; nt += 4) {
                            float4 four;
                            four.x = o[mt][nt][2 * r + x] * factor, four.y = o[mt][nt + 1][2 * r + x] * factor;
                            four.z = o[mt][nt + 2][2 * r + x] * factor, four.w = o[mt][nt + 3][2 * r + x] * factor;
                            const int element = DP < 128 ? (2 * t + x) * 8 + nt : (nt >> 4) * 128 + (t + 4 * x) * 16 + (nt & 15);
                            *reinterpret_cast<float4 *>(to + element) = four;
                        }
                    }
                }
            }
            __syncthreads();
            const int live = min(16, rows - 16 * mt);
            for (int i = int(threadIdx.x); i < live * (DP / 4); i += kWarps * 32) {
                const int row = i / (DP / 4), d = (i - row * (DP / 4)) * 4;
                float4 y = {};
                float top = -INFINITY, weights = 0.f;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    top = fmaxf(top, joinMax[v][16 * mt + row]);
                    const float4 a = *reinterpret_cast<const float4 *>(results + (v * 16 + row) * kPitch + d);
                    y.x += a.x, y.y += a.y, y.z += a.z, y.w += a.w;
                }
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    const float m = joinMax[v][16 * mt + row];
                    weights += joinSum[v][16 * mt + row] * (top == -INFINITY ? 1.f : exp2Fast(m - top));
                }
                if (whole) {
                    writeOut<T>(p, w.q.first, firstRow + 16 * mt + row, head, d, y, weights);
                } else {
                    float *to = partialRow<DP>(p, blockIdx.x, at == begin ? 0 : 1, 16 * mt + row, ROWS);
                    *reinterpret_cast<float4 *>(to + 4 + d) = y;
                    if (d == 0) {
                        to[0] = top, to[1] = weights;
                    }
                }
            }
            __syncthreads();
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the ring is filled by copies again
        __syncthreads();
        at += lastStep - firstStep;
    }
}

// Joins the pieces of one row of one tile (blockIdx.y: the row).
template <int DP, int MT, bool HALF>
__global__ void __launch_bounds__(kWarps * 32) pagedAttentionFewJoin(const AttendParams p, const int count) {
    constexpr int ROWS = 16 * MT;
    using T = typename std::conditional<HALF, __half, __nv_bfloat16>::type;
    __shared__ int parts[2][kWarps];
    dependencySync();
    // the tiles of all sequences in a row, those of a sequence without work included: ceil(max_new * group / ROWS) * heads each
    const int perSequence = int(gridDim.x) / p.batch.sequences;
    const int index = int(blockIdx.x) / perSequence, tile = int(blockIdx.x) - index * perSequence;
    const FewWork w = fewWorkOf<ROWS>(p, index);
    const int row = int(blockIdx.y), head = tile % p.cache.heads, firstRow = tile / p.cache.heads * ROWS;
    if (tile >= w.tiles || row >= w.q.fresh * p.group - firstRow || w.steps < 2) { // (the whole block)
        return;
    }
    // the steps of all sequences, and of those in front of this one
    int all = 0, front = 0;
    for (int b = int(threadIdx.x); b < p.batch.sequences; b += kWarps * 32) {
        const int work = fewWorkOf<ROWS>(p, b).work;
        all += work;
        front += b < index ? work : 0;
    }
    all = __reduce_add_sync(0xffffffffu, all), front = __reduce_add_sync(0xffffffffu, front);
    if ((threadIdx.x & 31) == 0) {
        parts[0][threadIdx.x >> 5] = all, parts[1][threadIdx.x >> 5] = front;
    }
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
        total += parts[0][v], before += parts[1][v];
    }
    const Pieces pieces(total, count);
    const int x0 = before + tile * w.steps, c0 = pieces.of(x0), c1 = pieces.of(x0 + w.steps - 1);
    if (c0 == c1) {
        return; // written by that piece
    }
    const int first = x0 == pieces.start(c0) ? 0 : 1; // where piece c0 left it: as its first tile, or as its last
    float top = -INFINITY;
    for (int c = c0; c <= c1; ++c) {
        top = fmaxf(top, partialRow<DP>(p, c, c == c0 ? first : 0, row, ROWS)[0]);
    }
    for (int d = int(threadIdx.x) * 4; d < DP; d += kWarps * 32 * 4) {
        float4 y = {};
        float sum = 0.f;
        for (int c = c0; c <= c1; ++c) {
            const float *from = partialRow<DP>(p, c, c == c0 ? first : 0, row, ROWS);
            const float factor = top == -INFINITY ? 1.f : exp2Fast(from[0] - top);
            const float4 a = *reinterpret_cast<const float4 *>(from + 4 + d);
            y.x += a.x * factor, y.y += a.y * factor, y.z += a.z * factor, y.w += a.w * factor;
            sum += from[1] * factor;
        }
        writeOut<T>(p, w.q.first, firstRow + row, head, d, y, sum);
    }
}

int paddedHead(int headDim) { return headDim <= 64 ? 64 : headDim <= 128 ? 128 : 256; }

template <int DP, int MT, bool HALF> int launchFew(const AttendParams &p, const FewPlan &plan, cudaStream_t s) {
    using Shape = FewShape<DP>;
    CUtensorMap k, v;
    if (!makeCacheMap(&k, p.cache.keys, p.cache, Shape::kPanel, kGroup, true) ||
        !makeCacheMap(&v, p.cache.values, p.cache, Shape::kPanel, kGroup, true)) {
        return MLEL_ERROR_DEVICE;
    }
    constexpr size_t smemBytes = Shape::kRing + 1024;
    const auto kernel = pagedAttentionFewKernel<DP, MT, HALF>;
    if (!allowDynamicSmem(reinterpret_cast<const void *>(kernel), smemBytes)) {
        return MLEL_ERROR_DEVICE;
    }
    cudaError_t err = launchOverlapped(kernel, dim3(unsigned(plan.blocks)), kWarps * 32, smemBytes, s, k, v, p);
    if (err == cudaSuccess && plan.joins) {
        const int64_t rows = int64_t(p.batch.maxNew) * p.group, tiles = (rows + 16 * MT - 1) / (16 * MT) * p.cache.heads;
        const dim3 grid(unsigned(tiles * p.batch.sequences), unsigned(std::min<int64_t>(rows, 16 * MT)));
        err = launchOverlapped(pagedAttentionFewJoin<DP, MT, HALF>, grid, kWarps * 32, 0, s, p, plan.blocks);
    }
    return launchStatus("mlel_cuda_paged_attention", err);
}

template <int DP, int MT> int launchFewType(const AttendParams &p, const FewPlan &plan, cudaStream_t s) {
    return p.halves ? launchFew<DP, MT, true>(p, plan, s) : launchFew<DP, MT, false>(p, plan, s);
}

} // namespace

FewPlan pagedAttentionFewPlan(const AttendParams &p) {
    FewPlan plan{};
    const int dp = paddedHead(p.cache.headDim);
    const int64_t rows = int64_t(p.batch.maxNew) * p.group;
    plan.rows = rows <= 16 || dp == 256 ? 16 : 32;
    // the most steps that the batch can have
    const int64_t steps = (int64_t(p.batch.maxLength) + kGroup * kWarps - 1) / (kGroup * kWarps);
    const int64_t work = steps * ((rows + plan.rows - 1) / plan.rows) * p.cache.heads * p.batch.sequences;
    const int resident = dp == 256 || plan.rows == 32 ? 2 : 3;
    if (work > 0x7fffffff) {
        refuse("mlel_cuda_paged_attention", "sequences, tokens and lengths give too much work for one call");
    }
    plan.blocks = int(std::max<int64_t>(1, std::min<int64_t>(work, int64_t(resident) * smCount())));
    plan.joins = steps > 1 && plan.blocks > 1;
    plan.workspace = plan.joins ? uint64_t(plan.blocks) * 2 * uint64_t(plan.rows) * uint64_t(dp + 4) * 4 : 0;
    return plan;
}

int pagedAttentionFew(const AttendParams &p, const FewPlan &plan, cudaStream_t s) {
    const int dp = paddedHead(p.cache.headDim);
    if (dp == 256) {
        return launchFewType<256, 1>(p, plan, s);
    }
    if (dp == 128) {
        return plan.rows == 16 ? launchFewType<128, 1>(p, plan, s) : launchFewType<128, 2>(p, plan, s);
    }
    return plan.rows == 16 ? launchFewType<64, 1>(p, plan, s) : launchFewType<64, 2>(p, plan, s);
}

int takePagedErrorFew() { return takePagedError(); }
int fewAttentionErrorWord() { return tc::readErrorWord(); }

} // namespace mlel
