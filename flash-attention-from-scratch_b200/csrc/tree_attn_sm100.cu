// Attention of a tree of drafted tokens over the paged cache.
//
//   O_t = sum_j e^(s_tj) v_j / sum_j e^(s_tj),   s_tj = scale q_t.k_j over the context (through a window and
//   sinks) and those nodes that are t itself or its ancestors
//
// The rows of a kv head, its query heads times the nodes, share every key, so an item is (sequence, kv head, up to 256
// rows) and its keys come once: 128 at a time by TMA, a copy a page, whatever the pages' size. Up to 16 rows are a matrix
// instruction's worth of rows for the cached attention's kernel, which takes them (kFewRows). More go to the tensor cores,
// 128 rows a product: S = Q K^T in tensor memory, its rows' softmax in registers with a running maximum and sum, P back to
// tensor memory and P V from there. Q, K and V of 16-bit caches are multiplied as they are. Over an e4m3 cache K's codes
// are multiplied as they are, too, by queries that are taken apart into e4m3 terms (2 for bfloat16, 3 for float16), whose
// products the tensor cores sum in float32: 2 (3) products at twice the rate instead of a K that would have to be widened.
// V is widened to float16 by four warps, exactly, since P has more bits than e4m3 holds. Scales join the scores:
// w = e^(s) v_scale is 2^(factor k_scale x + log2 v_scale), so that the maximum that is subtracted bounds what is summed,
// and the sum takes w / v_scale. P is rounded to 16 bits as a matrix operand (float16 over an e4m3 cache, where it is at
// most 2^15; else the type of V), the sum is not.
//
// 16 warps: 2 x 4 softmax (a thread a row), 4 that ready V, one for S, one for P V, two that list key tiles and copy them. The
// softmax warpgroups have a row tile each (more than 128 rows), or take key tiles in turn and join their sums at the
// end. There is one S, which a warpgroup takes into registers at once: its place is free for the other's while it computes.
//
// What bounds it: a step (128 rows x 128 keys) takes 2100 to 2350 cycles, of which the products need 1024 (scores in two
// e4m3 terms, P V) and the exponentials, in a unit of their own, 1024 too. Two warpgroups take steps in turn, yet the chain
// scores -> registers -> P -> product of one overlaps the other's only in part, with 40% of the issue slots taken and
// many waits for instructions that are not in their cache.
// DRAM takes a quarter to a half of the time. Items are laid end to end and cut into equal ranges, one an SM: an item a CTA
// would leave SMs idle, and a cut costs a record of 128 or 256 rows (22 MB written and read for the second case below).
//
// Measured (D 128, bf16 queries, 32 heads on 8 kv heads, in a captured graph): over e4m3 pages of 64 tokens, 32 contexts
// of 4096 to 8192 tokens: 8 nodes 130 us (62 for the cache's bytes), up to 64 nodes 217 (66; 80 for the products);
// 4 contexts of 118000 to 131000, 32 nodes: 287 (155; 157). 16-bit pages of 32, 61 nodes on 16 contexts of 10000 to
// 20000, window 4096: 98 (44; 40). Other forms of the first two: float16 queries (three terms) 142 and 243, pages of 16 or 8
// (scores read twice) 175 and 342, both 210 and 386; 16-bit caches 140 to 144 (122) and 215 to 221 (127; 80).
// Scores and products issued by one warp: 203 us where two take 182. The wait for a step's list behind that for its
// scores instead of before: 238 for 229, 298 for 290.

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "softmax_common.cuh"
#include "sm100_ptx.cuh"
#include "stream_internal.h"
#include "tma_host.h"

namespace fa_sm100 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMinScale = 7.888609052210118e-31f;  // 2^-100: values of smaller scales, which are below 2^-91, count as zeros
constexpr float kLeastFactor = 1e-37f;               // of a score: what is hidden (-inf) stays so
// A weight is at most 2^this, relative to the maximum in use, before O and the sum are rescaled. 2^6 took 221 us for 64 nodes on
// 32 contexts where this takes 217; 2^15 was not faster.
constexpr float kLazy = 8.0f;
constexpr int kMostNodes = 256;
constexpr int kMaskWords = kMostNodes / 32;

constexpr int kTile = 128;  // query rows, and keys, of a product
constexpr int kBox = 128 * 128;  // bytes of 128 rows of 64 16-bit values, 128-byte swizzle

constexpr int kSoftmaxWarps = 8;
constexpr int kValueWarps = 4;
constexpr int kScoreWarp = kSoftmaxWarps + kValueWarps;  // issues Q K^T
constexpr int kMmaWarp = kScoreWarp + 1;                 // issues P V, owns tensor memory
constexpr int kListWarp = kMmaWarp + 1;  // and the one after it: the list of key tiles, and their copies
// Tiles are the list warps' in turn. A warp that waits for a ring's slot has seen the slot `kListWarps` tiles before it
// consumed; with no more warps than a ring has slots the phase it waits for is then never two behind.
constexpr int kListWarps = 2;
constexpr int kWarps = kScoreWarp + 4;  // whole warpgroups: registers are handed over between those
constexpr int kThreads = kWarps * 32;
// Registers: launched with 128 a thread, 512 for a lane of the four warpgroups.
// 192 and 200 for the softmax were within 2%.
constexpr int kRegsSoftmax = 184;
constexpr int kRegsOther = 72;
static_assert(2 * kRegsSoftmax + 2 * kRegsOther <= 4 * 128, "no more than the launch has");

constexpr int kListed = 4;           // key tiles listed ahead
constexpr int kGroups = kTile / 8;   // keys that surely share a page
constexpr int kMostStages = 4;
constexpr int kParts = 2;  // pieces listed, the one at hand and the next

template <int D_, bool BF16_, bool E4M3_, bool COARSE_, int NR_>
struct Cfg {
    static constexpr int D = D_;
    static constexpr bool BF16 = BF16_;  // queries and output
    static constexpr bool E4M3 = E4M3_;
    static constexpr bool COARSE = COARSE_;  // 32 keys on end share a page
    static constexpr int NR = NR_;  // row tiles of an item: 1 (key tiles alternate between the softmax warpgroups) or 2
    static constexpr bool kMmaBf16 = BF16 && !E4M3;  // type of P and V (and of Q and K, over a 16-bit cache)
    // P is 2^kUp times a weight. float16's steps end at 2^-24, so a weight is off by 2^-32 of the largest at most: a flat tail of
    // 2^20 keys beside an attention sink is there to float16's own precision. Weights as they are (kUp 0) made 0.0078 of a tail's
    // share of 0.0054 (131000 keys 17 nats below the sink) and 0 of 0.0036 (17.4 nats). Same time. bfloat16 has float32's range
    // at the small end and needs it at the large one: P is at most 1, so that the unnormalised O of values near the end of that
    // range does not overflow by P.
    static constexpr float kUp = kMmaBf16 ? -kLazy : 7.0f;
    // What the sum takes of P: over an e4m3 cache, where P / v_scale may be large, the weight itself.
    static constexpr float kDown = E4M3 ? 1.0f / 128.0f : 1.0f;
    static_assert(!E4M3 || kUp == 7.0f, "kDown undoes kUp");
    static constexpr int kElem = E4M3 ? 1 : 2;
    // e4m3 terms that a query is the sum of: bfloat16 has 8 bits, float16 11, a term 4.
    static constexpr int kTerms = E4M3 ? (BF16 ? 2 : 3) : 1;
    static constexpr int kRaw = kTile * D * kElem;      // bytes of a tile as the cache holds it
    static constexpr int kWide = kTile * D * 2;         // of a tile of 16-bit values
    static constexpr int kQTile = kTerms * kRaw;
    // Rings: K as it is; V as it is and, e4m3, widened.
    static constexpr int kKStages = E4M3 ? (NR == 1 ? 4 : (BF16 ? 3 : 2)) : (NR == 1 ? 3 : 2);
    static constexpr int kRStages = E4M3 && NR == 1 && BF16 ? 3 : 2;
    static constexpr int kVStages = 2;
    static_assert(kKStages >= kListWarps && kRStages >= kListWarps && kVStages >= kListWarps && kListed >= kListWarps, "see kListWarps");
    static constexpr int kSmemQ = 0;
    static constexpr int kSmemK = NR * kQTile;
    static constexpr int kSmemV = kSmemK + kKStages * kRaw;
    static constexpr int kSmemR = kSmemV + kVStages * kWide;
    static constexpr int kSmemShared = kSmemR + (E4M3 ? kRStages * kRaw : 0);
    static constexpr int kRows = NR * kTile;
    // Tensor memory: one tile's scores, which a warpgroup takes into registers at once, so that the next tile's follow while it
    // computes; P and the sums of either warpgroup.
    static constexpr uint32_t kTmemS = 0;
    static constexpr uint32_t kTmemP = kTile;
    static constexpr uint32_t kTmemO = 2 * kTile;
};

struct Listed {             // a key tile
    float4 group[kGroups];  // e4m3: K's scale, log2 of V's, kDown / V's
    uint4 shown;            // bits of the rows that some row of the call sees and that have a page
    int key0;               // first position; -1: the list's end
    uint32_t gone;          // bits of groups that are shown and have no page
    uint32_t tiny;          // bits of groups whose values count as zeros
    int mixed;              // rows may differ in what they see
    int full;               // all rows see all of it
};

// A piece of an item, for the softmax and the products: what its walk would keep in their registers.
struct Part {
    int n;  // key tiles; 0: the end
    int b, kvh, block;
    int record;           // -1: a whole item
    int context, count;   // of its sequence
    int last;
    // A node's way up in runs: `low` the first node of the run of nodes, each the parent of the next, that ends with the
    // node; `up` the parent of that first one, 255 for none.
    uint8_t low[kMostNodes], up[kMostNodes];
};

struct alignas(16) Shared {
    Listed list[kListed];
    Part part[kParts];
    uint64_t part_full[kParts], part_empty[kParts];
    uint64_t list_full[kListed], list_empty[kListed];
    uint64_t k_full[kMostStages], k_empty[kMostStages], v_full[2], v_empty[2], r_full[kMostStages], r_empty[kMostStages];
    uint64_t s_full[2], s_free[2], p_full[2], p_free[2];  // by warpgroup
    uint64_t q_full, q_empty, done, o_free, ml_full, mma_idle;
    long long warp_sum[kWarps];
    long long found_base;
    int found;
    uint32_t tmem_base;
    int abort;
    int odd;
};

// NR 1: what the warpgroups tell each other of the rows they share.
struct Exchange {
    float factor[2][kTile];  // of two items in turn
    float2 ml[2][kTile];
};

template <class C>
constexpr int smem_bytes() {
    constexpr int bytes = C::kSmemShared + static_cast<int>(sizeof(Shared)) + (C::NR == 1 ? static_cast<int>(sizeof(Exchange)) : 0);
    static_assert(bytes <= 227 * 1024 && sizeof(Shared) % 16 == 0);
    return bytes;
}

template <bool BF16>
__device__ __forceinline__ float widen16(uint16_t x) {
    if constexpr (BF16) {
        return __uint_as_float(static_cast<uint32_t>(x) << 16);
    } else {
        return __half2float(__ushort_as_half(x));
    }
}

__device__ __forceinline__ int held(const FaCache& c) { return c.max_pages * c.page_size; }

// A sequence's context [0, context) and nodes, which are at [context, context + count) in the cache.
struct Drafted {
    int context;  // negative where lengths and counts contradict each other
    int count;
};

__device__ __forceinline__ Drafted drafted(const FaCache& c, int b) {
    Drafted s;
    s.count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
    s.context = max(c.lengths[b], 0) - s.count;
    return s;
}

// One row on its own: warps take its visible keys in turn, lanes the dims. What it does not see is not looked at.
constexpr int kRowWarps = 8;

template <int D, bool BF16, bool E4M3>
__device__ __forceinline__ void attend_row(const FaTreeParams& p, DeviceStatus* status, int b, int h, int t) {
    constexpr int kPer = D / 32;
    const FaCache& c = p.cache;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const Drafted s = drafted(c, b);
    uint16_t* out = static_cast<uint16_t*>(p.o) + ((static_cast<int64_t>(b) * p.heads + h) * c.tokens + t) * D;
    if (t >= s.count) {
        for (int d = static_cast<int>(threadIdx.x); d < D; d += kRowWarps * 32) {
            out[d] = 0;
        }
        return;
    }
    __shared__ uint32_t mask[kMaskWords];
    __shared__ int depth_of_row;
    __shared__ float2 all_ml[kRowWarps];
    __shared__ float all_o[kRowWarps][D];
    if (threadIdx.x < kMaskWords) {
        mask[threadIdx.x] = 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const int32_t* parents = p.parents + b * p.parent_stride;
        int depth = 0;
        for (int at = t;; ++depth) {
            mask[at / 32] |= 1u << (at % 32);
            const int up = __ldg(parents + at);
            if (up < -1 || up >= at) {
                atomicOr(&status->code, kStatusBadPage);
                break;
            }
            if (up == -1) {
                break;
            }
            at = up;
        }
        depth_of_row = depth;
        if (s.context < 0 || s.context + s.count > held(c)) {
            atomicOr(&status->code, kStatusBadPage);
        }
    }
    __syncthreads();
    const int kvh = h / (p.heads / c.kv_heads);
    const int position = s.context + depth_of_row;
    const int limit = held(c);  // positions that the table has a place for
    const int end = max(min(s.context, limit), 0);
    const int first = min(window_first(max(position, 0), p.window), end);
    const int sinks = min(p.sinks, first);
    const int shown = sinks + end - first;

    const uint16_t* q = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] + h * p.q_stride[1] + t * p.q_stride[2];
    float qf[kPer], o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        qf[i] = widen16<BF16>(q[lane * kPer + i]) * (p.softmax_scale * kLog2e);
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int log2_page = 31 - __clz(c.page_size);
    auto value = [&](const void* base, int64_t at) {
        if constexpr (E4M3) {
            return unpack_half2(e4m3x2_to_half2(static_cast<const uint8_t*>(base)[at])).x;
        } else {
            return widen16<BF16>(static_cast<const uint16_t*>(base)[at]);
        }
    };
    for (int i = warp; i < shown + t + 1; i += kRowWarps) {
        int key = i < sinks ? i : first + i - sinks;
        if (i >= shown) {
            const int node = i - shown;
            key = s.context + node;
            if (!((mask[node / 32] >> (node % 32)) & 1u) || key < 0 || key >= limit) {
                continue;
            }
        }
        const int id = __ldg(c.page_table + b * c.table_stride + (key >> log2_page));
        if (id < 0 || id >= c.num_pages) {
            if (lane == 0) {
                atomicOr(&status->code, kStatusBadPage);
            }
            continue;
        }
        const int64_t slot = static_cast<int64_t>(key & (c.page_size - 1)) * D + lane * kPer;
        const int64_t k_at = id * c.k_stride[0] + kvh * c.k_stride[1] + slot;
        const int64_t v_at = id * c.v_stride[0] + kvh * c.v_stride[1] + slot;
        float ks = 1.0f, vs = 1.0f;
        if constexpr (E4M3) {
            ks = c.k_scale[static_cast<int64_t>(id) * c.kv_heads + kvh];
            vs = c.v_scale[static_cast<int64_t>(id) * c.kv_heads + kvh];
        }
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            x = fmaf(qf[e], value(c.k, k_at + e), x);
        }
#pragma unroll
        for (int step = 16; step > 0; step >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, step);
        }
        x *= ks;
        const float now = fmax_nan(m, x);
        const float used = now == -INFINITY ? 0.0f : now;
        const float alpha = ex2_approx(m - used);
        const float w = ex2_approx(x - used);
        m = now;
        l = fmaf(l, alpha, w);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            o[e] = fmaf(o[e], alpha, w * (value(c.v, v_at + e) * vs));
        }
    }
    if (lane == 0) {
        all_ml[warp] = make_float2(m, l);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        all_o[warp][lane * kPer + e] = o[e];
    }
    __syncthreads();
    for (int d = 2 * static_cast<int>(threadIdx.x); d < D; d += 2 * kRowWarps * 32) {
        float top = -INFINITY, sum = 0.0f, x0 = 0.0f, x1 = 0.0f;
        for (int w = 0; w < kRowWarps; ++w) {
            top = fmax_nan(top, all_ml[w].x);
        }
        top = top == -INFINITY ? 0.0f : top;
        for (int w = 0; w < kRowWarps; ++w) {
            const float f = ex2_approx(all_ml[w].x - top);
            sum = fmaf(all_ml[w].y, f, sum);
            x0 = fmaf(all_o[w][d], f, x0);
            x1 = fmaf(all_o[w][d + 1], f, x1);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<uint32_t*>(out + d) = pack2<BF16>(x0 * inv, x1 * inv);
    }
}

// What a sequence shows its nodes, as a list of key tiles: those of the sinks, then from the earliest window (that of a
// node on the context) to the last token that the table has.
struct Sequence : Drafted {
    int first, last;  // positions; last is -1 if there is none
    int sink_tiles, first_tile, tiles;
};

__device__ __forceinline__ Sequence sequence(const FaTreeParams& p, int b) {
    Sequence s;
    static_cast<Drafted&>(s) = drafted(p.cache, b);
    const int limit = held(p.cache);
    s.first = min(window_first(max(s.context, 0), p.window), limit);
    s.last = s.count > 0 ? min(s.context + s.count, limit) - 1 : -1;
    s.first_tile = s.first / kTile;
    s.sink_tiles = min((min(p.sinks, s.first) + kTile - 1) / kTile, s.first_tile);
    // A sequence that shows nothing keeps one (hidden) tile, so that its rows are written.
    s.tiles = s.last < 0 ? 1 : max(s.sink_tiles + s.last / kTile - s.first_tile + 1, 1);
    return s;
}

__device__ __forceinline__ int tile_key(const Sequence& s, int v) { return (v < s.sink_tiles ? v : v - s.sink_tiles + s.first_tile) * kTile; }

// How a call is cut: items are (sequence, kv head, block of rows), each a list of key tiles. `whole`: an item a CTA. Else
// the lists are laid end to end, each behind the few units that an item costs beside its tiles, and cut into equal ranges,
// one a CTA; parts of cut items go to records, which a second kernel joins. Heads of 0, 4, 8 units: 8 nodes on 32 contexts 155,
// 146, 147 us, 64 nodes 245, 238, 241, the window of 4096 108, 107, 115.
constexpr int kItemHead = 4;

struct Split {
    int whole;
    int grid;
    int row_blocks;
    int items;  // of a sequence
};

// The item that a CTA's range begins within, for the join: pieces of it are records of CTAs c0 to c1. None (c1 = 0) where the
// range begins with an item, or another CTA's range begins within the same one before.
struct Cut {
    int b, kvh, block;
    int c0, c1;
    int first;  // the record of c0
};

struct Record {
    float* o;    // [2 grid][D / 4][rows of an item][4]
    float2* ml;  // [2 grid][rows of an item]
    Cut* cut;    // [grid]
    int* odd;    // [grid]: values that are not finite where some rows do not see them
};

struct Range {
    long long total, per;  // key tiles of all items, of a CTA
    long long found_base;  // start of the sequence found
    int found;             // -1: beyond the end
};

// The work list's length, and the sequence that holds unit `at(per)` of it. All threads of a CTA of WARPS warps call.
template <int WARPS, class At>
__device__ __forceinline__ Range locate(const FaTreeParams& p, const Split& split, long long* warp_sum, long long* found_base,
                                        int* found, At at) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int share = (p.cache.batch + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = min(static_cast<int>(threadIdx.x) * share, p.cache.batch);
    const int b1 = min(b0 + share, p.cache.batch);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        mine += sequence(p, b).tiles + kItemHead;
    }
    mine *= split.items;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        incl += lane >= o ? up : 0;
    }
    if (lane == 31) {
        warp_sum[warp] = incl;
    }
    if (threadIdx.x == 0) {
        *found = -1;
    }
    __syncthreads();
    Range r;
    r.total = 0;
    long long before = incl - mine;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? warp_sum[w] : 0;
        r.total += warp_sum[w];
    }
    r.per = (r.total + split.grid - 1) / split.grid;
    const long long target = at(r.per);
    if (target >= before && target < before + mine) {
        long long base = before;
        for (int b = b0; b < b1; ++b) {
            const long long n = static_cast<long long>(sequence(p, b).tiles + kItemHead) * split.items;
            if (target < base + n) {
                *found = b;
                *found_base = base;
                break;
            }
            base += n;
        }
    }
    __syncthreads();
    r.found = *found;
    r.found_base = *found_base;
    return r;
}

// A CTA's range as pieces of items, in order.
struct Walk {
    Sequence s;
    int b, item, v;
    long long left;    // units from here on
    int record;        // of the next cut piece
};

// Found at the start of a CTA's range, by one thread.
__device__ __forceinline__ Cut cut_at(const Split& split, const Range& range, const Walk& w, int cta) {
    Cut cut{};
    if (range.found >= 0 && w.left > 0 && w.v > 0) {
        const long long head = range.found_base + static_cast<long long>(w.item) * (w.s.tiles + kItemHead);
        const long long start = head + kItemHead;  // of its tiles
        const int c0 = static_cast<int>(start / range.per);
        if (c0 == cta - 1) {
            cut.b = w.b;
            cut.kvh = w.item / split.row_blocks;
            cut.block = w.item - cut.kvh * split.row_blocks;
            cut.c0 = c0;
            cut.c1 = static_cast<int>((start + w.s.tiles - 1) / range.per);
            // A CTA's first piece is its record 0, its last one its record 1.
            cut.first = 2 * c0 + (c0 * range.per >= head ? 0 : 1);
        }
    }
    return cut;
}

struct Piece {
    int b, kvh, block, v0, v1;
    int record;  // -1: a whole item
};

__device__ __forceinline__ Walk start_walk(const FaTreeParams& p, const Split& split, const Range& range, int cta) {
    Walk w;
    if (split.whole) {
        w.b = cta / split.items;
        w.item = cta - w.b * split.items;
        w.v = 0;
        w.s = sequence(p, w.b);
        w.left = w.s.tiles;
    } else if (range.found < 0) {
        w.b = w.item = w.v = 0;
        w.left = 0;
        w.s = Sequence{};
    } else {
        const long long at = cta * range.per;
        w.b = range.found;
        w.s = sequence(p, w.b);
        const long long in_seq = at - range.found_base;
        w.item = static_cast<int>(in_seq / (w.s.tiles + kItemHead));
        w.v = static_cast<int>(in_seq - static_cast<long long>(w.item) * (w.s.tiles + kItemHead)) - kItemHead;
        w.left = min(range.per, range.total - at);
        if (w.v < 0 && w.left <= -w.v) {
            w.left = 0;
        }
    }
    w.record = 2 * cta;
    return w;
}

// The piece at hand; `s` is its sequence. False at the end.
__device__ __forceinline__ bool next_piece(const FaTreeParams& p, const Split& split, Walk& w, Piece& piece, Sequence& s) {
    if (w.left <= 0) {
        return false;
    }
    if (w.v < 0) {  // what an item costs beside its tiles
        w.left += w.v;
        w.v = 0;
    }
    s = w.s;
    piece.b = w.b;
    piece.kvh = w.item / split.row_blocks;
    piece.block = w.item - piece.kvh * split.row_blocks;
    piece.v0 = w.v;
    const int take = static_cast<int>(min(static_cast<long long>(s.tiles - w.v), w.left));
    piece.v1 = w.v + take;
    piece.record = w.v == 0 && take == s.tiles ? -1 : w.record;
    w.record = 2 * static_cast<int>(blockIdx.x) + 1;  // a range has a cut piece at its start and at its end
    w.left -= take;
    w.v = -kItemHead;
    if (w.left > 0 && ++w.item == split.items) {
        w.item = 0;
        w.s = sequence(p, ++w.b);
    }
    if (w.left <= kItemHead) {
        w.left = 0;  // the range ends before the item's first tile
    }
    return true;
}

// What a wait that was given up leaves word of.
struct Waits {
    volatile int* abort;  // of the CTA, in shared memory
    unsigned* code;
};

// A bounded wait of a whole warp: 2^20 polls, 20 ms at the least, where a healthy wait is a tile's time. In few instructions,
// for there are many of them and the kernel's loops have to fit the instruction cache (with a look at the clock in each,
// 32 nodes on 4 long contexts took 411 us instead of 299). False: given up, by this warp or another of the CTA.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, int phase, const Waits& waits, unsigned code) {
    const uint32_t at = smem_u32(bar);
    const uint32_t parity = static_cast<uint32_t>(phase) & 1u;
    bool there = false;
#pragma unroll 1
    for (int i = 0; i < (1 << 20); ++i) {
        there = mbar_try_wait(at, parity);
        if (there || *waits.abort != 0) {
            break;
        }
    }
    there = __all_sync(0xffffffffu, there) != 0;
    if (!there && *waits.abort == 0) {
        *waits.abort = 1;
        atomicOr(waits.code, code);
    }
    return there;
}

// Nonzero if a word of cache elements holds one that is not finite.
template <class C>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    if constexpr (C::E4M3) {
        return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // e4m3 has NaN (all ones) and no infinity
    } else if constexpr (C::BF16) {
        return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    } else {
        return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    }
}

// Two e4m3 pairs of a word, widened exactly.
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

// Byte offset of 16-byte chunk `c` (8 dims) of row `r` in a tile of 64-dim boxes with the 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * kBox + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// The same in a tile of e4m3 values: rows of 128 bytes with the 128-byte swizzle, or of 64 with the 64-byte one.
template <int D>
__device__ __forceinline__ uint32_t code_offset(int r, int c) {
    return D == 128 ? static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)) : static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// Two of P: at most 2^(kLazy + kUp), which float16 holds twice over; more where scores pass 2^23 and the maximum is rounded to
// whole powers of two, and then float16's largest value rather than infinity.
template <bool BF16>
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
    if constexpr (BF16) {
        return pack_bf162(lo, hi);
    } else {
        uint32_t r;
        asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
}

__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
    return w;
}

// A piece listed for the softmax and the products; n = 0: the end.
__device__ __forceinline__ bool list_part(const FaTreeParams& p, DeviceStatus* status, Shared& sh, int part, const Piece& piece, const Sequence& s,
                                          int n, const Waits& waits) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    Part& to = sh.part[part % kParts];
    if (!warp_wait(&sh.part_empty[part % kParts], part / kParts + 1, waits, kStatusTimeoutProducer)) {
        return false;
    }
    if (n > 0) {
        const int32_t* parents = p.parents + piece.b * p.parent_stride;
        bool bad = s.count > 0 && (s.context < 0 || s.context > held(p.cache) - s.count);
        int start = 0;  // of the run at the end of the nodes before
        for (int t0 = 0; t0 < s.count; t0 += 32) {
            const int t = t0 + lane;
            int up = t < s.count ? __ldg(parents + t) : -1;
            if (up < -1 || up >= t) {
                bad = true;
                up = -1;
            }
            int low = t > 0 && up == t - 1 ? -1 : t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int before = __shfl_up_sync(0xffffffffu, low, o);
                low = lane >= o ? max(low, before) : low;
            }
            low = max(low, start);
            start = __shfl_sync(0xffffffffu, low, 31);
            if (t < s.count) {
                to.low[t] = static_cast<uint8_t>(low);
                // The first node's parent: the entry of the run's first node, which is its own.
                if (low == t) {
                    to.up[t] = up < 0 ? 255 : static_cast<uint8_t>(up);
                }
            }
        }
        if (bad) {
            atomicOr(&status->code, kStatusBadPage);
        }
    }
    if (lane == 0) {
        to.n = n;
        to.b = piece.b;
        to.kvh = piece.kvh;
        to.block = piece.block;
        to.record = piece.record;
        to.context = s.context;
        to.count = s.count;
        to.last = s.last;
    }
    __syncwarp();
    if (lane == 0) {
        mbar_arrive(smem_u32(&sh.part_full[part % kParts]));
    }
    return true;
}

// The range's key tiles: listed for the others, and copied, K and V, a copy a page. Every second tile is this warp's, so
// that the loads of pages and scales of two tiles are on their way at once.
template <class C>
__device__ __forceinline__ void list_tiles(const FaTreeParams& p, const CUtensorMap* tm_k, const CUtensorMap* tm_v, const Split& split,
                                           DeviceStatus* status, Walk walk, Shared& sh, uint32_t smem, int which, const Waits& waits) {
    const FaCache& c = p.cache;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int log2_page = 31 - __clz(c.page_size);
    const int log2_span = min(log2_page, 7);
    constexpr int kVRing = C::E4M3 ? C::kRStages : C::kVStages;
    uint64_t* v_free = C::E4M3 ? sh.r_empty : sh.v_empty;
    Piece piece;
    Sequence s;
    piece.v1 = 0;
    int n = -1;  // the tile at hand
    int v = -1;
    int turn = which;  // the tile that is this warp's
    int parts = 0;
    auto wait = [&](uint64_t* bar, int phase) {
        return warp_wait(bar, phase + 1, waits, kStatusTimeoutProducer);
    };
    while (true) {
        bool more = true;
        if (++v >= piece.v1) {
            more = next_piece(p, split, walk, piece, s);
            v = piece.v0;
            if (which == 0 && !list_part(p, status, sh, parts++, piece, s, more ? piece.v1 - piece.v0 : 0, waits)) {
                return;
            }
        }
        if (++n != turn) {
            if (!more) {
                return;  // the end is another warp's
            }
            continue;
        }
        turn += kListWarps;
        Listed& to = sh.list[n % kListed];
        if (!more) {
            if (wait(&sh.list_empty[n % kListed], n / kListed) && lane == 0) {
                to.key0 = -1;
                mbar_arrive(smem_u32(&sh.list_full[n % kListed]));
            }
            return;
        }
        const int key0 = tile_key(s, v);
        // Lane i's span: what lies in one page.
        const int span_key = key0 + (lane << log2_span);
        int id = -1;
        if (lane < (kTile >> log2_span) && span_key >= 0 && span_key <= s.last &&
            (span_key + (1 << log2_span) > s.first || span_key < p.sinks)) {
            id = __ldg(c.page_table + piece.b * c.table_stride + (span_key >> log2_page));
            if (id < 0 || id >= c.num_pages) {
                id = -1;
                atomicOr(&status->code, kStatusBadPage);
            }
        }
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, id >= 0)) * (static_cast<uint32_t>(C::D * C::kElem) << log2_span);
        const int y = span_key & (c.page_size - 1);
        const uint32_t row = static_cast<uint32_t>(lane) << log2_span;
        auto copy = [&](uint32_t tile, const CUtensorMap* map, uint64_t* full) {
            if (lane == 0) {
                mbar_arrive_expect_tx(smem_u32(full), bytes);
            }
            __syncwarp();
            if (id >= 0) {
                if constexpr (C::E4M3) {
                    tma_load_4d(tile + row * C::D, map, smem_u32(full), 0, y, piece.kvh, id);
                } else {
#pragma unroll
                    for (int box = 0; box < C::D / 64; ++box) {
                        tma_load_4d(tile + box * kBox + row * 128, map, smem_u32(full), 64 * box, y, piece.kvh, id);
                    }
                }
            }
        };
        if (!wait(&sh.k_empty[n % C::kKStages], n / C::kKStages)) {
            return;
        }
        copy(smem + C::kSmemK + (n % C::kKStages) * C::kRaw, tm_k, &sh.k_full[n % C::kKStages]);
        // The groups' pages and scales.
        const int group = lane % kGroups;
        const int key = key0 + 8 * group;
        const int page = __shfl_sync(0xffffffffu, id, (8 * group) >> log2_span);
        const bool wanted = key >= 0 && key <= s.last && (key + 7 >= s.first || key < p.sinks);
        float ks = 1.0f, vs = 1.0f;
        if (C::E4M3 && page >= 0) {
            const int64_t at = static_cast<int64_t>(page) * c.kv_heads + piece.kvh;
            ks = __ldg(c.k_scale + at);
            vs = __ldg(c.v_scale + at);
        }
        if (!wait(&v_free[n % kVRing], n / kVRing)) {
            return;
        }
        copy(smem + (C::E4M3 ? C::kSmemR : C::kSmemV) + (n % kVRing) * C::kRaw, tm_v, &sh.r_full[n % kVRing]);
        if (!wait(&sh.list_empty[n % kListed], n / kListed)) {
            return;
        }
        bool tiny = false;
        if constexpr (C::E4M3) {
            tiny = vs < kMinScale;
            const float used = tiny ? kMinScale : vs;
            if (lane < kGroups) {
                to.group[lane] = make_float4(ks, __log2f(used), __fdividef(C::kDown, used), 0.0f);
            }
        }
        const uint32_t paged = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
        const uint32_t gone = __ballot_sync(0xffffffffu, wanted && page < 0) & 0xffffu;
        const uint32_t tiny_bits = __ballot_sync(0xffffffffu, tiny) & 0xffffu;
        if (lane < 4) {
            const int kb = key0 + 32 * lane;
            uint32_t bits = bits_up_to(s.last - kb) & (~bits_up_to(s.first - 1 - kb) | bits_up_to(p.sinks - 1 - kb));
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                bits &= (paged >> (4 * lane + g)) & 1u ? 0xffffffffu : ~(0xffu << (8 * g));
            }
            reinterpret_cast<uint32_t*>(&to.shown)[lane] = bits;
        }
        if (lane == 0) {
            to.key0 = key0;
            to.gone = gone;
            to.tiny = tiny_bits;
            const int near = window_first(max(s.context, 0) + s.count, p.window);
            to.mixed = c.tokens > 1 && (key0 > s.context - kTile || (p.window > 0 && key0 < near));
            to.full = gone == 0 && key0 <= min(s.context - 1, s.last) - (kTile - 1) && (p.window == 0 || key0 >= near || key0 <= p.sinks - kTile);
        }
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(smem_u32(&sh.list_full[n % kListed]));
        }
    }
}

// V's tiles made ready: e4m3 values widened to float16 and laid out for the product, rows that no row of the call sees made
// zeros (0 times what lies there could be NaN), and what is not finite noticed where rows differ in what they see.
template <class C>
__device__ __forceinline__ void ready_values(const FaTreeParams& p, Shared& sh, uint32_t smem, const Waits& waits) {
    constexpr int kRing = C::E4M3 ? C::kRStages : C::kVStages;
    constexpr int kChunks = C::D * C::kElem / 16;  // 16-byte words of a row
    const int lt = static_cast<int>(threadIdx.x) % 128;
    const int lane = lt % 32;
    const int warp = lt / 32;
    auto wait = [&](uint64_t* bar, int phase) {
        return warp_wait(bar, phase, waits, kStatusTimeoutProducer);
    };
    bool odd = false;
    for (int n = 0;; ++n) {
        if (!wait(&sh.list_full[n % kListed], n / kListed)) {
            break;
        }
        const Listed& t = sh.list[n % kListed];
        if (t.key0 < 0) {
            break;
        }
        const bool mixed = t.mixed != 0;
        [[maybe_unused]] const uint32_t tiny = t.tiny;
        const bool whole = (t.shown.x & t.shown.y & t.shown.z & t.shown.w) == 0xffffffffu;
        const uint32_t* shown = reinterpret_cast<const uint32_t*>(&t.shown);
        if (!wait(&sh.r_full[n % kRing], n / kRing)) {
            break;
        }
        const uint32_t wide = smem + C::kSmemV + (n % C::kVStages) * C::kWide;
        if constexpr (C::E4M3) {
            const uint32_t raw = smem + C::kSmemR + (n % C::kRStages) * C::kRaw;
            if (!wait(&sh.v_empty[n % C::kVStages], n / C::kVStages + 1)) {
                break;
            }
            if (mixed || !whole || tiny != 0) {
                // The warp's rows as the cache holds them, in place (wherever the swizzle has a word in its row).
                uint32_t any = 0;
#pragma unroll 1
                for (int i = warp * 32 * kChunks + lane; i < (warp + 1) * 32 * kChunks; i += 32) {
                    const int r = i / kChunks;
                    uint4 w = load_shared16(raw + i * 16);
                    if (!((shown[r >> 5] >> (r & 31)) & 1u)) {
                        w = make_uint4(0u, 0u, 0u, 0u);
                    } else if ((tiny >> (r >> 3)) & 1u) {  // NaN stays
                        w = make_uint4(w.x & (not_finite<C>(w.x) >> 7) * 255u, w.y & (not_finite<C>(w.y) >> 7) * 255u,
                                       w.z & (not_finite<C>(w.z) >> 7) * 255u, w.w & (not_finite<C>(w.w) >> 7) * 255u);
                    }
                    any |= not_finite<C>(w.x) | not_finite<C>(w.y) | not_finite<C>(w.z) | not_finite<C>(w.w);
                    store_shared16(raw + i * 16, w.x, w.y, w.z, w.w);
                }
                odd = odd || (mixed && any != 0);
                __syncwarp();
            }
            // Words of 8 lanes that load and store together: D = 128, half a row of rows r and r ^ 5, which the swizzles of
            // 128-byte rows (codes: by r, values: two chunks apart) put into different banks; D = 64, two rows.
            constexpr int kPasses = kTile * kChunks / 128;
#pragma unroll 1
            for (int i0 = 0; i0 < kPasses; i0 += 4) {
                uint4 w[4];
                uint32_t to[4];
                const int chunk = C::D == 128 ? (lane & 3) + ((lane >> 1) & 4) : lane & 3;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int r;
                    if constexpr (C::D == 128) {
                        const int a = 2 * (i & 1) + (lane >> 4);
                        r = warp * 32 + ((i0 + i) >> 1) * 8 + ((lane & 4) != 0 ? a ^ 5 : a);
                        w[i] = load_shared16(raw + code_offset<128>(r, chunk));
                    } else {
                        r = warp * 32 + (i0 + i) * 8 + (lane >> 2);
                        w[i] = load_shared16(raw + r * 64 + chunk * 16);
                    }
                    to[i] = wide + tile_offset(r, 2 * chunk);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t h[8];
                    widen4(w[i].x, h[0], h[1]);
                    widen4(w[i].y, h[2], h[3]);
                    widen4(w[i].z, h[4], h[5]);
                    widen4(w[i].w, h[6], h[7]);
                    store_shared16(to[i], h[0], h[1], h[2], h[3]);
                    store_shared16(to[i] ^ 16u, h[4], h[5], h[6], h[7]);  // the odd chunk of the pair
                }
            }
            fence_proxy_async_smem();
        } else if (mixed || !whole) {
            uint32_t any = 0;
#pragma unroll 1
            for (int i = lt; i < kTile * kChunks; i += 128) {
                const int r = i / kChunks;
                const uint32_t at = wide + tile_offset(r, i % kChunks);
                if (!((shown[r >> 5] >> (r & 31)) & 1u)) {
                    store_shared16(at, 0u, 0u, 0u, 0u);
                } else {
                    const uint4 w = load_shared16(at);
                    any |= not_finite<C>(w.x) | not_finite<C>(w.y) | not_finite<C>(w.z) | not_finite<C>(w.w);
                }
            }
            odd = odd || (mixed && any != 0);
            fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(smem_u32(&sh.v_full[n % C::kVStages]));
            if constexpr (C::E4M3) {
                mbar_arrive(smem_u32(&sh.r_empty[n % C::kRStages]));
            }
            mbar_arrive(smem_u32(&sh.list_empty[n % kListed]));
        }
    }
    if (odd) {
        sh.odd = 1;
    }
}

template <class C>
__device__ __forceinline__ void issue_scores(uint32_t d, uint64_t a, uint64_t b) {
    // kind::f8f6f4 with e4m3 operands has the instruction descriptor of kind::f16 with float16.
    constexpr uint32_t idesc = make_idesc_f16(kTile, kTile, true, false, C::kMmaBf16);
    if constexpr (C::E4M3) {
#pragma unroll
        for (int term = 0; term < C::kTerms; ++term) {
#pragma unroll
            for (int k = 0; k < C::D / 32; ++k) {
                umma_ss_f8(d, a + static_cast<uint64_t>((term * C::kRaw + 32 * k) >> 4), b + static_cast<uint64_t>((32 * k) >> 4), idesc,
                           term + k > 0 ? 1u : 0u);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < C::D / 16; ++k) {
            const uint64_t off = static_cast<uint64_t>(((k / 4) * kBox + (k % 4) * 32) >> 4);
            umma_ss(d, a + off, b + off, idesc, k > 0 ? 1u : 0u);
        }
    }
}

template <class C>
__device__ __forceinline__ void issue_product(uint32_t acc, uint32_t w, uint64_t t, bool first) {
    constexpr uint32_t idesc = make_idesc_f16(kTile, C::D, true, true, C::kMmaBf16);
#pragma unroll
    for (int k = 0; k < kTile / 16; ++k) {
        umma_ts(acc, w + k * 8, t + static_cast<uint64_t>(k * (2048 >> 4)), idesc, (first && k == 0) ? 0u : 1u);
    }
}

// Products, scores and P V by a warp each: a warp's waits on barriers, which queue behind the products' own traffic in shared
// memory, come to about 300 cycles even for what is there, so that one warp for both is what the kernel would wait for. Step
// s is key tile s (NR 1) or row tile s % 2 of key tile s / 2 (NR 2), warpgroup s % 2's.
template <class C, class Scores>
__device__ __forceinline__ bool walk_parts(Shared& sh, const Waits& waits, Scores take) {
    for (int items = 0, tiles = 0;; ++items) {
        if (!warp_wait(&sh.part_full[items % kParts], items / kParts, waits, kStatusTimeoutMma)) {
            return false;
        }
        const int n = sh.part[items % kParts].n;
        if (n == 0) {
            return true;
        }
        __syncwarp();
        if (elect_one()) {
            mbar_arrive(smem_u32(&sh.part_empty[items % kParts]));
        }
        __syncwarp();
        if (!take(items, tiles, n * C::NR)) {
            return false;
        }
        tiles += n;
    }
}

__device__ __forceinline__ bool mma_wait(uint64_t* bar, int parity, const Waits& waits) {
    const bool there = warp_wait(bar, parity, waits, kStatusTimeoutMma);
    tc_fence_after();
    return there;
}

template <class C>
__device__ __forceinline__ void score_warp(Shared& sh, uint32_t smem, const Waits& waits) {
    constexpr int NR = C::NR;
    auto kmajor = [](uint32_t at) { return C::E4M3 && C::D == 64 ? make_desc_kmajor_sw64(at) : make_desc_kmajor_sw128(at); };
    const uint64_t q = kmajor(smem + C::kSmemQ);
    const uint64_t k = kmajor(smem + C::kSmemK);
    auto off = [](int tile, int bytes) { return static_cast<uint64_t>(tile * (bytes >> 4)); };
    int done0 = 0, done1 = 0;  // scores of either warpgroup
    int last = -1;             // whose were the last
    walk_parts<C>(sh, waits, [&](int items, int tiles, int steps) {
        if (!mma_wait(&sh.q_full, items, waits)) {
            return false;
        }
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            const int tile = tiles + (NR == 1 ? step : step >> 1);
            const int w = step & 1;
            if ((NR == 1 || w == 0) && !mma_wait(&sh.k_full[tile % C::kKStages], tile / C::kKStages, waits)) {
                return false;
            }
            if (last >= 0 && !mma_wait(&sh.s_free[last], (last == 0 ? done0 : done1) - 1, waits)) {
                return false;
            }
            if (elect_one()) {
                issue_scores<C>(C::kTmemS, q + off(NR == 1 ? 0 : w, C::kQTile), k + off(tile % C::kKStages, C::kRaw));
                umma_commit(smem_u32(&sh.s_full[w]));
                if (NR == 1 || w == 1) {
                    umma_commit(smem_u32(&sh.k_empty[tile % C::kKStages]));
                }
                if (step == steps - 1) {
                    umma_commit(smem_u32(&sh.q_empty));
                }
            }
            __syncwarp();
            last = w;
            done0 += 1 - w;
            done1 += w;
        }
        return true;
    });
    // Every product issued must be complete before tensor memory is released.
    if (elect_one()) {
        umma_commit(smem_u32(&sh.mma_idle));
    }
    __syncwarp();
}

template <class C>
__device__ __forceinline__ void product_warp(Shared& sh, uint32_t smem, const Waits& waits) {
    constexpr int NR = C::NR;
    const uint64_t v = make_desc_mnmajor_sw128(smem + C::kSmemV, kBox);
    int taken0 = 0, taken1 = 0;  // P of either warpgroup
    walk_parts<C>(sh, waits, [&](int items, int tiles, int steps) {
        if (items > 0 && !mma_wait(&sh.o_free, items - 1, waits)) {
            return false;
        }
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            const int tile = tiles + (NR == 1 ? step : step >> 1);
            const int w = step & 1;
            if ((NR == 1 || w == 0) && !mma_wait(&sh.v_full[tile % C::kVStages], tile / C::kVStages, waits)) {
                return false;
            }
            if (!mma_wait(&sh.p_full[w], w == 0 ? taken0++ : taken1++, waits)) {
                return false;
            }
            if (elect_one()) {
                issue_product<C>(C::kTmemO + w * C::D, C::kTmemP + w * (kTile / 2),
                                 v + static_cast<uint64_t>((tile % C::kVStages) * (C::kWide >> 4)), step < 2);
                umma_commit(smem_u32(&sh.p_free[w]));
                if (NR == 1 || w == 1) {
                    umma_commit(smem_u32(&sh.v_empty[tile % C::kVStages]));
                }
                if (step == steps - 1) {
                    umma_commit(smem_u32(&sh.done));
                }
            }
            __syncwarp();
        }
        return true;
    });
    if (elect_one()) {
        umma_commit(smem_u32(&sh.mma_idle));
    }
    __syncwarp();
    unsigned unused = 0;  // no other CTA listens
    mbar_wait_drain(smem_u32(&sh.mma_idle), 0, WaitCtx{&sh.abort, waits.code, &unused, 0}, kStatusTimeoutTeardown);
    __syncwarp();
}

// A thread's query row.
struct Row {
    bool real;          // a node's (else padding, or beyond the rows)
    int token;
    int first;          // first position of its window
    float factor;       // of a score, in log2 units
};

// A warp's rows of Q's tile (NR 1: half of its 32, the other warpgroup has the others), 16 dims a lane: as they are, or, over
// an e4m3 cache, as sums of e4m3 terms (each the nearest to what the ones before leave), a row brought to [2^8, 448] by a
// power of two that its factor takes back. e4m3's steps end at 2^-9: two terms hold bfloat16 exactly down to 2^-10 of the row's
// largest value, three float16 down to 2^-7 of it, and what is smaller is off by 2^-18 of the largest at most. `at`, `real`: the lane's own row; ready() waits until the tile may be written. Returns the factor of
// the lane's own row (NR 1: in `factors` by row, for both warpgroups).
template <class C, class Ready>
__device__ __forceinline__ float bring_queries(const FaTreeParams& p, const uint16_t* at, bool real, uint32_t tile, int quarter, int w,
                                               float* factors, Ready ready) {
    constexpr int kLanes = C::D / 16;     // of a row
    constexpr int kAtOnce = 32 / kLanes;  // rows
    constexpr int kPasses = kLanes / (C::NR == 1 ? 2 : 1);
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int part = lane % kLanes;
    const int row0 = (C::NR == 1 ? 16 * w : 0) + lane / kLanes;
    const uint32_t sign = p.softmax_scale < 0.0f ? 0x80008000u : 0u;  // the factor stays positive
    const float scale = fmaxf(fabsf(p.softmax_scale) * kLog2e, kLeastFactor);
    float factor = scale;
    uint4 word[2][2], next[2][2];
    auto load = [&](int pass, uint4 (&to)[2]) {
        const uint64_t from = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(at), (row0 + pass * kAtOnce) & 31);
        const bool there = __shfl_sync(0xffffffffu, static_cast<int>(real), (row0 + pass * kAtOnce) & 31) != 0;
        const uint4* src = reinterpret_cast<const uint4*>(from) + 2 * part;
        to[0] = there ? __ldg(src) : make_uint4(0u, 0u, 0u, 0u);
        to[1] = there ? __ldg(src + 1) : make_uint4(0u, 0u, 0u, 0u);
    };
    load(0, next[0]);
    load(1, next[1]);
    if (!ready()) {
        return factor;
    }
#pragma unroll 1
    for (int pass0 = 0; pass0 < kPasses; pass0 += 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            word[e][0] = next[e][0];
            word[e][1] = next[e][1];
            if (pass0 + 2 < kPasses) {
                load(pass0 + 2 + e, next[e]);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = pass0 + half;
            const int owner = row0 + i * kAtOnce;
            const int r = quarter * 32 + owner;
            const uint32_t x[8] = {word[half][0].x ^ sign, word[half][0].y ^ sign, word[half][0].z ^ sign, word[half][0].w ^ sign,
                                   word[half][1].x ^ sign, word[half][1].y ^ sign, word[half][1].z ^ sign, word[half][1].w ^ sign};
            if constexpr (!C::E4M3) {
                store_shared16(tile + tile_offset(r, 2 * part), x[0], x[1], x[2], x[3]);
                store_shared16(tile + tile_offset(r, 2 * part + 1), x[4], x[5], x[6], x[7]);
            } else {
                uint32_t top = 0;  // of the values' bits without sign: their order is that of the sizes
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    top = max(top, max(x[e] & 0x7fffu, (x[e] >> 16) & 0x7fffu));
                }
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) {
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                }
                // 2^(8 - exponent of the largest), one less where that would pass 448: from 2^-120 on, and to 2^100, so that the
                // factor, which takes it back, stays above kLeastFactor; 1 for zeros. A row with an infinity or NaN becomes NaN:
                // e4m3 has no infinity.
                const uint32_t most = __float_as_uint(widen16<C::BF16>(static_cast<uint16_t>(top)));
                const int e = static_cast<int>(most >> 23);
                const int shift = (e == 0 || e == 255) ? 0 : min(135 - e - ((most & 0x7fffffu) > 0x600000u ? 1 : 0), 100);
                const float up = e == 255 ? NAN : __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
                const float back = fmaxf(scale * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23), kLeastFactor);
                if constexpr (C::NR == 1) {
                    if (part == 0) {
                        factors[r] = back;
                    }
                } else {
                    const float rows_own = __shfl_sync(0xffffffffu, back, (lane % kAtOnce) * kLanes);
                    factor = lane / kAtOnce == i ? rows_own : factor;
                }
                float f[16];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    f[2 * j] = widen16<C::BF16>(static_cast<uint16_t>(x[j] & 0xffffu)) * up;
                    f[2 * j + 1] = widen16<C::BF16>(static_cast<uint16_t>(x[j] >> 16)) * up;
                }
#pragma unroll
                for (int term = 0; term < C::kTerms; ++term) {
                    uint32_t code[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t lo = pack_e4m3x2(f[4 * j], f[4 * j + 1]);
                        const uint32_t hi = pack_e4m3x2(f[4 * j + 2], f[4 * j + 3]);
                        code[j] = lo | (hi << 16);
                        const float2 u = unpack_half2(e4m3x2_to_half2(lo));
                        const float2 v = unpack_half2(e4m3x2_to_half2(hi));
                        f[4 * j] -= u.x;
                        f[4 * j + 1] -= u.y;
                        f[4 * j + 2] -= v.x;
                        f[4 * j + 3] -= v.y;
                    }
                    store_shared16(tile + term * C::kRaw + code_offset<C::D>(r, part), code[0], code[1], code[2], code[3]);
                }
            }
        }
    }
    fence_proxy_async_smem();
    return factor;
}

// A tile's columns that a row sees, as bits.
__device__ __forceinline__ uint4 kept_columns(const FaTreeParams& p, const Part& s, const Row& row, int key0, uint32_t gone) {
    uint32_t keep[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int kb = key0 + 32 * i;
        keep[i] = bits_up_to(s.context - 1 - kb);
        if (p.window > 0) {
            keep[i] &= ~bits_up_to(row.first - 1 - kb) | bits_up_to(p.sinks - 1 - kb);
        }
    }
    if (key0 > s.context - kTile) {
        const int column = s.context - key0;  // of node 0
        for (int at = row.real ? row.token : -1; at >= 0;) {
            const int low = s.low[at];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                keep[i] |= bits_up_to(column + at - 32 * i) & ~bits_up_to(column + low - 1 - 32 * i);
            }
            const int up = s.up[low];
            at = up == 255 ? -1 : up;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // 4 groups of 8 keys, and the end of the table.
        const uint32_t pages = ~(gone >> (4 * i));
        keep[i] &= bits_up_to(s.last - (key0 + 32 * i));
        keep[i] &= ((pages & 1u) * 0xffu) | (((pages >> 1) & 1u) * 0xff00u) | (((pages >> 2) & 1u) * 0xff0000u) | (((pages >> 3) & 1u) * 0xff000000u);
        keep[i] = row.real ? keep[i] : 0u;
    }
    return make_uint4(keep[0], keep[1], keep[2], keep[3]);
}

// The largest of one group of GROUP scores.
template <int GROUP, int N>
__device__ __forceinline__ float group_most(const uint32_t (&x)[N], int at) {
    float most[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        most[i] = fmax_nan(u2f(x[at + i]), u2f(x[at + 4 + i]));
    }
#pragma unroll
    for (int j = 8; j < GROUP; j += 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            most[i] = fmax3(most[i], u2f(x[at + j + i]), u2f(x[at + j + 4 + i]));
        }
    }
    return fmax_nan(fmax3(most[0], most[1], most[2]), most[3]);
}

// P of one group, in pairs of 16 bits, and its share of the sum.
template <class C, int GROUP, int N>
__device__ __forceinline__ void group_exponentials(const uint32_t (&x)[N], int at, uint32_t* packed, float f, float add, float inv, float& l) {
    const float2 f2 = make_float2(f, f), add2 = make_float2(add, add);
    float2 sum[4];
#pragma unroll
    for (int i = 0; i < GROUP / 2; ++i) {
        float2 y = __ffma2_rn(make_float2(u2f(x[at + 2 * i]), u2f(x[at + 2 * i + 1])), f2, add2);
        y = make_float2(ex2_approx(y.x), ex2_approx(y.y));
        sum[i & 3] = i < 4 ? y : __fadd2_rn(sum[i & 3], y);
        packed[i] = pack_weights<C::kMmaBf16>(y.x, y.y);
    }
    const float2 all = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
    l = fmaf(all.x + all.y, inv, l);
}

// The new maximum, and what the sums so far shrink by.
__device__ __forceinline__ float raise(float top, float& m, float& l) {
    float alpha = 1.0f;
    if (!(top <= m + kLazy)) {  // NaN among it
        alpha = ex2_approx(m - top);
        m = top;
    }
    l *= alpha;
    return alpha;
}

// One row's scores turned into P: returns what the sums so far shrink by (l is done here). taken() once the scores are in
// registers for good. All 128 at once, so that the next tile's scores can follow, where 32 keys on
// end share a page and its scales (or there are none).
template <class C, class Taken>
__device__ __forceinline__ float exponentials(const Listed& aux, uint32_t tmem_s, uint32_t tmem_p, float factor, float& m, float& l, Taken taken) {
    uint32_t x[128];
    tmem_ld64_of128<0>(tmem_s, x);
    tmem_ld64_of128<64>(tmem_s + 64, x);
    tmem_wait_ld();
    taken();
    float top = -INFINITY;
    if constexpr (C::E4M3) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float2 a = *reinterpret_cast<const float2*>(&aux.group[4 * c]);
            top = fmax_nan(top, fmaf(group_most<32>(x, 32 * c), fmaxf(factor * a.x, kLeastFactor), a.y));
        }
    } else {
        top = row_extreme<true, 128>(x) * factor;
    }
    const float alpha = raise(top, m, l);
    const float used = (m == -INFINITY ? 0.0f : m) - C::kUp;
    __syncwarp();  // tensor memory is accessed by whole warps
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float f = factor, add = -used, inv = 1.0f;
        if constexpr (C::E4M3) {
            const float4 a = aux.group[4 * c];
            f = fmaxf(f * a.x, kLeastFactor);
            add = a.y - used;
            inv = a.z;
        }
        uint32_t packed[16];  // P of 32 keys takes 16 columns
        group_exponentials<C, 32>(x, 32 * c, packed, f, add, inv, l);
        tmem_st16(tmem_p + 16 * c, packed);
    }
    return alpha;
}

// The same over pages of 8 or 16 tokens, in few registers.
template <class C, class Taken>
__device__ __forceinline__ float exponentials_by_8(const Listed& aux, uint32_t tmem_s, uint32_t tmem_p, float factor, float& m, float& l, Taken taken) {
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t x[32];
        tmem_ld32(tmem_s + 32 * c, x);
        tmem_wait_ld();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float2 a = *reinterpret_cast<const float2*>(&aux.group[4 * c + g]);
            top = fmax_nan(top, fmaf(group_most<8>(x, 8 * g), fmaxf(factor * a.x, kLeastFactor), a.y));
        }
    }
    const float alpha = raise(top, m, l);
    const float used = (m == -INFINITY ? 0.0f : m) - C::kUp;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t x[32], packed[16];
        __syncwarp();
        tmem_ld32(tmem_s + 32 * c, x);
        tmem_wait_ld();
        if (c == 3) {
            taken();
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 a = aux.group[4 * c + g];
            group_exponentials<C, 8>(x, 8 * g, packed + 4 * g, fmaxf(factor * a.x, kLeastFactor), a.y - used, a.z, l);
        }
        tmem_st16(tmem_p + 16 * c, packed);
    }
    return alpha;
}

template <class C>
__device__ __forceinline__ void softmax(const FaTreeParams& p, Shared& sh, Exchange& ex, uint32_t smem, const Record& rec,
                                        const Waits& waits) {
    constexpr int D = C::D;
    constexpr int NR = C::NR;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int w = warp / 4;                  // warpgroup
    const int r = (warp % 4) * 32 + lane;    // row of its tile
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t tmem_s = lanes + C::kTmemS;
    const uint32_t tmem_p = lanes + C::kTmemP + w * (kTile / 2);
    const uint32_t tmem_o = lanes + C::kTmemO + w * D;
    const int group = p.heads / p.cache.kv_heads;
    const int rows = group * p.cache.tokens;
    auto wait = [&](uint64_t* bar, int parity) {
        const bool there = warp_wait(bar, parity, waits, kStatusTimeoutSoftmax);
        tc_fence_after();
        return there;
    };
    auto arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(smem_u32(bar));
        }
    };
    int tiles = 0;   // key tiles of the pieces before
    int steps = 0;   // scores taken
    float next_factor = 0.0f;
    // The queries of piece `items`, on their way while the piece before ends. False: given up.
    auto queries = [&](int items) {
        if (!wait(&sh.part_full[items % kParts], items / kParts)) {
            return false;
        }
        const Part& s = sh.part[items % kParts];
        if (s.n == 0) {
            return true;
        }
        const int row_index = s.block * C::kRows + (NR == 2 ? w * kTile : 0) + r;
        const int head = row_index / p.cache.tokens;
        const int token = row_index - head * p.cache.tokens;
        bool ok = true;
        next_factor = bring_queries<C>(
            p, static_cast<const uint16_t*>(p.q) + s.b * p.q_stride[0] + (s.kvh * group + head) * p.q_stride[1] + token * p.q_stride[2],
            row_index < rows && token < s.count, smem + C::kSmemQ + (NR == 2 ? w * C::kQTile : 0), warp % 4, w, ex.factor[items & 1],
            [&] { return ok = items == 0 || wait(&sh.q_empty, items - 1); });
        if (ok) {
            arrive(&sh.q_full);
        }
        return ok;
    };
    if (!queries(0)) {
        return;
    }
    for (int items = 0;; ++items) {
        const Part& s = sh.part[items % kParts];  // until the end of the piece
        const int n = s.n;
        if (n == 0) {
            return;
        }
        const int row_index = s.block * C::kRows + (NR == 2 ? w * kTile : 0) + r;
        Row row;
        row.token = row_index % p.cache.tokens;
        row.real = row_index < rows && row.token < s.count;
        row.factor = next_factor;
        if (NR == 1 && C::E4M3) {
            if (!wait(&sh.q_full, items)) {
                return;
            }
            row.factor = ex.factor[items & 1][r];
        }
        row.first = 0;
        if (p.window > 0) {
            int above = 0;  // ancestors
            for (int at = row.real ? row.token : -1; at >= 0;) {
                const int low = s.low[at];
                const int up = s.up[low];
                above += at - low + (up == 255 ? 0 : 1);
                at = up == 255 ? -1 : up;
            }
            row.first = window_first(max(s.context + above, 0), p.window);
            __syncwarp();
        }

        float m = -INFINITY, l = 0.0f;
        int mine = 0;  // scores of this piece taken
        for (int t = NR == 1 ? w : 0; t < n; t += NR == 1 ? 2 : 1, ++mine) {
            const int slot = (tiles + t) % kListed;
            // P's place is free and the tile listed by the time its scores are there, most of the time. From the scores on
            // every instruction counts: the next ones are not begun before these are in registers.
            if ((steps > 0 && !wait(&sh.p_free[w], steps - 1)) || !wait(&sh.list_full[slot], (tiles + t) / kListed)) {
                return;
            }
            const bool full = sh.list[slot].full != 0;
            if (!wait(&sh.s_full[w], steps)) {
                return;
            }
            ++steps;
            const Listed& aux = sh.list[slot];
            if (!full) {
                // What the row does not see becomes -inf.
                const uint4 keep4 = kept_columns(p, s, row, aux.key0, aux.gone);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t x[32];
                    __syncwarp();
                    tmem_ld32(tmem_s + 32 * c, x);
                    tmem_wait_ld();
                    const uint32_t keep = c == 0 ? keep4.x : c == 1 ? keep4.y : c == 2 ? keep4.z : keep4.w;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        x[i] = (keep >> i) & 1u ? x[i] : 0xff800000u;
                    }
                    tmem_st32(tmem_s + 32 * c, x);
                }
                tmem_wait_st();
            }
            auto taken = [&] {
                tc_fence_before();
                arrive(&sh.s_free[w]);
            };
            float alpha;
            if constexpr (C::E4M3 && !C::COARSE) {
                alpha = exponentials_by_8<C>(aux, tmem_s, tmem_p, row.factor, m, l, taken);
            } else {
                alpha = exponentials<C>(aux, tmem_s, tmem_p, row.factor, m, l, taken);
            }
            if (mine > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t x[32];
                    tmem_ld32(tmem_o + 32 * c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        x[i] = f2u(u2f(x[i]) * alpha);
                    }
                    tmem_st32(tmem_o + 32 * c, x);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            arrive(&sh.p_full[w]);
            arrive(&sh.list_empty[slot]);
        }
        tiles += n;

        // The end of the piece: rows of both warpgroups joined (NR 1), normalised or left in a record.
        if (!queries(items + 1) || !wait(&sh.done, items)) {
            return;
        }
        float own_weight = 1.0f, other_weight = 0.0f;
        if constexpr (NR == 1) {
            ex.ml[w][r] = make_float2(m, l);
            arrive(&sh.ml_full);
            if (!wait(&sh.ml_full, items)) {
                return;
            }
            const float2 other = ex.ml[1 - w][r];
            const float all = fmax_nan(m, other.x);
            const float base = all == -INFINITY ? 0.0f : all;
            own_weight = ex2_approx(m - base);
            other_weight = ex2_approx(other.x - base);
            l = l * own_weight + other.y * other_weight;
            m = all;
        }
        constexpr int kColumns = NR == 1 ? D / 2 : D;  // of this thread
        const int column0 = NR == 1 ? w * kColumns : 0;
        const bool other = NR == 1 && (n > 1 || w == 1);  // the other sum exists
        const bool self = NR == 2 || w == 0 || n > 1;     // this one does
        const bool in_rows = row_index < rows;
        const int record = s.record;
        const float inv = (record >= 0 ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l)) * C::kDown;
        own_weight = row.real ? own_weight * inv : 0.0f;
        other_weight = row.real ? other_weight * inv : 0.0f;
        // Rows of an item lie one after another in the output. In a record four columns of all rows do, so that the
        // rows' threads write whole lines.
        uint16_t* out = static_cast<uint16_t*>(p.o) + ((static_cast<int64_t>(s.b) * p.heads + s.kvh * group) * p.cache.tokens + row_index) * D + column0;
        float4* kept = reinterpret_cast<float4*>(rec.o) +
                       (static_cast<int64_t>(record) * (D / 4) + column0 / 4) * C::kRows + (NR == 2 ? w * kTile : 0) + r;
#pragma unroll 1
        for (int c = 0; c < kColumns / 32; ++c) {
            uint32_t x[32];
            __syncwarp();
            if (self) {
                tmem_ld32(tmem_o + column0 + 32 * c, x);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = row.real ? f2u(u2f(x[i]) * own_weight) : 0u;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = 0u;
                }
            }
            if (other) {
                uint32_t y[32];
                tmem_ld32(lanes + C::kTmemO + (1 - w) * D + column0 + 32 * c, y);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = row.real ? f2u(fmaf(u2f(y[i]), other_weight, u2f(x[i]))) : 0u;
                }
            }
            if (in_rows && record < 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    reinterpret_cast<uint4*>(out)[4 * c + i] = make_uint4(
                        pack2<C::BF16>(u2f(x[8 * i]), u2f(x[8 * i + 1])), pack2<C::BF16>(u2f(x[8 * i + 2]), u2f(x[8 * i + 3])),
                        pack2<C::BF16>(u2f(x[8 * i + 4]), u2f(x[8 * i + 5])), pack2<C::BF16>(u2f(x[8 * i + 6]), u2f(x[8 * i + 7])));
                }
            } else if (in_rows) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    kept[static_cast<int64_t>(8 * c + i) * C::kRows] =
                        make_float4(u2f(x[4 * i]), u2f(x[4 * i + 1]), u2f(x[4 * i + 2]), u2f(x[4 * i + 3]));
                }
            }
        }
        if (record >= 0 && in_rows && (NR == 2 || w == 0)) {
            rec.ml[static_cast<int64_t>(record) * C::kRows + (NR == 2 ? w * kTile : 0) + r] = row.real ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
        }
        tc_fence_before();
        arrive(&sh.o_free);
        arrive(&sh.part_empty[items % kParts]);
    }
}

template <class C>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const __grid_constant__ FaTreeParams p, const __grid_constant__ CUtensorMap tm_k,
                                                           const __grid_constant__ CUtensorMap tm_v, DeviceStatus* status, Split split,
                                                           Record rec) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = raw;  // on 1024 bytes: a kernel without static shared memory has it from there
    Shared& sh = *reinterpret_cast<Shared*>(smem + C::kSmemShared);
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const Waits waits{&sh.abort, &status->code};
    cudaTriggerProgrammaticLaunchCompletion();  // the second kernel's CTAs may take SMs as they get free
    if (threadIdx.x == 0) {
        sh.abort = 0;
        sh.odd = 0;
        for (int i = 0; i < kMostStages; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
            mbar_init(smem_u32(&sh.r_full[i]), 1);
            mbar_init(smem_u32(&sh.r_empty[i]), kValueWarps);
        }
        for (int i = 0; i < C::kVStages; ++i) {
            mbar_init(smem_u32(&sh.v_full[i]), kValueWarps);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
        }
        for (int i = 0; i < kListed; ++i) {
            mbar_init(smem_u32(&sh.list_full[i]), 1);
            mbar_init(smem_u32(&sh.list_empty[i]), kValueWarps + C::NR * kSoftmaxWarps / 2);
        }
        for (int i = 0; i < kParts; ++i) {
            mbar_init(smem_u32(&sh.part_full[i]), 1);
            mbar_init(smem_u32(&sh.part_empty[i]), kSoftmaxWarps + 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.s_full[i]), 1);
            mbar_init(smem_u32(&sh.s_free[i]), kSoftmaxWarps / 2);
            mbar_init(smem_u32(&sh.p_full[i]), kSoftmaxWarps / 2);
            mbar_init(smem_u32(&sh.p_free[i]), 1);
        }
        mbar_init(smem_u32(&sh.q_full), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.q_empty), 1);
        mbar_init(smem_u32(&sh.done), 1);
        mbar_init(smem_u32(&sh.o_free), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.ml_full), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.mma_idle), 2);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&sh.tmem_base), 512);
        tmem_relinquish();
    }
    Range range{};
    if (!split.whole) {
        range = locate<kWarps>(p, split, sh.warp_sum, &sh.found_base, &sh.found, [&](long long per) { return blockIdx.x * per; });
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Owning all 512 columns means owning them from 0, a constant for the products' operands.
    if (sh.tmem_base != 0 || (smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) {
            atomicOr(&status->code, kStatusTimeoutTeardown);
            if (!split.whole) {
                rec.cut[blockIdx.x] = Cut{};
            }
        }
    } else {
        if (warp < kSoftmaxWarps) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
            softmax<C>(p, sh, *reinterpret_cast<Exchange*>(&sh + 1), smem_u32(smem), rec, waits);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
            if (warp < kScoreWarp) {
                ready_values<C>(p, sh, smem_u32(smem), waits);
            } else if (warp == kScoreWarp) {
                score_warp<C>(sh, smem_u32(smem), waits);
            } else if (warp == kMmaWarp) {
                product_warp<C>(sh, smem_u32(smem), waits);
            } else {
                const Walk walk = start_walk(p, split, range, static_cast<int>(blockIdx.x));
                list_tiles<C>(p, &tm_k, &tm_v, split, status, walk, sh, smem_u32(smem), warp - kListWarp, waits);
                // Behind the list, not before it: 217 us for 240 of 64 nodes on 32 contexts.
                if (!split.whole && warp == kListWarp && threadIdx.x % 32 == 0) {
                    const Walk start = start_walk(p, split, range, static_cast<int>(blockIdx.x));
                    rec.cut[blockIdx.x] = cut_at(split, range, start, static_cast<int>(blockIdx.x));
                }
                // Copies in flight end by themselves; after a wait that was given up they get a millisecond.
                if (sh.abort != 0) {
                    const unsigned long long t0 = globaltimer_ns();
                    while (globaltimer_ns() - t0 < 1000000ull) {
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(sh.tmem_base, 512);
    }
    if (rec.odd != nullptr && threadIdx.x == 0) {
        rec.odd[blockIdx.x] = sh.odd;
    }
}

// The second kernel. Its first CTAs join the records of cut items, always in the same order. The others, `fixers` of them,
// compute rows anew, one by one, of items in whose tiles infinities or NaN are hidden from some rows (0 times them would be
// NaN there).
template <class C>
__global__ void __launch_bounds__(kRowWarps * 32) tree_finish_kernel(const __grid_constant__ FaTreeParams p, DeviceStatus* status,
                                                                     Split split, Record rec, int joins, int fixers) {
    constexpr int D = C::D;
    __shared__ long long warp_sum[kRowWarps];
    __shared__ long long found_base;
    __shared__ int found;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int group = p.heads / p.cache.kv_heads;
    const int rows = group * p.cache.tokens;
    // One CTA waits whatever it finds to do, so that this kernel's end stands for the end of the one before.
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        cudaGridDependencySynchronize();
    }
    if (static_cast<int>(blockIdx.x) < joins) {
        cudaGridDependencySynchronize();  // the records are there
        const Cut cut = rec.cut[blockIdx.x + 1];
        // Out of range is what calls that share a workspace at a time make of it.
        if (cut.c1 <= 0 || cut.c1 >= split.grid || cut.c0 < 0 || cut.first < 0 || cut.first >= 2 * split.grid || cut.b < 0 ||
            cut.b >= p.cache.batch || cut.kvh < 0 || cut.kvh >= p.cache.kv_heads || cut.block < 0 || cut.block >= split.row_blocks) {
            return;
        }
        // A warp takes 32 rows and 8 columns, a lane a row.
        constexpr int kAcross = D / 8;
        const int unit = static_cast<int>(blockIdx.y) * kRowWarps + warp;
        const int r = unit / kAcross * 32 + lane;
        const int eight = unit % kAcross;
        const int row_index = cut.block * C::kRows + r;
        if (r >= C::kRows || row_index >= rows) {
            return;
        }
        float m = -INFINITY, l = 0.0f;
        float o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        bool odd = false;
#pragma unroll 4
        for (int c = cut.c0; c <= cut.c1; ++c) {
            const int64_t record = c == cut.c0 ? cut.first : 2 * c;
            odd = odd || (rec.odd != nullptr && rec.odd[c] != 0);
            const float2 ml = rec.ml[record * C::kRows + r];
            const float4* from = reinterpret_cast<const float4*>(rec.o) + (record * (D / 4) + 2 * eight) * C::kRows + r;
            const float4 y0 = from[0];
            const float4 y1 = from[C::kRows];
            const float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
            const float now = fmax_nan(m, ml.x);
            const float used = now == -INFINITY ? 0.0f : now;
            const float a = ex2_approx(m - used);
            const float f = ex2_approx(ml.x - used);
            m = now;
            l = fmaf(ml.y, f, l * a);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                o[i] = fmaf(y[i], f, o[i] * a);
            }
        }
        if (odd) {
            return;  // its rows are computed anew
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = static_cast<uint16_t*>(p.o) + ((static_cast<int64_t>(cut.b) * p.heads + cut.kvh * group) * p.cache.tokens + row_index) * D;
        reinterpret_cast<uint4*>(out)[eight] = make_uint4(pack2<C::BF16>(o[0] * inv, o[1] * inv), pack2<C::BF16>(o[2] * inv, o[3] * inv),
                                                          pack2<C::BF16>(o[4] * inv, o[5] * inv), pack2<C::BF16>(o[6] * inv, o[7] * inv));
        return;
    }
    if (blockIdx.y > 0) {
        return;
    }
    cudaGridDependencySynchronize();
    const int fixer = static_cast<int>(blockIdx.x) - joins;
    bool any = false;
    for (int i = static_cast<int>(threadIdx.x); i < split.grid; i += kRowWarps * 32) {
        any = any || rec.odd[i] != 0;
    }
    if (__syncthreads_or(any) == 0) {
        return;
    }
    for (int cta = 0; cta < split.grid; ++cta) {
        if (rec.odd[cta] == 0) {
            continue;
        }
        Range range{};
        if (!split.whole) {
            range = locate<kRowWarps>(p, split, warp_sum, &found_base, &found, [&](long long per) { return cta * per; });
        }
        Walk walk = start_walk(p, split, range, cta);
        Piece piece;
        Sequence s;
        while (next_piece(p, split, walk, piece, s)) {
            for (int r = fixer; r < C::kRows; r += fixers) {
                const int row_index = piece.block * C::kRows + r;
                if (row_index < rows) {
                    const int head = row_index / p.cache.tokens;
                    __syncthreads();  // the shared memory of the row before is free
                    attend_row<D, C::BF16, C::E4M3>(p, status, piece.b, piece.kvh * group + head, row_index - head * p.cache.tokens);
                }
            }
        }
        __syncthreads();
    }
}

// A map of k or v over {head dim, slot, head, page}: boxes of a page's tokens, at most a tile of them.
CUresult encode_pool_map(CUtensorMap* map, const FaCache& c, void* base, const int64_t (&stride)[2], bool bf16, CUtensorMapSwizzle swizzle) {
    auto fn = tensor_map_encoder();
    if (fn == nullptr) {
        return CUDA_ERROR_NOT_SUPPORTED;
    }
    const bool e4m3 = c.dtype == FA_DTYPE_FLOAT8_E4M3;
    const cuuint64_t elem = e4m3 ? 1 : 2;
    const cuuint64_t row = c.head_dim * elem;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size),
                                static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.num_pages)};
    // The stride of a dim of one element is never used and may be 0.
    const cuuint64_t strides[3] = {row, c.kv_heads > 1 ? static_cast<cuuint64_t>(stride[1]) * elem : row,
                                   c.num_pages > 1 ? static_cast<cuuint64_t>(stride[0]) * elem : row};
    const cuuint32_t box[4] = {e4m3 ? static_cast<cuuint32_t>(c.head_dim) : 64u, static_cast<cuuint32_t>(std::min(c.page_size, kTile)), 1, 1};
    const cuuint32_t elem_strides[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                          : (bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
    return fn(map, type, 4, base, dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Launches after the kernel before it has started to end: it waits for its results itself.
template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

constexpr int kFixers = 64;
constexpr int kFewRows = 16;
constexpr int kShort = 16;     // key tiles of a short list
constexpr int kJoinTiles = 5;  // what the records and their join cost, in key tiles of 1.15 us

// Whether a kv head's rows are better taken 16 at a time, by warps of their own: 16 rows on one context of 777 tokens take
// 15.5 us there and 17.1 here, 32 rows (8 nodes, above) 168 there and 141 here.
bool few_rows(const FaTreeParams& p) { return p.heads / p.cache.kv_heads * p.cache.tokens <= kFewRows; }

// Key tiles that a sequence has at most.
long long most_tiles(const FaCache& c, int window, int sinks) {
    long long shown = static_cast<long long>(c.max_pages) * c.page_size;
    if (window > 0) {
        shown = std::min<long long>(shown, static_cast<long long>(window) + sinks + c.tokens + 3 * kTile);
    }
    return (shown + kTile - 1) / kTile;
}

// Two row tiles an item, for which a key tile is copied and widened once, or one, of which both softmax warpgroups work on
// key tiles in turn. One where there are no more rows (32 nodes on 32 contexts of up to 8192 tokens: 148 us, padded to two
// 232), and where lists are short and SMs would stay idle (64 nodes on 1000 tokens: 19.6 and 25.1); else two (64 nodes on
// 32 contexts: 248 and 288; 128 nodes on 4 of up to 8192, 86 and 88).
int row_tiles(const FaTreeParams& p, int sm_count) {
    const long long rows = static_cast<long long>(p.heads / p.cache.kv_heads) * p.cache.tokens;
    const long long blocks = (rows + kTile - 1) / kTile;
    const bool is_short = most_tiles(p.cache, p.window, p.sinks) <= kShort;
    return blocks == 1 || (is_short && blocks * p.cache.kv_heads * p.cache.batch <= sm_count) ? 1 : 2;
}

// Short lists are not cut where every item has an SM and the cut would not pay for the records: 16 nodes on 16 contexts of
// 1024 tokens 21.0 us whole and 30.5 cut, of 2048 30.2 and 39.6; on 4 of 512 15.8 and 16.9, of 1024 20.1 and 19.2, of 2048
// 28.7 and 22.3; on one of 1024 20.2 and 16.5. Lengths are on the device, so a list is as short as the table is narrow: behind a
// table of 131072 places 16 nodes on 16 contexts of 1024 take 30.6 us (21.5 behind one of 1024), 64 nodes on 1000 26.4 (19.7).
Split split_for(const FaTreeParams& p, int sm_count) {
    const FaCache& c = p.cache;
    const long long rows = static_cast<long long>(p.heads / c.kv_heads) * c.tokens;
    const long long block = static_cast<long long>(row_tiles(p, sm_count)) * kTile;
    const long long row_blocks = (rows + block - 1) / block;
    const long long items = static_cast<long long>(c.kv_heads) * row_blocks;
    const long long tiles = most_tiles(c, p.window, p.sinks);
    Split s;
    s.row_blocks = static_cast<int>(row_blocks);
    s.items = static_cast<int>(items);
    s.whole = tiles <= kShort && items * c.batch <= sm_count && (tiles - kJoinTiles) * sm_count <= items * c.batch * (tiles + kItemHead);
    s.grid = static_cast<int>(s.whole ? items * c.batch : std::min<long long>(sm_count, items * c.batch * tiles));
    return s;
}

template <class C>
cudaError_t launch(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    const Split split = split_for(p, sm_count);
    constexpr auto kernel = tree_kernel<C>;
    cudaError_t err = ensure_smem_limit<kernel>(smem_bytes<C>());
    if (err != cudaSuccess) {
        return err;
    }
    Record rec{};
    int* odd = static_cast<int*>(workspace);
    if (!split.whole) {
        const size_t rows = static_cast<size_t>(split.grid) * 2 * C::kRows;
        rec.o = static_cast<float*>(workspace);
        rec.ml = reinterpret_cast<float2*>(rec.o + rows * C::D);
        rec.cut = reinterpret_cast<Cut*>(rec.ml + rows);
        odd = reinterpret_cast<int*>(rec.cut + split.grid);
    }
    rec.odd = p.cache.tokens > 1 ? odd : nullptr;
    CUtensorMap tm_k, tm_v;
    const CUtensorMapSwizzle raw_k = C::E4M3 && C::D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    const CUtensorMapSwizzle raw_v = C::E4M3 && C::D == 64 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
    if (encode_pool_map(&tm_k, p.cache, p.cache.k, p.cache.k_stride, C::BF16, raw_k) != CUDA_SUCCESS ||
        encode_pool_map(&tm_v, p.cache, p.cache.v, p.cache.v_stride, C::BF16, raw_v) != CUDA_SUCCESS) {
        return cudaErrorInvalidValue;
    }
    kernel<<<static_cast<unsigned>(split.grid), kThreads, smem_bytes<C>(), stream>>>(p, tm_k, tm_v, status, split, rec);
    err = cudaGetLastError();
    const int joins = split.whole ? 0 : split.grid - 1;
    const int fixers = rec.odd != nullptr ? kFixers : 0;
    if (err == cudaSuccess && joins + fixers > 0) {
        const int rows = std::min(C::kRows, p.heads / p.cache.kv_heads * p.cache.tokens);
        const dim3 grid(static_cast<unsigned>(joins + fixers), static_cast<unsigned>(joins > 0 ? ((rows + 31) / 32 * (C::D / 8) + kRowWarps - 1) / kRowWarps : 1));
        err = launch_early(tree_finish_kernel<C>, grid, kRowWarps * 32, stream, p, status, split, rec, joins, fixers);
    }
    return err;
}

template <int D, bool BF16, bool E4M3, bool COARSE>
cudaError_t launch_rows(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    return row_tiles(p, sm_count) == 1 ? launch<Cfg<D, BF16, E4M3, COARSE, 1>>(p, status, workspace, sm_count, stream)
                             : launch<Cfg<D, BF16, E4M3, COARSE, 2>>(p, status, workspace, sm_count, stream);
}

// Pages of 8 or 16 tokens matter to an e4m3 cache alone, by their scales. (One kernel for both took 271 us for 64 nodes on
// 32 contexts where this takes 239: what it runs has to fit the instruction cache.)
template <int D, bool BF16>
cudaError_t launch_types(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    if (p.cache.dtype != FA_DTYPE_FLOAT8_E4M3) {
        return launch_rows<D, BF16, false, true>(p, status, workspace, sm_count, stream);
    }
    return p.cache.page_size >= 32 ? launch_rows<D, BF16, true, true>(p, status, workspace, sm_count, stream)
                                   : launch_rows<D, BF16, true, false>(p, status, workspace, sm_count, stream);
}

template <int D>
cudaError_t launch_dim(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    return p.dtype == FA_DTYPE_BFLOAT16 ? launch_types<D, true>(p, status, workspace, sm_count, stream)
                                        : launch_types<D, false>(p, status, workspace, sm_count, stream);
}

}  // namespace

unsigned long long tree_workspace_bytes(const FaTreeParams& p, int sm_count) {
    if (few_rows(p)) {
        return small_tree_workspace_bytes(p, sm_count);
    }
    const Split split = split_for(p, sm_count);
    const unsigned long long records =
        split.whole ? 0 : static_cast<unsigned long long>(split.grid) * (2ull * row_tiles(p, sm_count) * kTile * (p.cache.head_dim + 2) * 4 + sizeof(Cut));
    return records + (p.cache.tokens > 1 ? 4ull * split.grid : 0);
}

cudaError_t launch_tree(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    if (few_rows(p)) {
        return launch_small_tree(p, status, workspace, sm_count, stream);
    }
    return p.cache.head_dim == 64 ? launch_dim<64>(p, status, workspace, sm_count, stream)
                                  : launch_dim<128>(p, status, workspace, sm_count, stream);
}

}  // namespace fa_sm100
