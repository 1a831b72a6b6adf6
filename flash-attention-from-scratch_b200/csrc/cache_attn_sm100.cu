// Attention of the newest tokens of every sequence over the paged cache (flash decoding).
//
//   O = sum_j e^(s_j) v_j / sum_j e^(s_j),   s_j = scale q.k_j over the visible positions j
//
// Every cache element is read once for a tile of 16 query rows (the query heads that share a kv
// head, times the tokens), so the kernel is bound by DRAM bytes; what it needs is many loads in
// flight, equal work for every SM whatever the lengths, and few instructions a byte.
//
// Split. The work is a list of (sequence, kv head, row tile) items of as many key tiles as the
// sequence shows, laid end to end in units of key tiles and cut into equal ranges, one for each
// CTA of a grid that fills the GPU. Lengths are on the device, so every CTA adds them up itself. A
// CTA walks its range; an item that lies within it is written at once, one that was cut
// leaves its unnormalised rows with (max, sum) in the workspace, at most two records a CTA, and a
// second kernel (started early, by programmatic launch) joins them in order: no atomics.
//
// Within a CTA each of 4 warps takes every fourth key tile through a ring of its own, filled with
// 16-byte cp.async copies: no CTA barrier until the item's end, where the warps' rows are joined in
// shared memory. A key tile is 4 KB of K and 4 KB of V: 32 tokens of 128 e4m3 values, 16 of 128
// 16-bit ones. Rings of 2 tiles and 3 CTAs an SM (168 registers a thread) keep 96 KB in flight; 6.5 TB/s
// at about 1 us needs 44. (3 tiles and 2 CTAs: 136 us where this takes 87, for want of warps.)
//
// Measured, 32 query heads on 8, D 128, e4m3, pages of 64, one state replayed in bursts: 32 sequences of 4000 to 8000
// tokens 78 us (5.1 TB/s), 4 of 120000 to 131000 168 us (6.0 TB/s), 64 x 4 drafted tokens over a window of 4096 and 4
// sinks 112 us (4.8 TB/s); calls in turn under load that lasts, at the power cap, 80, 182 and 116 us. With 16-bit
// values 126, 305 and 178 us, at the copy's rate. What is left: the instructions of a tile (about 730, half of the
// issue slots), and for short ranges the start of an item, its join in shared memory and the second launch. A long
// chunk of tokens is slow: a sequence has one list of key tiles, from its first query's window to its last
// query, for all its row tiles, and from 16 tokens on a row tile is one head's, so that a group's heads read
// the tiles each for itself (4000 tokens on nothing before them 1.6 ms, where the dense window forward takes 0.18).
//
// Products are mma.sync m16n8k16: with 16 rows of queries and two operations a byte of K
// or V an M = 128 tcgen05 tile would be seven eighths padding, and dequantised operands would have to
// go back to shared memory for it. e4m3 widens exactly to float16; bfloat16 queries are brought
// into float16's range by a power of two per row: the largest in [2^13, 2^14), steps of 2^-24, so that values
// down to 2^-30 of the row's largest are exact; smaller ones round to those steps and vanish from 2^-38 on. Both
// products permute their contraction (head dim, keys) and output columns so that a lane's fragments are whole
// 16-byte words of the cache's own rows.
//
// e4m3's value scales. With w_j = e^(s_j) vs_j (vs_j: the scale of j's page) O = sum w_j c_j / sum
// (w_j / vs_j) over the codes c_j. The running maximum is taken over log2 w_j = s_j log2 e + log2
// vs_j, so P <= 1 keeps its 11 bits where the output comes from, whatever the scales of other
// pages; the sum takes P / vs_j in fp32. Scales below 2^-60 (0 among them) enter as 2^-60 with P
// scaled down.

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;          // query rows of an item: the M of the matrix instruction
constexpr int kStages = 2;         // key tiles of a warp's ring
constexpr int kTileBytes = 4096;   // K (or V) of a key tile
constexpr int kAuxFloats = 16;     // of a stage: 8 K scales, 8 V scales
constexpr int kCtasPerSm = 3;
constexpr int kMinTiles = kWarps;  // least key tiles of a CTA: one for each warp
constexpr int kWholeTiles = 8;     // up to this many key tiles in the table's capacity items are not cut
constexpr float kMinScale = 8.673617379884035e-19f;  // 2^-60
constexpr int kSmem = kWarps * kStages * (2 * kTileBytes + kAuxFloats * 4);

// Values that are not finite, of keys that some of an item's rows see and some do not, in bits of (row, dim): NaN,
// +inf and -inf. See attend().
struct Apart {
    uint32_t bits[3][kRows][128 / 32];
};

__device__ __forceinline__ float not_finite_sum(const Apart& a, int row, int dim) {
    const uint32_t bit = 1u << (dim % 32);
    float sum = 0.0f;
    sum += (a.bits[0][row][dim / 32] & bit) != 0 ? NAN : 0.0f;
    sum += (a.bits[1][row][dim / 32] & bit) != 0 ? INFINITY : 0.0f;
    sum += (a.bits[2][row][dim / 32] & bit) != 0 ? -INFINITY : 0.0f;
    return sum;
}

constexpr int kSmemCareful = kSmem + static_cast<int>(sizeof(Apart));

template <int D_, bool BF16_, bool E4M3_, bool ONE_PAGE_>
struct Cfg {
    static constexpr bool ONE_PAGE = ONE_PAGE_;  // a key tile lies within one page
    static constexpr int D = D_;
    static constexpr bool BF16 = BF16_;  // queries and output
    static constexpr bool E4M3 = E4M3_;
    static constexpr bool kMmaBf16 = BF16 && !E4M3;
    static constexpr int kElem = E4M3 ? 1 : 2;
    static constexpr int kRowBytes = D * kElem;
    static constexpr int kKeys = kTileBytes / kRowBytes;  // 16, 32 or 64
    static constexpr int kChunks = kRowBytes / 16;
    static constexpr int kSteps = D / 16;   // k steps of Q K^T
    static constexpr int kNTiles = kKeys / 8;
    static constexpr int kOTiles = D / 8;
    static constexpr bool kNarrow = kRowBytes == 64;  // two rows in a 128-byte line
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// Two e4m3 pairs of a word, widened exactly.
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
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

// Byte offsets of chunk `c` (16 bytes) of token `r` in a K and in a V tile. The swizzles make the
// fragment reads below free of bank conflicts: a K read takes chunks t, t + 4, .. of tokens g
// (lane = 4 g + t), a V read chunk g of tokens 2 t, 2 t + 1.
template <class C>
__device__ __forceinline__ uint32_t k_offset(int r, int c) {
    return static_cast<uint32_t>(r * C::kRowBytes + (C::kNarrow ? c : c ^ ((r & 1) << 2)) * 16);
}
template <class C>
__device__ __forceinline__ uint32_t v_offset(int r, int c) {
    if constexpr (C::kNarrow) {
        const int row = (r & ~3) | ((r & 1) << 1) | ((r >> 1) & 1);
        return static_cast<uint32_t>(row * 64 + (c ^ ((r >> 1) & 2)) * 16);
    } else {
        return static_cast<uint32_t>(r * C::kRowBytes + (c ^ (r & 7)) * 16);
    }
}

// Positions that the page tables have a place for (below 2^31).
__device__ __forceinline__ int held(const FaCache& c) { return c.max_pages * c.page_size; }

// What a sequence shows its queries: positions [0, sinks) and [first, last], as a list of key tiles. The list
// ends with the page table, whatever length the device holds, so that a call's work is bounded by its arguments.
struct Sequence {
    int pos0;    // position of its first query (may be negative)
    int count;   // queries
    int last;    // last position any query sees and the table has, -1 if none
    int first;   // first position of the earliest window, at most the table's end
    int sink_tiles, first_tile, tiles;
};

template <class C>
__device__ __forceinline__ Sequence sequence(const FaCachedParams& p, int b) {
    Sequence s;
    const int len = max(p.cache.lengths[b], 0);
    s.count = p.cache.counts != nullptr ? min(max(p.cache.counts[b], 0), p.cache.tokens) : p.cache.tokens;
    s.pos0 = len - s.count;
    s.last = s.count > 0 ? min(len, held(p.cache)) - 1 : -1;
    s.first = min(window_first(max(s.pos0, 0), p.window), held(p.cache));
    s.first_tile = s.first / C::kKeys;
    s.sink_tiles = min((min(p.sinks, s.first) + C::kKeys - 1) / C::kKeys, s.first_tile);
    // A sequence that shows nothing keeps one (hidden) tile, so that its rows are written.
    s.tiles = s.last < 0 ? 1 : max(s.sink_tiles + s.last / C::kKeys - s.first_tile + 1, 1);
    return s;
}

struct Range {
    long long total, per;   // key tiles of all items, of a CTA
    long long found_base;   // start of the sequence found
    int found;
};

// The work list's length, and the sequence that holds unit `at(per)` of it. All threads call.
template <class C, class At>
__device__ __forceinline__ Range locate(const FaCachedParams& p, int grid, At at) {
    __shared__ long long warp_sum[kWarps];
    __shared__ long long found_base;
    __shared__ int found;
    const int heads_rows = p.cache.kv_heads * ((p.heads / p.cache.kv_heads * p.cache.tokens + kRows - 1) / kRows);
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int share = (p.cache.batch + kThreads - 1) / kThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * share, p.cache.batch);
    const int b1 = min(b0 + share, p.cache.batch);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
        mine += sequence<C>(p, b).tiles;
    }
    mine *= heads_rows;
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
        found = -1;
    }
    __syncthreads();
    Range r;
    r.total = 0;
    long long before = incl - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        before += w < warp ? warp_sum[w] : 0;
        r.total += warp_sum[w];
    }
    r.per = max((r.total + grid - 1) / grid, static_cast<long long>(kMinTiles));
    const long long target = at(r.per);
    if (target >= before && target < before + mine) {
        long long base = before;
        for (int b = b0; b < b1; ++b) {
            const long long n = static_cast<long long>(sequence<C>(p, b).tiles) * heads_rows;
            if (target < base + n) {
                found = b;
                found_base = base;
                break;
            }
            base += n;
        }
    }
    __syncthreads();
    r.found = found;
    r.found_base = found_base;
    return r;
}

// Takes what is not finite out of 16 bytes `at` of a V tile (chunk `chunk` of the token at position `key`) and notes it for
// the rows of the item that see it.
template <class C>
__device__ __forceinline__ void set_apart(const FaCachedParams& p, const Sequence& s, Apart& apart, uint8_t* at, int row0, int key,
                                       int chunk) {
    const int rows = p.heads / p.cache.kv_heads * p.cache.tokens;
    for (int e = 0; e < 16 / C::kElem; ++e) {
        int kind = 0;
        if constexpr (C::E4M3) {
            if ((at[e] & 0x7f) != 0x7f) {
                continue;
            }
            at[e] = 0;
        } else {
            uint16_t* x = reinterpret_cast<uint16_t*>(at) + e;
            constexpr uint32_t kInf = C::BF16 ? 0x7f80u : 0x7c00u;
            if ((*x & 0x7fffu) < kInf) {
                continue;
            }
            kind = (*x & 0x7fffu) > kInf ? 0 : (*x >> 15) + 1;
            *x = 0;
        }
        const int dim = chunk * (16 / C::kElem) + e;
        for (int row = 0; row < kRows && row0 + row < rows; ++row) {
            const int token = (row0 + row) % p.cache.tokens;
            const int gap = s.pos0 + token - key;
            if (token < s.count && gap >= 0 && (p.window == 0 || gap < p.window || key < p.sinks)) {
                atomicOr(&apart.bits[kind][row][dim / 32], 1u << (dim % 32));
            }
        }
    }
}

struct Record {  // of a cut item's rows in the workspace
    float* o;    // [record][16][D]
    float2* ml;  // [record][16]
    int* odd;    // [CTA], several tokens: whether a result of its range is not finite
};

// One range of key tiles [v0, v1) of an item.
//
// Several tokens: where not all rows see all of a tile, 0 times an infinite or NaN value is NaN in rows that it is hidden from
// (a drafted token's, in the rows of the tokens before it). A CTA with a result that is not finite says so, and a second
// kernel takes its range again, CAREFUL: such values are taken out of those tiles, and added to the rows that see
// them when the rows are joined. (In this loop, which has no registers left, looking for them in every such tile, or
// keeping rows apart in the product, cost drafted tokens 3 to 50%.)
template <class C, bool CAREFUL>
__device__ __forceinline__ void attend(const FaCachedParams& p, DeviceStatus* status, uint8_t* smem, const Sequence& s,
                                       int b, int kvh, int row0, int v0, int v1, Record rec, long long record) {
    constexpr int D = C::D;
    const FaCache& c = p.cache;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int g = lane / 4;
    const int t = lane % 4;
    const int group = p.heads / c.kv_heads;
    const int rows = group * c.tokens;
    uint8_t* ring = smem + warp * kStages * 2 * kTileBytes;
    float* aux = reinterpret_cast<float*>(smem + kWarps * kStages * 2 * kTileBytes) + warp * kStages * kAuxFloats;
    [[maybe_unused]] Apart& apart = *reinterpret_cast<Apart*>(smem + kSmem);
    if constexpr (CAREFUL) {
        uint32_t* words = &apart.bits[0][0][0];
        for (int i = static_cast<int>(threadIdx.x); i < static_cast<int>(sizeof(Apart) / 4); i += kThreads) {
            words[i] = 0;
        }
        __syncthreads();
    }

    if (threadIdx.x == 0 && s.count > 0 && s.pos0 + s.count > held(c)) {
        atomicOr(&status->code, kStatusBadPage);  // positions that the table has no place for are left out
    }

    // Pages of a key tile: `spans` of them (at most 8), 2^log2_span tokens each.
    const int log2_page = 31 - __clz(c.page_size);
    const int log2_span = C::ONE_PAGE ? 31 - __clz(C::kKeys) : log2_page;
    const int spans = C::kKeys >> log2_span;

    auto tile_key = [&](int v) { return (v < s.sink_tiles ? v : v - s.sink_tiles + s.first_tile) * C::kKeys; };
    auto shown = [&](int key) { return key <= s.last && (key >= s.first || key < p.sinks); };
    // The page of the tile (ONE_PAGE: in every lane) or of its span number `lane`; -1 for one that is
    // outside the pool or hidden.
    const int32_t* table = c.page_table + b * c.table_stride;
    auto fetch = [&](int v) {
        int id = -1;
        if (v < v1 && (C::ONE_PAGE || lane < spans)) {
            const int key = tile_key(v) + (C::ONE_PAGE ? 0 : lane << log2_span);
            const int end = key + (1 << log2_span) - 1;
            if (key <= s.last && (end >= s.first || key < p.sinks)) {
                id = __ldg(table + (key >> log2_page));
                if (id < 0 || id >= c.num_pages) {
                    id = -1;
                    atomicOr(&status->code, kStatusBadPage);
                }
            }
        }
        return id;
    };
    const int chunk = lane % C::kChunks;
    constexpr int kStep = 32 / C::kChunks;  // tokens of one copy of the warp
    const int r0 = lane / C::kChunks;
    const uint8_t* kbase = static_cast<const uint8_t*>(c.k) + kvh * c.k_stride[1] * C::kElem + chunk * 16;
    const uint8_t* vbase = static_cast<const uint8_t*>(c.v) + kvh * c.v_stride[1] * C::kElem + chunk * 16;
    const int64_t kpage = c.k_stride[0] * C::kElem;
    const int64_t vpage = c.v_stride[0] * C::kElem;
    float next_ks = -1.0f, next_vs = 1.0f;  // ONE_PAGE: scales of the tile last asked for (K: below 0, hidden)
    auto issue = [&](int v, int stage, int ids) {
        if (v < v1) {
            const int key0 = tile_key(v);
            const uint32_t ks = smem_u32(ring) + stage * 2 * kTileBytes;
            const uint32_t vs = ks + kTileBytes;
            const int last = key0 + C::kKeys - 1;
            const bool shows_all = last <= s.last && (key0 >= s.first || last < p.sinks);
            if (!C::ONE_PAGE && shows_all && __all_sync(0xffffffffu, ids >= 0 || lane >= spans)) {
                // All of the tile is shown, in several pages.
                const int in_page = c.page_size - 1;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = i * kStep + r0;
                    const int id = __shfl_sync(0xffffffffu, ids, r >> log2_span);
                    const int slot = ((key0 + r) & in_page) * C::kRowBytes;
                    cp_async16(ks + k_offset<C>(r, chunk), kbase + (id * kpage + slot), true);
                    cp_async16(vs + v_offset<C>(r, chunk), vbase + (id * vpage + slot), true);
                }
            } else if (C::ONE_PAGE && shows_all && ids >= 0) {
                // The usual tile: all of it shown, contiguous in its page.
                const int64_t slot = static_cast<int64_t>((key0 & (c.page_size - 1)) + r0) * C::kRowBytes;
                const uint8_t* ksrc = kbase + ids * kpage + slot;
                const uint8_t* vsrc = vbase + ids * vpage + slot;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    cp_async16(ks + k_offset<C>(i * kStep + r0, chunk), ksrc + i * kStep * C::kRowBytes, true);
                    cp_async16(vs + v_offset<C>(i * kStep + r0, chunk), vsrc + i * kStep * C::kRowBytes, true);
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                    const int r = i * kStep + r0;
                    const int id = C::ONE_PAGE ? ids : __shfl_sync(0xffffffffu, ids, r >> log2_span);
                    const int key = key0 + r;
                    const bool real = id >= 0 && shown(key);
                    const int64_t slot = static_cast<int64_t>(key & (c.page_size - 1)) * C::kRowBytes;
                    cp_async16(ks + k_offset<C>(r, chunk), real ? kbase + id * kpage + slot : kbase, real);
                    cp_async16(vs + v_offset<C>(r, chunk), real ? vbase + id * vpage + slot : vbase, real);
                }
            }
            if constexpr (C::ONE_PAGE) {
                next_ks = ids >= 0 ? 1.0f : -1.0f;
                next_vs = 1.0f;
                if (C::E4M3 && ids >= 0) {
                    const int64_t n = static_cast<int64_t>(ids) * c.kv_heads + kvh;
                    next_ks = __ldg(c.k_scale + n);
                    next_vs = __ldg(c.v_scale + n);
                }
            } else if (lane < spans) {
                float* at = aux + stage * kAuxFloats + lane;
                if (C::E4M3 && ids >= 0) {
                    const int64_t n = static_cast<int64_t>(ids) * c.kv_heads + kvh;
                    cp_async4(smem_u32(at), c.k_scale + n);
                    cp_async4(smem_u32(at + 8), c.v_scale + n);
                } else {
                    at[0] = ids >= 0 ? 1.0f : -1.0f;
                    at[8] = 1.0f;
                }
            }
        }
        cp_commit();
    };

    // The warp's first tiles are on their way while the queries are read.
    int next = v0 + warp;
    int ids = fetch(next);
    static_assert(kStages == 2, "the scales of one tile ahead are kept");
    {
        const int ahead = fetch(next + kWarps);
        issue(next, 0, ids);
        ids = ahead;
        next += kWarps;
    }

    // Query fragments: rows g and g + 8; a k step takes 4 dims of every lane t.
    uint32_t q[C::kSteps][4];
    float factor[2];  // scale * log2 e, and the row's power of two taken back
    int pos[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = row0 + g + 8 * half;
        const int head = r / c.tokens;
        const int token = r - head * c.tokens;
        const bool real = r < rows && token < s.count;
        pos[half] = real ? s.pos0 + token : -1;
        const uint16_t* src = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] +
                              static_cast<int64_t>(kvh * group + head) * p.q_stride[1] + token * p.q_stride[2];
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < C::kSteps; ++k) {
            const int d = C::E4M3 ? 16 * (t + 4 * (k / 4)) + 4 * (k % 4) : 8 * (t + 4 * (k / 2)) + 4 * (k % 2);
            const uint2 w = real ? __ldg(reinterpret_cast<const uint2*>(src + d)) : make_uint2(0u, 0u);
            q[k][half] = w.x;
            q[k][2 + half] = w.y;
            if constexpr (C::E4M3 && C::BF16) {
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(__uint_as_float(w.x << 16)), fabsf(__uint_as_float(w.x & 0xFFFF0000u))),
                                         fmaxf(fabsf(__uint_as_float(w.y << 16)), fabsf(__uint_as_float(w.y & 0xFFFF0000u)))));
            }
        }
        factor[half] = p.softmax_scale * 1.4426950408889634f;
        if constexpr (C::E4M3 && C::BF16) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // 2^(13 - exponent of amax), both it and its inverse normal; 1 for zeros, inf and NaN.
            const int e = static_cast<int>(__float_as_uint(amax) >> 23);
            const int shift = (e == 0 || e == 255) ? 0 : min(max(140 - e, -100), 100);
            const float up = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
            factor[half] *= __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
            for (int k = 0; k < C::kSteps; ++k) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t x = q[k][2 * w + half];
                    q[k][2 * w + half] = pack_half2(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xFFFF0000u) * up);
                }
            }
        }
    }

    float o[C::kOTiles][4];
#pragma unroll
    for (int i = 0; i < C::kOTiles; ++i) {
        o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    }
    float m[2] = {-INFINITY, -INFINITY};
    float l[2] = {0.0f, 0.0f};

    int stage = 0;
    for (int v = v0 + warp; v < v1; v += kWarps) {
        cp_wait<kStages - 2>();
        __syncwarp();  // the tile is there, and every lane has left the stage that is refilled next
        const float page_ks = next_ks;
        const float page_vs = next_vs;
        {
            const int ahead = fetch(next + kWarps);
            issue(next, stage ^ 1, ids);
            ids = ahead;
            next += kWarps;
        }
        const uint8_t* ks = ring + stage * 2 * kTileBytes;
        const uint8_t* vs = ks + kTileBytes;
        const float* sc = aux + stage * kAuxFloats;
        const int key0 = tile_key(v);

        // Scores: keys 8 n + g of the tile, lane t's dims.
        float x[C::kNTiles][4];
#pragma unroll
        for (int n = 0; n < C::kNTiles; ++n) {
            x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
#pragma unroll
            for (int cc = 0; cc < C::kChunks / 4; ++cc) {
                const uint4 w4 = *reinterpret_cast<const uint4*>(ks + k_offset<C>(8 * n + g, t + 4 * cc));
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                if constexpr (C::E4M3) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t lo, hi;
                        widen4(w[i], lo, hi);
                        mma16816<false>(x[n], q[4 * cc + i], lo, hi);
                    }
                } else {
                    mma16816<C::kMmaBf16>(x[n], q[2 * cc], w[0], w[1]);
                    mma16816<C::kMmaBf16>(x[n], q[2 * cc + 1], w[2], w[3]);
                }
            }
        }

        // log2 of the weights, and what is hidden.
        const bool whole = key0 + C::kKeys - 1 <= s.pos0 &&
                           (p.window == 0 || s.pos0 + s.count - 1 - key0 < p.window || key0 + C::kKeys <= p.sinks);
        float inv_vs[C::kNTiles];
        float shrink = 1.0f;  // of P, for scales below 2^-60
        float tile_shrink[C::kNTiles];
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < C::kNTiles; ++n) {
            const int span = (8 * n) >> log2_span;
            const float kscale = C::ONE_PAGE ? page_ks : sc[span];
            float lv = kscale < 0.0f ? -INFINITY : 0.0f;
            inv_vs[n] = 1.0f;
            tile_shrink[n] = 1.0f;
            if constexpr (C::E4M3) {
                const float vscale = C::ONE_PAGE ? page_vs : sc[8 + span];
                const float used = fmaxf(vscale, kMinScale);
                inv_vs[n] = __fdividef(1.0f, used);
                lv += __log2f(used);
                tile_shrink[n] = vscale >= kMinScale ? 1.0f : vscale * inv_vs[n];
                shrink = fminf(shrink, tile_shrink[n]);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float f = factor[half] * (C::E4M3 ? fabsf(kscale) : 1.0f);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float y = fmaf(x[n][2 * half + e], f, lv);
                    if (!whole) {
                        const int key = key0 + 8 * n + 2 * t + e;
                        const int gap = pos[half] - key;
                        const bool seen = gap >= 0 && (p.window == 0 || gap < p.window || key < p.sinks);
                        y = seen ? y : -INFINITY;
                    }
                    x[n][2 * half + e] = y;
                    top[half] = fmaxf(top[half], y);
                }
            }
        }
        float used[2];
        bool grew = false;
        float alpha[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
            top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
            const float now = fmaxf(m[half], top[half]);
            used[half] = now == -INFINITY ? 0.0f : now;
            alpha[half] = ex2_approx(m[half] - used[half]);
            grew = grew || now > m[half];
            m[half] = now;
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                l[half] *= alpha[half];
#pragma unroll
                for (int i = 0; i < C::kOTiles; ++i) {
                    o[i][2 * half] *= alpha[half];
                    o[i][2 * half + 1] *= alpha[half];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < C::kNTiles; ++n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float p0 = ex2_approx(x[n][2 * half] - used[half]);
                const float p1 = ex2_approx(x[n][2 * half + 1] - used[half]);
                l[half] = C::E4M3 ? fmaf(p0 + p1, inv_vs[n], l[half]) : l[half] + (p0 + p1);
                x[n][2 * half] = p0;
                x[n][2 * half + 1] = p1;
            }
        }
        if (C::E4M3 && shrink != 1.0f) {
#pragma unroll
            for (int n = 0; n < C::kNTiles; ++n) {
                x[n][0] *= tile_shrink[n];
                x[n][1] *= tile_shrink[n];
                x[n][2] *= tile_shrink[n];
                x[n][3] *= tile_shrink[n];
            }
        }

        if (CAREFUL && !whole) {
            for (int i = 0; i < 8; ++i) {
                const int r = i * kStep + r0;
                uint8_t* at = ring + stage * 2 * kTileBytes + kTileBytes + v_offset<C>(r, chunk);
                const uint4 y = *reinterpret_cast<const uint4*>(at);
                if ((not_finite<C>(y.x) | not_finite<C>(y.y) | not_finite<C>(y.z) | not_finite<C>(y.w)) != 0) {
                    set_apart<C>(p, s, apart, at, row0, key0 + r, chunk);
                }
            }
            __syncwarp();
        }

        // O += P V, 16 keys a step: lane (g, t) brings keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 and
        // the dims of its chunk g, byte i of it for output tile i.
#pragma unroll
        for (int k = 0; k < C::kKeys / 16; ++k) {
            uint32_t a[4];
            a[0] = pack2<C::kMmaBf16>(x[2 * k][0], x[2 * k][1]);
            a[1] = pack2<C::kMmaBf16>(x[2 * k][2], x[2 * k][3]);
            a[2] = pack2<C::kMmaBf16>(x[2 * k + 1][0], x[2 * k + 1][1]);
            a[3] = pack2<C::kMmaBf16>(x[2 * k + 1][2], x[2 * k + 1][3]);
            const int r = 16 * k + 2 * t;
            if constexpr (C::E4M3) {
                constexpr int W = C::kNarrow ? 2 : 4;  // words of a lane's dims
                uint32_t w[4][W];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = r + (i & 1) + 8 * (i >> 1);
                    if constexpr (C::kNarrow) {
                        const uint2 y = *reinterpret_cast<const uint2*>(vs + v_offset<C>(key, g >> 1) + (g & 1) * 8);
                        w[i][0] = y.x;
                        w[i][1] = y.y;
                    } else {
                        const uint4 y = *reinterpret_cast<const uint4*>(vs + v_offset<C>(key, g));
                        w[i][0] = y.x;
                        w[i][1] = y.y;
                        w[i][2] = y.z;
                        w[i][3] = y.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const uint32_t lo0 = __byte_perm(w[0][j], w[1][j], 0x5140);
                    const uint32_t hi0 = __byte_perm(w[0][j], w[1][j], 0x7362);
                    const uint32_t lo1 = __byte_perm(w[2][j], w[3][j], 0x5140);
                    const uint32_t hi1 = __byte_perm(w[2][j], w[3][j], 0x7362);
                    uint32_t b0[4], b1[4];
                    widen4(lo0, b0[0], b0[1]);
                    widen4(hi0, b0[2], b0[3]);
                    widen4(lo1, b1[0], b1[1]);
                    widen4(hi1, b1[2], b1[3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mma16816<false>(o[4 * j + i], a, b0[i], b1[i]);
                    }
                }
            } else {
#pragma unroll
                for (int cc = 0; cc < C::kChunks / 8; ++cc) {
                    uint4 y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[i] = *reinterpret_cast<const uint4*>(vs + v_offset<C>(r + (i & 1) + 8 * (i >> 1), g + 8 * cc));
                    }
                    const uint32_t w[4][4] = {{y[0].x, y[0].y, y[0].z, y[0].w},
                                              {y[1].x, y[1].y, y[1].z, y[1].w},
                                              {y[2].x, y[2].y, y[2].z, y[2].w},
                                              {y[3].x, y[3].y, y[3].z, y[3].w}};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma16816<C::kMmaBf16>(o[8 * cc + 2 * j], a, __byte_perm(w[0][j], w[1][j], 0x5410),
                                              __byte_perm(w[2][j], w[3][j], 0x5410));
                        mma16816<C::kMmaBf16>(o[8 * cc + 2 * j + 1], a, __byte_perm(w[0][j], w[1][j], 0x7632),
                                              __byte_perm(w[2][j], w[3][j], 0x7632));
                    }
                }
            }
        }
        stage ^= 1;
    }
    cp_wait<0>();
    __syncthreads();

    // Join the warps' rows: [warp][16][D] floats over the rings, then [warp][16] (max, sum). Groups
    // of 4 dims are swizzled by their row and 32-dim block against bank conflicts.
    float4* all_o = reinterpret_cast<float4*>(smem);
    float2* all_ml = reinterpret_cast<float2*>(smem + kWarps * kRows * D * 4);
    static_assert(kWarps * kRows * (D * 4 + 8) <= kSmem, "the joined rows fit over the rings");
    auto place = [](int row, int four) { return row * (D / 4) + (four ^ (((four >> 3) & 3) | ((row & 1) << 2))); };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        const int row = g + 8 * half;
        if (t == 0) {
            all_ml[warp * kRows + row] = make_float2(m[half], l[half]);
        }
        // Column c of output tile i is dim W c + i of its block of 8 W dims (W output tiles).
        constexpr int W = C::E4M3 ? C::kOTiles : 8;
#pragma unroll
        for (int i = 0; i < C::kOTiles; i += 4) {
            const int block = i / W * 8 * W;
            const int d0 = block + W * (2 * t) + i % W;
            const int d1 = d0 + W;
            all_o[warp * (kRows * D / 4) + place(row, d0 / 4)] =
                make_float4(o[i][2 * half], o[i + 1][2 * half], o[i + 2][2 * half], o[i + 3][2 * half]);
            all_o[warp * (kRows * D / 4) + place(row, d1 / 4)] =
                make_float4(o[i][2 * half + 1], o[i + 1][2 * half + 1], o[i + 2][2 * half + 1], o[i + 3][2 * half + 1]);
        }
    }
    __syncthreads();
    constexpr int kLanes = kThreads / kRows;  // 8 threads a row, D / 8 dims each
    const int row = static_cast<int>(threadIdx.x) / kLanes;
    const int part = static_cast<int>(threadIdx.x) % kLanes;
    const int r = row0 + row;
    bool odd = false;
    if (r < rows) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            top = fmaxf(top, all_ml[w * kRows + row].x);
        }
        const float used = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
        float weight[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            weight[w] = ex2_approx(all_ml[w * kRows + row].x - used);
            sum = fmaf(all_ml[w * kRows + row].y, weight[w], sum);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int head = r / c.tokens;
        const int token = r - head * c.tokens;
        const bool real = token < s.count;  // else padding: zeros (its row saw unmasked tiles, too)
        const long long out_row =
            (static_cast<long long>(b) * p.heads + kvh * group + head) * c.tokens + token;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int four = part * (D / 32) + i;
            float4 sum4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float4 y = all_o[w * (kRows * D / 4) + place(row, four)];
                sum4.x = fmaf(y.x, weight[w], sum4.x);
                sum4.y = fmaf(y.y, weight[w], sum4.y);
                sum4.z = fmaf(y.z, weight[w], sum4.z);
                sum4.w = fmaf(y.w, weight[w], sum4.w);
            }
            if constexpr (CAREFUL) {
                sum4.x += not_finite_sum(apart, row, four * 4);
                sum4.y += not_finite_sum(apart, row, four * 4 + 1);
                sum4.z += not_finite_sum(apart, row, four * 4 + 2);
                sum4.w += not_finite_sum(apart, row, four * 4 + 3);
            } else {
                odd = odd || !(fabsf(sum4.x) + fabsf(sum4.y) + fabsf(sum4.z) + fabsf(sum4.w) < INFINITY);
            }
            if (record < 0) {
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.o) + out_row * D + four * 4) =
                    real ? make_uint2(pack2<C::BF16>(sum4.x * inv, sum4.y * inv), pack2<C::BF16>(sum4.z * inv, sum4.w * inv))
                         : make_uint2(0u, 0u);
            } else {
                reinterpret_cast<float4*>(rec.o)[(record * kRows + row) * (D / 4) + four] =
                    real ? sum4 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        if (record >= 0 && part == 0) {
            rec.ml[record * kRows + row] = real ? make_float2(top, sum) : make_float2(-INFINITY, 0.0f);
        }
    }
    const bool any_odd = __syncthreads_or(odd) != 0;  // ... and the rings are free for the next item
    if (!CAREFUL && any_odd && s.count > 1 && threadIdx.x == 0) {
        rec.odd[blockIdx.x] = 1;
    }
}

// Calls take(i) for the ranges (or whole items) of this CTA: its own in the first kernel, one for each CTA; in the second
// (CAREFUL), whose few CTAs look at all answers of the first, those of results that were not finite.
template <bool CAREFUL, class Take>
__device__ __forceinline__ void take_ranges(const FaCachedParams& p, const Record& rec, int ranges, Take take) {
    cudaTriggerProgrammaticLaunchCompletion();  // the next kernel's CTAs may take SMs as they get free
    if constexpr (CAREFUL) {
        cudaGridDependencySynchronize();  // the answers are there
        bool any = false;
        for (long long i = blockIdx.x + static_cast<long long>(threadIdx.x) * gridDim.x; i < ranges; i += static_cast<long long>(kThreads) * gridDim.x) {
            any = any || rec.odd[i] != 0;
        }
        if (__syncthreads_or(any) != 0) {
            for (long long i = blockIdx.x; i < ranges; i += gridDim.x) {
                if (rec.odd[i] != 0) {
                    take(static_cast<int>(i));
                }
            }
        }
    } else {
        if (p.cache.tokens > 1 && threadIdx.x == 0) {
            rec.odd[blockIdx.x] = 0;
        }
        take(static_cast<int>(blockIdx.x));
    }
}

// Items that are never cut, one a CTA.
template <class C, bool CAREFUL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) cached_whole_kernel(const __grid_constant__ FaCachedParams p,
                                                                            DeviceStatus* status, Record rec, int ranges) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int row_tiles = (p.heads / p.cache.kv_heads * p.cache.tokens + kRows - 1) / kRows;
    const int items = p.cache.kv_heads * row_tiles;
    take_ranges<CAREFUL>(p, rec, ranges, [&](int range) {
        const int b = range / items;
        const int item = range - b * items;
        const Sequence s = sequence<C>(p, b);
        attend<C, CAREFUL>(p, status, smem, s, b, item / row_tiles, (item % row_tiles) * kRows, 0, s.tiles, rec, -1);
    });
}

template <class C, bool CAREFUL>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) cached_kernel(const __grid_constant__ FaCachedParams p,
                                                                      DeviceStatus* status, Record rec, int ranges) {
    extern __shared__ __align__(128) uint8_t smem[];
    take_ranges<CAREFUL>(p, rec, ranges, [&](int cta) {
        const Range range = locate<C>(p, ranges, [&](long long per) { return cta * per; });
        if (range.found < 0) {
            return;  // past the end of the list
        }
        const int row_tiles = (p.heads / p.cache.kv_heads * p.cache.tokens + kRows - 1) / kRows;
        const int items = p.cache.kv_heads * row_tiles;
        long long at = cta * range.per;
        const long long end = min(at + range.per, range.total);
        int b = range.found;
        Sequence s = sequence<C>(p, b);
        long long in_seq = at - range.found_base;
        int item = static_cast<int>(in_seq / s.tiles);
        int v = static_cast<int>(in_seq - static_cast<long long>(item) * s.tiles);
        bool first = true;
        while (at < end) {
            const int take = static_cast<int>(min(static_cast<long long>(s.tiles - v), end - at));
            const bool whole = v == 0 && take == s.tiles;
            attend<C, CAREFUL>(p, status, smem, s, b, item / row_tiles, (item % row_tiles) * kRows, v, v + take, rec,
                               whole ? -1 : 2ll * cta + (first ? 0 : 1));
            first = false;
            at += take;
            v = 0;
            if (at < end && ++item == items) {
                item = 0;
                s = sequence<C>(p, ++b);
            }
        }
    });
}

// Joins the records of the item that was cut at unit k per, k = blockIdx.x + 1, if that is its first
// cut, always in the same order. SPREAD: a row a CTA, its 4 warps taking the records in turn and joining in
// order, where all those CTAs are resident at once or an item has many records (few, long sequences). Else a
// warp a row, 4 rows a CTA (64 sequences x 4 tokens: 122 us a call with SPREAD, 110 without; one token
// over 777: 10.3 us with, 12.7 without).
template <class C, bool SPREAD>
__global__ void __launch_bounds__(kThreads) cached_join_kernel(const __grid_constant__ FaCachedParams p, Record rec,
                                                               int grid) {
    constexpr int D = C::D;
    constexpr int PER = D / 32;
    const long long k = blockIdx.x + 1;
    const Range range = locate<C>(p, grid, [&](long long per) { return k * per; });
    // One CTA waits whatever it finds to do, so that this kernel's end stands for the end of the one before.
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        cudaGridDependencySynchronize();
    }
    if (range.found < 0) {
        return;
    }
    const int group = p.heads / p.cache.kv_heads;
    const int rows = group * p.cache.tokens;
    const int row_tiles = (rows + kRows - 1) / kRows;
    const Sequence s = sequence<C>(p, range.found);
    const long long item = (k * range.per - range.found_base) / s.tiles;
    const long long start = range.found_base + item * s.tiles;
    const int row0 = static_cast<int>(item % row_tiles) * kRows;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int row = SPREAD ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.y) * kWarps + warp;
    const int row_first = SPREAD ? row : static_cast<int>(blockIdx.y) * kWarps;
    if (start == k * range.per || start / range.per != k - 1 || row0 + row_first >= rows) {
        return;
    }
    const long long c0 = start / range.per;
    const long long c1 = (start + s.tiles - 1) / range.per;
    cudaGridDependencySynchronize();  // the records are there
    float m = -INFINITY, l = 0.0f;
    float o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        o[i] = 0.0f;
    }
    if (row < kRows) {
#pragma unroll 4
        for (long long c = c0 + (SPREAD ? warp : 0); c <= c1; c += SPREAD ? kWarps : 1) {
            // A CTA's first stretch is its record 0; the item starts in c0, as its second unless there.
            const long long record = (2 * c + (c * range.per >= start ? 0 : 1)) * kRows + row;
            const float2 ml = rec.ml[record];
            float y[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                y[i] = rec.o[record * D + lane * PER + i];
            }
            const float now = fmaxf(m, ml.x);
            const float used = now == -INFINITY ? 0.0f : now;
            const float a = ex2_approx(m - used);
            const float w = ex2_approx(ml.x - used);
            m = now;
            l = fmaf(ml.y, w, l * a);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                o[i] = fmaf(y[i], w, o[i] * a);
            }
        }
    }
    if constexpr (SPREAD) {
        __shared__ float2 all_ml[kWarps];
        __shared__ float all_o[kWarps][D];
        if (lane == 0) {
            all_ml[warp] = make_float2(m, l);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            all_o[warp][lane * PER + i] = o[i];
        }
        __syncthreads();
        if (warp > 0) {
            return;
        }
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            m = fmaxf(m, all_ml[w].x);
        }
        const float used = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            o[i] = 0.0f;
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ex2_approx(all_ml[w].x - used);
            l = fmaf(all_ml[w].y, f, l);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                o[i] = fmaf(all_o[w][lane * PER + i], f, o[i]);
            }
        }
    }
    if (row >= kRows || row0 + row >= rows) {
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int kvh = static_cast<int>(item / row_tiles);
    const int head = (row0 + row) / p.cache.tokens;
    const int token = row0 + row - head * p.cache.tokens;
    const long long out_row =
        (static_cast<long long>(range.found) * p.heads + kvh * group + head) * p.cache.tokens + token;
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
        reinterpret_cast<uint32_t*>(p.o)[(out_row * D + lane * PER + i) / 2] =
            pack2<C::BF16>(o[i] * inv, o[i + 1] * inv);
    }
}

int tile_keys(const FaCache& c) { return kTileBytes / (c.head_dim * (c.dtype == FA_DTYPE_FLOAT8_E4M3 ? 1 : 2)); }

// How a call is cut. Short contexts (by the table's capacity, since lengths are on the device): an item is
// one CTA's, two key tiles a warp, in one launch. Longer ones: the CTAs that fill the GPU, or
// fewer where the capacity is less work, and a second launch to join (one token over 777 in 25
// tiles of 16 heads: 10.3 us so, 14.0 us with a CTA a head and 7 tiles a warp).
struct Split {
    bool whole;
    long long grid;
    long long items;
};

Split split_for(const FaCachedParams& p, int sm_count) {
    const FaCache& c = p.cache;
    const int keys = tile_keys(c);
    const long long rows = static_cast<long long>(p.heads / c.kv_heads) * c.tokens;
    const long long items = static_cast<long long>(c.batch) * c.kv_heads * ((rows + kRows - 1) / kRows);
    long long shown = static_cast<long long>(c.max_pages) * c.page_size;
    if (p.window > 0) {
        shown = std::min<long long>(shown, static_cast<long long>(p.window) + p.sinks + c.tokens + 2 * keys);
    }
    const long long tiles = shown / keys + 1;
    if (tiles <= kWholeTiles) {
        return {true, items, items};
    }
    return {false, std::min<long long>(kCtasPerSm * sm_count, (items * tiles + kMinTiles - 1) / kMinTiles), items};
}

// Launches after the kernel before it has started to end: it waits for its results itself.
template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

template <class C>
cudaError_t launch_join(const FaCachedParams& p, const Record& rec, const Split& split, int sm_count, cudaStream_t stream) {
    const int grid = static_cast<int>(split.grid);
    const int rows = std::min(kRows, p.heads / p.cache.kv_heads * p.cache.tokens);
    constexpr int kResident = 16;  // CTAs of the join on an SM
    const bool spread = static_cast<long long>(grid - 1) * rows <= kResident * sm_count || grid > 8 * split.items;
    const dim3 join_grid(static_cast<unsigned>(grid - 1), static_cast<unsigned>(spread ? rows : (rows + kWarps - 1) / kWarps));
    return spread ? launch_early(cached_join_kernel<C, true>, join_grid, 0, stream, p, rec, grid)
                  : launch_early(cached_join_kernel<C, false>, join_grid, 0, stream, p, rec, grid);
}

// All items or ranges; with several tokens, those that have to be taken carefully; the join of what was cut.
template <class C, bool WHOLE>
cudaError_t launch_kernels(const FaCachedParams& p, DeviceStatus* status, const Record& rec, const Split& split, int sm_count,
                           cudaStream_t stream) {
    constexpr auto kernel = WHOLE ? cached_whole_kernel<C, false> : cached_kernel<C, false>;
    constexpr auto careful = WHOLE ? cached_whole_kernel<C, true> : cached_kernel<C, true>;
    const int ranges = static_cast<int>(split.grid);
    cudaError_t err = ensure_smem_limit<kernel>(kSmem);
    if (err == cudaSuccess && p.cache.tokens > 1) {
        err = ensure_smem_limit<careful>(kSmemCareful);
    }
    if (err != cudaSuccess) {
        return err;
    }
    kernel<<<ranges, kThreads, kSmem, stream>>>(p, status, rec, ranges);
    err = cudaGetLastError();
    if (err == cudaSuccess && p.cache.tokens > 1) {
        // Half as many CTAs as SMs: they find room while the first kernel's last ranges run, and the join's CTAs after
        // them (64 sequences x 4 tokens: 112.5 us, with a CTA for each range 115, without this kernel 110).
        err = launch_early(careful, dim3(static_cast<unsigned>(std::min(ranges, std::max(sm_count / 2, 1)))), kSmemCareful, stream,
                           p, status, rec, ranges);
    }
    if (err == cudaSuccess && !WHOLE && ranges > 1) {
        err = launch_join<C>(p, rec, split, sm_count, stream);
    }
    return err;
}

template <class C>
cudaError_t launch(const FaCachedParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    const Split split = split_for(p, sm_count);
    if (split.grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    Record rec{};
    if (split.whole) {
        rec.odd = static_cast<int*>(workspace);
        return launch_kernels<C, true>(p, status, rec, split, sm_count, stream);
    }
    const size_t rows = static_cast<size_t>(split.grid) * 2 * kRows;
    rec.o = static_cast<float*>(workspace);
    rec.ml = reinterpret_cast<float2*>(rec.o + rows * C::D);
    rec.odd = reinterpret_cast<int*>(rec.ml + rows);
    return launch_kernels<C, false>(p, status, rec, split, sm_count, stream);
}

template <int D, bool ONE_PAGE>
cudaError_t launch_pages(const FaCachedParams& p, DeviceStatus* status, void* workspace, int sm_count,
                         cudaStream_t stream) {
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.cache.dtype == FA_DTYPE_FLOAT8_E4M3) {
        return bf16 ? launch<Cfg<D, true, true, ONE_PAGE>>(p, status, workspace, sm_count, stream)
                    : launch<Cfg<D, false, true, ONE_PAGE>>(p, status, workspace, sm_count, stream);
    }
    return bf16 ? launch<Cfg<D, true, false, ONE_PAGE>>(p, status, workspace, sm_count, stream)
                : launch<Cfg<D, false, false, ONE_PAGE>>(p, status, workspace, sm_count, stream);
}

template <int D>
cudaError_t launch_dim(const FaCachedParams& p, DeviceStatus* status, void* workspace, int sm_count,
                       cudaStream_t stream) {
    return p.cache.page_size >= tile_keys(p.cache) ? launch_pages<D, true>(p, status, workspace, sm_count, stream)
                                                   : launch_pages<D, false>(p, status, workspace, sm_count, stream);
}

}  // namespace

unsigned long long cached_workspace_bytes(const FaCachedParams& p, int sm_count) {
    const Split split = split_for(p, sm_count);
    const unsigned long long records = split.whole ? 0 : static_cast<unsigned long long>(split.grid) * 2 * kRows * (p.cache.head_dim + 2) * 4;
    return records + (p.cache.tokens > 1 ? 4ull * split.grid : 0);
}

cudaError_t launch_cached(const FaCachedParams& p, DeviceStatus* status, void* workspace, int sm_count,
                          cudaStream_t stream) {
    return p.cache.head_dim == 64 ? launch_dim<64>(p, status, workspace, sm_count, stream)
                                  : launch_dim<128>(p, status, workspace, sm_count, stream);
}

}  // namespace fa_sm100
