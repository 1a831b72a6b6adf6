// Backward of window attention with sinks for B200 (sm_100a): tcgen05.mma into tensor memory, TMA
// rings, softmax warpgroups with one row a thread.
//
//   S = scale Q K^T (masked), P = e^(S - LSE), delta = rowsum(dO o O), dP = dO V^T,
//   dS = P o (dP - delta),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
//
// P and dS are rounded to 16 bits for their products; in float16, whose range is short, times a power of two
// (head_power).
//
// Three passes: delta by rows (bound by DRAM bytes); dK and dV by key tiles; dQ by query tiles. The last
// two recompute P, seven products a tile pair where one pass over both would take five, but every
// sum then has one owner: no atomics, no float32 dQ in memory, the same bits every time. They are
// one kernel, written for a resident pair of tiles (R0, R1) and streamed pairs (X, Y):
//
//                 R0  R1  X  Y    S            dP            products
//   DKV           K   V   Q  dO   K Q^T = S^T  V dO^T = dP^T  dV += P^T Y,  dK += dS^T X
//   dQ            Q   dO  K  V    Q K^T        dO V^T                       dQ += dS X
//
// Tensor memory (columns): S 0..127, dP 128..255, the products' accumulators from 256. P and dS are
// 16-bit matrix operands read from tensor memory. dQ has room for two dS of its own. DKV with d =
// 128 has none left: P(i) lies in the first half of dP's columns until dV(i) has read it, then dP(i) takes
// them all, and once every warp has read dP(i), dS(i) goes to the second half and P(i + 1) to the first.
// The tensor pipe is kept busy by the order of issue. DKV: S(i + 1) as soon as S(i) is in registers; with
// P(i) and dS(i - 1) in hand dV(i), dK(i - 1), dP(i), under which the exponentials of tile i + 1 run. dQ: S(i + 1) as
// early, and with dS(i) in hand dP(i + 1), dQ(i).
//
// Warps: two warpgroups share a tile's 128 x 128 scores, 64 columns each (thread = row); a third has the TMA
// producer, the issuer of S, the issuer of the other products (issuing holds a warp until the tensor pipe
// takes its products) and (DKV) the loader of LSE and delta of the streamed rows. Every role walks the
// same items with running barrier phases, so that the next item's loads and first products run under an
// item's last tile and its stores.
//
// Split. A resident tile's list of streamed tiles (DKV: the query tiles of its window, of every head
// of its group; keys with sinks take all later ones) makes an item; the items laid end to end are cut
// into equal ranges of streamed tiles, one a CTA, one CTA an SM. Whole lists in turn left up to a
// quarter of the SMs idle (254 lists of 132 tiles on 148 SMs). A cut list's parts leave float32
// sums in the workspace, at most two a CTA, and a last kernel adds them up in order.

// Measured, bf16, D 128 (of 1689 TFLOP/s), in bursts: 16 x 8191 on 4 kv heads, window 1024 + 4 sinks 280 us, 8 x 16384 on
// 2, window 4096 780 us (770 TFLOP/s of the 5 products of visible pairs, 1080 of the 7 computed); float16 290 and 810 us. A
// DKV step is 2048 cycles of products and 2400 of shared memory (192 KB of operands, 64 KB arriving, the columns' LSE and
// delta), a dQ step 1536 and 1800, which is what bounds them: without the exponentials they take as long. Tiles
// shared by two SMs (cta_group::2) would halve the streamed operands. At d = 64 the softmax bounds them (2 x 16 x 8192 on 4
// kv heads, window 1024: 420 us), and its loop is about as long as the SM fetches in time: a few dozen instructions more
// took up to 18% of the dK, dV pass, with the stalls for want of an instruction up from 0.25 to 0.44 an issue.

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "softmax_common.cuh"
#include "stream_internal.h"
#include "tma_host.h"

namespace fa_sm100 {

namespace {

constexpr int kTile = 128;             // rows of every tile
constexpr int kBox = kTile * 128;      // one TMA box: 128 rows x 128 bytes
constexpr int kXStages = 3;
constexpr int kYStages = 2;
// Items whose powers are kept (float16). The loader is at most three streamed tiles ahead of the products, and an
// item's products wait for the sums of the one before to be read, so that four are never overwritten too early.
constexpr int kPowers = 4;
static_assert(kPowers > kXStages, "an item's power stays until its sums are read");
constexpr int kBwdThreads = 384;
constexpr int kSoftmaxWarps = 8;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kLoaderWarp = 10;
constexpr int kScoreWarp = 11;  // issues S; kMmaWarp the other products
// Registers: 8 softmax warps take 224 and the other four keep 56, the launch's 384 x 168 in all (P of two tiles
// in float32: 208 and 88 spill more and take 2% longer).
constexpr int kRegsSoftmax = 224;
constexpr int kRegsOther = 56;
static_assert(256 * kRegsSoftmax + 128 * kRegsOther <= kBwdThreads * 168, "register split");
constexpr int kEmuPer8 = 3;  // column pairs of 8 whose 2^x runs on the FMA pipe (1: 2% slower, 4: the same)
__host__ __device__ constexpr bool emulated(int column) { return (column / 2) % 8 < kEmuPer8; }

struct BwdArgs {
    int batch, heads, kv_heads, group;
    int q_len, k_len, shift, window, sinks;
    int tiles;              // resident tiles of a head (DKV: key tiles of a kv head)
    int grid;               // CTAs
    long long head_steps;   // streamed tiles of a head's lists
    long long steps;        // of all heads'
    long long per;          // of a CTA
    float scale, scale_log2;
    const float* lse;       // [batch * heads][q_len]
    const float* delta;
    const float* do_size;   // float16: largest |dO|_2 of kSlotRows query rows, [batch * heads][q_slots]
    const float* v_size;    // ... |V|_2 of key rows, [batch * kv_heads][k_slots]
    int q_slots, k_slots;   // of a head
    float* parts;           // cut lists' sums, [part][outputs][D / 4][128 rows][4]
    void* out0;             // DKV: dV
    void* out1;             // dK or dQ
    int64_t out0_stride[3], out1_stride[3];
    FastDiv div_heads, div_group;  // heads of the lists (DKV: kv heads)
    unsigned epoch;
    DeviceStatus* status;
};

template <int D_, bool BF16_, bool DKV_>
struct BwdCfg {
    static constexpr int D = D_;
    static constexpr bool BF16 = BF16_;
    static constexpr bool DKV = DKV_;
    static constexpr bool kLoads = DKV_ || !BF16_;  // there is work for the loader warp
    static constexpr int kBoxes = D / 64;
    static constexpr int kTileBytes = kTile * D * 2;
    static constexpr int kSmemR0 = 0;
    static constexpr int kSmemR1 = kTileBytes;
    static constexpr int kSmemX = 2 * kTileBytes;
    static constexpr int kSmemY = kSmemX + kXStages * kTileBytes;
    static constexpr int kSmemShared = kSmemY + kYStages * kTileBytes;
    static constexpr int kTmemS = 0;
    static constexpr int kTmemDP = 128;
    static constexpr int kTmemAcc0 = 256;              // DKV: dV
    static constexpr int kTmemAcc1 = DKV ? 256 + D : 256;  // dK or dQ
    // Columns of the 16-bit operands (64 each): DKV with d = 128 over dP's (see above).
    static constexpr bool kOverDP = DKV && D == 128;
    static constexpr int kTmemP = kOverDP ? kTmemDP : 384;
    static constexpr int kTmemDS = kOverDP ? kTmemDP + 64 : (DKV ? 448 : 384);
    static constexpr int kTmemDS2 = DKV ? kTmemDS : 448;  // of odd tiles
    static constexpr int kTmemCols = 512;
};

struct BwdShared {
    uint64_t r0_full, r0_empty, r1_full, r1_empty;
    uint64_t x_full[kXStages], x_empty[kXStages];
    uint64_t y_full[kYStages], y_empty[kYStages];
    uint64_t s_read[2];  // of alternate tiles
    uint64_t s_full, dp_full, ds_full, acc_done, acc_free, mma_idle;
    uint32_t tmem_base;
    int abort;
    int tile, offset;  // where the CTA's range starts
    long long warp_sum[kBwdThreads / 32];
    // DKV: of the streamed rows: minus LSE in log2 units (-inf: P = 0), minus delta.
    alignas(16) float lse2[2][kTile];
    alignas(16) float delta[kXStages][kTile];
    float power[kPowers];  // float16: head_power
};

// No static shared memory: the tiles start the dynamic window, 1024-byte aligned, and with d = 128 leave
// 3 KB of the 227 for the rest.
template <class Cfg>
constexpr int bwd_smem() {
    static_assert(Cfg::kSmemShared + sizeof(BwdShared) <= 227 * 1024, "shared memory budget");
    static_assert(Cfg::kSmemShared + sizeof(BwdShared) > 114 * 1024, "one CTA an SM: it owns all of tensor memory");
    return Cfg::kSmemShared + static_cast<int>(sizeof(BwdShared));
}

struct BwdItem {
    int b, kvh, head;   // head: dQ
    int row0;           // of the resident tiles
    int total;          // streamed tiles of the list
    int first, n;       // this CTA's part of it
    long long part;     // record of the part's sums, -1: it is the whole list
    int q0, per;        // DKV: the list is query tiles [q0, q0 + per) of every head of the group
    int sink_tiles, first_tile;  // dQ: the list is key tiles [0, sink_tiles), [first_tile, ..]
};

// Rows of a delta block, and of a slot of do_size and v_size.
constexpr int kDeltaThreads = 256;
constexpr int kDeltaRows = 4;  // of a thread
template <int D>
constexpr int kSlotRows = kDeltaThreads / (D / 8) * kDeltaRows;

// The power of two, 2^15 at most, that brings `bound` below 2^16; 1 where it is 0 or not finite.
__device__ __forceinline__ float power_for(float bound) {
    const int e = static_cast<int>(__float_as_uint(bound) >> 23);  // bound < 2^(e - 126)
    return __uint_as_float(static_cast<uint32_t>((e == 0 || e >= 255) ? 127 : 127 + max(min(142 - e, 15), -100)) << 23);
}
__device__ __forceinline__ float inverse_power(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }
__device__ __forceinline__ float exponent(float p) { return static_cast<float>(static_cast<int>(__float_as_uint(p) >> 23) - 127); }

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    }
    return x;
}

// The list of resident tile `tile`: its length, and what it is made of. A tile with nothing to see
// keeps one streamed tile, all hidden, so that its zeros are written.
template <bool DKV>
__host__ __device__ inline void tile_list(const BwdArgs& a, int tile, BwdItem& it) {
    it.row0 = tile * kTile;
    if (DKV) {
        const long long k0 = it.row0;
        const long long lo = k0 - a.shift > 0 ? k0 - a.shift : 0;
        const long long k_last = (k0 + kTile < a.k_len ? k0 + kTile : a.k_len) - 1;
        long long hi = k0 < a.sinks ? a.q_len - 1 : k_last + a.window - 1 - a.shift;
        hi = hi < a.q_len - 1 ? hi : a.q_len - 1;
        it.q0 = static_cast<int>(lo / kTile);
        it.per = hi >= lo ? static_cast<int>(hi / kTile) - it.q0 + 1 : 0;
        it.total = it.per > 0 ? it.per * a.group : 1;
        it.per = it.per > 0 ? it.per : 1;
    } else {
        const int lo_pos = it.row0 + a.shift > 0 ? it.row0 + a.shift : 0;
        const int end = it.row0 + kTile < a.q_len ? it.row0 + kTile : a.q_len;
        const int hi_pos = end - 1 + a.shift > 0 ? end - 1 + a.shift : 0;
        it.first_tile = lo_pos - a.window + 1 > 0 ? (lo_pos - a.window + 1) / kTile : 0;
        const int sinks = (a.sinks + kTile - 1) / kTile;
        it.sink_tiles = sinks < it.first_tile ? sinks : it.first_tile;
        it.total = it.sink_tiles + hi_pos / kTile - it.first_tile + 1;
    }
}

template <bool DKV>
__device__ __forceinline__ int list_length(const BwdArgs& a, int tile) {
    BwdItem it;
    tile_list<DKV>(a, tile, it);
    return it.total;
}

// The resident tile whose list holds streamed tile `at` of a head's lists, and its place in the list.
// All THREADS of a block call; the result is in *tile, *offset after the next barrier.
template <bool DKV, int THREADS>
__device__ __forceinline__ void locate_tile(const BwdArgs& a, long long at, long long* warp_sum, int* tile, int* offset) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int share = (a.tiles + THREADS - 1) / THREADS;
    const int t0 = min(static_cast<int>(threadIdx.x) * share, a.tiles);
    const int t1 = min(t0 + share, a.tiles);
    long long mine = 0;
    for (int t = t0; t < t1; ++t) {
        mine += list_length<DKV>(a, t);
    }
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        incl += lane >= o ? up : 0;
    }
    if (lane == 31) {
        warp_sum[warp] = incl;
    }
    __syncthreads();
    long long before = incl - mine;
    for (int w = 0; w < warp; ++w) {
        before += warp_sum[w];
    }
    if (at >= before && at < before + mine) {
        for (int t = t0; t < t1; ++t) {
            const int n = list_length<DKV>(a, t);
            if (at < before + n) {
                *tile = t;
                *offset = static_cast<int>(at - before);
                break;
            }
            before += n;
        }
    }
}

// Walks a CTA's range, list by list.
struct Cursor {
    int bx, tile, offset;  // head of the lists, resident tile, place in its list
    long long left;
    long long record;      // of the next part
};

template <bool DKV>
__device__ __forceinline__ bool next_item(const BwdArgs& a, Cursor& c, BwdItem& it) {
    if (c.left <= 0) {
        return false;
    }
    tile_list<DKV>(a, c.tile, it);
    it.b = a.div_heads.div(c.bx);
    const int h = c.bx - it.b * static_cast<int>(a.div_heads.d);
    it.head = h;
    it.kvh = DKV ? h : a.div_group.div(h);
    it.first = c.offset;
    it.n = static_cast<int>(min(static_cast<long long>(it.total - c.offset), c.left));
    it.part = it.n == it.total ? -1 : c.record;
    c.record |= 1;  // a CTA's range has at most two parts: its first list's and its last's
    c.left -= it.n;
    c.offset = 0;
    if (++c.tile == a.tiles) {
        c.tile = 0;
        ++c.bx;
    }
    return true;
}

// Streamed tile i of an item: its first row, and (DKV) its head.
template <class Cfg>
__device__ __forceinline__ void stream_tile(const BwdArgs& a, const BwdItem& it, int i, int& row, int& head) {
    const int at = it.first + i;
    if constexpr (Cfg::DKV) {
        const int g = at / it.per;
        row = (it.q0 + at - g * it.per) * kTile;
        head = it.kvh * a.group + g;
    } else {
        row = (at < it.sink_tiles ? at : at - it.sink_tiles + it.first_tile) * kTile;
        head = it.kvh;
    }
}

// float16: the power of two that P and dS carry, by the exponent of P, and the sums give back; one for a kv head and its
// group. With delta = sum_k P_k dP_k, |dS_j| = P_j |dP_j - delta| <= P_j (1 - P_j) 2 max|dP| <= max|dO|_2 max|V|_2 / 2, so that
// neither P nor dS overflows with it (a tenth is left for what P, O and the norms round). Without, dS of ordinary
// small dO (P is about 1 / window) fell among float16's subnormals: with a window of 1024 and dO of 1e-3 the gradients
// were off by 0.13%, of 1e-4 by 1.3%; and large ones overflowed. A power below 1 costs small P of dV bits instead;
// rows whose dO is 10^4 below the largest still have normal dS. (A factor on dS alone, in the streamed delta and an FMA,
// took 17% of the dK, dV pass at d = 64; a power for each item, from its own list, 7 to 18%. This, with the norms,
// takes 1 to 3% of the whole.) bfloat16 has float32's range and needs none. The whole loader warp calls.
__device__ __forceinline__ float head_power(const BwdArgs& a, int b, int kvh) {
    const float* d_o = a.do_size + (static_cast<long long>(b) * a.heads + kvh * a.group) * a.q_slots;
    const float* v = a.v_size + (static_cast<long long>(b) * a.kv_heads + kvh) * a.k_slots;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    float most = 0.0f, value = 0.0f;
    const long long n = static_cast<long long>(a.group) * a.q_slots;
#pragma unroll 8
    for (long long i = lane; i < n; i += 32) {
        most = fmaxf(most, __ldg(d_o + i));
    }
#pragma unroll 4
    for (int i = lane; i < a.k_slots; i += 32) {
        value = fmaxf(value, __ldg(v + i));
    }
    return power_for(0.55f * warp_max(most) * warp_max(value));
}

// D (128 x 128) = A B^T, both operands 128 rows of the head dim in shared memory.
template <class Cfg>
__device__ __forceinline__ void issue_scores(uint32_t d, uint64_t a, uint64_t b) {
    constexpr uint32_t idesc = make_idesc_f16(kTile, kTile, true, false, Cfg::BF16);
#pragma unroll
    for (int k = 0; k < Cfg::D / 16; ++k) {
        const uint64_t off = static_cast<uint64_t>(((k / 4) * kBox + (k % 4) * 32) >> 4);
        umma_ss(d, a + off, b + off, idesc, k > 0 ? 1u : 0u);
    }
}

// acc (128 x D) += W T: W (128 x 128, 16-bit) in tensor memory, 64 columns from `w`; T the 128 rows of a
// streamed tile.
template <class Cfg>
__device__ __forceinline__ void issue_product(uint32_t acc, uint32_t w, uint64_t t, bool first) {
    constexpr uint32_t idesc = make_idesc_f16(kTile, Cfg::D, true, true, Cfg::BF16);
#pragma unroll
    for (int k = 0; k < kTile / 16; ++k) {
        umma_ts(acc, w + k * 8, t + static_cast<uint64_t>(k * (2048 >> 4)), idesc,
                     (first && k == 0) ? 0u : 1u);
    }
}

// hide_columns with rows = keys: kept are the columns [from, from + span).
__device__ __forceinline__ void hide_key_columns(uint32_t (&x)[64], int from, int span) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const uint32_t keep = bits_up_to(from + span - 1 - 32 * g) & ~bits_up_to(from - 1 - 32 * g);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            x[32 * g + c] = (keep >> c) & 1u ? x[32 * g + c] : 0xff800000u;
        }
    }
}

template <class Cfg>
__global__ void __launch_bounds__(kBwdThreads, 1)
    window_bwd_kernel(const __grid_constant__ CUtensorMap tm_r0, const __grid_constant__ CUtensorMap tm_r1,
                      const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_y,
                      const __grid_constant__ BwdArgs args) {
    constexpr int D = Cfg::D;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    BwdShared& sh = *reinterpret_cast<BwdShared*>(smem_raw + Cfg::kSmemShared);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0);
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const uint32_t smem = smem_u32(smem_raw);
    if ((smem & 1023u) != 0) {  // the swizzled layouts need it; the driver places the window so
        atomicOr(&args.status->code, kStatusTimeoutTeardown);
        return;
    }
    const long long start = static_cast<long long>(blockIdx.x) * args.per;
    const int first_head = static_cast<int>(start / args.head_steps);
    const WaitCtx wctx{&sh.abort, &args.status->code, &args.status->epoch_aborted, args.epoch};

    if (threadIdx.x == 0) {
        sh.abort = 0;
        mbar_init(smem_u32(&sh.r0_full), 1);
        mbar_init(smem_u32(&sh.r0_empty), 1);
        mbar_init(smem_u32(&sh.r1_full), 1);
        mbar_init(smem_u32(&sh.r1_empty), 1);
        for (int s = 0; s < kXStages; ++s) {
            mbar_init(smem_u32(&sh.x_full[s]), Cfg::kLoads ? 2 : 1);  // the copy, and the loader's
            mbar_init(smem_u32(&sh.x_empty[s]), 1);
        }
        for (int s = 0; s < kYStages; ++s) {
            mbar_init(smem_u32(&sh.y_full[s]), 1);
            mbar_init(smem_u32(&sh.y_empty[s]), 1);
        }
        mbar_init(smem_u32(&sh.s_read[0]), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.s_read[1]), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.s_full), 1);
        mbar_init(smem_u32(&sh.dp_full), 1);
        mbar_init(smem_u32(&sh.ds_full), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.acc_done), 1);
        mbar_init(smem_u32(&sh.acc_free), kSoftmaxWarps);
        mbar_init(smem_u32(&sh.mma_idle), 2);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&sh.tmem_base), Cfg::kTmemCols);
        tmem_relinquish();
    }
    locate_tile<Cfg::DKV, kBwdThreads>(args, start - first_head * args.head_steps, sh.warp_sum, &sh.tile, &sh.offset);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Owning all 512 columns means owning them from 0: a constant, like the shared-memory addresses.
    constexpr uint32_t tmem = 0;
    if (sh.tmem_base != tmem) {
        if (threadIdx.x == 0) {
            atomicOr(&args.status->code, kStatusTimeoutTeardown);
        }
        __syncthreads();
        if (warp == kMmaWarp) {
            tmem_dealloc(sh.tmem_base, Cfg::kTmemCols);
        }
        return;
    }
    Cursor cursor;
    cursor.bx = first_head;
    cursor.tile = __shfl_sync(0xffffffffu, sh.tile, 0);  // the same in all lanes, known to be
    cursor.offset = __shfl_sync(0xffffffffu, sh.offset, 0);
    cursor.left = min(args.per, args.steps - start);
    cursor.record = 2 * static_cast<long long>(blockIdx.x);
    if constexpr (Cfg::DKV) {
        cudaGridDependencySynchronize();  // delta is there
        cudaTriggerProgrammaticLaunchCompletion();  // the dQ pass may take SMs as they get free
    }

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    }

    if (warp < kSoftmaxWarps) {
        // ================================== softmax ====================================
        const int wg = warp / 4;
        const int row = (warp % 4) * 32 + lane;
        const int col0 = wg * 64;
        const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const uint32_t t_s = tmem + lanes + Cfg::kTmemS + col0;
        const uint32_t t_dp = tmem + lanes + Cfg::kTmemDP + col0;
        const uint32_t t_p = tmem + lanes + Cfg::kTmemP + wg * 32;
        const uint32_t t_ds = tmem + lanes + Cfg::kTmemDS + wg * 32;
        const float scale_log2 = args.scale_log2;
        int g = 0;      // streamed tiles whose S was read so far
        int gd = 0;     // ... whose dP was
        int done = 0;   // accumulations read out so far
        bool ok = true;
        auto arrive = [&](uint64_t* bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(bar));
            }
        };
        BwdItem it, next;
        bool more = next_item<Cfg::DKV>(args, cursor, next);
        float next_lse2, next_delta;
        auto statistics = [&]() {  // dQ: of this thread's row of the next item, negated
            next_lse2 = -INFINITY;
            next_delta = 0.0f;
            if (!Cfg::DKV && more && next.row0 + row < args.q_len) {
                const long long at =
                    (static_cast<long long>(next.b) * args.heads + next.head) * args.q_len + next.row0 + row;
                const float lse = __ldg(args.lse + at);
                next_lse2 = lse == -INFINITY ? -INFINITY : lse * -1.4426950408889634f;
                next_delta = -__ldg(args.delta + at);
            }
        };
        statistics();
        while (more) {
            it = next;
            float row_lse2 = next_lse2;
            const float row_delta = next_delta;
            more = next_item<Cfg::DKV>(args, cursor, next);
            statistics();
            // P of tile i in float32 from S. It is rounded to 16 bits for dV's product alone; dS is made of P and dP
            // in float32 and rounded once, for its own products. (With the rounded P in dS dK was off by twice
            // what rounding dK itself costs; this takes 3% longer.)
            auto probabilities = [&](int i, uint32_t (&p)[64]) {
                int tile_row, head;
                stream_tile<Cfg>(args, it, i, tile_row, head);
                ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.s_full), g & 1, wctx, kStatusTimeoutSoftmax));
                if (!ok) {
                    return;
                }
                tc_fence_after();
                if constexpr (!Cfg::DKV && !Cfg::BF16) {
                    if (i == 0) {
                        row_lse2 += exponent(sh.power[done % kPowers]);
                    }
                }
                tmem_ld64(t_s, p);
                // Half of the columns' LSE comes meanwhile: shared memory is busy with the products' operands.
                [[maybe_unused]] float4 early[8];
                if constexpr (Cfg::DKV) {
#pragma unroll
                    for (int c4 = 0; c4 < 8; ++c4) {
                        early[c4] = *reinterpret_cast<const float4*>(&sh.lse2[g % 2][col0 + 4 * c4]);
                    }
                }
                tmem_wait_ld();
                if constexpr (!Cfg::DKV) {
                    arrive(&sh.s_read[g % 2]);  // S is in registers: the next scores may take its columns
                }
#pragma unroll
                for (int c4 = 0; c4 < 16; ++c4) {
                    float2 neg[2];
                    if constexpr (Cfg::DKV) {
                        const float4 l4 =
                            c4 < 8 ? early[c4 % 8] : *reinterpret_cast<const float4*>(&sh.lse2[g % 2][col0 + 4 * c4]);
                        neg[0] = make_float2(l4.x, l4.y);
                        neg[1] = make_float2(l4.z, l4.w);
                    } else {
                        neg[0] = neg[1] = make_float2(row_lse2, row_lse2);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c = 4 * c4 + 2 * h;
                        const float2 x = __ffma2_rn(make_float2(u2f(p[c]), u2f(p[c + 1])),
                                                    make_float2(scale_log2, scale_log2), neg[h]);
                        p[c] = f2u(x.x);
                        p[c + 1] = f2u(x.y);
                    }
                }
                if constexpr (Cfg::DKV) {
                    arrive(&sh.s_read[g % 2]);  // ... and the LSE of tile i + 2 its slot
                }
                // Masks: query position minus key position in [0, window), or the key a sink.
                const int q_row = Cfg::DKV ? tile_row : it.row0;
                const int k_row = Cfg::DKV ? it.row0 : tile_row;
                const int gap = q_row + args.shift - k_row;  // of the tiles' first rows
                if (gap < kTile - 1 || (gap + kTile - 1 >= args.window && k_row + kTile > args.sinks)) {
                    if constexpr (Cfg::DKV) {
                        // Row = key: it is seen by the columns [from, from + window), a sink by all from
                        // `from` on.
                        hide_key_columns(p, row - gap - col0, k_row + row < args.sinks ? kNoWindow : args.window);
                    } else {
                        // Row = query: it sees the columns (to - window, to], and the sinks.
                        hide_columns<64>(p, gap + row - col0, args.window, args.sinks - k_row - col0, 0xff800000u);
                    }
                }
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float2 x = make_float2(u2f(p[c]), u2f(p[c + 1]));
                    const float2 e = emulated(c) ? exp2_poly2(x)
                                                 : make_float2(ex2_approx(x.x), ex2_approx(x.y));
                    p[c] = f2u(e.x);
                    p[c + 1] = f2u(e.y);
                }
            };
            // dS of the tile whose dP is next, from its P.
            auto gradients = [&](const auto& p, uint32_t (&w)[32]) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.dp_full), gd & 1, wctx, kStatusTimeoutSoftmax));
                if (!ok) {
                    return;
                }
                tc_fence_after();
                uint32_t dp[32];
                [[maybe_unused]] const float* delta = sh.delta[gd % kXStages] + col0;
#pragma unroll
                for (int c4 = 0; c4 < 16; ++c4) {
                    if (c4 % 8 == 0) {
                        tmem_ld32(t_dp + 4 * c4, dp);
                        tmem_wait_ld();
                    }
                    float2 d[2];
                    if constexpr (Cfg::DKV) {
                        const float4 d4 = *reinterpret_cast<const float4*>(delta + 4 * c4);
                        d[0] = make_float2(d4.x, d4.y);
                        d[1] = make_float2(d4.z, d4.w);
                    } else {
                        d[0] = d[1] = make_float2(row_delta, row_delta);
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c = 4 * c4 + 2 * h;
                        const float2 y = __fmul2_rn(make_float2(u2f(p[c]), u2f(p[c + 1])), __fadd2_rn(make_float2(u2f(dp[c % 32]), u2f(dp[c % 32 + 1])), d[h]));
                        w[c / 2] = pack2<Cfg::BF16>(y.x, y.y);
                    }
                }
            };
            if constexpr (Cfg::DKV) {
                // Step i: P of tile i, dS of tile i - 1.
                uint32_t p_last[64];
                for (int i = 0; i <= it.n; ++i) {
                    uint32_t p[64], w[32];
                    if (i < it.n) {
                        probabilities(i, p);
                        ++g;
                    }
                    if (i > 0) {
                        gradients(p_last, w);
                        ++gd;
                        if constexpr (Cfg::kOverDP) {
                            // Every warp has dP in registers; its columns take dS and the next P. (Warps that
                            // gave up come here, too.)
                            asm volatile("bar.sync 1, 256;" ::: "memory");
                        }
                        if (ok) {
                            tmem_st32(t_ds, w);
                        }
                    }
                    if (i < it.n) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            w[c] = pack2<Cfg::BF16>(u2f(p[2 * c]), u2f(p[2 * c + 1]));
                        }
                        if (ok) {
                            tmem_st32(t_p, w);
                        }
#pragma unroll
                        for (int c = 0; c < 64; ++c) {
                            p_last[c] = p[c];
                        }
                    }
                    if (ok) {
                        tmem_wait_st();
                        arrive(&sh.ds_full);
                    }
                }
            } else {
                for (int i = 0; i < it.n; ++i, ++g, ++gd) {
                    uint32_t p[64], w[32];
                    probabilities(i, p);
                    gradients(p, w);
                    if (ok) {
                        tmem_st32(t_ds + (g % 2) * (Cfg::kTmemDS2 - Cfg::kTmemDS), w);
                        tmem_wait_st();
                        arrive(&sh.ds_full);
                    }
                }
            }

            // The item's sums: DKV: warpgroup 0 stores dV, 1 dK; dQ: a half of the columns each.
            ok = ok && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.acc_done), done & 1, wctx, kStatusTimeoutSoftmax));
            ++done;
            if (!ok) {
                continue;
            }
            tc_fence_after();
            constexpr int kCols = Cfg::DKV ? D : D / 2;
            const int out_col = Cfg::DKV ? 0 : wg * kCols;
            const uint32_t t_acc = tmem + lanes + ((Cfg::DKV && wg == 0) ? Cfg::kTmemAcc0 : Cfg::kTmemAcc1) + out_col;
            float factor = (Cfg::DKV && wg == 0) ? 1.0f : args.scale;
            if constexpr (!Cfg::BF16) {
                factor *= inverse_power(sh.power[(done - 1) % kPowers]);
            }
            const int rows = Cfg::DKV ? args.k_len : args.q_len;
            const bool first_out = Cfg::DKV && wg == 0;
            const int64_t* st = first_out ? args.out0_stride : args.out1_stride;
            uint16_t* dst = static_cast<uint16_t*>(first_out ? args.out0 : args.out1) + it.b * st[0] +
                            (Cfg::DKV ? it.kvh : it.head) * st[1] + static_cast<int64_t>(it.row0 + row) * st[2] + out_col;
            float4* part = reinterpret_cast<float4*>(args.parts) +
                           (Cfg::DKV ? (it.part * 2 + wg) * (D / 4) : it.part * (D / 4) + out_col / 4) * kTile + row;
#pragma unroll
            for (int c = 0; c < kCols / 32; ++c) {
                uint32_t x[32];
                tmem_ld32(t_acc + c * 32, x);
                tmem_wait_ld();
                if (c == kCols / 32 - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(smem_u32(&sh.acc_free));
                    }
                }
                if (it.part >= 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        part[(c * 8 + e) * kTile] = make_float4(u2f(x[4 * e]) * factor, u2f(x[4 * e + 1]) * factor,
                                                                u2f(x[4 * e + 2]) * factor, u2f(x[4 * e + 3]) * factor);
                    }
                } else if (it.row0 + row < rows) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t h[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            h[k] = pack2<Cfg::BF16>(u2f(x[8 * e + 2 * k]) * factor, u2f(x[8 * e + 2 * k + 1]) * factor);
                        }
                        *reinterpret_cast<uint4*>(dst + c * 32 + e * 8) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
            }
        }
    } else if (warp == kProducerWarp) {
        // ================================ TMA producer =================================
        if (lane == 0) {
            bool ok = true;
            int g = 0;      // streamed tiles so far
            int items = 0;  // resident pairs so far
            BwdItem it;
            while (ok && next_item<Cfg::DKV>(args, cursor, it)) {
                const int r_head = Cfg::DKV ? it.kvh : it.head;
                auto load = [&](uint32_t dst, const CUtensorMap* map, uint64_t* bar, int row, int head) {
                    mbar_arrive_expect_tx(smem_u32(bar), Cfg::kTileBytes);
#pragma unroll
                    for (int b = 0; b < Cfg::kBoxes; ++b) {
                        tma_load_4d(dst + b * kBox, map, smem_u32(bar), b * 64, row, head, it.b);
                    }
                };
                for (int i = 0; ok && i < it.n; ++i, ++g) {
                    int row, head;
                    stream_tile<Cfg>(args, it, i, row, head);
                    const int xs = g % kXStages;
                    const int ys = g % kYStages;
                    if (i == 0) {
                        // R0 is free after the item's last scores, R1 after its last dP.
                        ok = items == 0 ||
                             mbar_wait(smem_u32(&sh.r0_empty), (items - 1) & 1, wctx, kStatusTimeoutProducer);
                        if (ok) {
                            load(smem + Cfg::kSmemR0, &tm_r0, &sh.r0_full, it.row0, r_head);
                        }
                    }
                    ok = ok && mbar_wait(smem_u32(&sh.x_empty[xs]), ((g / kXStages) & 1) ^ 1, wctx, kStatusTimeoutProducer);
                    if (ok) {
                        load(smem + Cfg::kSmemX + xs * Cfg::kTileBytes, &tm_x, &sh.x_full[xs], row, head);
                    }
                    if (i == 0) {
                        ok = ok && (items == 0 ||
                                    mbar_wait(smem_u32(&sh.r1_empty), (items - 1) & 1, wctx, kStatusTimeoutProducer));
                        if (ok) {
                            load(smem + Cfg::kSmemR1, &tm_r1, &sh.r1_full, it.row0, r_head);
                            ++items;
                        }
                    }
                    ok = ok && mbar_wait(smem_u32(&sh.y_empty[ys]), ((g / kYStages) & 1) ^ 1, wctx, kStatusTimeoutProducer);
                    if (ok) {
                        load(smem + Cfg::kSmemY + ys * Cfg::kTileBytes, &tm_y, &sh.y_full[ys], row, head);
                    }
                }
            }
            if (!ok) {
                // Copies in flight end by themselves within microseconds; give them that long before
                // the CTA's shared memory is released.
                const unsigned long long t0 = globaltimer_ns();
                while (globaltimer_ns() - t0 < 1000000ull) {
                }
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // =============================== MMA issuers ===================================
        // The whole warp walks in step, one elected lane issues. This one: dP and the sums.
        bool ok = true;
        int g = 0;
        int items = 0;
        const uint64_t r1 = make_desc_kmajor_sw128(smem + Cfg::kSmemR1);
        const uint64_t xn = make_desc_mnmajor_sw128(smem + Cfg::kSmemX, kBox);
        const uint64_t yk = make_desc_kmajor_sw128(smem + Cfg::kSmemY);
        const uint64_t yn = make_desc_mnmajor_sw128(smem + Cfg::kSmemY, kBox);
        auto off = [](int stage) { return static_cast<uint64_t>(stage * (Cfg::kTileBytes >> 4)); };
        auto wait = [&](uint64_t* bar, int parity) {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity & 1, wctx, kStatusTimeoutMma)) != 0;
        };
        auto dscores = [&](int at, bool last) {  // dP, the last use of Y
            const uint64_t y = yk + off(at % kYStages);
            if (elect_one()) {
                issue_scores<Cfg>(tmem + Cfg::kTmemDP, r1, y);
                umma_commit(smem_u32(&sh.dp_full));
                umma_commit(smem_u32(&sh.y_empty[at % kYStages]));
                if (last) {
                    umma_commit(smem_u32(&sh.r1_empty));
                }
            }
            __syncwarp();
        };
        auto dproduct = [&](int at, bool first, bool last) {  // dK or dQ, the last use of X
            const uint64_t x = xn + off(at % kXStages);
            const uint32_t ds = tmem + ((at & 1) ? Cfg::kTmemDS2 : Cfg::kTmemDS);
            if (elect_one()) {
                issue_product<Cfg>(tmem + Cfg::kTmemAcc1, ds, x, first);
                umma_commit(smem_u32(&sh.x_empty[at % kXStages]));
                if (last) {
                    umma_commit(smem_u32(&sh.acc_done));
                }
            }
            __syncwarp();
        };
        int steps = 0;  // completions of ds_full so far
        BwdItem it;
        while (ok && next_item<Cfg::DKV>(args, cursor, it)) {
            const int n = it.n;
            ok = wait(&sh.r1_full, items);
            if (!Cfg::DKV) {
                ok = ok && wait(&sh.y_full[g % kYStages], g / kYStages);
                if (ok) {
                    tc_fence_after();
                    dscores(g, n == 1);
                }
            }
            for (int i = 0; ok && i < (Cfg::DKV ? n + 1 : n); ++i) {
                const int at = g + i;
                const int y_next = Cfg::DKV ? i : i + 1;  // the tile whose dP comes now
                if (y_next < n) {
                    ok = wait(&sh.y_full[(g + y_next) % kYStages], (g + y_next) / kYStages);
                }
                if (ok && i == 0 && items > 0) {
                    ok = wait(&sh.acc_free, items - 1);  // the item before has left the accumulators
                }
                ok = ok && wait(&sh.ds_full, steps++);
                if (!ok) {
                    break;
                }
                tc_fence_after();
                if constexpr (Cfg::DKV) {
                    if (i < n) {
                        const uint64_t y = yn + off(at % kYStages);
                        if (elect_one()) {
                            issue_product<Cfg>(tmem + Cfg::kTmemAcc0, tmem + Cfg::kTmemP, y, i == 0);
                        }
                        __syncwarp();
                    }
                    if (i > 0) {
                        dproduct(at - 1, i == 1, i == n);
                    }
                    if (i < n) {
                        dscores(at, i + 1 == n);
                    }
                } else {
                    if (i + 1 < n) {
                        dscores(at + 1, i + 2 == n);
                    }
                    dproduct(at, i == 0, i + 1 == n);
                }
            }
            g += n;
            ++items;
        }
        // Every MMA issued must be complete before tensor memory is released.
        if (elect_one()) {
            umma_commit(smem_u32(&sh.mma_idle));
        }
        __syncwarp();
        mbar_wait_drain(smem_u32(&sh.mma_idle), 0, wctx, kStatusTimeoutTeardown);
        __syncwarp();
    } else if (warp == kScoreWarp) {
        // S of every streamed tile, as soon as the one before is in registers. In a warp of its own, since issuing
        // holds a warp until the tensor pipe takes its products.
        bool ok = true;
        int g = 0;
        int items = 0;
        const uint64_t r0 = make_desc_kmajor_sw128(smem + Cfg::kSmemR0);
        const uint64_t xk = make_desc_kmajor_sw128(smem + Cfg::kSmemX);
        auto wait = [&](uint64_t* bar, int parity) {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity & 1, wctx, kStatusTimeoutMma)) != 0;
        };
        BwdItem it;
        while (ok && next_item<Cfg::DKV>(args, cursor, it)) {
            ok = wait(&sh.r0_full, items);
            for (int i = 0; ok && i < it.n; ++i, ++g) {
                ok = wait(&sh.x_full[g % kXStages], g / kXStages) &&
                     (g == 0 || wait(&sh.s_read[(g - 1) % 2], (g - 1) / 2));
                if (!ok) {
                    break;
                }
                tc_fence_after();
                const uint64_t x = xk + static_cast<uint64_t>((g % kXStages) * (Cfg::kTileBytes >> 4));
                const bool last = i + 1 == it.n;
                if (elect_one()) {
                    issue_scores<Cfg>(tmem + Cfg::kTmemS, r0, x);
                    umma_commit(smem_u32(&sh.s_full));
                    if (last) {
                        umma_commit(smem_u32(&sh.r0_empty));
                    }
                }
                __syncwarp();
            }
            ++items;
        }
        if (elect_one()) {
            umma_commit(smem_u32(&sh.mma_idle));
        }
        __syncwarp();
        mbar_wait_drain(smem_u32(&sh.mma_idle), 0, wctx, kStatusTimeoutTeardown);
        __syncwarp();
    } else if (Cfg::kLoads && warp == kLoaderWarp) {
        // ========== LSE and delta of the streamed query rows (DKV), the items' powers (float16) ==========
        bool ok = true;
        int g = 0;
        int items = 0;
        [[maybe_unused]] float power = 1.0f;  // of kv head `power_of`
        [[maybe_unused]] int power_of = -1;
        BwdItem it;
        while (ok && next_item<Cfg::DKV>(args, cursor, it)) {
            if (!Cfg::BF16 && it.b * args.kv_heads + it.kvh != power_of) {
                power_of = it.b * args.kv_heads + it.kvh;
                power = head_power(args, it.b, it.kvh);
            }
            for (int i = 0; ok && i < it.n; ++i, ++g) {
                [[maybe_unused]] float lse[4], delta[4];
                if constexpr (Cfg::DKV) {
                    int row, head;
                    stream_tile<Cfg>(args, it, i, row, head);
                    const long long base = (static_cast<long long>(it.b) * args.heads + head) * args.q_len;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = row + k * 32 + lane;
                        lse[k] = r < args.q_len ? __ldg(args.lse + base + r) : -INFINITY;
                        delta[k] = r < args.q_len ? __ldg(args.delta + base + r) : 0.0f;
                    }
                }
                // LSE has two slots, free when tile g - 2 has been read; delta three, like X.
                ok = mbar_wait(smem_u32(&sh.x_empty[g % kXStages]), ((g / kXStages) & 1) ^ 1, wctx, kStatusTimeoutProducer);
                if (Cfg::DKV && g >= 2) {
                    ok = ok && mbar_wait(smem_u32(&sh.s_read[g % 2]), ((g - 2) / 2) & 1, wctx, kStatusTimeoutProducer);
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) {
                    break;
                }
                if constexpr (Cfg::DKV) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        // A row whose LSE is NaN (a NaN score) makes P NaN: in the columns of the software 2^x, +inf does.
                        const float x = lse[k] * -1.4426950408889634f + (Cfg::BF16 ? 0.0f : exponent(power));
                        const float nan = emulated(lane) ? INFINITY : x;
                        sh.lse2[g % 2][k * 32 + lane] = lse[k] == -INFINITY ? -INFINITY : (x != x ? nan : x);
                        sh.delta[g % kXStages][k * 32 + lane] = -delta[k];
                    }
                }
                if (!Cfg::BF16 && i == 0 && lane == 0) {
                    sh.power[items % kPowers] = power;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&sh.x_full[g % kXStages]));
                }
            }
            ++items;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
    if constexpr (!Cfg::DKV) {
        // The dQ pass needs delta, which was complete before any of its CTAs could start, and nothing of the
        // dK, dV pass beside it; but its own end stands for both.
        cudaGridDependencySynchronize();
    }
}

// delta[row] = dO.O, a row by D / 8 lanes, kDeltaRows rows a thread of head blockIdx.y. Bound by DRAM bytes. float16:
// also what bounds dS, the largest |dO| of the block's rows, and |V| (blockIdx.z = 1).
template <int D, bool BF16>
__global__ void __launch_bounds__(kDeltaThreads) delta_kernel(const __grid_constant__ FaWindowParams p, float* delta, float* do_size,
                                                              float* v_size, int q_slots, int k_slots) {
    constexpr int C = D / 8;
    constexpr int kGroups = kDeltaThreads / C;
    const bool values = !BF16 && blockIdx.z != 0;
    const int heads = values ? p.kv_heads : p.heads;
    const int len = values ? p.k_len : p.q_len;
    const int chunk = static_cast<int>(threadIdx.x) % C;
    const int bh = static_cast<int>(blockIdx.y);
    const int b = bh / heads;
    const int h = bh - b * heads;
    if (!BF16 && (b >= p.batch || static_cast<int>(blockIdx.x) >= (values ? k_slots : q_slots))) {
        return;
    }
    const int64_t* d_st = values ? p.v_stride : p.do_stride;
    const uint16_t* o_head = static_cast<const uint16_t*>(p.o) + b * p.o_stride[0] + h * p.o_stride[1] + chunk * 8;
    const uint16_t* d_head = static_cast<const uint16_t*>(values ? p.v : p.d_o) + b * d_st[0] + h * d_st[1] + chunk * 8;
    const int row0 = static_cast<int>(blockIdx.x) * kSlotRows<D> + static_cast<int>(threadIdx.x) / C;
    uint4 o[kDeltaRows], d[kDeltaRows];
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i) {
        const int64_t row = row0 + i * kGroups;
        o[i] = d[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < len) {
            if (!values) {
                o[i] = __ldg(reinterpret_cast<const uint4*>(o_head + row * p.o_stride[2]));
            }
            d[i] = __ldg(reinterpret_cast<const uint4*>(d_head + row * d_st[2]));
        }
    }
    [[maybe_unused]] float most = 0.0f;
#pragma unroll
    for (int i = 0; i < kDeltaRows; ++i) {
        const uint32_t ow[4] = {o[i].x, o[i].y, o[i].z, o[i].w};
        const uint32_t dw[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
        float sum = 0.0f;
        [[maybe_unused]] float square = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (BF16) {
                sum = fmaf(u2f(ow[k] << 16), u2f(dw[k] << 16), sum);
                sum = fmaf(u2f(ow[k] & 0xFFFF0000u), u2f(dw[k] & 0xFFFF0000u), sum);
            } else {
                const float2 x = unpack_half2(ow[k]);
                const float2 y = unpack_half2(dw[k]);
                sum = fmaf(x.x, y.x, sum);
                sum = fmaf(x.y, y.y, sum);
                square = fmaf(y.x, y.x, square);
                square = fmaf(y.y, y.y, square);
            }
        }
#pragma unroll
        for (int k = C / 2; k > 0; k >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, k);
            if constexpr (!BF16) {
                square += __shfl_xor_sync(0xffffffffu, square, k);
            }
        }
        const int row = row0 + i * kGroups;
        if (!values && row < len && chunk == 0) {
            delta[static_cast<long long>(bh) * len + row] = sum;
        }
        if constexpr (!BF16) {
            most = fmaxf(most, square);
        }
    }
    if constexpr (!BF16) {
        __shared__ float all[kDeltaThreads / 32];
        most = warp_max(most);
        if (threadIdx.x % 32 == 0) {
            all[threadIdx.x / 32] = most;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kDeltaThreads / 32; ++w) {
                most = fmaxf(most, all[w]);
            }
            (values ? v_size + static_cast<long long>(bh) * k_slots : do_size + static_cast<long long>(bh) * q_slots)[blockIdx.x] = sqrtf(most);
        }
    }
}

// Adds up the parts of the list that is cut at the end of CTA `boundary`'s range (of the dK, dV pass, then
// of the dQ pass), if that is its first cut; a quarter of the dims of dV (which 0), dK or dQ (1). Lanes take 8 rows x 4 groups of 4 dims: 128-byte reads, 32-byte writes.
constexpr int kJoinThreads = 256;

template <int D, bool BF16, bool DKV>
__device__ __forceinline__ void join(const BwdArgs& a, int boundary, int which, int quarter) {
    __shared__ long long warp_sum[kJoinThreads / 32];
    __shared__ int tile, offset;
    const long long cut = (boundary + 1) * a.per;
    const int bx = static_cast<int>(cut / a.head_steps);
    locate_tile<DKV, kJoinThreads>(a, cut - bx * a.head_steps, warp_sum, &tile, &offset);
    __syncthreads();
    const long long begin = cut - offset;
    if (offset == 0 || begin / a.per != boundary) {
        return;
    }
    BwdItem it;
    tile_list<DKV>(a, tile, it);
    const long long last = (begin + it.total - 1) / a.per;
    const int b = a.div_heads.div(bx);
    const int h = bx - b * static_cast<int>(a.div_heads.d);
    const bool first_out = DKV && which == 0;
    const int64_t* st = first_out ? a.out0_stride : a.out1_stride;
    uint16_t* dst = static_cast<uint16_t*>(first_out ? a.out0 : a.out1) + b * st[0] + h * st[1];
    const int rows = DKV ? a.k_len : a.q_len;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    constexpr int kOutputs = DKV ? 2 : 1;
    // All of a thread's pieces of a part are on their way at once.
    constexpr int kPieces = (D / 64) * (kTile / 8) / (kJoinThreads / 32);
    float4 sum[kPieces];
    int at[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int u = static_cast<int>(threadIdx.x) / 32 + i * (kJoinThreads / 32);
        const int row = u / (D / 64) * 8 + lane % 8;
        const int four = quarter * (D / 16) + u % (D / 64) * 4 + lane / 8;
        at[i] = four * kTile + row;
        sum[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (long long c = boundary; c <= last; ++c) {
        // The list is its first CTA's last part unless it starts that CTA's range; else a first part.
        const long long record = 2 * c + (c * a.per >= begin ? 0 : 1);
        const float4* src = reinterpret_cast<const float4*>(a.parts) + (record * kOutputs + (DKV ? which : 0)) * (D / 4) * kTile;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const float4 x = __ldcg(src + at[i]);
            sum[i].x += x.x;
            sum[i].y += x.y;
            sum[i].z += x.z;
            sum[i].w += x.w;
        }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int row = at[i] % kTile;
        if (it.row0 + row < rows) {
            *reinterpret_cast<uint2*>(dst + static_cast<int64_t>(it.row0 + row) * st[2] + at[i] / kTile * 4) =
                make_uint2(pack2<BF16>(sum[i].x, sum[i].y), pack2<BF16>(sum[i].z, sum[i].w));
        }
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kJoinThreads) window_bwd_join_kernel(const __grid_constant__ BwdArgs dkv,
                                                                       const __grid_constant__ BwdArgs dq) {
    cudaGridDependencySynchronize();
    const int quarter = static_cast<int>(blockIdx.x) % 4;
    const int unit = static_cast<int>(blockIdx.x) / 4;
    const int dkv_units = 2 * (dkv.grid - 1);
    if (unit < dkv_units) {
        join<D, BF16, true>(dkv, unit / 2, unit % 2, quarter);
    } else {
        join<D, BF16, false>(dq, unit - dkv_units, 1, quarter);
    }
}

constexpr int kMinSteps = 4;  // least streamed tiles of a CTA's range

// The sizes of a pass, and its cut into ranges.
template <bool DKV>
BwdArgs bwd_args(const FaWindowParams& p, int sm_count) {
    BwdArgs a{};
    a.batch = p.batch;
    a.heads = p.heads;
    a.kv_heads = p.kv_heads;
    a.group = p.heads / p.kv_heads;
    a.q_len = p.q_len;
    a.k_len = p.k_len;
    a.shift = p.k_len - p.q_len;
    a.window = p.window == 0 ? kNoWindow : std::min(p.window, kNoWindow);
    a.sinks = std::min(p.sinks, p.k_len);
    a.tiles = ((DKV ? p.k_len : p.q_len) + kTile - 1) / kTile;
    for (int t = 0; t < a.tiles; ++t) {
        BwdItem it;
        tile_list<DKV>(a, t, it);
        a.head_steps += it.total;
    }
    a.steps = a.head_steps * p.batch * (DKV ? p.kv_heads : p.heads);
    a.per = std::max<long long>(kMinSteps, (a.steps + sm_count - 1) / sm_count);
    a.grid = static_cast<int>((a.steps + a.per - 1) / a.per);
    a.scale = p.softmax_scale;
    a.scale_log2 = static_cast<float>(static_cast<double>(p.softmax_scale) * M_LOG2E);
    a.div_heads = FastDiv(DKV ? p.kv_heads : p.heads);
    a.div_group = FastDiv(a.group);
    return a;
}

template <bool DKV>
unsigned long long part_bytes(const BwdArgs& a, int head_dim) {
    return a.grid > 1 ? 2ull * a.grid * (DKV ? 2 : 1) * kTile * head_dim * 4 : 0;
}

// Where the row statistics lie in the workspace.
struct Statistics {
    int q_slots, k_slots;
    unsigned long long do_size, v_size, bytes;  // delta is first
};

Statistics statistics_of(const FaWindowParams& p) {
    const auto up = [](unsigned long long n) { return (n + 255) / 256 * 256; };
    const int slot_rows = p.head_dim == 64 ? kSlotRows<64> : kSlotRows<128>;
    Statistics s{};
    s.bytes = up(4ull * p.batch * p.heads * p.q_len);
    if (p.dtype == FA_DTYPE_FLOAT16) {
        s.q_slots = (p.q_len + slot_rows - 1) / slot_rows;
        s.k_slots = (p.k_len + slot_rows - 1) / slot_rows;
        s.do_size = s.bytes;
        s.v_size = s.do_size + up(4ull * p.batch * p.heads * s.q_slots);
        s.bytes = s.v_size + up(4ull * p.batch * p.kv_heads * s.k_slots);
    }
    return s;
}

// Launches after the kernel before it has started to end: it waits for its results itself.
template <class Kernel, class... Args>
cudaError_t launch_early(Kernel kernel, dim3 grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

template <int D, bool BF16>
cudaError_t bwd(const FaWindowParams& p, DeviceStatus* status, unsigned epoch, void* workspace, int sm_count,
                cudaStream_t stream) {
    BwdArgs dkv = bwd_args<true>(p, sm_count);
    BwdArgs dq = bwd_args<false>(p, sm_count);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    float* delta = static_cast<float*>(workspace);
    dkv.epoch = dq.epoch = epoch;
    dkv.status = dq.status = status;
    dkv.lse = dq.lse = p.lse;
    dkv.delta = dq.delta = delta;
    const Statistics st = statistics_of(p);
    float* do_size = reinterpret_cast<float*>(ws + st.do_size);
    float* v_size = reinterpret_cast<float*>(ws + st.v_size);
    dkv.do_size = dq.do_size = do_size;
    dkv.v_size = dq.v_size = v_size;
    dkv.q_slots = dq.q_slots = st.q_slots;
    dkv.k_slots = dq.k_slots = st.k_slots;
    dkv.parts = reinterpret_cast<float*>(ws + st.bytes);
    dq.parts = reinterpret_cast<float*>(ws + st.bytes + part_bytes<true>(dkv, D));
    dkv.out0 = p.dv;
    dkv.out1 = p.dk;
    dq.out1 = p.dq;
    auto strides = [](int64_t(&to)[3], const int64_t(&from)[3]) { std::copy(from, from + 3, to); };
    strides(dkv.out0_stride, p.dv_stride);
    strides(dkv.out1_stride, p.dk_stride);
    strides(dq.out1_stride, p.dq_stride);
    const int delta_blocks = BF16 ? (p.q_len + kSlotRows<D> - 1) / kSlotRows<D> : std::max(st.q_slots, st.k_slots);
    const dim3 delta_grid(static_cast<unsigned>(delta_blocks), static_cast<unsigned>(p.batch * p.heads), BF16 ? 1 : 2);
    CUtensorMap q, k, v, d_o;
    if (encode_strided_map(&q, p.q, p.q_stride, p.batch, p.heads, p.q_len, D, kTile, BF16) != CUDA_SUCCESS ||
        encode_strided_map(&k, p.k, p.k_stride, p.batch, p.kv_heads, p.k_len, D, kTile, BF16) != CUDA_SUCCESS ||
        encode_strided_map(&v, p.v, p.v_stride, p.batch, p.kv_heads, p.k_len, D, kTile, BF16) != CUDA_SUCCESS ||
        encode_strided_map(&d_o, p.d_o, p.do_stride, p.batch, p.heads, p.q_len, D, kTile, BF16) != CUDA_SUCCESS) {
        return cudaErrorInvalidValue;
    }
    using Dkv = BwdCfg<D, BF16, true>;
    using Dq = BwdCfg<D, BF16, false>;
    cudaError_t err = ensure_smem_limit<window_bwd_kernel<Dkv>>(bwd_smem<Dkv>());
    if (err == cudaSuccess) {
        err = ensure_smem_limit<window_bwd_kernel<Dq>>(bwd_smem<Dq>());
    }
    if (err != cudaSuccess) {
        return err;
    }
    delta_kernel<D, BF16><<<delta_grid, kDeltaThreads, 0, stream>>>(p, delta, do_size, v_size, st.q_slots, st.k_slots);
    err = cudaGetLastError();
    if (err != cudaSuccess) {
        return err;
    }
    err = launch_early(window_bwd_kernel<Dkv>, dim3(static_cast<unsigned>(dkv.grid)), kBwdThreads, bwd_smem<Dkv>(),
                       stream, k, v, q, d_o, dkv);
    if (err == cudaSuccess) {
        err = launch_early(window_bwd_kernel<Dq>, dim3(static_cast<unsigned>(dq.grid)), kBwdThreads, bwd_smem<Dq>(),
                           stream, q, d_o, k, v, dq);
    }
    const int units = 2 * (dkv.grid - 1) + dq.grid - 1;  // outputs of lists that may be cut
    if (err == cudaSuccess && units > 0) {
        err = launch_early(window_bwd_join_kernel<D, BF16>, dim3(static_cast<unsigned>(4 * units)), kJoinThreads, 0, stream,
                           dkv, dq);
    }
    return err;
}

}  // namespace

unsigned long long window_bwd_workspace_bytes(const FaWindowParams& p, int sm_count) {
    return statistics_of(p).bytes + part_bytes<true>(bwd_args<true>(p, sm_count), p.head_dim) +
           part_bytes<false>(bwd_args<false>(p, sm_count), p.head_dim);
}

cudaError_t launch_window_bwd(const FaWindowParams& p, DeviceStatus* status, unsigned epoch, void* workspace,
                              int sm_count, cudaStream_t stream) {
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.head_dim == 64) {
        return bf16 ? bwd<64, true>(p, status, epoch, workspace, sm_count, stream)
                    : bwd<64, false>(p, status, epoch, workspace, sm_count, stream);
    }
    return bf16 ? bwd<128, true>(p, status, epoch, workspace, sm_count, stream)
                : bwd<128, false>(p, status, epoch, workspace, sm_count, stream);
}

}  // namespace fa_sm100
