// Appending to the paged cache: new queries and keys are rotated by their positions, keys and
// values stored into the pages of their sequences, 16-bit or e4m3 with a scale for every page
// and head.
//
// Rotation of a pair at position p with angle a_i(p) (tables of cos and sin):
//   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin)
// in fp32 with every product rounded (no contraction), so that the stored codes do not depend on
// how a compiler fuses them, and rounded once: to the tensors' type, or to e4m3.
//
// The e4m3 scale is 2^k with the smallest k >= -60 for which the block's largest finite value is
// at most 448 * 2^k. e4m3 is a floating format, so a power of two costs no precision against
// amax / 448, and growing the scale of a page that already holds tokens multiplies their codes by
// a power of two: exact but for codes that become subnormal.
//
// Work split: a CTA per (sequence, page touched, kv head, K or V), so that a scale has one owner
// and no atomics, alternating with CTAs for the rows of q, whose threads keep one token's angles over the heads.
// A row is D / 8 lanes of 16 bytes, at most 4 rows a thread, kept in registers between the block's maximum
// and the store: one pass over the data. Measured, 32 query heads, 8 kv heads, D 128, bf16 to e4m3 pages of
// 64: 10875 tokens of 4 prompts 58 us (4.3 TB/s; bound by the latency of a page's loads, maximum and store at
// 32 warps an SM), a decode step of 128 sequences 3.9 us (one launch's latency).

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

constexpr int kRowsPerThread = 4;
constexpr int kMaxThreads = 1024;  // a page of 256 tokens x 128 dims; leaves 64 registers a thread

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 f = unpack_half2(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]),
                      pack2<BF16>(x[6], x[7]));
}

// How pairs are turned.
enum : int { kNoTurn = 0, kHalves = 1, kInterleaved = 2 };

// cos and sin of the 8 dims of `chunk` (dims 8 chunk ...) at a position: one value a dim with
// halves (sin negated in the first), one a pair (4 of the 8) when interleaved.
struct Angles {
    float c[8], s[8];
};

template <int TURN>
__device__ __forceinline__ void load_angles(Angles& a, int chunk, int pos, bool live, const FaAppendParams& p) {
    const int half = p.rotary_dim / 2;
    const int hc = half / 8;  // chunks of a half
    const bool first = TURN == kInterleaved || chunk < hc;
    const long long at = static_cast<long long>(pos) * half +
                         (TURN == kInterleaved ? chunk * 4 : (first ? chunk : chunk - hc) * 8);
    const uint32_t sign = TURN == kHalves && first ? 0x80000000u : 0u;
#pragma unroll
    for (int q = 0; q < (TURN == kInterleaved ? 1 : 2); ++q) {
        float4 c = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (live && chunk < 2 * hc) {
            c = __ldg(reinterpret_cast<const float4*>(p.cos + at + 4 * q));
            s = __ldg(reinterpret_cast<const float4*>(p.sin + at + 4 * q));
        }
        a.c[4 * q] = c.x;
        a.c[4 * q + 1] = c.y;
        a.c[4 * q + 2] = c.z;
        a.c[4 * q + 3] = c.w;
        a.s[4 * q] = __uint_as_float(__float_as_uint(s.x) ^ sign);
        a.s[4 * q + 1] = __uint_as_float(__float_as_uint(s.y) ^ sign);
        a.s[4 * q + 2] = __uint_as_float(__float_as_uint(s.z) ^ sign);
        a.s[4 * q + 3] = __uint_as_float(__float_as_uint(s.w) ^ sign);
    }
}

// Rotates the 8 dims of `chunk` of a row (16-bit in `raw`, widened to x). The lanes of a row are
// consecutive; with halves a lane's partner dims are in the lane rotary / 16 chunks away, so whole
// warps call. Dims beyond rotary_dim stay as they are.
template <int TURN, bool BF16>
__device__ __forceinline__ void rotate8(float (&x)[8], const uint4& raw, const Angles& a, int chunk, int hc) {
    const bool turns = chunk < 2 * hc;
    if constexpr (TURN == kInterleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float u = x[2 * i];
            const float v = x[2 * i + 1];
            x[2 * i] = turns ? __fsub_rn(__fmul_rn(u, a.c[i]), __fmul_rn(v, a.s[i])) : u;
            x[2 * i + 1] = turns ? __fadd_rn(__fmul_rn(v, a.c[i]), __fmul_rn(u, a.s[i])) : v;
        }
    } else {
        const int lane = static_cast<int>(threadIdx.x) & 31;
        const int src = (chunk < hc ? lane + hc : lane - hc) & 31;
        uint4 other;
        other.x = __shfl_sync(0xffffffffu, raw.x, src);
        other.y = __shfl_sync(0xffffffffu, raw.y, src);
        other.z = __shfl_sync(0xffffffffu, raw.z, src);
        other.w = __shfl_sync(0xffffffffu, raw.w, src);
        float y[8];
        unpack8<BF16>(other, y);
        if (turns) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // The first half's sines are negated: x1 c + x2 (-s) is x1 c - x2 s, to the bit. (The
                // paired forms of these two are contracted to one rounding, so they stay scalar.)
                x[i] = __fadd_rn(__fmul_rn(x[i], a.c[i]), __fmul_rn(y[i], a.s[i]));
            }
        }
    }
}

// 2^k, the smallest k >= -60 with amax <= 448 * 2^k (448 = 1.75 * 2^8).
__device__ __forceinline__ float block_scale(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = static_cast<int>(bits >> 23) - 127;  // amax = 1.f * 2^e
    const int k = max(((bits & 0x7FFFFFu) <= 0x600000u) ? e - 8 : e - 7, -60);
    return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

template <int D, bool BF16, bool E4M3, int TURN>
__device__ __forceinline__ void store_page(const FaAppendParams& p, DeviceStatus* status, int unit, bool is_v,
                                           int spans, int log2_page) {
    constexpr int C = D / 8;  // lanes of a row
    const FaCache& c = p.cache;
    const int h = unit % c.kv_heads;
    unit /= c.kv_heads;
    const int span = unit % spans;
    const int b = unit / spans;
    const int len = max(c.lengths[b], 0);
    const int count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
    const int start = len - count;
    const int page = (max(start, 0) >> log2_page) + span;
    const int base = static_cast<int>(static_cast<unsigned>(page) << log2_page);  // negative: a page beyond 2^31 tokens
    const int lo = max(start, base);
    int hi = base < 0 ? 0 : (len - base > c.page_size ? base + c.page_size : len);
    const bool leader = threadIdx.x == 0 && h == 0 && !is_v;
    if (leader && span == 0 && start < 0 && count > 0) {
        atomicOr(&status->code, kStatusBadPage);
    }
    if (lo >= hi) {
        return;
    }
    int id = -1;
    if (page < c.max_pages) {
        id = c.page_table[b * c.table_stride + page];
    }
    const bool short_table = p.cos != nullptr && hi > p.table_rows;
    if (id < 0 || id >= c.num_pages || short_table) {
        if (leader) {
            atomicOr(&status->code, kStatusBadPage);
        }
        hi = short_table ? min(hi, p.table_rows) : hi;
        if (id < 0 || id >= c.num_pages || lo >= hi) {
            return;
        }
    }

    const int chunk = static_cast<int>(threadIdx.x) % C;
    const int group = static_cast<int>(threadIdx.x) / C;
    const int groups = static_cast<int>(blockDim.x) / C;
    const int64_t* st = is_v ? p.v_new_stride : p.k_new_stride;
    const uint16_t* src = static_cast<const uint16_t*>(is_v ? p.v_new : p.k_new) + b * st[0] + h * st[1] + chunk * 8;
    const int hc = p.rotary_dim / 16;
    const int rows = hi - lo;

    uint4 raw[kRowsPerThread];
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        const int r = i * groups + group;
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows) {
            raw[i] = __ldg(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(lo + r - start) * st[2]));
        }
    }
    float x[kRowsPerThread][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        if (i * groups < rows) {
            const int r = i * groups + group;
            unpack8<BF16>(raw[i], x[i]);
            if constexpr (TURN != kNoTurn) {
                Angles a;
                load_angles<TURN>(a, chunk, lo + r, r < rows, p);
                rotate8<TURN, BF16>(x[i], raw[i], a, chunk, hc);
            }
            if constexpr (E4M3) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    amax = fmaxf(amax, fabsf(x[i][e]));  // NaN passes by
                }
            }
        }
    }
    if (E4M3 && amax > FLT_MAX) {  // infinities do not count either
        amax = 0.0f;
        for (int i = 0; i < kRowsPerThread && i * groups < rows; ++i) {
            for (int e = 0; e < 8; ++e) {
                const float v = fabsf(x[i][e]);
                amax = fmaxf(amax, v <= FLT_MAX ? v : 0.0f);
            }
        }
    }
    const int64_t* ps = is_v ? c.v_stride : c.k_stride;
    const int64_t slot0 = id * ps[0] + h * ps[1] + chunk * 8;
    const int in_page = lo - base;  // tokens the page held before
    if constexpr (!E4M3) {
        uint16_t* dst = static_cast<uint16_t*>(is_v ? c.v : c.k) + slot0;
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int r = i * groups + group;
            if (r < rows) {
                *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(in_page + r) * D) = pack8<BF16>(x[i]);
            }
        }
    } else {
        __shared__ float warp_max[kMaxThreads / 32];
        float* scale = (is_v ? c.v_scale : c.k_scale) + static_cast<int64_t>(id) * c.kv_heads + h;
        const float before = in_page > 0 ? *scale : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        }
        if (threadIdx.x % 32 == 0) {
            warp_max[threadIdx.x / 32] = amax;
        }
        __syncthreads();  // every thread has read `before`, too
        for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) {
            amax = fmaxf(amax, warp_max[w]);
        }
        const float s = fmaxf(block_scale(amax), before);
        if (threadIdx.x == 0) {
            *scale = s;
        }
        // s is a power of two unless a caller brought other scales: then the quotient is divided.
        const bool pow2 = (__float_as_uint(s) & 0x7FFFFFu) == 0;
        const float inv = 1.0f / s;
        uint8_t* dst = static_cast<uint8_t*>(is_v ? c.v : c.k) + slot0;
        if (in_page > 0 && s > before) {
            const float ratio = before / s;
            for (int r = group; r < in_page; r += groups) {
                uint2* at = reinterpret_cast<uint2*>(dst + static_cast<int64_t>(r) * D);
                uint2 w = *at;
                uint32_t v[2] = {w.x, w.y};
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float2 a = unpack_half2(e4m3x2_to_half2(v[q] & 0xFFFFu));
                    const float2 d = unpack_half2(e4m3x2_to_half2(v[q] >> 16));
                    v[q] = pack_e4m3x2(a.x * ratio, a.y * ratio) | (pack_e4m3x2(d.x * ratio, d.y * ratio) << 16);
                }
                *at = make_uint2(v[0], v[1]);
            }
        }
        auto store = [&](auto quotient) {
#pragma unroll
            for (int i = 0; i < kRowsPerThread; ++i) {
                const int r = i * groups + group;
                if (r < rows) {
                    uint32_t w[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        w[q] = pack_e4m3x2(quotient(x[i][4 * q]), quotient(x[i][4 * q + 1])) |
                               (pack_e4m3x2(quotient(x[i][4 * q + 2]), quotient(x[i][4 * q + 3])) << 16);
                    }
                    *reinterpret_cast<uint2*>(dst + static_cast<int64_t>(in_page + r) * D) = make_uint2(w[0], w[1]);
                }
            }
        };
        if (pow2) {
            store([&](float v) { return v * inv; });
        } else {
            store([&](float v) { return __fdiv_rn(v, s); });
        }
    }
}

// How the rows of q go over the threads: a CTA has `tokens` tokens (a power of two) of as many
// heads at a time as its rows allow, and takes `heads` of them in turn, so that a thread stays
// with one token and reads its angles once.
struct QuerySplit {
    int log2_tokens, heads, token_blocks, head_blocks;
};

template <int D, bool BF16, int TURN>
__device__ __forceinline__ void rotate_queries(const FaAppendParams& p, DeviceStatus* status, int block,
                                               const QuerySplit& split) {
    constexpr int C = D / 8;
    constexpr int kAtOnce = 4;  // loads in flight of a thread
    const FaCache& c = p.cache;
    const int chunk = static_cast<int>(threadIdx.x) % C;
    const int row = static_cast<int>(threadIdx.x) / C;
    const int head_step = (static_cast<int>(blockDim.x) / C) >> split.log2_tokens;
    const int hb = block % split.head_blocks;
    const int tb = block / split.head_blocks % split.token_blocks;
    const int b = block / split.head_blocks / split.token_blocks;
    const int t = (tb << split.log2_tokens) + (row & ((1 << split.log2_tokens) - 1));
    const int h_end = min((hb + 1) * split.heads, p.heads);
    const int h0 = hb * split.heads + (row >> split.log2_tokens);
    const int count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
    const int pos = max(c.lengths[b], 0) - count + t;
    const bool mine = t < c.tokens;
    bool live = t < count;
    if (live && (pos < 0 || (p.cos != nullptr && pos >= p.table_rows))) {
        live = false;
        atomicOr(&status->code, kStatusBadPage);
    }
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] + t * p.q_stride[2] + chunk * 8;
    uint16_t* dst = static_cast<uint16_t*>(p.q_out) + (static_cast<int64_t>(b) * p.heads * c.tokens + t) * D + chunk * 8;
    const int64_t src_step = p.q_stride[1] * head_step;
    const int64_t dst_step = static_cast<int64_t>(head_step) * c.tokens * D;
    const int hc = p.rotary_dim / 16;
    src += h0 * p.q_stride[1];
    dst += static_cast<int64_t>(h0) * c.tokens * D;
    Angles a;
    if constexpr (TURN != kNoTurn) {
        load_angles<TURN>(a, chunk, pos, live, p);
    }
    const bool any_live = __any_sync(0xffffffffu, live);
    for (int h = h0; __any_sync(0xffffffffu, h < h_end); h += kAtOnce * head_step) {
        uint4 raw[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            raw[i] = make_uint4(0u, 0u, 0u, 0u);
            if (live && h + i * head_step < h_end) {
                raw[i] = __ldg(reinterpret_cast<const uint4*>(src + i * src_step));
            }
        }
        if (TURN != kNoTurn && any_live) {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                // Padding beside a real token: zeros, which turn into zeros.
                float x[8];
                unpack8<BF16>(raw[i], x);
                rotate8<TURN, BF16>(x, raw[i], a, chunk, hc);
                raw[i] = pack8<BF16>(x);
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (mine && h + i * head_step < h_end) {
                *reinterpret_cast<uint4*>(dst + i * dst_step) = raw[i];
            }
        }
        src += kAtOnce * src_step;
        dst += kAtOnce * dst_step;
    }
}

template <int D, bool BF16, bool E4M3, int TURN>
__global__ void __launch_bounds__(kMaxThreads) append_kernel(const __grid_constant__ FaAppendParams p,
                                                             DeviceStatus* status, unsigned long long page_share, int spans,
                                                             int log2_page, QuerySplit split) {
    // Pages and rows of q alternate in proportion, so that one's stores run beside the other's waits: page
    // blocks before block b are floor(b pages / blocks), kept as a 32-bit fraction rounded up.
    const unsigned long long b = blockIdx.x;
    const int before = static_cast<int>((b * page_share) >> 32);
    const bool is_page = static_cast<int>(((b + 1) * page_share) >> 32) > before;
    if (!is_page) {
        rotate_queries<D, BF16, TURN>(p, status, static_cast<int>(b) - before, split);
    } else if ((before & 1) == 0) {
        store_page<D, BF16, E4M3, TURN>(p, status, before >> 1, false, spans, log2_page);
    } else {
        store_page<D, BF16, E4M3, kNoTurn>(p, status, before >> 1, true, spans, log2_page);
    }
}

template <int D, bool BF16, bool E4M3, int TURN>
cudaError_t launch(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    const FaCache& c = p.cache;
    // Every page a sequence's tokens can touch, from any place in the first one.
    const int spans = (c.tokens + c.page_size - 2) / c.page_size + 1;
    const long long pages = static_cast<long long>(c.batch) * spans * c.kv_heads * 2;
    // A page's new rows are at most kRowsPerThread a thread. A decode step has one: with a warp a CTA all
    // of them run at once (128 sequences x 8 heads: 10.3 us with the threads of a whole page, 3.9 us with a warp).
    int rows_most = 1;
    while (rows_most < std::min(c.page_size, c.tokens)) {
        rows_most *= 2;
    }
    const int threads = std::min(kMaxThreads, std::max(32, rows_most * (D / 8) / kRowsPerThread));
    QuerySplit split{};
    long long query_blocks = 0;
    if (p.q != nullptr) {
        const int rows = threads / (D / 8);
        while ((1 << split.log2_tokens) < std::min(rows, c.tokens)) {
            ++split.log2_tokens;
        }
        // Heads of a CTA: 4 loads in flight a thread, twice (with few tokens once: more CTAs).
        split.heads = (rows >> split.log2_tokens) * (split.log2_tokens > 0 ? 8 : 4);
        split.token_blocks = (c.tokens + (1 << split.log2_tokens) - 1) >> split.log2_tokens;
        split.head_blocks = (p.heads + split.heads - 1) / split.heads;
        query_blocks = static_cast<long long>(c.batch) * split.token_blocks * split.head_blocks;
    }
    const long long blocks = pages + query_blocks;
    if (blocks > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    const unsigned long long page_share = ((static_cast<unsigned long long>(pages) << 32) + blocks - 1) / blocks;
    int log2_page = 0;
    while ((1 << log2_page) < c.page_size) {
        ++log2_page;
    }
    append_kernel<D, BF16, E4M3, TURN><<<static_cast<unsigned>(blocks), threads, 0, stream>>>(
        p, status, page_share, spans, log2_page, split);
    return cudaGetLastError();
}

template <int D, int TURN>
cudaError_t launch_types(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.cache.dtype == FA_DTYPE_FLOAT8_E4M3) {
        return bf16 ? launch<D, true, true, TURN>(p, status, stream) : launch<D, false, true, TURN>(p, status, stream);
    }
    return bf16 ? launch<D, true, false, TURN>(p, status, stream) : launch<D, false, false, TURN>(p, status, stream);
}

template <int D>
cudaError_t launch_dim(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    if (p.cos == nullptr) {
        return launch_types<D, kNoTurn>(p, status, stream);
    }
    return p.interleaved ? launch_types<D, kInterleaved>(p, status, stream)
                         : launch_types<D, kHalves>(p, status, stream);
}

}  // namespace

cudaError_t launch_append(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    return p.cache.head_dim == 64 ? launch_dim<64>(p, status, stream) : launch_dim<128>(p, status, stream);
}

}  // namespace fa_sm100
