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
// and no atomics; then CTAs for the rows of q. A row is D / 8 lanes of 16 bytes, at most 8
// rows a thread, kept in registers between the block's maximum and the store: one pass over the
// data. Bound by DRAM bytes for prompts, by one launch for a decode step.

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

constexpr int kRowsPerThread = 8;
constexpr int kMaxThreads = 512;

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

// Rotates the 8 dims of `chunk` (dims 8 chunk ...) of a row at `pos`. The lanes of a row are
// consecutive; with halves a lane's partner dims are in the lane rotary / 16 chunks away. Called
// by whole warps; `live` lanes have a valid position.
__device__ __forceinline__ void rotate8(float (&x)[8], int chunk, int pos, bool live, const FaAppendParams& p) {
    const int half = p.rotary_dim / 2;
    if (p.interleaved) {
        if (live && chunk * 8 < p.rotary_dim) {
            const long long at = static_cast<long long>(pos) * half + chunk * 4;
            const float4 c = *reinterpret_cast<const float4*>(p.cos + at);
            const float4 s = *reinterpret_cast<const float4*>(p.sin + at);
            const float cc[4] = {c.x, c.y, c.z, c.w};
            const float ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = x[2 * i];
                const float b = x[2 * i + 1];
                x[2 * i] = __fsub_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, ss[i]));
                x[2 * i + 1] = __fadd_rn(__fmul_rn(b, cc[i]), __fmul_rn(a, ss[i]));
            }
        }
        return;
    }
    const int lane = static_cast<int>(threadIdx.x) & 31;
    const int hc = half / 8;  // chunks of a half
    const bool first = chunk < hc;
    const int src = first ? lane + hc : lane - hc;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = __shfl_sync(0xffffffffu, x[i], src & 31);
    }
    if (live && chunk < 2 * hc) {
        const long long at = static_cast<long long>(pos) * half + (first ? chunk : chunk - hc) * 8;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float4 c = *reinterpret_cast<const float4*>(p.cos + at + 4 * q);
            const float4 s = *reinterpret_cast<const float4*>(p.sin + at + 4 * q);
            const float cc[4] = {c.x, c.y, c.z, c.w};
            const float ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = __fmul_rn(x[4 * q + i], cc[i]);
                const float b = __fmul_rn(y[4 * q + i], ss[i]);
                x[4 * q + i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
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

template <int D, bool BF16, bool E4M3>
__device__ __forceinline__ void store_page(const FaAppendParams& p, DeviceStatus* status, int unit, int spans,
                                           int log2_page) {
    constexpr int C = D / 8;  // lanes of a row
    const FaCache& c = p.cache;
    const bool is_v = (unit & 1) != 0;
    unit >>= 1;
    const int h = unit % c.kv_heads;
    unit /= c.kv_heads;
    const int span = unit % spans;
    const int b = unit / spans;
    const int len = c.lengths[b];
    const int count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
    const int start = len - count;
    const int page = (max(start, 0) >> log2_page) + span;
    const int base = page << log2_page;
    const int lo = max(start, base);
    int hi = min(len, base + c.page_size);
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
    const bool turn = !is_v && p.cos != nullptr;
    const int rows = hi - lo;

    float x[kRowsPerThread][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kRowsPerThread; ++i) {
        if (i * groups < rows) {
            const int r = i * groups + group;
            const bool live = r < rows;
            uint4 raw = make_uint4(0u, 0u, 0u, 0u);
            if (live) {
                raw = __ldg(reinterpret_cast<const uint4*>(src + static_cast<int64_t>(lo + r - start) * st[2]));
            }
            unpack8<BF16>(raw, x[i]);
            if (turn) {
                rotate8(x[i], chunk, lo + r, live, p);
            }
            if constexpr (E4M3) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float a = fabsf(x[i][e]);
                    amax = fmaxf(amax, a <= FLT_MAX ? a : 0.0f);
                }
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
        auto code = [&](float v) { return pow2 ? v * inv : __fdiv_rn(v, s); };
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
#pragma unroll
        for (int i = 0; i < kRowsPerThread; ++i) {
            const int r = i * groups + group;
            if (r < rows) {
                uint32_t w[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    w[q] = pack_e4m3x2(code(x[i][4 * q]), code(x[i][4 * q + 1])) |
                           (pack_e4m3x2(code(x[i][4 * q + 2]), code(x[i][4 * q + 3])) << 16);
                }
                *reinterpret_cast<uint2*>(dst + static_cast<int64_t>(in_page + r) * D) = make_uint2(w[0], w[1]);
            }
        }
    }
}

template <int D, bool BF16>
__device__ __forceinline__ void rotate_queries(const FaAppendParams& p, DeviceStatus* status, int block) {
    constexpr int C = D / 8;
    const FaCache& c = p.cache;
    const int chunk = static_cast<int>(threadIdx.x) % C;
    const int groups = static_cast<int>(blockDim.x) / C;
    const long long total = static_cast<long long>(c.batch) * p.heads * c.tokens;
    const long long row0 = static_cast<long long>(block) * groups * kRowsPerThread + threadIdx.x / C;
#pragma unroll 2
    for (int i = 0; i < kRowsPerThread; ++i) {
        const long long row = row0 + static_cast<long long>(i) * groups;
        bool live = row < total;
        int t = 0, h = 0, b = 0, pos = 0;
        if (live) {
            const int bh = static_cast<int>(row / c.tokens);
            t = static_cast<int>(row - static_cast<long long>(bh) * c.tokens);
            b = bh / p.heads;
            h = bh - b * p.heads;
        }
        const bool mine = live;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (live) {
            const int count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
            pos = c.lengths[b] - count + t;
            live = t < count;
            if (live && (pos < 0 || (p.cos != nullptr && pos >= p.table_rows))) {
                live = false;
                if (chunk == 0 && h == 0) {
                    atomicOr(&status->code, kStatusBadPage);
                }
            }
        }
        if (live) {
            raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + b * p.q_stride[0] +
                                                       h * p.q_stride[1] + t * p.q_stride[2] + chunk * 8));
        }
        if (p.cos != nullptr) {
            float x[8];
            unpack8<BF16>(raw, x);
            rotate8(x, chunk, pos, live, p);
            raw = live ? pack8<BF16>(x) : make_uint4(0u, 0u, 0u, 0u);
        }
        if (mine) {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.q_out) + row * D + chunk * 8) = raw;
        }
    }
}

template <int D, bool BF16, bool E4M3>
__global__ void __launch_bounds__(kMaxThreads) append_kernel(const __grid_constant__ FaAppendParams p,
                                                             DeviceStatus* status, int page_blocks, int spans,
                                                             int log2_page) {
    if (static_cast<int>(blockIdx.x) < page_blocks) {
        store_page<D, BF16, E4M3>(p, status, static_cast<int>(blockIdx.x), spans, log2_page);
    } else {
        rotate_queries<D, BF16>(p, status, static_cast<int>(blockIdx.x) - page_blocks);
    }
}

template <int D, bool BF16, bool E4M3>
cudaError_t launch(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    const FaCache& c = p.cache;
    // Every page a sequence's tokens can touch, from any place in the first one.
    const int spans = (c.tokens + c.page_size - 2) / c.page_size + 1;
    const long long pages = static_cast<long long>(c.batch) * spans * c.kv_heads * 2;
    // A page is at most kRowsPerThread rows a thread.
    const int threads = std::min(kMaxThreads, std::max(32, c.page_size * (D / 8) / kRowsPerThread));
    const long long rows = p.q != nullptr ? static_cast<long long>(c.batch) * p.heads * c.tokens : 0;
    const int rows_per_block = threads / (D / 8) * kRowsPerThread;
    const long long blocks = pages + (rows + rows_per_block - 1) / rows_per_block;
    if (blocks > 0x7fffffffLL || rows / c.tokens > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    int log2_page = 0;
    while ((1 << log2_page) < c.page_size) {
        ++log2_page;
    }
    append_kernel<D, BF16, E4M3><<<static_cast<unsigned>(blocks), threads, 0, stream>>>(
        p, status, static_cast<int>(pages), spans, log2_page);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_dim(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.cache.dtype == FA_DTYPE_FLOAT8_E4M3) {
        return bf16 ? launch<D, true, true>(p, status, stream) : launch<D, false, true>(p, status, stream);
    }
    return bf16 ? launch<D, true, false>(p, status, stream) : launch<D, false, false>(p, status, stream);
}

}  // namespace

cudaError_t launch_append(const FaAppendParams& p, DeviceStatus* status, cudaStream_t stream) {
    return p.cache.head_dim == 64 ? launch_dim<64>(p, status, stream) : launch_dim<128>(p, status, stream);
}

}  // namespace fa_sm100
