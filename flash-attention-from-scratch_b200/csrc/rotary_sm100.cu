// Rotation of queries and keys by positions on several axes.
//
//   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin),   cos, sin of pair i at row positions[axis(i)][b][t], column i
//
// (inverse: sin negated), each product and their sum rounded to float32, the result once more: to the
// bit what append_kv stores. Every row is read and written once, so the kernel is bound by DRAM bytes:
// angles are looked up once for a token and kept in registers over the heads.
//
// A thread owns 16 dims of a row that turn among themselves: 8 pairs as two 16-byte words (halves:
// dims 8 c .. of either half; interleaved: 16 dims on end), so nothing is exchanged between lanes, and 8
// cosines and sines are all it keeps. Dims that do not turn are copied by threads of their own. A CTA
// has a power of two of tokens and as many heads at a time as its threads hold; heads are parted among CTAs until
// there are some for every SM.
//
// Measured, bf16, D 128, tokens with their heads on end: 2 x 4999 tokens of 32 + 8 heads, 3 axes, 36.7 us (5.7 TB/s); 16384 of
// 16 + 4 heads, half of the dims turned, 35.9 us (4.7 TB/s). CTAs of 256 threads took 40.0 and 43.6 (longer last waves), half
// or twice as many parts 46.8 or 41.0 and 33.8 or 35.9; angles a value at a time 37.5 and 38.0. The second shape's rate is that of
// its layout (a head's tokens on end): interleaved or not, half or all of the dims turned, it takes 36.2 to 36.8.

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

constexpr int kThreads = 128;

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (BF16) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    } else {
        return unpack_half2(w);
    }
}

struct RotarySplit {
    int log2_tokens;   // tokens of a CTA
    int token_blocks;  // of a sequence
    int head_parts;    // CTAs that share a token block's heads
    int heads_of_part;
    unsigned one_axis;  // bits of a row's threads whose 8 pairs turn by one axis: their angles are whole words
};

template <int D, bool BF16, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ FaRotaryParams p, DeviceStatus* status,
                                                          RotarySplit split) {
    constexpr int kLanes = D / 16;             // threads of a row
    constexpr int kSlots = kThreads / kLanes;  // rows at a time
    const int lane = static_cast<int>(threadIdx.x) % kLanes;
    const int slot = static_cast<int>(threadIdx.x) / kLanes;
    const int head_step = kSlots >> split.log2_tokens;
    int unit = static_cast<int>(blockIdx.x);
    const int part = unit % split.head_parts;
    unit /= split.head_parts;
    const int b = unit / split.token_blocks;
    const int token = ((unit - b * split.token_blocks) << split.log2_tokens) + (slot & ((1 << split.log2_tokens) - 1));
    if (token >= p.tokens) {
        return;
    }
    int pos[4] = {0, 0, 0, 0};
    bool real = true;
    bool bad = false;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        if (a < p.axes) {
            pos[a] = __ldg(p.positions + a * p.position_stride[0] + b * p.position_stride[1] + token * p.position_stride[2]);
            real = real && pos[a] >= 0;
            bad = bad || pos[a] >= p.table_rows;
        }
    }
    if (real && bad && part == 0 && threadIdx.x % kLanes == 0) {
        atomicOr(&status->code, kStatusBadPage);
    }
    real = real && !bad;

    const int turning = p.rotary_dim / 16;  // threads of a row that turn
    const int half = p.rotary_dim / 2;
    const bool turns = lane < turning;
    // Dims of the thread's two words.
    const int d0 = turns && !INTERLEAVED ? 8 * lane : 16 * lane;
    const int d1 = turns && !INTERLEAVED ? 8 * lane + half : 16 * lane + 8;
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        c[i] = 1.0f;
        s[i] = 0.0f;
    }
    auto row_of = [&](int axis) { return axis == 0 ? pos[0] : axis == 1 ? pos[1] : axis == 2 ? pos[2] : pos[3]; };
    if (turns && real) {
        if ((split.one_axis >> lane) & 1u) {
            const int64_t at = static_cast<int64_t>(row_of(p.axis_of_pair[8 * lane])) * half + 8 * lane;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 u = __ldg(reinterpret_cast<const float4*>(p.cos + at) + i);
                const float4 v = __ldg(reinterpret_cast<const float4*>(p.sin + at) + i);
                c[4 * i] = u.x;
                c[4 * i + 1] = u.y;
                c[4 * i + 2] = u.z;
                c[4 * i + 3] = u.w;
                s[4 * i] = v.x;
                s[4 * i + 1] = v.y;
                s[4 * i + 2] = v.z;
                s[4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int pair = 8 * lane + i;
                const int64_t at = static_cast<int64_t>(row_of(p.axis_of_pair[pair])) * half + pair;
                c[i] = __ldg(p.cos + at);
                s[i] = __ldg(p.sin + at);
            }
        }
        if (p.inverse) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[i] = -s[i];
            }
        }
    }

    const int first = part * split.heads_of_part + (slot >> split.log2_tokens);
    const int end = min((part + 1) * split.heads_of_part, p.heads + p.kv_heads);
#pragma unroll 4
    for (int h = first; h < end; h += head_step) {
        const bool is_k = h >= p.heads;
        const int head = is_k ? h - p.heads : h;
        const int64_t* st = is_k ? p.k_stride : p.q_stride;
        const uint16_t* src = static_cast<const uint16_t*>(is_k ? p.k : p.q) + b * st[0] + head * st[1] + token * st[2];
        uint16_t* dst = static_cast<uint16_t*>(is_k ? p.k_out : p.q_out) +
                        ((static_cast<int64_t>(b) * (is_k ? p.kv_heads : p.heads) + head) * p.tokens + token) * D;
        const uint4 lo = __ldg(reinterpret_cast<const uint4*>(src + d0));
        const uint4 hi = __ldg(reinterpret_cast<const uint4*>(src + d1));
        uint32_t u[4] = {lo.x, lo.y, lo.z, lo.w};
        uint32_t v[4] = {hi.x, hi.y, hi.z, hi.w};
        if (!real) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u[i] = v[i] = 0u;
            }
        } else if (turns) {
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t& w = i < 4 ? u[i & 3] : v[i & 3];
                    const float2 x = unpack2<BF16>(w);
                    w = pack2<BF16>(__fsub_rn(__fmul_rn(x.x, c[i]), __fmul_rn(x.y, s[i])),
                                    __fadd_rn(__fmul_rn(x.y, c[i]), __fmul_rn(x.x, s[i])));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 x = unpack2<BF16>(u[i]);
                    const float2 y = unpack2<BF16>(v[i]);
                    u[i] = pack2<BF16>(__fsub_rn(__fmul_rn(x.x, c[2 * i]), __fmul_rn(y.x, s[2 * i])),
                                       __fsub_rn(__fmul_rn(x.y, c[2 * i + 1]), __fmul_rn(y.y, s[2 * i + 1])));
                    v[i] = pack2<BF16>(__fadd_rn(__fmul_rn(y.x, c[2 * i]), __fmul_rn(x.x, s[2 * i])),
                                       __fadd_rn(__fmul_rn(y.y, c[2 * i + 1]), __fmul_rn(x.y, s[2 * i + 1])));
                }
            }
        }
        *reinterpret_cast<uint4*>(dst + d0) = make_uint4(u[0], u[1], u[2], u[3]);
        *reinterpret_cast<uint4*>(dst + d1) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

template <int D, bool BF16, bool INTERLEAVED>
cudaError_t launch(const FaRotaryParams& p, DeviceStatus* status, int sm_count, cudaStream_t stream) {
    constexpr int kSlots = kThreads / (D / 16);
    const int heads = p.heads + p.kv_heads;
    RotarySplit split;
    split.log2_tokens = 0;
    while ((1 << split.log2_tokens) < std::min(kSlots, p.tokens)) {
        ++split.log2_tokens;
    }
    const int tokens = 1 << split.log2_tokens;
    split.token_blocks = (p.tokens + tokens - 1) / tokens;
    // As many CTAs as fill the GPU a few times over, whole passes of heads each.
    const long long blocks = static_cast<long long>(p.batch) * split.token_blocks;
    const int step = kSlots / tokens;
    const int passes = (heads + step - 1) / step;
    const long long want = (8ll * sm_count + blocks - 1) / blocks;
    const int passes_of_part = std::max(1, passes / static_cast<int>(std::min<long long>(want, passes)));
    split.heads_of_part = passes_of_part * step;
    split.head_parts = (heads + split.heads_of_part - 1) / split.heads_of_part;
    split.one_axis = 0;
    for (int lane = 0; lane < p.rotary_dim / 16; ++lane) {
        const uint8_t* axis = p.axis_of_pair + 8 * lane;
        split.one_axis |= static_cast<unsigned>(std::all_of(axis, axis + 8, [&](uint8_t a) { return a == axis[0]; })) << lane;
    }
    const long long grid = blocks * split.head_parts;
    if (grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    rotary_kernel<D, BF16, INTERLEAVED><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p, status, split);
    return cudaGetLastError();
}

template <int D, bool BF16>
cudaError_t launch_pairs(const FaRotaryParams& p, DeviceStatus* status, int sm_count, cudaStream_t stream) {
    return p.interleaved ? launch<D, BF16, true>(p, status, sm_count, stream) : launch<D, BF16, false>(p, status, sm_count, stream);
}

}  // namespace

cudaError_t launch_rotary(const FaRotaryParams& p, DeviceStatus* status, int sm_count, cudaStream_t stream) {
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.head_dim == 64) {
        return bf16 ? launch_pairs<64, true>(p, status, sm_count, stream) : launch_pairs<64, false>(p, status, sm_count, stream);
    }
    return bf16 ? launch_pairs<128, true>(p, status, sm_count, stream) : launch_pairs<128, false>(p, status, sm_count, stream);
}

}  // namespace fa_sm100
