// Attention of a tree of drafted tokens over the paged cache.
//
//   O_t = sum_j e^(s_tj) v_j / sum_j e^(s_tj),   s_tj = scale q_t.k_j over the context (through a window and
//   sinks) and those nodes that are t itself or its ancestors

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMostNodes = 256;
constexpr int kMaskWords = kMostNodes / 32;

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
constexpr int kRowWarps = 4;

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

template <int D, bool BF16, bool E4M3>
__global__ void __launch_bounds__(kRowWarps * 32) tree_row_kernel(const __grid_constant__ FaTreeParams p, DeviceStatus* status) {
    const long long row = blockIdx.x;
    const int t = static_cast<int>(row % p.cache.tokens);
    const long long head = row / p.cache.tokens;
    attend_row<D, BF16, E4M3>(p, status, static_cast<int>(head / p.heads), static_cast<int>(head % p.heads), t);
}

template <int D, bool BF16, bool E4M3>
cudaError_t launch(const FaTreeParams& p, DeviceStatus* status, void*, int, cudaStream_t stream) {
    const long long grid = static_cast<long long>(p.cache.batch) * p.heads * p.cache.tokens;
    if (grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    tree_row_kernel<D, BF16, E4M3><<<static_cast<unsigned>(grid), kRowWarps * 32, 0, stream>>>(p, status);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_types(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.cache.dtype == FA_DTYPE_FLOAT8_E4M3) {
        return bf16 ? launch<D, true, true>(p, status, workspace, sm_count, stream)
                    : launch<D, false, true>(p, status, workspace, sm_count, stream);
    }
    return bf16 ? launch<D, true, false>(p, status, workspace, sm_count, stream)
                : launch<D, false, false>(p, status, workspace, sm_count, stream);
}

}  // namespace

unsigned long long tree_workspace_bytes(const FaTreeParams&, int) { return 0; }

cudaError_t launch_tree(const FaTreeParams& p, DeviceStatus* status, void* workspace, int sm_count, cudaStream_t stream) {
    return p.cache.head_dim == 64 ? launch_types<64>(p, status, workspace, sm_count, stream)
                                  : launch_types<128>(p, status, workspace, sm_count, stream);
}

}  // namespace fa_sm100
