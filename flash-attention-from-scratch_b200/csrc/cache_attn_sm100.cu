// Attention of the newest tokens of every sequence over the paged cache.
//
// One warp per query row, the head dim over the lanes, keys one after the other with a running
// maximum and sum: O = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m).

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

template <bool BF16>
__device__ __forceinline__ float widen(uint16_t x) {
    if constexpr (BF16) {
        return __uint_as_float(static_cast<uint32_t>(x) << 16);
    } else {
        return __half2float(__ushort_as_half(x));
    }
}

template <int D, bool BF16, bool E4M3>
__global__ void __launch_bounds__(128) cached_rows_kernel(const __grid_constant__ FaCachedParams p,
                                                          DeviceStatus* status) {
    constexpr int PER = D / 32;
    const FaCache& c = p.cache;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const long long row = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / 32;
    if (row >= static_cast<long long>(c.batch) * p.heads * c.tokens) {
        return;
    }
    const int bh = static_cast<int>(row / c.tokens);
    const int t = static_cast<int>(row - static_cast<long long>(bh) * c.tokens);
    const int b = bh / p.heads;
    const int h = bh - b * p.heads;
    const int kvh = h / (p.heads / c.kv_heads);
    const int len = c.lengths[b];
    const int count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
    const int pos = t < count ? len - count + t : -1;
    float q[PER], acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        q[i] = widen<BF16>(static_cast<const uint16_t*>(p.q)[b * p.q_stride[0] + h * p.q_stride[1] +
                                                             t * p.q_stride[2] + lane * PER + i]);
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int first = window_first(pos, p.window);
    int j = p.sinks > 0 ? 0 : first;
    for (; j <= pos; ++j) {
        if (j == p.sinks && j < first) {
            j = first;
        }
        const int page = j / c.page_size;
        const int id = page < c.max_pages ? c.page_table[b * c.table_stride + page] : -1;
        if (id < 0 || id >= c.num_pages) {
            if (lane == 0) {
                atomicOr(&status->code, kStatusBadPage);
            }
            continue;
        }
        const int64_t slot = static_cast<int64_t>(j % c.page_size) * D + lane * PER;
        const int64_t ka = id * c.k_stride[0] + kvh * c.k_stride[1] + slot;
        const int64_t va = id * c.v_stride[0] + kvh * c.v_stride[1] + slot;
        float kx[PER], vx[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if constexpr (E4M3) {
                const int64_t s = static_cast<int64_t>(id) * c.kv_heads + kvh;
                kx[i] = unpack_half2(e4m3x2_to_half2(static_cast<const uint8_t*>(c.k)[ka + i])).x * c.k_scale[s];
                vx[i] = unpack_half2(e4m3x2_to_half2(static_cast<const uint8_t*>(c.v)[va + i])).x * c.v_scale[s];
            } else {
                kx[i] = widen<BF16>(static_cast<const uint16_t*>(c.k)[ka + i]);
                vx[i] = widen<BF16>(static_cast<const uint16_t*>(c.v)[va + i]);
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s = fmaf(q[i], kx[i], s);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
        }
        s *= p.softmax_scale;
        const float top = fmaxf(m, s);
        const float used = top == -INFINITY ? 0.0f : top;
        const float a = __expf(m - used);
        const float w = __expf(s - used);
        m = top;
        l = fmaf(l, a, w);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            acc[i] = fmaf(acc[i], a, w * vx[i]);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        static_cast<uint16_t*>(p.o)[row * D + lane * PER + i] =
            static_cast<uint16_t>(pack2<BF16>(acc[i] * inv, 0.0f) & 0xFFFFu);
    }
}

template <int D>
cudaError_t launch_dim(const FaCachedParams& p, DeviceStatus* status, cudaStream_t stream) {
    const long long rows = static_cast<long long>(p.cache.batch) * p.heads * p.cache.tokens;
    if ((rows + 3) / 4 > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.cache.dtype == FA_DTYPE_FLOAT8_E4M3) {
        if (bf16) {
            cached_rows_kernel<D, true, true><<<grid, 128, 0, stream>>>(p, status);
        } else {
            cached_rows_kernel<D, false, true><<<grid, 128, 0, stream>>>(p, status);
        }
    } else if (bf16) {
        cached_rows_kernel<D, true, false><<<grid, 128, 0, stream>>>(p, status);
    } else {
        cached_rows_kernel<D, false, false><<<grid, 128, 0, stream>>>(p, status);
    }
    return cudaGetLastError();
}

}  // namespace

unsigned long long cached_workspace_bytes(const FaCachedParams&, int) { return 0; }

cudaError_t launch_cached(const FaCachedParams& p, DeviceStatus* status, void*, int, cudaStream_t stream) {
    return p.cache.head_dim == 64 ? launch_dim<64>(p, status, stream) : launch_dim<128>(p, status, stream);
}

}  // namespace fa_sm100
