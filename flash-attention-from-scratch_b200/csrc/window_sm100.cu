// Window attention with sinks over dense tensors, forward and backward: one warp per row.
//
// Forward, row i:  s_j = scale q.k_j over the visible j, O = sum_j p_j v_j, LSE = ln sum_j e^s_j.
// Backward:        p_j = e^(s_j - LSE), delta = dO.O, ds_j = p_j (dO.v_j - delta) scale,
//                  dq = sum_j ds_j k_j, dk_j = sum_i ds_ij q_i, dv_j = sum_i p_ij dO_i,
// dq by query rows (which also write delta), dk and dv by key rows over the queries of every
// head of the group, in order: no atomics.

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

template <int D, bool BF16>
struct Row {
    static constexpr int PER = D / 32;
    float x[PER];
    __device__ __forceinline__ void load(const void* base, const int64_t (&st)[3], int b, int h, int n, int lane) {
        const uint16_t* src = static_cast<const uint16_t*>(base) + b * st[0] + h * st[1] + n * st[2] + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            x[i] = BF16 ? __uint_as_float(static_cast<uint32_t>(src[i]) << 16) : __half2float(__ushort_as_half(src[i]));
        }
    }
    __device__ __forceinline__ void store(void* base, const int64_t (&st)[3], int b, int h, int n, int lane) const {
        uint16_t* dst = static_cast<uint16_t*>(base) + b * st[0] + h * st[1] + n * st[2] + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            dst[i] = static_cast<uint16_t>(pack2<BF16>(x[i], 0.0f) & 0xFFFFu);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            x[i] = 0.0f;
        }
    }
    __device__ __forceinline__ float dot(const Row& o) const {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s = fmaf(x[i], o.x[i], s);
        }
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, k);
        }
        return s;
    }
    __device__ __forceinline__ void axpy(float a, const Row& o) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            x[i] = fmaf(a, o.x[i], x[i]);
        }
    }
};

template <int D, bool BF16, bool BWD>
__global__ void __launch_bounds__(128) query_rows_kernel(const __grid_constant__ FaWindowParams p, float* delta_out) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const long long row = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / 32;
    if (row >= static_cast<long long>(p.batch) * p.heads * p.q_len) {
        return;
    }
    const int bh = static_cast<int>(row / p.q_len);
    const int i = static_cast<int>(row - static_cast<long long>(bh) * p.q_len);
    const int b = bh / p.heads;
    const int h = bh - b * p.heads;
    const int kvh = h / (p.heads / p.kv_heads);
    const int pos = p.k_len - p.q_len + i;
    Row<D, BF16> q, k, v, acc, dout;
    q.load(p.q, p.q_stride, b, h, i, lane);
    acc.zero();
    float m = -INFINITY, l = 0.0f, delta = 0.0f, lse = 0.0f;
    if constexpr (BWD) {
        dout.load(p.d_o, p.do_stride, b, h, i, lane);
        v.load(p.o, p.o_stride, b, h, i, lane);
        delta = dout.dot(v);
        lse = p.lse[row];
        if (lane == 0) {
            delta_out[row] = delta;
        }
    }
    const int first = window_first(pos, p.window);
    for (int j = p.sinks > 0 ? 0 : first; j <= pos; ++j) {
        if (j == p.sinks && j < first) {
            j = first;
        }
        k.load(p.k, p.k_stride, b, kvh, j, lane);
        v.load(p.v, p.v_stride, b, kvh, j, lane);
        const float s = q.dot(k) * p.softmax_scale;
        if constexpr (BWD) {
            acc.axpy(__expf(s - lse) * (dout.dot(v) - delta) * p.softmax_scale, k);
        } else {
            const float top = fmaxf(m, s);
            const float used = top == -INFINITY ? 0.0f : top;
            const float a = __expf(m - used);
            const float w = __expf(s - used);
            m = top;
            l = fmaf(l, a, w);
#pragma unroll
            for (int e = 0; e < acc.PER; ++e) {
                acc.x[e] = fmaf(acc.x[e], a, w * v.x[e]);
            }
        }
    }
    if constexpr (BWD) {
        acc.store(p.dq, p.dq_stride, b, h, i, lane);
    } else {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int e = 0; e < acc.PER; ++e) {
            acc.x[e] *= inv;
        }
        acc.store(p.o, p.o_stride, b, h, i, lane);
        if (lane == 0 && p.lse != nullptr) {
            p.lse[row] = l > 0.0f ? m + logf(l) : -INFINITY;
        }
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(128) key_rows_kernel(const __grid_constant__ FaWindowParams p, const float* delta) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const long long row = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / 32;
    if (row >= static_cast<long long>(p.batch) * p.kv_heads * p.k_len) {
        return;
    }
    const int bh = static_cast<int>(row / p.k_len);
    const int j = static_cast<int>(row - static_cast<long long>(bh) * p.k_len);
    const int b = bh / p.kv_heads;
    const int kvh = bh - b * p.kv_heads;
    const int group = p.heads / p.kv_heads;
    const int shift = p.k_len - p.q_len;
    Row<D, BF16> k, v, q, dout, dk, dv;
    k.load(p.k, p.k_stride, b, kvh, j, lane);
    v.load(p.v, p.v_stride, b, kvh, j, lane);
    dk.zero();
    dv.zero();
    const long long last = (p.window == 0 || j < p.sinks) ? p.k_len : min(static_cast<long long>(p.k_len), static_cast<long long>(j) + p.window);
    for (int h = kvh * group; h < (kvh + 1) * group; ++h) {
        for (int i = max(0, j - shift); i + shift < last; ++i) {
            q.load(p.q, p.q_stride, b, h, i, lane);
            dout.load(p.d_o, p.do_stride, b, h, i, lane);
            const long long at = (static_cast<long long>(b) * p.heads + h) * p.q_len + i;
            const float w = __expf(q.dot(k) * p.softmax_scale - p.lse[at]);
            dv.axpy(w, dout);
            dk.axpy(w * (dout.dot(v) - delta[at]) * p.softmax_scale, q);
        }
    }
    dk.store(p.dk, p.dk_stride, b, kvh, j, lane);
    dv.store(p.dv, p.dv_stride, b, kvh, j, lane);
}

unsigned blocks(long long rows) { return static_cast<unsigned>((rows + 3) / 4); }

}  // namespace

unsigned long long window_bwd_workspace_bytes(const FaWindowParams& p, int) {
    return 4ull * p.batch * p.heads * p.q_len;
}

template <int D, bool BF16>
static cudaError_t bwd(const FaWindowParams& p, float* delta, cudaStream_t stream) {
    query_rows_kernel<D, BF16, true><<<blocks(static_cast<long long>(p.batch) * p.heads * p.q_len), 128, 0, stream>>>(p, delta);
    key_rows_kernel<D, BF16><<<blocks(static_cast<long long>(p.batch) * p.kv_heads * p.k_len), 128, 0, stream>>>(p, delta);
    return cudaGetLastError();
}

cudaError_t launch_window_bwd(const FaWindowParams& p, DeviceStatus*, unsigned, void* workspace, int, cudaStream_t stream) {
    float* delta = static_cast<float*>(workspace);
    const bool bf16 = p.dtype == FA_DTYPE_BFLOAT16;
    if (p.head_dim == 64) {
        return bf16 ? bwd<64, true>(p, delta, stream) : bwd<64, false>(p, delta, stream);
    }
    return bf16 ? bwd<128, true>(p, delta, stream) : bwd<128, false>(p, delta, stream);
}

}  // namespace fa_sm100
