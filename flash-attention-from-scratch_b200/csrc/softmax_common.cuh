#pragma once
// Softmax building blocks of the forward kernel (flash_fwd_sm100.cu).

#include <cstdint>

#include "sm100_ptx.cuh"

namespace fa_sm100 {

__device__ __forceinline__ float u2f(uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ uint32_t f2u(float x) { return __float_as_uint(x); }

// Bits 0 .. x of a word (none for x < 0, all for x >= 31).
__device__ __forceinline__ uint32_t bits_up_to(int x) {
    return x < 0 ? 0u : (x >= 31 ? 0xffffffffu : (2u << x) - 1u);
}

// Hides columns of one row's N scores (N a multiple of 32): kept are (to - span, to] and those up to
// `to` before `sinks`; the others become `hidden`. The bounds become one word of bits for 32 columns,
// so that a column costs a select and a share of a bit-to-predicate move: testing every column against
// three bounds instead cost the forward kernel a fifth of its time at a window of 1024. (Leaving out
// groups that are all kept or all hidden by branches costs more: the row no longer stays in registers.)
template <int N>
__device__ __forceinline__ void hide_columns(uint32_t (&x)[N], int to, int span, int sinks, uint32_t hidden) {
#pragma unroll
    for (int g = 0; g < N / 32; ++g) {
        const int c0 = 32 * g;
        const uint32_t keep = bits_up_to(to - c0) & (~bits_up_to(to - span - c0) | bits_up_to(sinks - 1 - c0));
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            x[c0 + c] = (keep >> c) & 1u ? x[c0 + c] : hidden;
        }
    }
}

// Row max (or min, for a negative scale) of N scores (N = 64 or 128): eight independent
// three-input chains over columns 8 .. N-9, then the last eight columns. A NaN among them is the result: the
// software 2^x that some columns take would lose it, while a NaN maximum makes the whole row NaN.
template <bool MAX, int N>
__device__ __forceinline__ float row_extreme(const uint32_t (&sr)[N]) {
    static_assert(N % 16 == 0 && N >= 32, "row_extreme covers N = 16 k columns");
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m[i] = u2f(sr[i]);
    }
#pragma unroll
    for (int c = 8; c + 16 <= N; c += 16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = MAX ? fmax3(m[i], u2f(sr[c + i]), u2f(sr[c + 8 + i]))
                       : fmin3(m[i], u2f(sr[c + i]), u2f(sr[c + 8 + i]));
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m[i] = MAX ? fmax_nan(m[i], u2f(sr[N - 8 + i])) : fmin_nan(m[i], u2f(sr[N - 8 + i]));
    }
    return MAX ? fmax3(fmax3(m[0], m[1], m[2]), fmax3(m[3], m[4], m[5]), fmax_nan(m[6], m[7]))
               : fmin3(fmin3(m[0], m[1], m[2]), fmin3(m[3], m[4], m[5]), fmin_nan(m[6], m[7]));
}

}  // namespace fa_sm100
