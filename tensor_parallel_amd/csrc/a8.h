// What the files of products of two 8-bit operands share: launch parameters and the arithmetic behind the sums.
#pragma once
#include "common.h"

namespace tpamd {

// y[m][n] = act(s_x[m] s_w[n] sum_k x[m][k] w[n][k] + bias[n]) (+ addend), or the gated pair; sums exact in int32.
struct A8Params {
    const char *x, *w, *w2;            // codes: rows, weights (pair: gate), up weights
    const float *sx, *sw, *sw2;        // a scale for each row, column
    const char *bias, *addend;         // of the outputs' dtype, or NULL
    char *y;
    int64_t copy;                      // every output is stored a second time that many bytes on (0: once)
    int M, N, K;
    int64_t ldx, ldw, ldadd, ldy;      // elements
    int act;
};

constexpr int64_t A8_MAX_K = 131071;   // 128 * 128 * K < 2^31

// From a sum to the value before it is rounded: in fp32 behind the exact sum (the int32 is rounded to 24 bits, 2^-24 of it).
__device__ __forceinline__ float a8_scaled(int sum, float sx, float sw) { return static_cast<float>(sum) * sw * sx; }

// SiLU(g) u, rounded once by the caller: both factors stay in fp32 (the 16-bit pair rounds g, u, SiLU(g) and the product as its four separate operations would;
// here no 16-bit operation is stood in for, and one rounding is 2.3 times closer to the definition).
__device__ __forceinline__ float a8_gated(float g, float u) { return silu_f32(g) * u; }

// Rounded to the outputs' dtype as an fp32 value of its own: a product and its conversion to fp16 may otherwise become one instruction that rounds once, in some kernels and not in
// others, and a row's bits would depend on the kernel that its batch selects.
template <int DT>
__device__ __forceinline__ uint16_t a8_round(float v) {
    asm("" : "+v"(v));
    return f32_to_half<DT>(v);
}

}  // namespace tpamd
