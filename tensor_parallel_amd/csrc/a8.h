// What the files of products of two 8-bit operands share: launch parameters and the arithmetic behind the sums.
#pragma once
#include "common.h"

namespace tpamd {

// y[m][n] = act((s_x[m] s_w[n]) sum_k x[m][k] w[n][k] + bias[n]) (+ addend), or the gated pair; sums exact in int32.
struct A8Params {
    const char *x, *w, *w2;            // codes: rows, weights (pair: gate), up weights
    const float *sx, *sw, *sw2;        // a scale for each row, column
    const char *bias, *addend;         // of the outputs' dtype, or NULL
    char *y;
    int64_t copy;                      // every output is stored a second time that many bytes on (0: once)
    int M, N, K;
    int64_t ldx, ldw, ldadd, ldy;      // elements
    int act;
    struct { int64_t x, w, w2, sx, sw, sw2, bias, y; } to;  // byte distances to a second rank's operands
};

constexpr int64_t A8_MAX_K = 131071;   // 128 * 128 * K < 2^31

// An fp32 value of its own: products, sums and conversions to fp16 would otherwise become one instruction that rounds once in some kernels and not in others, and a
// row's bits would depend on the kernel that its batch selects.
__device__ __forceinline__ float a8_value(float v) {
    asm("" : "+v"(v));
    return v;
}

// From a sum to the value before it is rounded, in fp32: the sum converted (24 bits of it), times the product of the scales, and the bias in the same operation.
__device__ __forceinline__ float a8_linear(int sum, float sx, float sw, float bias) { return a8_value(fmaf(static_cast<float>(sum), a8_value(sx * sw), bias)); }
__device__ __forceinline__ float a8_act(float v, int act) { return act == TPAMD_ACT_GELU ? a8_value(gelu_erf(v)) : v; }

// SiLU(g) u, rounded once by the caller: both factors stay in fp32 (the 16-bit pair rounds g, u, SiLU(g) and the product as its four separate operations would;
// here no 16-bit operation is stood in for, and one rounding leaves 1.66e-3 of normally distributed g and u in bf16 where four leave 3.56e-3).
__device__ __forceinline__ float a8_gated(float g, float u) { return a8_value(a8_value(silu_f32(g)) * u); }

template <int DT>
__device__ __forceinline__ uint16_t a8_round(float v) { return f32_to_half<DT>(v); }
template <int DT>
__device__ __forceinline__ uint32_t a8_round2(float a, float b) { return pack2_half<DT>(a, b); }

// Where the fast kernels take operands: pieces of 16 codes in the rows of x and w, rows within reach of 32-bit offsets.
static inline bool a8_fast(const A8Params &p) {
    return p.K >= 16 && p.K % 16 == 0 && p.ldx % 16 == 0 && p.ldw % 16 == 0 && p.ldx < (1ll << 22) && p.ldw < (1ll << 22) && aligned(p.x, 16) && aligned(p.w, 16) && aligned(p.w2, 16);
}
// gemm_a8.hip: tiles of 64 * tm x-rows by 64 * tn w-rows (a pair: 32 * tn columns), K in at most `splits` ranges. stream_a8.hip: up to 64 rows on one block per CU. Operands of a8_fast.
int gemm_a8(const A8Params &p, bool pair, int dtype, int tm, int tn, int splits, hipStream_t s);
bool stream_a8_takes(const A8Params &p, bool pair, int ranks, int cus);
float stream_a8_us(const A8Params &p, bool pair, int cus);  // predicted
int stream_a8(const A8Params &p, bool pair, int dtype, int ranks, int cus, hipStream_t s);  // ranks: 1, or 2 (no addend)

}  // namespace tpamd
