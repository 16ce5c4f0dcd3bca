// Rows of an activation in 8 bits with a scale each, on their own or behind an RMS norm (with or without the residual's addition), and the way back.
//
//   p = x, or t w of the norm's input t (round(r + x) with a residual);  a = max |p| over the row
//   codes  round_half_even(127 p / a)     scale  a f / 127, f = 1 or rsqrt(mean t^2 + eps)
// The norm's factor is the same for a whole row, so it is in the scale alone: a row's codes do not depend on how its squares are summed, the maximum is found in
// the pass that sums them, and one meeting of the block serves both. The scale does not depend on the launch's number of rows either (block_sum_max); rows off the boundaries of quantize_kernel
// sum in an order of their own, and theirs may differ by rounding.
// A code is the integer nearest to the exact quotient: in rows of 16-bit values many quotients lie on a half (a value of half the largest is 63.5), which a product with a
// rounded 127 / a would put on either side. What the product leaves within 2^-15 of a half (its error is below 127 * 2 * 2^-24: one rounding each of 127 / a and of the product) is
// compared with the half exactly; p is exact in fp32 (two 16-bit significands). Eight codes ask once whether one is that near.
// A row that holds an infinity or NaN has no scale: it gets NaN, and codes of 0, so that products with it are NaN. One without a value of 2^-100 or more gets 1 and codes of 0.
//
// Bound: at a few rows by the latency of a launch (2.1-2.3 us in a graph, 1 x 4096; the shortest launches here take 1.7), else by HBM (x, r read once; sum and codes written once) and, as all rows of up to some 2000 are under way at
// once, by the instructions between their loads and their stores. In a graph, operands and results rotated through more memory than the caches hold, bf16: 2103 x 4096 quantised in 9.3 us (2.8 TB/s), normed 8.7,
// with the addition 14.5 (4.1); 4096 x 8192 21.2 (4.8), 21.3 and 42 (5.6); 4096 x 16384 37.7 (5.3), 37.9 and 83 (5.7), the way back of those to fp32 56.6 (5.9). Rows off the boundaries, single values at a time:
// 2103 x 4098 24, 25 and 49 us; rows above 16384 values 4096 x 28672 216, 220 and 400 (1.6-2.1 TB/s), 1 x 32768 35, 37 and 96.
#include "gemm_tile.h"

namespace tpamd {
namespace {

struct QuantParams {
    const char *x, *w, *r;
    char *s, *q;
    float *scale;
    int64_t ldx, ldr, lds, ldq;  // elements between rows
    int D;
    float eps;
    struct { int64_t x, w, r, s, q, scale; } to;  // blockIdx.y = 1: byte distances to a second rank's operands
};

// What a row has in common: its scale, 127 / a, and a (0: codes of 0).
struct RowCode {
    float scale, inv, most;
};
__device__ __forceinline__ RowCode row_code(uint32_t most_bits, float factor) {
    RowCode c;
    c.most = __uint_as_float(most_bits);
    if (most_bits >= 0x7f800000u) {  // an infinity or NaN: the integer maximum keeps both
        c.scale = __uint_as_float(0x7fc00000u);
        c.most = 0.f;
    } else if (c.most < 0x1p-100f) {
        c.scale = 1.f;
        c.most = 0.f;
    } else {
        c.scale = c.most * factor / 127.f;
    }
    c.inv = c.most != 0.f ? 127.f / c.most : 0.f;
    return c;
}
// p * inv rounded by an addition of 1.5 * 2^23, whose low byte is then the code, and how far that integer is from p * inv.
constexpr float CODE_MAGIC = 12582912.f;
__device__ __forceinline__ float code_bits(float p, float inv, float &off) {
    const float m = fmaf(p, inv, CODE_MAGIC);
    off = fmaf(p, inv, CODE_MAGIC - m);
    return m;
}
constexpr float CODE_NEAR = 0.5f - 0x1p-15f;
// A quotient that near to h, `whole` + 1/2 or - 1/2 on the side of `off`: 127 p against h a, both divided by 256 against overflow. h a is t + low exactly; 127 p lies within 2^-13 a of it and both are
// multiples of 2^-33 a, so their difference from t is exact as well. On a tie the rounding of h itself takes the even side.
__device__ __forceinline__ float code_bits_exact(float p, float m, float off, float most) {
    const float h = m - CODE_MAGIC + (off > 0.f ? 0.5f : -0.5f), a = most * 0x1p-8f;
    const float t = h * a, low = fmaf(h, a, -t), d = fmaf(127.f, p * 0x1p-8f, -t);
    return CODE_MAGIC + rintf(h + (d > low ? 0.25f : d < low ? -0.25f : 0.f));
}
__device__ __forceinline__ int code_of(float p, const RowCode &c) {
    if (c.most == 0.f) return 0;
    float off, m = code_bits(p, c.inv, off);
    if (fabsf(off) > CODE_NEAR) m = code_bits_exact(p, m, off, c.most);
    return static_cast<int8_t>(__float_as_uint(m));
}
// Eight codes; whether one of them lies near a half is asked once.
__device__ __forceinline__ uint2 codes8(const float (&p)[8], const RowCode &c) {
    float m[8], off[8], far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = code_bits(p[j], c.inv, off[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j) far = fmaxf(far, fabsf(off[j]));
    if (far > CODE_NEAR) {
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = fabsf(off[j]) > CODE_NEAR ? code_bits_exact(p[j], m[j], off[j], c.most) : m[j];
    }
    uint32_t o[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(m[4 * h + 1]), __float_as_uint(m[4 * h]), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(m[4 * h + 3]), __float_as_uint(m[4 * h + 2]), 0x0c0c0400u);
        o[h] = c.most != 0.f ? lo | hi << 16 : 0;
    }
    return make_uint2(o[0], o[1]);
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Steps of a butterfly over the wavefront, between halves, rows of 16 lanes and inside rows: no trip through LDS. Swapping halves (or odd rows with even ones) of two registers and adding them up
// also makes one of two values, each in the lanes of its half (of its rows), for the price of one.
__device__ __forceinline__ float add_halves(float a, float b) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}
__device__ __forceinline__ float add_rows(float a, float b) {
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}
template <int S>
__device__ __forceinline__ uint32_t partner_in_row(uint32_t v) {
    constexpr int CTRL = S == 0 ? 0xB1 : S == 1 ? 0x4E : S == 2 ? 0x141 : 0x140;  // quads 1 0 3 2, 2 3 0 1; halves of a row and rows mirrored
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_in_rows(float v) {
    unrolled<4>([&](auto stage) { v += __uint_as_float(partner_in_row<decltype(stage)::value>(__float_as_uint(v))); });
    return v;
}
__device__ __forceinline__ uint32_t most_of_wave(uint32_t v) {
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(halves[0], halves[1]);
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(rows[0], rows[1]);
    unrolled<4>([&](auto stage) { v = max(v, partner_in_row<decltype(stage)::value>(v)); });
    return v;
}

// Sum (SUM) and maximum over the block, the same in every thread. A thread has CH sums, of chunks that lie 64 * WAVES apart: each is added up over the wavefront, and the results, one for every 64
// chunks of the row, as a tree: the row's two halves first, then halves of halves, its neighbours last. So a row's sum does not depend on how many wavefronts hold it, which a launch's number of
// rows decides, and the tree's first steps are those inside a wavefront in every form.
template <int WAVES, bool SUM, int CH>
__device__ __forceinline__ float block_sum_max(const float (&sum)[CH], uint32_t &most) {
    static_assert(CH == 1 || CH == 2 || CH == 4, "halves and rows of a wavefront");
    __shared__ uint2 part[WAVES];
    most = most_of_wave(most);
    float s = 0.f;
    if constexpr (SUM) {
        if constexpr (CH == 1) s = add_halves(sum[0], sum[0]), s = add_in_rows(add_rows(s, s));
        if constexpr (CH == 2) s = add_halves(sum[0], sum[1]), s = add_in_rows(add_rows(s, s)), s = add_halves(s, s);  // sums 0 and 1 in the halves
        if constexpr (CH == 4) s = add_in_rows(add_rows(add_halves(sum[0], sum[1]), add_halves(sum[2], sum[3]))), s = add_rows(s, s), s = add_halves(s, s);  // sums 0, 2, 1, 3 in the rows
    }
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_uint2(__float_as_uint(s), most);
        __syncthreads();
        float t[WAVES];
        most = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const uint2 v = part[i];
            t[i] = __uint_as_float(v.x);
            most = max(most, v.y);
        }
        if constexpr (SUM) {
#pragma unroll
            for (int n = WAVES / 2; n > 0; n /= 2)
#pragma unroll
                for (int i = 0; i < n; ++i) t[i] += t[i + n];
            s = t[0];
        }
    }
    return s;
}

// Rows of D elements, D a multiple of 8 and at most 64 * WAVES * CH * 8, every row of x, r, s on a 16-byte boundary and of q on an 8-byte one. A block holds its row in registers.
template <int DT, int WAVES, int CH, bool NORM, bool ADD>
__global__ __launch_bounds__(64 * WAVES) void quantize_kernel(QuantParams p) {
    constexpr int T = 64 * WAVES;
    if (blockIdx.y != 0) {
        p.x += p.to.x; p.w += p.to.w; p.r += p.to.r; p.s += p.to.s; p.q += p.to.q;
        p.scale = reinterpret_cast<float *>(reinterpret_cast<char *>(p.scale) + p.to.scale);
    }
    const int64_t row = blockIdx.x;
    const uint4 *x = reinterpret_cast<const uint4 *>(p.x + row * p.ldx * 2);
    const uint4 *w = reinterpret_cast<const uint4 *>(p.w);
    const int n = p.D / 8;
    uint4 v[CH], wv[NORM ? CH : 1];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = threadIdx.x + c * T;
        v[c] = i < n ? x[i] : make_uint4(0, 0, 0, 0);
    }
    if constexpr (NORM) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = threadIdx.x + c * T;
            wv[c] = i < n ? w[i] : make_uint4(0, 0, 0, 0);
        }
    }
    if constexpr (ADD) {
        const uint4 *r = reinterpret_cast<const uint4 *>(p.r + row * p.ldr * 2);
        uint4 *s = reinterpret_cast<uint4 *>(p.s + row * p.lds * 2);
        uint4 rv[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = threadIdx.x + c * T;
            rv[c] = i < n ? r[i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = threadIdx.x + c * T;
            v[c] = make_uint4(add_packed2<DT>(rv[c].x, v[c].x), add_packed2<DT>(rv[c].y, v[c].y), add_packed2<DT>(rv[c].z, v[c].z), add_packed2<DT>(rv[c].w, v[c].w));
            if (i < n) s[i] = v[c];
        }
    }
    float f[CH][8], sum[CH], zero = -0.f;
    asm("" : "+v"(zero));  // products by fused operations that take their factors from 16 bits (fp16), instead of two conversions and a multiplication
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t u[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
        const uint32_t g[4] = {wv[NORM ? c : 0].x, wv[NORM ? c : 0].y, wv[NORM ? c : 0].z, wv[NORM ? c : 0].w};
        sum[c] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a = lo_half_to_f32<DT>(u[j]), b = hi_half_to_f32<DT>(u[j]);
            if constexpr (NORM) {
                sum[c] = fmaf(a, a, fmaf(b, b, sum[c]));
                a = fmaf(a, lo_half_to_f32<DT>(g[j]), zero);
                b = fmaf(b, hi_half_to_f32<DT>(g[j]), zero);
            }
            f[c][2 * j] = a;
            f[c][2 * j + 1] = b;
            most = max(most, max(abs_bits(a), abs_bits(b)));
        }
    }
    const float squares = block_sum_max<WAVES, NORM>(sum, most);
    const RowCode code = row_code(most, NORM ? rsqrtf(squares / static_cast<float>(p.D) + p.eps) : 1.f);
    if (threadIdx.x == 0) p.scale[row] = code.scale;
    uint2 *q = reinterpret_cast<uint2 *>(p.q + row * p.ldq);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = threadIdx.x + c * T;
        if (i >= n) continue;
        q[i] = codes8(f[c], code);
    }
}

// Any length and alignment: element loads, x (ADD: the stored sum, by the thread that stored it) read twice.
template <int DT, bool NORM, bool ADD>
__global__ __launch_bounds__(256) void quantize_any_kernel(QuantParams p) {
    const int64_t row = blockIdx.x;
    const uint16_t *x = reinterpret_cast<const uint16_t *>(p.x) + row * p.ldx, *w = reinterpret_cast<const uint16_t *>(p.w);
    const uint16_t *r = reinterpret_cast<const uint16_t *>(p.r) + row * p.ldr;
    uint16_t *s = reinterpret_cast<uint16_t *>(p.s) + row * p.lds;
    float sum[1] = {0.f};
    uint32_t most = 0;
    for (int i = threadIdx.x; i < p.D; i += 256) {
        float a = half_to_f32<DT>(x[i]);
        if constexpr (ADD) {
            s[i] = f32_to_half<DT>(half_to_f32<DT>(r[i]) + a);
            a = half_to_f32<DT>(s[i]);
        }
        sum[0] = fmaf(a, a, sum[0]);
        if constexpr (NORM) a *= half_to_f32<DT>(w[i]);
        most = max(most, abs_bits(a));
    }
    const float squares = block_sum_max<4, NORM>(sum, most);
    const RowCode code = row_code(most, NORM ? rsqrtf(squares / static_cast<float>(p.D) + p.eps) : 1.f);
    if (threadIdx.x == 0) p.scale[row] = code.scale;
    for (int i = threadIdx.x; i < p.D; i += 256) {
        const float a = half_to_f32<DT>(ADD ? s[i] : x[i]);
        p.q[row * p.ldq + i] = static_cast<char>(code_of(NORM ? a * half_to_f32<DT>(w[i]) : a, code));
    }
}

// Without the addition, rows of a large launch are held by fewer wavefronts with four chunks a lane: more rows are under way on a CU, and a row's meeting costs less. Quantised / normed, us:
// 2103 x 4096 9.6 -> 9.3 / 9.0 -> 8.6, 4096 x 5504 15.6 -> 16.0 / 17.2 -> 16.3, 4096 x 16384 37.7 -> 37.5 / 41.2 -> 38.1, 1024 x 11008 10.7 -> 10.5 / 11.4 -> 10.6; smaller ones lose, 1024 x 4096
// 6.5 -> 6.9 / 6.0 -> 6.3, 2048 x 2048 6.7 -> 6.8 / 6.0 -> 6.4, 512 x 8192 5.9 -> 6.6 / 5.8 -> 6.3. With the addition the form made no difference worth having (4096 x 8192 37.8 and 38.3).
constexpr int64_t MANY_VALUES = 1 << 23;

template <int DT, bool NORM, bool ADD>
void launch_rows(const QuantParams &p, int64_t rows, int ranks, bool vec, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(ranks));
    const int n = p.D / 8;  // 16-byte chunks per row
    if constexpr (!ADD) {
        if (vec && n > 64 && rows * p.D > MANY_VALUES) {
            if (n <= 256) hipLaunchKernelGGL((quantize_kernel<DT, 1, 4, NORM, ADD>), grid, dim3(64), 0, s, p);
            else if (n <= 512) hipLaunchKernelGGL((quantize_kernel<DT, 2, 4, NORM, ADD>), grid, dim3(128), 0, s, p);
            else if (n <= 1024) hipLaunchKernelGGL((quantize_kernel<DT, 4, 4, NORM, ADD>), grid, dim3(256), 0, s, p);
            else hipLaunchKernelGGL((quantize_kernel<DT, 8, 4, NORM, ADD>), grid, dim3(512), 0, s, p);
            return;
        }
    }
    if (!vec) hipLaunchKernelGGL((quantize_any_kernel<DT, NORM, ADD>), grid, dim3(256), 0, s, p);
    else if (n <= 64) hipLaunchKernelGGL((quantize_kernel<DT, 1, 1, NORM, ADD>), grid, dim3(64), 0, s, p);
    else if (n <= 256) hipLaunchKernelGGL((quantize_kernel<DT, 4, 1, NORM, ADD>), grid, dim3(256), 0, s, p);
    else if (n <= 512) hipLaunchKernelGGL((quantize_kernel<DT, 8, 1, NORM, ADD>), grid, dim3(512), 0, s, p);
    else if (n <= 1024) hipLaunchKernelGGL((quantize_kernel<DT, 8, 2, NORM, ADD>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((quantize_kernel<DT, 16, 2, NORM, ADD>), grid, dim3(1024), 0, s, p);
}

// A launch has at most 2^32 - 1 threads; further rows go into further launches.
constexpr int64_t ROWS_PER_LAUNCH = 1ll << 20;

template <int DT, bool NORM, bool ADD>
int launch(QuantParams p, int64_t rows, int ranks, bool vec, hipStream_t s) {
    for (; rows > 0; rows -= ROWS_PER_LAUNCH) {
        launch_rows<DT, NORM, ADD>(p, rows < ROWS_PER_LAUNCH ? rows : ROWS_PER_LAUNCH, ranks, vec, s);
        TPAMD_HIP(hipGetLastError());
        p.x += ROWS_PER_LAUNCH * p.ldx * 2;
        p.q += ROWS_PER_LAUNCH * p.ldq;
        p.scale += ROWS_PER_LAUNCH;
        if constexpr (ADD) {
            p.r += ROWS_PER_LAUNCH * p.ldr * 2;
            p.s += ROWS_PER_LAUNCH * p.lds * 2;
        }
    }
    return TPAMD_OK;
}

template <bool NORM, bool ADD>
int quantize_check(const char *who, const QuantParams &p, int64_t rows, int64_t D, int dtype) {
    TPAMD_REQUIRE(rows >= 0 && D >= 0 && rows < (1ll << 31) && D < (1ll << 30), "%s: dimension negative or too large (rows=%lld D=%lld)", who, (long long)rows, (long long)D);
    TPAMD_REQUIRE(dtype == TPAMD_BF16 || dtype == TPAMD_F16, "%s: rows of bfloat16 or float16 are quantised, not dtype %d", who, dtype);
    if (rows == 0) return TPAMD_OK;
    TPAMD_REQUIRE(p.scale != nullptr && (D == 0 || (p.x != nullptr && p.q != nullptr && (!NORM || p.w != nullptr) && (!ADD || (p.r != nullptr && p.s != nullptr)))),
                  "%s: null pointer", who);
    TPAMD_REQUIRE(p.ldx >= D && p.ldq >= D && (!ADD || (p.ldr >= D && p.lds >= D)), "%s: leading dimension smaller than the row (ldx=%lld ldr=%lld lds=%lld ldq=%lld)", who,
                  (long long)p.ldx, (long long)p.ldr, (long long)p.lds, (long long)p.ldq);
    TPAMD_REQUIRE(aligned(p.x, 2) && aligned(p.w, 2) && aligned(p.r, 2) && aligned(p.s, 2) && aligned(p.scale, 4), "%s: a pointer is not aligned to its type", who);
    return TPAMD_OK;
}

// Rows for quantize_kernel.
template <bool NORM, bool ADD>
bool quantize_vec(const QuantParams &p, int64_t D) {
    return D > 0 && D % 8 == 0 && D <= 16384 && aligned(p.x, 16) && p.ldx % 8 == 0 && aligned(p.q, 8) && p.ldq % 8 == 0 && (!NORM || aligned(p.w, 16)) &&
                     (!ADD || (aligned(p.r, 16) && p.ldr % 8 == 0 && aligned(p.s, 16) && p.lds % 8 == 0));
}

template <bool NORM, bool ADD>
int quantize_entry(const char *who, const QuantParams &p, int64_t rows, int64_t D, int dtype, void *stream, int ranks = 1) {
    if (int rc = quantize_check<NORM, ADD>(who, p, rows, D, dtype); rc != TPAMD_OK || rows == 0) return rc;
    const bool vec = quantize_vec<NORM, ADD>(p, D);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == TPAMD_BF16 ? launch<TPAMD_BF16, NORM, ADD>(p, rows, ranks, vec, s) : launch<TPAMD_F16, NORM, ADD>(p, rows, ranks, vec, s);
}

// Several ranks' rows, two in a launch where quantize_kernel takes both.
template <bool NORM, bool ADD>
int quantize_ranks(const char *who, int n, const tpamd_q8_rank *ranks, const QuantParams &form, int64_t rows, int64_t D, int dtype, void *stream) {
    auto params = [&](const tpamd_q8_rank &r) {
        QuantParams p = form;
        p.x = static_cast<const char *>(r.x); p.w = static_cast<const char *>(r.w); p.r = static_cast<const char *>(r.r);
        p.s = static_cast<char *>(r.sum); p.q = static_cast<char *>(r.q); p.scale = static_cast<float *>(r.scale);
        return p;
    };
    for (int i = 0; i < n; ++i)
        if (int rc = quantize_check<NORM, ADD>(who, params(ranks[i]), rows, D, dtype); rc != TPAMD_OK) return rc;
    for (int i = 0; i < n; ++i) {
        QuantParams p = params(ranks[i]);
        int together = 1;
        if (i + 1 < n) {
            const QuantParams q = params(ranks[i + 1]);
            if (quantize_vec<NORM, ADD>(p, D) && quantize_vec<NORM, ADD>(q, D)) {
                p.to = {bytes_from(p.x, q.x), bytes_from(p.w, q.w), bytes_from(p.r, q.r), bytes_from(p.s, q.s), bytes_from(p.q, q.q), bytes_from(p.scale, q.scale)};
                together = 2;
                ++i;
            }
        }
        if (int rc = quantize_entry<NORM, ADD>(who, p, rows, D, dtype, stream, together); rc != TPAMD_OK) return rc;
    }
    return TPAMD_OK;
}

// A product as an fp32 value of its own: the compiler would otherwise make one instruction of it and its conversion to fp16, which rounds once where the packed conversion behind
// the product rounds twice, and a row's bits would depend on its alignment.
__device__ __forceinline__ float product(float a, float b) {
    float v = a * b;
    asm("" : "+v"(v));
    return v;
}

// y = q * scale in fp32, rounded to the dtype: blockIdx.y takes every gridDim.y-th row; VEC (rows of q on boundaries of V, of y on 16 bytes, D a multiple of V): a thread
// has V codes, 16 bytes of y, 256 V further on once more.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void dequantize_kernel(const char *q, const float *scale, char *y, int64_t rows, int D, int64_t ldq, int64_t ldy) {
    constexpr int V = !VEC ? 1 : DT == TPAMD_F32 ? 4 : 8, U = VEC ? 2 : 1;
    const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * (U * 256) + threadIdx.x) * V;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float f = scale[row];
        if constexpr (VEC) {
            uint2 u[U];
#pragma unroll
            for (int h = 0; h < U; ++h) {
                const int64_t i = i0 + h * (256 * V);
                u[h] = make_uint2(0, 0);
                if (i < D) {
                    if constexpr (V == 8) u[h] = *reinterpret_cast<const uint2 *>(q + row * ldq + i);
                    else u[h].x = *reinterpret_cast<const uint32_t *>(q + row * ldq + i);
                }
            }
#pragma unroll
            for (int h = 0; h < U; ++h) {
                const int64_t i = i0 + h * (256 * V);
                if (i >= D) break;
                const uint32_t a[2] = {u[h].x, u[h].y};
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = product(static_cast<float>(static_cast<int8_t>(a[e >> 2] >> (8 * (e & 3)))), f);
                if constexpr (DT == TPAMD_F32)
                    *reinterpret_cast<float4 *>(y + (row * ldy + i) * 4) = make_float4(v[0], v[1], v[2], v[3]);
                else
                    *reinterpret_cast<uint4 *>(y + (row * ldy + i) * 2) =
                        make_uint4(pack2_half<DT>(v[0], v[1]), pack2_half<DT>(v[2], v[3]), pack2_half<DT>(v[4], v[5]), pack2_half<DT>(v[6], v[7]));
            }
        } else if (i0 < D) {
            const float v = product(static_cast<float>(static_cast<int8_t>(q[row * ldq + i0])), f);
            if constexpr (DT == TPAMD_F32) reinterpret_cast<float *>(y)[row * ldy + i0] = v;
            else reinterpret_cast<uint16_t *>(y)[row * ldy + i0] = f32_to_half<DT>(v);
        }
    }
}

template <int DT>
void launch_dequantize(const char *q, const float *scale, char *y, int64_t rows, int D, int64_t ldq, int64_t ldy, bool vec, hipStream_t s) {
    const int64_t per = !vec ? 256 : DT == TPAMD_F32 ? 2048 : 4096;
    const unsigned columns = static_cast<unsigned>((D + per - 1) / per);
    // rows in turn once 2^22 blocks are out
    const int64_t most = (1 << 22) / columns > 0 ? (1 << 22) / columns : 1;
    const int64_t by = rows < 65535 ? rows : 65535;
    const dim3 grid(columns, static_cast<unsigned>(by < most ? by : most));
    if (vec) hipLaunchKernelGGL((dequantize_kernel<DT, true>), grid, dim3(256), 0, s, q, scale, y, rows, D, ldq, ldy);
    else hipLaunchKernelGGL((dequantize_kernel<DT, false>), grid, dim3(256), 0, s, q, scale, y, rows, D, ldq, ldy);
}

}  // namespace
}  // namespace tpamd

using namespace tpamd;

extern "C" int tpamd_quantize_rows(const void *x_dev, void *q_dev, void *scale_dev, int64_t rows, int64_t D, int64_t ldx, int64_t ldq, int dtype, void *stream) {
    QuantParams p{};
    p.x = static_cast<const char *>(x_dev); p.q = static_cast<char *>(q_dev); p.scale = static_cast<float *>(scale_dev);
    p.ldx = ldx; p.ldq = ldq; p.D = static_cast<int>(D);
    return quantize_entry<false, false>("tpamd_quantize_rows", p, rows, D, dtype, stream);
}

extern "C" int tpamd_rms_norm_q8(const void *x_dev, const void *w_dev, void *q_dev, void *scale_dev, int64_t rows, int64_t D, int64_t ldx, int64_t ldq, float eps, int dtype,
                                 void *stream) {
    QuantParams p{};
    p.x = static_cast<const char *>(x_dev); p.w = static_cast<const char *>(w_dev); p.q = static_cast<char *>(q_dev); p.scale = static_cast<float *>(scale_dev);
    p.ldx = ldx; p.ldq = ldq; p.D = static_cast<int>(D); p.eps = eps;
    return quantize_entry<true, false>("tpamd_rms_norm_q8", p, rows, D, dtype, stream);
}

extern "C" int tpamd_add_rms_norm_q8(const void *x_dev, const void *r_dev, const void *w_dev, void *sum_dev, void *q_dev, void *scale_dev, int64_t rows, int64_t D, int64_t ldx,
                                     int64_t ldr, int64_t ldsum, int64_t ldq, float eps, int dtype, void *stream) {
    QuantParams p{};
    p.x = static_cast<const char *>(x_dev); p.r = static_cast<const char *>(r_dev); p.w = static_cast<const char *>(w_dev);
    p.s = static_cast<char *>(sum_dev); p.q = static_cast<char *>(q_dev); p.scale = static_cast<float *>(scale_dev);
    p.ldx = ldx; p.ldr = ldr; p.lds = ldsum; p.ldq = ldq; p.D = static_cast<int>(D); p.eps = eps;
    return quantize_entry<true, true>("tpamd_add_rms_norm_q8", p, rows, D, dtype, stream);
}

extern "C" int tpamd_rows_q8_ranks(int n, const tpamd_q8_rank *ranks, int64_t rows, int64_t D, int64_t ldx, int64_t ldr, int64_t ldsum, int64_t ldq, float eps, int dtype, void *stream) {
    const char *who = "tpamd_rows_q8_ranks";
    TPAMD_REQUIRE(n >= 0 && (n == 0 || ranks != nullptr), "%s: null pointer", who);
    if (n == 0) return TPAMD_OK;
    for (int i = 1; i < n; ++i)
        TPAMD_REQUIRE((ranks[i].w == nullptr) == (ranks[0].w == nullptr) && (ranks[i].r == nullptr) == (ranks[0].r == nullptr), "%s: ranks of different forms", who);
    TPAMD_REQUIRE(ranks[0].w != nullptr || ranks[0].r == nullptr, "%s: an addition goes with a norm", who);
    QuantParams p{};
    p.ldx = ldx; p.ldr = ldr; p.lds = ldsum; p.ldq = ldq; p.D = static_cast<int>(D); p.eps = eps;
    if (ranks[0].w == nullptr) return quantize_ranks<false, false>(who, n, ranks, p, rows, D, dtype, stream);
    if (ranks[0].r == nullptr) return quantize_ranks<true, false>(who, n, ranks, p, rows, D, dtype, stream);
    return quantize_ranks<true, true>(who, n, ranks, p, rows, D, dtype, stream);
}

extern "C" int tpamd_dequantize_rows(const void *q_dev, const void *scale_dev, void *y_dev, int64_t rows, int64_t D, int64_t ldq, int64_t ldy, int dtype, void *stream) {
    const char *who = "tpamd_dequantize_rows";
    TPAMD_REQUIRE(rows >= 0 && D >= 0 && rows < (1ll << 31) && D < (1ll << 30), "%s: dimension negative or too large (rows=%lld D=%lld)", who, (long long)rows, (long long)D);
    TPAMD_REQUIRE(dtype == TPAMD_BF16 || dtype == TPAMD_F16 || dtype == TPAMD_F32, "%s: unknown dtype %d", who, dtype);
    if (rows == 0 || D == 0) return TPAMD_OK;
    TPAMD_REQUIRE(q_dev != nullptr && scale_dev != nullptr && y_dev != nullptr, "%s: null pointer", who);
    TPAMD_REQUIRE(ldq >= D && ldy >= D, "%s: leading dimension smaller than the row (ldq=%lld ldy=%lld)", who, (long long)ldq, (long long)ldy);
    TPAMD_REQUIRE(aligned(scale_dev, 4) && aligned(y_dev, dtype == TPAMD_F32 ? 4 : 2), "%s: a pointer is not aligned to its type", who);
    const char *q = static_cast<const char *>(q_dev);
    const float *scale = static_cast<const float *>(scale_dev);
    char *y = static_cast<char *>(y_dev);
    const int v = dtype == TPAMD_F32 ? 4 : 8;
    const bool vec = D % v == 0 && aligned(q, v) && ldq % v == 0 && aligned(y, 16) && ldy % v == 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int d = static_cast<int>(D);
    if (dtype == TPAMD_BF16) launch_dequantize<TPAMD_BF16>(q, scale, y, rows, d, ldq, ldy, vec, s);
    else if (dtype == TPAMD_F16) launch_dequantize<TPAMD_F16>(q, scale, y, rows, d, ldq, ldy, vec, s);
    else launch_dequantize<TPAMD_F32>(q, scale, y, rows, d, ldq, ldy, vec, s);
    TPAMD_HIP(hipGetLastError());
    return TPAMD_OK;
}
