#include "a8.h"
#include "a8_model.h"

namespace tpamd {
namespace {

// gemm_a8_any_kernel: any shape, pitch and alignment. 64 x 64 outputs a block, K in stages of 64 bytes that are read one byte at a time (what lies behind the ends is zero)
// and multiplied four at a time (v_dot4_i32_i8), 4 x 4 outputs a thread. Bound by the latency of those loads: 1 / 64 / 701 / 4096 rows of 4096 x 2750 338 / 483 / 415 / 1128 us, where the kernels that take
// whole pieces of 16 need 4.5 / 8.6 / 16.1 / 45.5 for a K of 2752 on rows in lines.
template <int DT, bool PAIR>
__global__ __launch_bounds__(256) void gemm_a8_any_kernel(A8Params p) {
    constexpr int B = 64, PITCH = 68, MATS = PAIR ? 2 : 1;
    __shared__ __align__(16) char xs[B * PITCH], ws[MATS][B * PITCH];
    const int64_t tiles_n = (p.N + B - 1) / B;
    const int64_t m0 = blockIdx.x / tiles_n * B, n0 = blockIdx.x % tiles_n * B;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    int acc[MATS][4][4] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += B) {
        for (int i = tid; i < B * B; i += 256) {
            const int row = i >> 6, c = i & 63;
            const bool kin = k0 + c < p.K;
            xs[row * PITCH + c] = kin && m0 + row < p.M ? p.x[(m0 + row) * p.ldx + k0 + c] : 0;
            ws[0][row * PITCH + c] = kin && n0 + row < p.N ? p.w[(n0 + row) * p.ldw + k0 + c] : 0;
            if constexpr (PAIR) ws[1][row * PITCH + c] = kin && n0 + row < p.N ? p.w2[(n0 + row) * p.ldw + k0 + c] : 0;
        }
        __syncthreads();
        for (int c = 0; c < B; c += 4) {
            int xv[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) xv[a] = *reinterpret_cast<const int *>(xs + (ty * 4 + a) * PITCH + c);
#pragma unroll
            for (int t = 0; t < MATS; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int wv = *reinterpret_cast<const int *>(ws[t] + (tx + 16 * b) * PITCH + c);
#pragma unroll
                    for (int a = 0; a < 4; ++a) acc[t][a][b] = __builtin_amdgcn_sdot4(xv[a], wv, acc[t][a][b], false);
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int64_t m = m0 + ty * 4 + a;
        if (m >= p.M) continue;
        const float sx = p.sx[m];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int64_t n = n0 + tx + 16 * b;
            if (n >= p.N) continue;
            uint16_t out;
            if constexpr (PAIR) {
                out = a8_round<DT>(a8_gated(a8_linear(acc[0][a][b], sx, p.sw[n], 0.f), a8_linear(acc[1][a][b], sx, p.sw2[n], 0.f)));
            } else {
                out = a8_round<DT>(a8_act(a8_linear(acc[0][a][b], sx, p.sw[n], p.bias != nullptr ? half_to_f32<DT>(reinterpret_cast<const uint16_t *>(p.bias)[n]) : 0.f), p.act));
                if (p.addend != nullptr)
                    out = f32_to_half<DT>(half_to_f32<DT>(out) + half_to_f32<DT>(reinterpret_cast<const uint16_t *>(p.addend)[m * p.ldadd + n]));
            }
            uint16_t *y = reinterpret_cast<uint16_t *>(p.y) + m * p.ldy + n;
            *y = out;
            if (p.copy != 0) *reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(y) + p.copy) = out;
        }
    }
}

template <bool PAIR>
int launch_any(const A8Params &p, int dtype, hipStream_t s) {
    const int64_t tiles = (static_cast<int64_t>(p.M) + 63) / 64 * ((static_cast<int64_t>(p.N) + 63) / 64);
    TPAMD_REQUIRE(tiles < (1ll << 24), "a8: too many tiles");  // 2^32 threads
    const dim3 grid(static_cast<unsigned>(tiles));
    if (dtype == TPAMD_BF16) hipLaunchKernelGGL((gemm_a8_any_kernel<TPAMD_BF16, PAIR>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((gemm_a8_any_kernel<TPAMD_F16, PAIR>), grid, dim3(256), 0, s, p);
    TPAMD_HIP(hipGetLastError());
    return TPAMD_OK;
}

// Whether operands of a8_fast go to the streaming kernel; else `tile` is the choice among tiles.
bool a8_streams(const A8Params &p, bool pair, int cus, A8Choice *tile) {
    const Tuning &t = tuning();
    const bool stream = t.stream != 0 && t.a8_tile == TUNE_UNSET && stream_a8_takes(p, pair, 1, cus);
    if (stream && t.stream == 1) return true;
    *tile = a8_choose(pair, p.M, p.N, p.K, cus, static_cast<int64_t>(scratch_reserve(cus)));
    // Tiles have to be predicted a sixth faster (the two models' errors at few rows): with that the choice is 1.2 % off the best of both in the geometric mean over 300 shapes of 1-64 rows, 1.0 % on
    // 150 others (worst 38 %), streaming always 1.9 and 2.6 (16384 x 1376 at 45 rows 13.8 us streamed, 9.2 on tiles; 5504 x 8192 the other way round at 62 rows)
    return stream && stream_a8_us(p, pair, cus) <= 1.2f * tile->us;
}

int a8_dispatch(const A8Params &p, bool pair, int dtype, hipStream_t s) {
    int dev = 0, cus = 256;
    TPAMD_HIP(hipGetDevice(&dev));
    if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
    if (a8_fast(p)) {
        A8Choice tile{};
        if (a8_streams(p, pair, cus, &tile)) return stream_a8(p, pair, dtype, 1, cus, s);
        const Tuning &t = tuning();
        if (t.a8_tile != TUNE_UNSET) tile = {t.a8_tile / 1000 / 64, t.a8_tile % 1000 / 64, 1, 0.f};
        if (t.a8_splits != TUNE_UNSET) tile.ranges = t.a8_splits < 1 ? 1 : t.a8_splits;
        return gemm_a8(p, pair, dtype, tile.tm, tile.tn, tile.ranges, s);
    }
    return pair ? launch_any<true>(p, dtype, s) : launch_any<false>(p, dtype, s);
}

int a8_check(const char *who, const A8Params &p, int64_t M, int64_t N, int64_t K, bool pair, int dtype) {
    TPAMD_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative dimension (M=%lld N=%lld K=%lld)", who, (long long)M, (long long)N, (long long)K);
    TPAMD_REQUIRE(M < (1ll << 30) && N < (1ll << 30), "%s: dimension of 2^30 or more (M=%lld N=%lld)", who, (long long)M, (long long)N);  // (indices of a tile behind the ends fit 32 bits)
    TPAMD_REQUIRE(dtype == TPAMD_BF16 || dtype == TPAMD_F16, "%s: outputs are bfloat16 or float16, not dtype %d", who, dtype);
    if (K > A8_MAX_K) {
        set_error("%s: K=%lld products of 8-bit codes may not fit 32 bits (at most %lld do)", who, (long long)K, (long long)A8_MAX_K);
        return TPAMD_ERR_UNSUPPORTED;
    }
    if (M == 0 || N == 0) return TPAMD_OK;
    TPAMD_REQUIRE(p.sx != nullptr && p.sw != nullptr && p.y != nullptr && (K == 0 || (p.x != nullptr && p.w != nullptr)), "%s: null pointer", who);
    TPAMD_REQUIRE(!pair || (p.sw2 != nullptr && (K == 0 || p.w2 != nullptr)), "%s: null pointer", who);
    TPAMD_REQUIRE(p.ldx >= K && p.ldw >= K && p.ldy >= N && (p.addend == nullptr || p.ldadd >= N),
                  "%s: leading dimension smaller than the row (ldx=%lld ldw=%lld ldadd=%lld ldy=%lld)", who, (long long)p.ldx, (long long)p.ldw, (long long)p.ldadd, (long long)p.ldy);
    TPAMD_REQUIRE(aligned(p.sx, 4) && aligned(p.sw, 4) && aligned(p.sw2, 4) && aligned(p.bias, 2) && aligned(p.addend, 2) && aligned(p.y, 2) && p.copy % 2 == 0,
                  "%s: a pointer is not aligned to its type", who);
    return TPAMD_OK;
}

int linear_a8(const char *who, const void *x, const void *sx, const void *w, const void *sw, const void *bias, const void *addend, int64_t ldadd, void *y, void *copy, int64_t M,
              int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldy, int dtype, int act, void *stream) {
    A8Params p{};
    p.x = static_cast<const char *>(x); p.w = static_cast<const char *>(w);
    p.sx = static_cast<const float *>(sx); p.sw = static_cast<const float *>(sw);
    p.bias = static_cast<const char *>(bias); p.addend = static_cast<const char *>(addend);
    p.y = static_cast<char *>(y); p.copy = bytes_from(y, copy);
    p.ldx = ldx; p.ldw = ldw; p.ldadd = ldadd; p.ldy = ldy; p.act = act;
    if (int rc = a8_check(who, p, M, N, K, false, dtype); rc != TPAMD_OK) return rc;
    TPAMD_REQUIRE(act == TPAMD_ACT_NONE || act == TPAMD_ACT_GELU, "%s: unknown activation %d", who, act);
    if (M == 0 || N == 0) return TPAMD_OK;
    p.M = static_cast<int>(M); p.N = static_cast<int>(N); p.K = static_cast<int>(K);
    return a8_dispatch(p, false, dtype, static_cast<hipStream_t>(stream));
}

// Several ranks' products of one form, two in a launch where each by itself would stream and half the CUs hold a rank's columns; else one after another. 216 random shapes of 1-64 rows, time of one
// launch for both in that of two: Linears 0.61, pairs 0.70, none above 1.01.
int a8_ranks(const char *who, int n, const tpamd_a8_rank *ranks, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldy, bool pair, int dtype, int act, hipStream_t s) {
    TPAMD_REQUIRE(n >= 0 && (n == 0 || ranks != nullptr), "%s: null pointer", who);
    TPAMD_REQUIRE(act == TPAMD_ACT_NONE || act == TPAMD_ACT_GELU, "%s: unknown activation %d", who, act);
    auto params = [&](const tpamd_a8_rank &r) {
        A8Params p{};
        p.x = static_cast<const char *>(r.x); p.w = static_cast<const char *>(r.w); p.w2 = pair ? static_cast<const char *>(r.w2) : nullptr;
        p.sx = static_cast<const float *>(r.xscale); p.sw = static_cast<const float *>(r.wscale); p.sw2 = pair ? static_cast<const float *>(r.w2scale) : nullptr;
        p.bias = pair ? nullptr : static_cast<const char *>(r.bias); p.y = static_cast<char *>(r.y);
        p.ldx = ldx; p.ldw = ldw; p.ldy = ldy; p.act = act;
        return p;
    };
    for (int i = 0; i < n; ++i)
        if (int rc = a8_check(who, params(ranks[i]), M, N, K, pair, dtype); rc != TPAMD_OK) return rc;
    if (M == 0 || N == 0) return TPAMD_OK;
    int dev = 0, cus = 256;
    TPAMD_HIP(hipGetDevice(&dev));
    if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
    for (int i = 0; i < n; ++i) {
        A8Params p = params(ranks[i]), q = params(ranks[i + 1 < n ? i + 1 : i]);
        p.M = q.M = static_cast<int>(M); p.N = q.N = static_cast<int>(N); p.K = q.K = static_cast<int>(K);
        A8Choice tile{};
        if (i + 1 < n && a8_fast(p) && a8_fast(q) && (p.bias == nullptr) == (q.bias == nullptr) && stream_a8_takes(p, pair, 2, cus) && a8_streams(p, pair, cus, &tile)) {
            p.to = {bytes_from(p.x, q.x), bytes_from(p.w, q.w), bytes_from(p.w2, q.w2), bytes_from(p.sx, q.sx), bytes_from(p.sw, q.sw), bytes_from(p.sw2, q.sw2),
                    bytes_from(p.bias, q.bias), bytes_from(p.y, q.y)};
            if (int rc = stream_a8(p, pair, dtype, 2, cus, s); rc != TPAMD_OK) return rc;
            ++i;
        } else if (int rc = a8_dispatch(p, pair, dtype, s); rc != TPAMD_OK) {
            return rc;
        }
    }
    return TPAMD_OK;
}

}  // namespace
}  // namespace tpamd

using namespace tpamd;

extern "C" int tpamd_linear_a8(const void *x_dev, const void *xscale_dev, const void *w_dev, const void *wscale_dev, const void *bias_dev, void *y_dev, int64_t M, int64_t N,
                               int64_t K, int64_t ldx, int64_t ldw, int64_t ldy, int dtype, int act, void *stream) {
    return linear_a8("tpamd_linear_a8", x_dev, xscale_dev, w_dev, wscale_dev, bias_dev, nullptr, 0, y_dev, nullptr, M, N, K, ldx, ldw, ldy, dtype, act, stream);
}

extern "C" int tpamd_linear_a8_add(const void *x_dev, const void *xscale_dev, const void *w_dev, const void *wscale_dev, const void *bias_dev, const void *addend_dev, void *y_dev,
                                   void *copy_dev, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldadd, int64_t ldy, int dtype, int act, void *stream) {
    const char *who = "tpamd_linear_a8_add";
    TPAMD_REQUIRE(addend_dev != nullptr || M == 0 || N == 0, "%s: addend is NULL", who);
    TPAMD_REQUIRE(copy_dev == nullptr || copy_dev != y_dev, "%s: the copy is y", who);
    return linear_a8(who, x_dev, xscale_dev, w_dev, wscale_dev, bias_dev, addend_dev, ldadd, y_dev, copy_dev, M, N, K, ldx, ldw, ldy, dtype, act, stream);
}

extern "C" int tpamd_swiglu_up_a8(const void *x_dev, const void *xscale_dev, const void *wg_dev, const void *gscale_dev, const void *wu_dev, const void *uscale_dev, void *h_dev,
                                  int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldh, int dtype, void *stream) {
    A8Params p{};
    p.x = static_cast<const char *>(x_dev); p.w = static_cast<const char *>(wg_dev); p.w2 = static_cast<const char *>(wu_dev);
    p.sx = static_cast<const float *>(xscale_dev); p.sw = static_cast<const float *>(gscale_dev); p.sw2 = static_cast<const float *>(uscale_dev);
    p.y = static_cast<char *>(h_dev);
    p.ldx = ldx; p.ldw = ldw; p.ldy = ldh;
    if (int rc = a8_check("tpamd_swiglu_up_a8", p, M, N, K, true, dtype); rc != TPAMD_OK) return rc;
    if (M == 0 || N == 0) return TPAMD_OK;
    p.M = static_cast<int>(M); p.N = static_cast<int>(N); p.K = static_cast<int>(K);
    return a8_dispatch(p, true, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int tpamd_linear_a8_ranks(int n, const tpamd_a8_rank *ranks, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldy, int dtype, int act, void *stream) {
    return a8_ranks("tpamd_linear_a8_ranks", n, ranks, M, N, K, ldx, ldw, ldy, false, dtype, act, static_cast<hipStream_t>(stream));
}

extern "C" int tpamd_swiglu_up_a8_ranks(int n, const tpamd_a8_rank *ranks, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldh, int dtype, void *stream) {
    return a8_ranks("tpamd_swiglu_up_a8_ranks", n, ranks, M, N, K, ldx, ldw, ldh, true, dtype, TPAMD_ACT_NONE, static_cast<hipStream_t>(stream));
}
