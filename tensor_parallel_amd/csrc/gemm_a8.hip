#include "a8.h"
#include "gemm_tile.h"

namespace tpamd {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

constexpr int A8_BK = 128;  // K elements (bytes of a row) per stage

struct A8Tiles {
    int tiles_m, tiles_n;
    int kt_per_split, splits;  // K tiles of a range, ranges
    int *ws;                   // partial tiles
    int store, add;            // bytes per access that the rows of the outputs and of the addend allow: 16, 8 or 2
};

// Four outputs n..n+3 of a row from their sums (u: the up sums of a pair), before the addend.
template <int DT, int MODE>
__device__ __forceinline__ uint2 a8_finish4(const A8Params &p, const i32x4 &g, const i32x4 &u, float sx, const float (&sw)[4], const float (&sw2)[4], const float (&bias)[4]) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = a8_scaled(g[j], sx, sw[j]);
        if constexpr (MODE == MODE_SWIGLU) {
            v[j] = a8_gated(v[j], a8_scaled(u[j], sx, sw2[j]));
        } else {
            v[j] = a8_linear(v[j], bias[j], p.act);
        }
    }
    return make_uint2(a8_round2<DT>(v[0], v[1]), a8_round2<DT>(v[2], v[3]));
}

// What four columns have in common (of those there are: the last one again behind it).
template <int DT, int MODE>
__device__ __forceinline__ void a8_columns(const A8Params &p, int n, float (&sw)[4], float (&sw2)[4], float (&bias)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = n + j < p.N ? n + j : p.N - 1;
        sw[j] = p.sw[c];
        sw2[j] = MODE == MODE_SWIGLU ? p.sw2[c] : 0.f;
        bias[j] = MODE == MODE_LINEAR && p.bias != nullptr ? half_to_f32<DT>(reinterpret_cast<const uint16_t *>(p.bias)[c]) : 0.f;
    }
}

// `count` (up to 8) values of a row from or to memory whose rows allow accesses of `bytes`.
__device__ __forceinline__ uint4 load_values(const char *from, int count, int bytes) {
    uint4 v = make_uint4(0, 0, 0, 0);
    uint32_t *e = &v.x;
    if (bytes == 16 && count == 8) return *reinterpret_cast<const uint4 *>(from);
    if (bytes >= 8 && (count == 8 || count == 4)) {
        const uint2 a = *reinterpret_cast<const uint2 *>(from);
        v.x = a.x; v.y = a.y;
        if (count == 8) {
            const uint2 b = *reinterpret_cast<const uint2 *>(from + 8);
            v.z = b.x; v.w = b.y;
        }
        return v;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < count) e[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(from)[j]) << (16 * (j & 1));
    return v;
}
__device__ __forceinline__ void store_values(char *to, uint4 v, int count, int bytes) {
    if (bytes == 16 && count == 8) {
        *reinterpret_cast<uint4 *>(to) = v;
    } else if (bytes >= 8 && (count == 8 || count == 4)) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(v.x, v.y);
        if (count == 8) *reinterpret_cast<uint2 *>(to + 8) = make_uint2(v.z, v.w);
    } else {
        const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) reinterpret_cast<uint16_t *>(to)[j] = static_cast<uint16_t>(e[j >> 1] >> (16 * (j & 1)));
    }
}
// Up to 8 outputs of row m from column n on, with the addend, to where they go.
template <int DT, int MODE>
__device__ __forceinline__ void a8_put(const A8Params &p, const A8Tiles &t, uint4 v, int m, int n, int most) {
    const int count = p.N - n < most ? p.N - n : most;
    if constexpr (MODE == MODE_LINEAR) {
        if (p.addend != nullptr) {
            const uint4 a = load_values(p.addend + (static_cast<int64_t>(m) * p.ldadd + n) * 2, count, t.add);
            v = make_uint4(add_packed2<DT>(v.x, a.x), add_packed2<DT>(v.y, a.y), add_packed2<DT>(v.z, a.z), add_packed2<DT>(v.w, a.w));
        }
    }
    char *y = p.y + (static_cast<int64_t>(m) * p.ldy + n) * 2;
    store_values(y, v, count, t.store);
    if constexpr (MODE == MODE_LINEAR) {
        if (p.copy != 0) store_values(y + p.copy, v, count, t.store);
    }
}

// gemm_a8_kernel: products of 8-bit rows on 32 * TMX x 32 * TNX tiles of 4 wavefronts (2 x 2, 16 * TMX x-rows by 16 * TNX w-rows each; a pair's w-rows: gate rows, then up
// rows), 128 elements of K a stage, v_mfma_i32_16x16x64_i8. A stage of 8-bit elements is 128 bytes a row as one of 64 16-bit elements is, and a lane's 16 bytes of a
// fragment lie where they do there, so the plan is that of the 16-bit tiles: NS unpadded stages (piece c of row r in slot c ^ ((r / 2) % 8): 16 rows that follow one another
// are conflict-free), filled by loads straight into LDS; a stage as two steps of TMX * TNX MFMAs, the fragments of the next step read behind those that use the
// present ones, one barrier a stage, the loads of stage g + NS spread over the second step.
// K ends in a multiple of 16: in the last stage the pieces of x behind it are asked for outside the descriptor's range, which gives zeros, and what stands in those of w
// (the next row, or the bytes between rows) counts for nothing.
// SPLIT: a block has one of t.splits ranges of K; its sums go to t.ws as they lie in the registers and are added by finish_a8_kernel.
template <int DT, int MODE, int TMX, int TNX, int NS, bool SPLIT>
__global__ __launch_bounds__(256) void gemm_a8_kernel(A8Params p, A8Tiles t) {
    constexpr int BM = 32 * TMX, BN = 32 * TNX, BN_OUT = MODE == MODE_SWIGLU ? BN / 2 : BN;
    constexpr int XREG = BM * 128, STAGE = (BM + BN) * 128;
    constexpr int LPT = TMX + TNX;  // global->LDS loads per wavefront and stage
    constexpr int MF = TMX * TNX, BAR = TNX;
    static_assert(NS >= 2 && NS * STAGE <= 160 * 1024 && 4 * 16 * EP_PITCH <= NS * STAGE, "LDS");
    static_assert(BAR + TNX + TMX <= MF && TMX + TNX <= 16 && (NS - 1) * LPT < 64, "reads of a step, and the counts in s_waitcnt");
    extern __shared__ __align__(16) char smem[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, lq = lane >> 4, wm = wave & 1, wn = wave >> 1;
    const int tiles = t.tiles_m * t.tiles_n;
    const int tile = SPLIT ? blockIdx.x % tiles : blockIdx.x, split = SPLIT ? blockIdx.x / tiles : 0;
    int tile_m, tile_n;
    tile_of_block(tile, tiles, t.tiles_m, t.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * BM, n0 = tile_n * BN_OUT;
    const int KT_ALL = (p.K + A8_BK - 1) / A8_BK, first = split * t.kt_per_split;
    const int KT = SPLIT ? (KT_ALL - first < t.kt_per_split ? KT_ALL - first : t.kt_per_split) : KT_ALL;
    const int last_kt = KT_ALL - 1 - first;  // the K tile of this range that K ends in
    const int pieces = (p.K - (KT_ALL - 1) * A8_BK) / 16;

    // ---- load addresses: rows past the end of an operand are clamped to its last one
    const int rb = lane >> 3;
    uint32_t x_off[TMX], w_off[TNX], behind[2];
#pragma unroll
    for (int i = 0; i < TMX; ++i) {
        const int row = (wave * TMX + i) * 8 + rb;
        const int r = m0 + row < p.M ? row : p.M - 1 - m0;
        x_off[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.ldx) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)  // by whether the 8 rows of a load are an odd or an even eighth
        behind[h] = static_cast<int>((lane & 7) ^ ((h * 4 + (rb >> 1)) & 7)) >= pieces ? 0x80000000u : 0u;
    const bool up = MODE == MODE_SWIGLU && wave >= 2;
#pragma unroll
    for (int i = 0; i < TNX; ++i) {
        const int row = (wave * TNX + i) * 8 + rb, wr = up ? row - BN / 2 : row;
        const int r = n0 + wr < p.N ? wr : p.N - 1 - n0;
        w_off[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.ldw) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    }
    const int x_rows = p.M - m0 < BM ? p.M - m0 : BM, w_rows = p.N - n0 < BN_OUT ? p.N - n0 : BN_OUT;
    const __amdgpu_buffer_rsrc_t x_rsrc =
        make_rsrc(p.x + static_cast<int64_t>(m0) * p.ldx, static_cast<uint32_t>(x_rows - 1) * static_cast<uint32_t>(p.ldx) + static_cast<uint32_t>(p.K));
    const __amdgpu_buffer_rsrc_t w_rsrc =
        make_rsrc((up ? p.w2 : p.w) + static_cast<int64_t>(n0) * p.ldw, static_cast<uint32_t>(w_rows - 1) * static_cast<uint32_t>(p.ldw) + static_cast<uint32_t>(p.K));
    auto load = [&](auto ic, int kt, int stage_off) {  // load number ic of K tile kt of this range
        constexpr int i = decltype(ic)::value;
        if constexpr (i < TMX) {
            const uint32_t end = kt == last_kt ? behind[(wave * TMX + i) & 1] : 0u;
            buffer_load16_to_lds(x_rsrc, x_off[i] | end, (first + kt) * A8_BK, smem + stage_off + (wave * TMX + i) * 1024);
        } else {
            buffer_load16_to_lds(w_rsrc, w_off[i - TMX], (first + kt) * A8_BK, smem + stage_off + XREG + (wave * TNX + i - TMX) * 1024);
        }
    };

    // ---- fragment addresses
    const uint32_t smem_base = lds_addr_of(smem);
    const uint32_t x_rd = smem_base + (wm * TMX * 16 + l16) * 128;
    const uint32_t w_rd = smem_base + XREG + (wn * (MODE == MODE_SWIGLU ? TNX * 8 : TNX * 16) + l16) * 128;
    const uint32_t kk_off[2] = {static_cast<uint32_t>((lq ^ (l16 >> 1)) * 16), static_cast<uint32_t>(((4 + lq) ^ (l16 >> 1)) * 16)};

    i32x4 acc[TMX][TNX];
    u32x4 xq[TMX], wq[2][TNX];
#pragma unroll
    for (int a = 0; a < TMX; ++a)
#pragma unroll
        for (int b = 0; b < TNX; ++b) acc[a][b] = i32x4{0, 0, 0, 0};
    auto read_w = [&](auto hc, auto bc, uint32_t addr) {
        constexpr int h = decltype(hc)::value, b = decltype(bc)::value;
        constexpr int off = MODE == MODE_SWIGLU && b >= TNX / 2 ? (BN / 2) * 128 + (b - TNX / 2) * 2048 : b * 2048;
        wq[h][b] = lds_read16<off>(addr);
    };
    auto fence = []() { __builtin_amdgcn_sched_barrier(0); };
    const std::integral_constant<int, 0> half0{};
    const std::integral_constant<int, 1> half1{};

    // ---- first stages
    unrolled<NS>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        const int kt = s < KT ? s : KT - 1;
        unrolled<LPT>([&](auto ic) { load(ic, kt, s * STAGE); });
    });
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * LPT) : "memory");
    unrolled<TNX>([&](auto bc) { read_w(half0, bc, w_rd + kk_off[0]); });
    unrolled<TMX>([&](auto ac) { xq[decltype(ac)::value] = lds_read16<decltype(ac)::value * 2048>(x_rd + kk_off[0]); });
    fence();

    int cur = 0, nxt = STAGE;  // offsets of the stages of K tiles g and g + 1
    for (int g = 0; g < KT; ++g) {
        {   // step A
            const uint32_t xa = x_rd + cur + kk_off[1], wa = w_rd + cur + kk_off[1];
            unrolled<MF>([&](auto mc) {
                constexpr int m = decltype(mc)::value, a = m / TNX, b = m % TNX;
                // younger than fragment a: the x fragments behind it and, from row 1 on, the w reads and a x reads of this step
                if constexpr (b == 0) {
                    reads_landed<a == 0 ? TMX - 1 : TMX - 1 + TNX>(xq[a]);
                    if constexpr (a == 0) unrolled<TNX>([&](auto bc) { already_landed(wq[0][decltype(bc)::value]); });
                    fence();
                }
                acc[a][b] = mfma_i8(wq[0][b], xq[a], acc[a][b]);
                fence();
                if constexpr (m < TNX) read_w(half1, std::integral_constant<int, (m < TNX ? m : 0)>{}, wa);
                if constexpr (b == TNX - 1) xq[a] = lds_read16<a * 2048>(xa);
                fence();
            });
        }
        {   // step B
            const uint32_t xa = x_rd + nxt + kk_off[0], wa = w_rd + nxt + kk_off[0];
            const int kload = g + NS < KT ? g + NS : KT - 1;  // past the end the last tile again, into a stage nobody reads any more
            unrolled<MF>([&](auto mc) {
                constexpr int m = decltype(mc)::value, a = m / TNX, b = m % TNX;
                if constexpr (m == BAR) {
                    // this wavefront has read tile g out, its part of tile g + 1 has landed; then everybody's
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * LPT) : "memory");
                    fence();
                }
                if constexpr (b == 0) {
                    if constexpr (m < BAR) reads_landed<TMX - 1 - a>(xq[a]);
                    else already_landed(xq[a]);
                    if constexpr (a == 0) unrolled<TNX>([&](auto bc) { already_landed(wq[1][decltype(bc)::value]); });
                    fence();
                }
                acc[a][b] = mfma_i8(wq[1][b], xq[a], acc[a][b]);
                fence();
                if constexpr (m >= BAR) {
                    if constexpr (m < BAR + TNX) read_w(half0, std::integral_constant<int, (m >= BAR && m < BAR + TNX ? m - BAR : 0)>{}, wa);
                    // x fragment r behind its last use and behind the w fragments, one per MFMA while behind
                    unrolled<TMX>([&](auto rc) {
                        constexpr int r = decltype(rc)::value, after = r * TNX + TNX - 1, turn = BAR + TNX + r;
                        if constexpr (m == (after > turn ? after : turn)) xq[r] = lds_read16<r * 2048>(xa);
                    });
                    constexpr int n = MF - BAR, l0 = (m - BAR) * LPT / n, l1 = (m + 1 - BAR) * LPT / n;
                    unrolled<(l1 > l0 ? l1 - l0 : 0)>([&](auto lc) { load(std::integral_constant<int, l0 + decltype(lc)::value>{}, kload, cur); });
                }
                fence();
            });
        }
        cur = nxt;
        nxt = nxt + STAGE == NS * STAGE ? 0 : nxt + STAGE;
    }
    // every load and fragment read of this wavefront is done before another use of the stages and registers
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    unrolled<TMX>([&](auto ac) { reads_landed<0>(xq[decltype(ac)::value]); });
    unrolled<TNX>([&](auto bc) { reads_landed<0>(wq[0][decltype(bc)::value]); });
#pragma unroll
    for (int a = 0; a < TMX; ++a)
#pragma unroll
        for (int b = 0; b < TNX; ++b) asm volatile("" : "+a"(acc[a][b]));
    fence();
    drain_and_barrier();

    if constexpr (SPLIT) {
        i32x4 *ws = reinterpret_cast<i32x4 *>(t.ws) + ((static_cast<int64_t>(split) * tiles + tile_m * t.tiles_n + tile_n) * 4 + wave) * (MF * 64) + lane;
#pragma unroll
        for (int a = 0; a < TMX; ++a) {
            if (m0 + (wm * TMX + a) * 16 >= p.M) break;  // the finishing pass reads rows that there are
#pragma unroll
            for (int b = 0; b < TNX; ++b) ws[(a * TNX + b) * 64] = acc[a][b];
        }
        return;
    }

    // ---- epilogue: 16 rows x (16 * GB) columns at a time through a slab of the wavefront's own, out as 16 bytes a lane
    constexpr int NB = MODE == MODE_SWIGLU ? TNX / 2 : TNX;  // 16-column groups of outputs
    constexpr int GB = NB % 4 == 0 ? 4 : NB % 3 == 0 ? 3 : NB % 2 == 0 ? 2 : 1, GROUPS = NB / GB;
    constexpr int LPR = GB * 2, READS = (16 * LPR + 63) / 64;
    char *slab = smem + wave * (16 * EP_PITCH);
    const int m_wave = m0 + wm * TMX * 16, n_wave = n0 + wn * NB * 16;
    float sx[TMX];
#pragma unroll
    for (int a = 0; a < TMX; ++a) {
        const int m = m_wave + a * 16 + l16;
        sx[a] = p.sx[m < p.M ? m : p.M - 1];
    }
    unrolled<GROUPS>([&](auto qc) {
        constexpr int q0 = decltype(qc)::value * GB;
        float sw[GB][4], sw2[GB][4], bias[GB][4];
#pragma unroll
        for (int bb = 0; bb < GB; ++bb) a8_columns<DT, MODE>(p, n_wave + (q0 + bb) * 16 + lq * 4, sw[bb], sw2[bb], bias[bb]);
#pragma unroll
        for (int a = 0; a < TMX; ++a) {
#pragma unroll
            for (int bb = 0; bb < GB; ++bb) {
                const uint2 o = a8_finish4<DT, MODE>(p, acc[a][q0 + bb], acc[a][MODE == MODE_SWIGLU ? NB + q0 + bb : 0], sx[a], sw[bb], sw2[bb], bias[bb]);
                *reinterpret_cast<uint2 *>(slab + l16 * EP_PITCH + bb * 32 + lq * 8) = o;
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int h = 0; h < READS; ++h) {
                const int row = (lane + 64 * h) / LPR, col = (lane + 64 * h) % LPR;
                const uint4 v = *reinterpret_cast<const uint4 *>(slab + (row & 15) * EP_PITCH + col * 16);
                const int m = m_wave + a * 16 + row, n = n_wave + q0 * 16 + col * 8;
                if (row < 16 && m < p.M && n < p.N) a8_put<DT, MODE>(p, t, v, m, n, 8);
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
    });
}

// The ranges' sums of a tile added up, in the registers' order: a wavefront has 16 rows x 16 columns (a pair: gate and up sums of the same ones).
template <int DT, int MODE, int TMX, int TNX>
__global__ __launch_bounds__(256) void finish_a8_kernel(A8Params p, A8Tiles t) {
    constexpr int MF = TMX * TNX, NB = MODE == MODE_SWIGLU ? TNX / 2 : TNX;
    const int lane = threadIdx.x & 63, l16 = lane & 15, lq = lane >> 4;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);  // ((tile, wave), a), b
    const int tiles = t.tiles_m * t.tiles_n;
    if (unit >= tiles * 4 * TMX * NB) return;
    const int b = unit % NB, a = unit / NB % TMX, wave = unit / (NB * TMX) % 4, tile = unit / (NB * TMX * 4);
    const int m0 = tile / t.tiles_n * (32 * TMX) + ((wave & 1) * TMX + a) * 16, n = tile % t.tiles_n * (2 * NB * 16) + ((wave >> 1) * NB + b) * 16 + lq * 4;
    if (m0 >= p.M) return;
    const int64_t step = static_cast<int64_t>(tiles) * 4 * MF * 64;
    const i32x4 *ws = reinterpret_cast<const i32x4 *>(t.ws) + (static_cast<int64_t>(tile) * 4 + wave) * (MF * 64) + (a * TNX + b) * 64 + lane;
    i32x4 g{0, 0, 0, 0}, u{0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < t.splits; ++s) {
        g += ws[s * step];
        if constexpr (MODE == MODE_SWIGLU) u += ws[s * step + NB * 64];
    }
    const int m = m0 + l16;
    if (m >= p.M || n >= p.N) return;
    float sw[4], sw2[4], bias[4];
    a8_columns<DT, MODE>(p, n, sw, sw2, bias);
    const uint2 o = a8_finish4<DT, MODE>(p, g, u, p.sx[m], sw, sw2, bias);
    a8_put<DT, MODE>(p, t, make_uint4(o.x, o.y, 0, 0), m, n, 4);
}

int row_access(const void *a, const void *b, int64_t ld) {  // (b may be NULL)
    if (aligned(a, 16) && aligned(b, 16) && ld % 8 == 0) return 16;
    return aligned(a, 8) && aligned(b, 8) && ld % 4 == 0 ? 8 : 2;
}

template <int DT, int MODE, int TMX, int TNX, int NS, bool SPLIT>
int launch_tiles(const A8Params &p, const A8Tiles &t, hipStream_t s) {
    constexpr int LDS = NS * 32 * (TMX + TNX) * 128;
    auto kern = gemm_a8_kernel<DT, MODE, TMX, TNX, NS, SPLIT>;
    static thread_local int configured_dev = -1;  // per instantiation and host thread
    int dev = 0;
    TPAMD_HIP(hipGetDevice(&dev));
    if (configured_dev != dev) {
        TPAMD_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
        configured_dev = dev;
    }
    const int64_t blocks = static_cast<int64_t>(t.tiles_m) * t.tiles_n * t.splits;
    TPAMD_REQUIRE(blocks < (1ll << 24), "a8: too many tiles");  // 2^32 threads
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks)), dim3(256), LDS, s, p, t);
    TPAMD_HIP(hipGetLastError());
    return TPAMD_OK;
}

template <int DT, int MODE, int TMX, int TNX, int NS>
int launch_a8(const A8Params &p, int splits, hipStream_t s) {
    constexpr int BM = 32 * TMX, BN_OUT = MODE == MODE_SWIGLU ? 16 * TNX : 32 * TNX, NB = MODE == MODE_SWIGLU ? TNX / 2 : TNX;
    A8Tiles t{};
    t.tiles_m = (p.M + BM - 1) / BM;
    t.tiles_n = (p.N + BN_OUT - 1) / BN_OUT;
    t.store = row_access(p.y, p.y + p.copy, p.ldy);
    t.add = row_access(p.addend, nullptr, p.ldadd);
    const int kt = (p.K + A8_BK - 1) / A8_BK;
    t.kt_per_split = (kt + splits - 1) / splits;
    t.splits = (kt + t.kt_per_split - 1) / t.kt_per_split;
    if (t.splits > 1) {
        int dev = 0, cus = 256;
        TPAMD_HIP(hipGetDevice(&dev));
        if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
        const size_t need = static_cast<size_t>(t.splits) * t.tiles_m * t.tiles_n * (BM * 32 * TNX) * sizeof(int);
        std::lock_guard<std::mutex> hold(splitk_mutex(dev));
        void *ws = nullptr;
        if (int rc = splitk_scratch(dev, s, need, scratch_reserve(cus), &ws); rc != TPAMD_OK) return rc;
        if (ws != nullptr) {
            t.ws = static_cast<int *>(ws);
            if (int rc = launch_tiles<DT, MODE, TMX, TNX, NS, true>(p, t, s); rc != TPAMD_OK) return rc;
            const int64_t units = static_cast<int64_t>(t.tiles_m) * t.tiles_n * 4 * TMX * NB;
            hipLaunchKernelGGL((finish_a8_kernel<DT, MODE, TMX, TNX>), dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), 0, s, p, t);
            TPAMD_HIP(hipGetLastError());
            return TPAMD_OK;
        }
        t.splits = 1;  // no scratch memory for the stream: all of K in a block
        t.kt_per_split = kt;
    }
    return launch_tiles<DT, MODE, TMX, TNX, NS, false>(p, t, s);
}

template <int DT, int MODE>
int launch_a8_tile(const A8Params &p, int tmx, int tnx, int splits, hipStream_t s) {
#define A8_TILE(tmx, tnx, stages) case tmx * 16 + tnx: return launch_a8<DT, MODE, tmx, tnx, stages>(p, splits, s)
    switch (tmx * 16 + tnx) {
        A8_TILE(3, 4, 4);
        A8_TILE(4, 4, 4);
        A8_TILE(4, 6, 4);
        A8_TILE(4, 8, 3);
        A8_TILE(6, 6, 3);
        A8_TILE(6, 8, 2);
        A8_TILE(8, 6, 2);
        A8_TILE(8, 8, 2);
    }
#undef A8_TILE
    set_error("a8: no tile of %d x %d rows", 32 * tmx, 32 * tnx);
    return TPAMD_ERR_UNSUPPORTED;
}

}  // namespace

// K a multiple of 16, at least 16; ldx, ldw multiples of 16 below 2^22; x, w, w2 on 16-byte boundaries.
int gemm_a8(const A8Params &p, bool pair, int dtype, int tmx, int tnx, int splits, hipStream_t s) {
    if (dtype == TPAMD_BF16) return pair ? launch_a8_tile<TPAMD_BF16, MODE_SWIGLU>(p, tmx, tnx, splits, s) : launch_a8_tile<TPAMD_BF16, MODE_LINEAR>(p, tmx, tnx, splits, s);
    return pair ? launch_a8_tile<TPAMD_F16, MODE_SWIGLU>(p, tmx, tnx, splits, s) : launch_a8_tile<TPAMD_F16, MODE_LINEAR>(p, tmx, tnx, splits, s);
}

}  // namespace tpamd
