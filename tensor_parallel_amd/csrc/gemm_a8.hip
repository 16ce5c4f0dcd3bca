#include "a8.h"
#include "gemm_tile.h"

namespace tpamd {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ i32x16 mfma_i8(u32x4 a, u32x4 b, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}
template <int Q>
__device__ __forceinline__ i32x4 quarter(const i32x16 &v) { return i32x4{v[4 * Q], v[4 * Q + 1], v[4 * Q + 2], v[4 * Q + 3]}; }

constexpr int A8_BK = 128;  // K elements (bytes of a row) per stage

struct A8Tiles {
    int tiles_m, tiles_n;
    int kt_per_split, splits;  // K tiles of a range, ranges
    int *ws;                   // partial tiles
    bool direct;               // the epilogue from the registers: no activation, rows of outputs and addend and the scales on 16-byte boundaries (bias: 8), N a multiple of 8, rows of the addend within reach of 32-bit offsets
    int store;                 // values of a row that outputs and addend are accessed by: 8 (N a multiple of 8), 2 (N even) or 1, as their rows allow
};

// What 8 columns from n on have in common (of those there are: the last one again behind it).
__device__ __forceinline__ void a8_scales(float (&v)[8], const float *s, int n, int N) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s[n + j < N ? n + j : N - 1];
}
template <int DT>
__device__ __forceinline__ void a8_bias(float (&v)[8], const char *bias, int n, int N) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bias == nullptr ? 0.f : half_to_f32<DT>(reinterpret_cast<const uint16_t *>(bias)[n + j < N ? n + j : N - 1]);
}
// 8 values of a row: read from, and (those of them that there are, `count`) written to memory accessed by `by` values.
__device__ __forceinline__ uint4 get8(const char *from, int count, int by) {
    if (by == 8) return *reinterpret_cast<const uint4 *>(from);
    uint32_t v[4] = {0, 0, 0, 0};
    if (by == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (2 * j < count) v[j] = reinterpret_cast<const uint32_t *>(from)[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) v[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(from)[j]) << (16 * (j & 1));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put8(char *to, uint4 u, int count, int by) {
    const uint32_t v[4] = {u.x, u.y, u.z, u.w};
    if (by == 8) {
        *reinterpret_cast<uint4 *>(to) = u;
    } else if (by == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (2 * j < count) reinterpret_cast<uint32_t *>(to)[j] = v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) reinterpret_cast<uint16_t *>(to)[j] = static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1)));
    }
}
template <int DT>
__device__ __forceinline__ uint4 add8(uint4 v, uint4 a) {
    return make_uint4(add_packed2<DT>(v.x, a.x), add_packed2<DT>(v.y, a.y), add_packed2<DT>(v.z, a.z), add_packed2<DT>(v.w, a.w));
}
// 8 outputs of a row from their sums (u: the up sums of a pair), before the addend.
template <int DT, int MODE>
__device__ __forceinline__ uint4 a8_finish8(const int (&g)[8], const int (&u)[8], float sx, const float (&sw)[8], const float (&sw2)[8], const float (&bias)[8], int act) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (MODE == MODE_SWIGLU) v[j] = a8_gated(a8_linear(g[j], sx, sw[j], 0.f), a8_linear(u[j], sx, sw2[j], 0.f));
        else v[j] = a8_linear(g[j], sx, sw[j], bias[j]);
    }
    if (MODE == MODE_LINEAR && act == TPAMD_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = a8_act(v[j], TPAMD_ACT_GELU);
    }
    return make_uint4(a8_round2<DT>(v[0], v[1]), a8_round2<DT>(v[2], v[3]), a8_round2<DT>(v[4], v[5]), a8_round2<DT>(v[6], v[7]));
}
// A quarter of an MFMA tile's sums from accumulation registers into LDS.
template <int OFFSET>
__device__ __forceinline__ void lds_write_acc(uint32_t addr, i32x4 v) {
    static_assert(OFFSET >= 0 && OFFSET < 65536, "ds offset field is 16 bits");
    asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(addr), "a"(v), "n"(OFFSET) : "memory");
}

// gemm_a8_kernel: products of 8-bit rows on 64 * TM x 64 * TN tiles of 4 wavefronts (2 x 2, 32 * TM x-rows by 32 * TN w-rows each), 128 elements of K a stage,
// v_mfma_i32_32x32x32_i8. That form alone has the pipe's rate: a loop of nothing else reaches 4.7 POP/s on constant operands and 3.6 on random ones, of
// v_mfma_i32_16x16x64_i8 2.3 on either.
// A lane gives 16 bytes of row lane % 32, those of K half lane / 32, and has D[n = 8 (i / 4) + 4 (lane / 32) + i % 4][m = lane % 32] with w first. A pair's w-rows lie in
// the stage as 16 gate rows, then the 16 up rows of the same columns: elements i and i + 8 of a lane are the two sums of one output.
// LDS: NS stages of (BM + BN) rows of 128 bytes without padding; piece c of row r is in slot c ^ ((r / 2) % 8), so 16 rows that follow one another are conflict-free.
// K tile g runs as four steps of TM * TN MFMAs on two sets of fragments; the reads of a step's fragments stand behind the first MFMAs of the step before. In the last step a
// barrier: tile g + 1 has landed, tile g is read out; the loads of tile g + NS go into its stage in the rest of that step and the first of the next tile.
// K ends in a multiple of 16: in the last stage the pieces of x behind it are asked for outside the descriptor's range, which gives zeros, and what stands in those of w
// (the next row, or the bytes between rows) counts for nothing.
// Bound: by the power that the matrix pipe takes on real codes: a K tile of a 256 x 256 tile takes 1.6 us with every CU at it (2.7 POP/s), 1.06 on zeros. 4096 x 4096 x 5504 in 78-86 us (2.15-2.35 POP/s; 86-91
// with an addend, most of it loaded under the last K tiles; 95 with the GELU, whose epilogue goes through LDS), 4096 x 16384 x 8192 in 439 (2.5; with the GELU 489), the pair of 4096 x 5504 x 4096 in 162 (2.28).
// Smaller tiles by what LDS and the L2 deliver: 645 x 6144 x 4096 on 128 x 192 tiles, one to a CU, 23 us, 25-28 on weights from memory; a fourth or fifth stage changes nothing. Rows that begin
// inside 128-byte lines cost 8-20 % more (each of their lines is asked for in two K tiles): the pair of 4096 x 5504 x 4112 198 us, in lines 170, 2048 x 4096 x 2752 30.2 and 27.9.
// SPLIT: a block has one of t.splits ranges of K; its sums go to t.ws as they lie in the registers and are added by finish_a8_kernel.
constexpr int a8_slab_rows(int tm, int tn) { return tm == 3 && tn == 4 ? 1 : tm == 4 ? 2 : tm; }  // MFMA tiles of rows
constexpr int a8_lds(int tm, int tn, int ns) {
    const int stages = ns * 64 * (tm + tn) * 128, slabs = 4 * (a8_slab_rows(tm, tn) * 32 * (tn * 128 + 16) + tm * 128);
    return stages > slabs ? stages : slabs;
}
template <int DT, int MODE, int TM, int TN, int NS, bool SPLIT, bool ADD>
__global__ __launch_bounds__(256) void gemm_a8_kernel(A8Params p, A8Tiles t) {
    constexpr int BM = 64 * TM, BN = 64 * TN, BN_OUT = MODE == MODE_SWIGLU ? BN / 2 : BN;
    constexpr int XREG = BM * 128, STAGE = (BM + BN) * 128;
    constexpr int XL = 2 * TM, WL = 2 * TN, LPT = XL + WL, HALF = LPT / 2;  // global->LDS loads per wavefront and stage
    constexpr int MF = TM * TN, READS = TM + TN, BAR = MF >= 8 ? 4 : MF / 2;
    // the epilogue's slab of a wavefront: the sums of 32 * AH rows, shifted by 4 banks a row, and the scales of all its rows
    constexpr int CB = MODE == MODE_SWIGLU ? 16 : 32, PITCH = TN * 128 + 16;  // (outputs in a row of an MFMA tile)
    constexpr int AH = a8_slab_rows(TM, TN), SLAB = AH * 32 * PITCH + TM * 128;
    static_assert(NS >= 2 && a8_lds(TM, TN, NS) <= 160 * 1024, "LDS");
    static_assert((NS - 2) * LPT + HALF < 64 && READS < 16, "the counts in s_waitcnt");
    extern __shared__ __align__(16) char smem[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l32 = lane & 31, lh = lane >> 5, wm = wave & 1, wn = wave >> 1;
    const int tiles = t.tiles_m * t.tiles_n;
    const int tile = SPLIT ? blockIdx.x % tiles : blockIdx.x, split = SPLIT ? blockIdx.x / tiles : 0;
    int tile_m, tile_n;
    tile_of_block(tile, tiles, t.tiles_m, t.tiles_n, tile_m, tile_n);
    const int m0 = tile_m * BM, n0 = tile_n * BN_OUT;
    const int KT_ALL = (p.K + A8_BK - 1) / A8_BK, first = split * t.kt_per_split;
    const int KT = SPLIT ? (KT_ALL - first < t.kt_per_split ? KT_ALL - first : t.kt_per_split) : KT_ALL;
    const int last_kt = KT_ALL - 1 - first;  // the K tile of this range that K ends in
    const int pieces = (p.K - (KT_ALL - 1) * A8_BK) / 16;

    // ---- load addresses: rows past the end of an operand lie outside the descriptors, whose extents are below 2^31
    const int rb = lane >> 3;
    uint32_t x_off[XL], w_off[WL], behind[2];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int row = (wave * XL + i) * 8 + rb;
        x_off[i] = m0 + row < p.M ? static_cast<uint32_t>(row) * static_cast<uint32_t>(p.ldx) + ((lane & 7) ^ ((row >> 1) & 7)) * 16 : 0x80000000u;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)  // by whether the 8 rows of a load are an odd or an even eighth
        behind[h] = static_cast<int>((lane & 7) ^ ((h * 4 + (rb >> 1)) & 7)) >= pieces ? 0x80000000u : 0u;
    auto is_up = [&](int i) { return MODE == MODE_SWIGLU && ((wave * WL + i) & 2) != 0; };  // 8-row group 2 or 3 of 32 staged rows
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int row = (wave * WL + i) * 8 + rb, wr = MODE == MODE_SWIGLU ? (row >> 5) * 16 + (row & 15) : row;
        w_off[i] = n0 + wr < p.N ? static_cast<uint32_t>(wr) * static_cast<uint32_t>(p.ldw) + ((lane & 7) ^ ((row >> 1) & 7)) * 16 : 0x80000000u;
    }
    const int x_rows = p.M - m0 < BM ? p.M - m0 : BM, w_rows = p.N - n0 < BN_OUT ? p.N - n0 : BN_OUT;
    const uint32_t w_extent = static_cast<uint32_t>(w_rows - 1) * static_cast<uint32_t>(p.ldw) + static_cast<uint32_t>(p.K);
    const __amdgpu_buffer_rsrc_t x_rsrc =
        make_rsrc(p.x + static_cast<int64_t>(m0) * p.ldx, static_cast<uint32_t>(x_rows - 1) * static_cast<uint32_t>(p.ldx) + static_cast<uint32_t>(p.K));
    const __amdgpu_buffer_rsrc_t w_rsrc = make_rsrc(p.w + static_cast<int64_t>(n0) * p.ldw, w_extent);
    const __amdgpu_buffer_rsrc_t w2_rsrc = MODE == MODE_SWIGLU ? make_rsrc(p.w2 + static_cast<int64_t>(n0) * p.ldw, w_extent) : w_rsrc;
    // the addend's rows of this wavefront (ADD), for the epilogue from the registers: EARLY slabs of 32 rows take the place of K tiles behind the last one. 4096 x 8192 x 4096 150 -> 140 us, 4096 x
    // 4096 x 5504 94 -> 90 against requests in the epilogue
    const int m_wave = m0 + wm * TM * 32, n_wave = n0 + wn * TN * CB;
    constexpr int SLAB_LOADS = 2 * TN, AHEAD = (NS - 1) * LPT + HALF, EARLY = AHEAD / SLAB_LOADS < TM ? AHEAD / SLAB_LOADS : TM;
    static_assert(TM - EARLY <= 1, "the rest of the addend is held in registers");
    const uint32_t add_pitch = static_cast<uint32_t>(p.ldadd) * 2;
    uint32_t add_extent = 0;
    if (ADD && t.direct && m_wave < p.M && n_wave < p.N)
        add_extent = static_cast<uint32_t>((p.M - m_wave < TM * 32 ? p.M - m_wave : TM * 32) - 1) * add_pitch + static_cast<uint32_t>(p.N - n_wave < TN * CB ? p.N - n_wave : TN * CB) * 2;
    const __amdgpu_buffer_rsrc_t add_rsrc = add_extent != 0 ? make_rsrc(p.addend + (static_cast<int64_t>(m_wave) * p.ldadd + n_wave) * 2, add_extent) : x_rsrc;
    auto slot = [&](int i) { return i < XL ? (wave * XL + i) * 1024 : XREG + (wave * WL + i - XL) * 1024; };  // of load i in its stage
    // load number ic of K tile kt of this range; behind the last one (which `inside` rules out) the same count of loads, of the addend or from outside the descriptors (with the uniform offset inside
    // their extents)
    auto load = [&](auto ic, int kt, int stage_off, auto inside) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        char *to = smem + stage_off + slot(i);
        const bool here = decltype(inside)::value || kt < KT;
        const uint32_t from = i < XL ? x_off[i < XL ? i : 0] | (kt == last_kt ? behind[i & 1] : 0u) : w_off[i < XL ? 0 : i - XL];  // (XL is even)
        const __amdgpu_buffer_rsrc_t rsrc = i < XL ? x_rsrc : is_up(i - XL) ? w2_rsrc : w_rsrc;
        if constexpr (decltype(inside)::value) {
            buffer_load16_to_lds(rsrc, from, (first + kt) * A8_BK, to);
        } else if constexpr (!ADD) {
            buffer_load16_to_lds(rsrc, here ? from : 0x80000000u, here ? (first + kt) * A8_BK : 0, to);
        } else {
            const uint32_t j = static_cast<uint32_t>(kt - KT) * LPT + i, a = j / SLAB_LOADS, at = a * 32 * add_pitch + j % SLAB_LOADS * 32;
            const bool there = a < EARLY && at < add_extent;
            const uint32_t lane_at = there ? static_cast<uint32_t>(l32) * add_pitch + static_cast<uint32_t>(lh) * 16 : 0x80000000u;
            buffer_load16_to_lds(here ? rsrc : add_rsrc, here ? from : lane_at, here ? (first + kt) * A8_BK : there ? static_cast<int>(at) : 0, to);
        }
    };

    // ---- fragment addresses
    const uint32_t smem_base = lds_addr_of(smem);
    const uint32_t x_rd = smem_base + (wm * TM * 32 + l32) * 128, w_rd = smem_base + XREG + (wn * TN * 32 + l32) * 128;
    uint32_t kk_off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) kk_off[k] = static_cast<uint32_t>(((k * 2 + lh) ^ ((l32 >> 1) & 7)) * 16);

    i32x16 acc[TM][TN];
    u32x4 xq[2][TM], wq[2][TN];
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] = i32x16{};
    auto read = [&](auto hc, auto rc, uint32_t xa, uint32_t wa) __attribute__((always_inline)) {  // fragment number rc of a step: w, then x
        constexpr int h = decltype(hc)::value, r = decltype(rc)::value;
        if constexpr (r < TN) wq[h][r] = lds_read16<r * 4096>(wa);
        else xq[h][r - TN] = lds_read16<(r - TN) * 4096>(xa);
    };
    auto fence = []() { __builtin_amdgcn_sched_barrier(0); };
    auto landed = [&](auto hc) __attribute__((always_inline)) {
        constexpr int h = decltype(hc)::value;
        reads_landed<0>(wq[h][0]);
        unrolled<TN>([&](auto bc) { already_landed(wq[h][decltype(bc)::value]); });
        unrolled<TM>([&](auto ac) { already_landed(xq[h][decltype(ac)::value]); });
    };
    const std::integral_constant<int, 0> set0{};
    const std::integral_constant<int, 1> set1{};

    float sx[TM];  // the scales of the lane's rows, asked for ahead of everything else
    if constexpr (!SPLIT) {
#pragma unroll
        for (int a = 0; a < TM; ++a) {
            const int m = m0 + (wm * TM + a) * 32 + l32;
            sx[a] = p.sx[m < p.M ? m : p.M - 1];
        }
    }
    // ---- first stages: the second half of the last one is loaded in the first step
    unrolled<NS>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        unrolled<(s < NS - 1 ? LPT : HALF)>([&](auto ic) { load(ic, s, s * STAGE, std::false_type{}); });
    });
    if constexpr (!SPLIT) {
#pragma unroll
        for (int a = 0; a < TM; ++a) asm volatile("" : "+v"(sx[a]));
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * LPT + HALF) : "memory");
    unrolled<READS>([&](auto rc) { read(set0, rc, x_rd + kk_off[0], w_rd + kk_off[0]); });
    fence();

    int cur = 0, nxt = STAGE, old = (NS - 1) * STAGE;  // offsets of the stages of K tiles g, g + 1 and g + NS - 1
    auto k_tile = [&](int g, auto inside) __attribute__((always_inline)) {
        const int k_old = g + NS - 1, k_cur = g + NS;
        unrolled<4>([&](auto sc) {
            constexpr int s = decltype(sc)::value, bar = s == 3 ? BAR : 0, slots = MF - bar, per = (READS + slots - 1) / slots;
            const uint32_t off = (s == 3 ? nxt : cur) + kk_off[(s + 1) & 3], xa = x_rd + off, wa = w_rd + off;
            const std::integral_constant<int, (s & 1)> now{};
            const std::integral_constant<int, ((s + 1) & 1)> then{};
            landed(now);
            fence();
            unrolled<MF>([&](auto mc) {
                constexpr int m = decltype(mc)::value, a = m / TN, b = m % TN;
                if constexpr (s == 3 && m == BAR) {
                    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 2) * LPT) : "memory");
                    fence();
                }
                acc[a][b] = mfma_i8(wq[s & 1][b], xq[s & 1][a], acc[a][b]);
                fence();
                if constexpr (m >= bar) {
                    constexpr int r0 = (m - bar) * per, r1 = r0 + per < READS ? r0 + per : READS;
                    unrolled<(r1 > r0 ? r1 - r0 : 0)>([&](auto rc) { read(then, std::integral_constant<int, r0 + decltype(rc)::value>{}, xa, wa); });
                    constexpr int l0 = (m - bar) * HALF / slots, l1 = (m + 1 - bar) * HALF / slots;
                    if constexpr (s == 3) unrolled<l1 - l0>([&](auto lc) { load(std::integral_constant<int, l0 + decltype(lc)::value>{}, k_cur, cur, inside); });
                    if constexpr (s == 0) unrolled<l1 - l0>([&](auto lc) { load(std::integral_constant<int, HALF + l0 + decltype(lc)::value>{}, k_old, old, inside); });
                }
                fence();
            });
        });
        old = cur;
        cur = nxt;
        nxt = nxt + STAGE == NS * STAGE ? 0 : nxt + STAGE;
    };
    // two loops: asked in every load, whether it lies behind the last K tile costs 8 % of a 256 x 256 tile's time
    int g = 0;
    for (; g < KT - NS; ++g) k_tile(g, std::true_type{});
    for (; g < KT; ++g) k_tile(g, std::false_type{});
    // every load and fragment read of this wavefront is done before another use of the stages and registers
    landed(set0);
    (void)set1;
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) asm volatile("" : "+a"(acc[a][b]));
    fence();
    drain_and_barrier();

    if constexpr (SPLIT) {
        i32x4 *ws = reinterpret_cast<i32x4 *>(t.ws) + ((static_cast<int64_t>(split) * tiles + tile_m * t.tiles_n + tile_n) * 4 + wave) * (MF * 256) + lane;
#pragma unroll
        for (int a = 0; a < TM; ++a) {
            if (m0 + (wm * TM + a) * 32 >= p.M) break;  // the finishing pass reads rows that there are
#pragma unroll
            for (int b = 0; b < TN; ++b)
                unrolled<4>([&](auto qc) { ws[((a * TN + b) * 4 + decltype(qc)::value) * 64] = quarter<decltype(qc)::value>(acc[a][b]); });
        }
        return;
    }

    // ---- epilogue from the registers, 32 rows at a time: two lanes exchange halves of groups of 8 columns, and a store has 32 bytes of 32 rows, which the L2 puts together.
    // A 256 x 256 tile takes 11000 cycles with it, 25000 with the loop over LDS below
    if (t.direct) {
        constexpr int CHUNKS = CB / 16;  // groups of 8 outputs that a lane has of an MFMA tile
        float4 sw[TN][4];
        uint2 braw[TN][4];
        uint4 rest[TN][CHUNKS];  // of the addend
        unrolled<TN>([&](auto bc) {
            constexpr int b = decltype(bc)::value;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = n_wave + b * CB + (MODE == MODE_SWIGLU ? q & 1 : q) * 8 + lh * 4, n = c < p.N ? c : 0;
                sw[b][q] = *reinterpret_cast<const float4 *>((MODE == MODE_SWIGLU && q >= 2 ? p.sw2 : p.sw) + n);
                braw[b][q] = MODE == MODE_LINEAR && p.bias != nullptr ? *reinterpret_cast<const uint2 *>(p.bias + static_cast<int64_t>(n) * 2) : make_uint2(0, 0);
            }
        });
        if constexpr (ADD && EARLY < TM) {
#pragma unroll
            for (int i = 0; i < TN * CHUNKS; ++i) {
                const int m = m_wave + EARLY * 32 + l32, n = n_wave + i * 16 + lh * 8;
                rest[i / CHUNKS][i % CHUNKS] = m < p.M && n < p.N ? *reinterpret_cast<const uint4 *>(p.addend + (static_cast<int64_t>(m) * p.ldadd + n) * 2) : make_uint4(0, 0, 0, 0);
            }
        }
        unrolled<TM>([&](auto ac) {
            constexpr int a = decltype(ac)::value;
            const int m = m_wave + a * 32 + l32;
            char *row = p.y + (static_cast<int64_t>(m) * p.ldy + n_wave + lh * 8) * 2;
            unrolled<TN>([&](auto bc) {
                constexpr int b = decltype(bc)::value;
                const i32x16 &v = acc[a][b];
                uint2 w[2 * CHUNKS];
#pragma unroll
                for (int q = 0; q < 2 * CHUNKS; ++q) {
                    const float4 f = sw[b][q], g = sw[b][(q + 2) & 3];
                    const uint2 r = braw[b][q];
                    float o[4];
                    if constexpr (MODE == MODE_SWIGLU) {
                        o[0] = a8_gated(a8_linear(v[4 * q], sx[a], f.x, 0.f), a8_linear(v[4 * q + 8], sx[a], g.x, 0.f));
                        o[1] = a8_gated(a8_linear(v[4 * q + 1], sx[a], f.y, 0.f), a8_linear(v[4 * q + 9], sx[a], g.y, 0.f));
                        o[2] = a8_gated(a8_linear(v[4 * q + 2], sx[a], f.z, 0.f), a8_linear(v[4 * q + 10], sx[a], g.z, 0.f));
                        o[3] = a8_gated(a8_linear(v[4 * q + 3], sx[a], f.w, 0.f), a8_linear(v[4 * q + 11], sx[a], g.w, 0.f));
                    } else {
                        o[0] = a8_linear(v[4 * q], sx[a], f.x, lo_half_to_f32<DT>(r.x));
                        o[1] = a8_linear(v[4 * q + 1], sx[a], f.y, hi_half_to_f32<DT>(r.x));
                        o[2] = a8_linear(v[4 * q + 2], sx[a], f.z, lo_half_to_f32<DT>(r.y));
                        o[3] = a8_linear(v[4 * q + 3], sx[a], f.w, hi_half_to_f32<DT>(r.y));
                    }
                    w[q] = make_uint2(a8_round2<DT>(o[0], o[1]), a8_round2<DT>(o[2], o[3]));
                }
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                    // lane / 32 = 0 gives its half of the second group for the other's half of the first
                    const auto x = __builtin_amdgcn_permlane32_swap(w[2 * c].x, w[2 * c + 1].x, false, false);
                    const auto y = __builtin_amdgcn_permlane32_swap(w[2 * c].y, w[2 * c + 1].y, false, false);
                    uint4 u = make_uint4(x[0], y[0], x[1], y[1]);
                    if constexpr (ADD) {
                        if constexpr (a < EARLY) {
                            constexpr int j = a * SLAB_LOADS + b * 2, behind_last = j / LPT;
                            const int stage_off = behind_last == 0 ? cur : behind_last == 1 ? nxt : old;  // (two stages: nxt is old)
                            u = add8<DT>(u, *reinterpret_cast<const uint4 *>(smem + stage_off + slot(j % LPT + c) + lane * 16));
                        } else {
                            u = add8<DT>(u, rest[b][c]);
                        }
                    }
                    if (m < p.M && n_wave + b * CB + c * 16 + lh * 8 < p.N) {
                        *reinterpret_cast<uint4 *>(row + b * CB * 2 + c * 32) = u;
                        if (MODE == MODE_LINEAR && p.copy != 0) *reinterpret_cast<uint4 *>(row + b * CB * 2 + c * 32 + p.copy) = u;
                    }
                }
            });
        });
        return;
    }

    // ---- epilogue: the sums of 32 * AH rows at a time through the wavefront's slab, from where a lane takes 8 columns of a row, the same ones of every row. Behind the registers it
    // is a loop: instructions come in at the pace of their misses, and unrolled over the accumulators these cost a 256 x 256 tile 12-18 us.
    constexpr int LPR = TN * CB / 8, RPP = 64 / LPR, ROWS = AH * 32;  // lanes to a row, rows at a time
    char *slab = smem + wave * SLAB;
    float *scales = reinterpret_cast<float *>(slab + ROWS * PITCH);
    const int my_row = lane / LPR, my_col = lane % LPR * 8;
    const int n = n_wave + my_col, count = my_row < RPP ? p.N - n : 0;
    const uint32_t to = lds_addr_of(slab) + l32 * PITCH + lh * 16;
    const char *from = slab + (MODE == MODE_SWIGLU ? (my_col >> 4) * 128 + (my_col & 15) * 4 : my_col * 4);
    float sw[8], sw2[8], bias[8];
    a8_scales(sw, p.sw, n, p.N);
    if constexpr (MODE == MODE_SWIGLU) a8_scales(sw2, p.sw2, n, p.N);
    else a8_bias<DT>(bias, p.bias, n, p.N);
#pragma unroll
    for (int a = 0; a < TM; ++a) scales[a * 32 + l32] = sx[a];
    constexpr int U = MODE == MODE_SWIGLU ? 2 : 4, STEP = U * RPP;  // rows of a lane at a time, of the wavefront
    uint4 ahead[U];
    auto request = [&](int r0) __attribute__((always_inline)) {  // the addend of the wavefront's rows from r0 on
        if constexpr (!ADD) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * RPP + my_row, m = m_wave + r;
            ahead[u] = r < TM * 32 && m < p.M && count > 0 ? get8(p.addend + (static_cast<int64_t>(m) * p.ldadd + n) * 2, count, t.store) : make_uint4(0, 0, 0, 0);
        }
    };
    request(0);
#pragma unroll 1
    for (int a0 = 0; a0 < TM; a0 += AH) {
        unrolled<TM / AH>([&](auto pc) {
            constexpr int ph = decltype(pc)::value;
            if (a0 == ph * AH)
                unrolled<AH * TN>([&](auto tc) {
                    constexpr int a = decltype(tc)::value / TN, b = decltype(tc)::value % TN;
                    unrolled<4>([&](auto qc) {
                        constexpr int q = decltype(qc)::value;
                        lds_write_acc<(a * 32 * PITCH + b * 128 + q * 32) % 65536>(to + (a * 32 * PITCH + b * 128 + q * 32) / 65536 * 65536, quarter<q>(acc[ph * AH + a][b]));
                    });
                });
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int r0 = 0; r0 < ROWS; r0 += STEP) {
            uint4 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * RPP + my_row < ROWS ? r0 + u * RPP + my_row : ROWS - 1;
                const i32x4 *sums = reinterpret_cast<const i32x4 *>(from + r * PITCH);
                const i32x4 g0 = sums[0], g1 = sums[1], u0 = MODE == MODE_SWIGLU ? sums[4] : g0, u1 = MODE == MODE_SWIGLU ? sums[5] : g1;
                const int g[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w}, up[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
                o[u] = a8_finish8<DT, MODE>(g, up, scales[a0 * 32 + r], sw, sw2, bias, p.act);
            }
            if constexpr (ADD) {
#pragma unroll
                for (int u = 0; u < U; ++u) o[u] = add8<DT>(o[u], ahead[u]);
                request(a0 * 32 + r0 + STEP < a0 * 32 + ROWS ? a0 * 32 + r0 + STEP : (a0 + AH) * 32);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * RPP + my_row, m = m_wave + a0 * 32 + r;
                if (r >= ROWS || m >= p.M || count <= 0) continue;
                char *y = p.y + (static_cast<int64_t>(m) * p.ldy + n) * 2;
                put8(y, o[u], count, t.store);
                if (MODE == MODE_LINEAR && p.copy != 0) put8(y + p.copy, o[u], count, t.store);
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    }
}

// The ranges' sums of a tile added up, in the registers' order: a wavefront has the 32 x 32 sums of an MFMA tile.
template <int DT, int MODE, int TM, int TN>
__global__ __launch_bounds__(256) void finish_a8_kernel(A8Params p, A8Tiles t) {
    constexpr int MF = TM * TN, CB = MODE == MODE_SWIGLU ? 16 : 32;
    __shared__ __align__(16) int slabs[4 * 32 * 36];  // 32 sums of a row, shifted by 4 banks a row
    const int lane = threadIdx.x & 63, l32 = lane & 31, lh = lane >> 5;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);  // ((tile, wave), a), b
    const int tiles = t.tiles_m * t.tiles_n;
    if (unit >= tiles * 4 * MF) return;
    const int b = unit % TN, a = unit / TN % TM, wave = unit / MF % 4, tile = unit / (MF * 4);
    const int m0 = tile / t.tiles_n * (64 * TM) + ((wave & 1) * TM + a) * 32, n0 = tile % t.tiles_n * (2 * TN * CB) + ((wave >> 1) * TN + b) * CB;
    if (m0 >= p.M) return;
    const int64_t step = static_cast<int64_t>(tiles) * 4 * MF * 256;
    const i32x4 *ws = reinterpret_cast<const i32x4 *>(t.ws) + (static_cast<int64_t>(tile) * 4 + wave) * (MF * 256) + (a * TN + b) * 256 + lane;
    i32x4 sum[4] = {};
#pragma unroll 2
    for (int s = 0; s < t.splits; ++s)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += ws[s * step + q * 64];
    int *slab = slabs + (threadIdx.x >> 6) * (32 * 36);
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<i32x4 *>(slab + l32 * 36 + q * 8 + lh * 4) = sum[q];
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
    constexpr int LPR = CB / 8, RPP = 64 / LPR;
    const int my_col = lane % LPR * 8, n = n0 + my_col, count = p.N - n;
    if (count <= 0) return;
    float sw[8], sw2[8], bias[8];
    a8_scales(sw, p.sw, n, p.N);
    if constexpr (MODE == MODE_SWIGLU) a8_scales(sw2, p.sw2, n, p.N);
    else a8_bias<DT>(bias, p.bias, n, p.N);
#pragma unroll
    for (int r = lane / LPR; r < 32; r += RPP) {
        const int m = m0 + r;
        if (m >= p.M) return;
        int g[8], u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            g[j] = slab[r * 36 + my_col + j];
            u[j] = MODE == MODE_SWIGLU ? slab[r * 36 + 16 + my_col + j] : 0;
        }
        uint4 o = a8_finish8<DT, MODE>(g, u, p.sx[m], sw, sw2, bias, p.act);
        if (MODE == MODE_LINEAR && p.addend != nullptr) o = add8<DT>(o, get8(p.addend + (static_cast<int64_t>(m) * p.ldadd + n) * 2, count, t.store));
        char *y = p.y + (static_cast<int64_t>(m) * p.ldy + n) * 2;
        put8(y, o, count, t.store);
        if (MODE == MODE_LINEAR && p.copy != 0) put8(y + p.copy, o, count, t.store);
    }
}

int values_by(const void *a, int64_t copy, int64_t ld, int N) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a) | static_cast<uintptr_t>(copy);
    if (N % 8 == 0 && ld % 8 == 0 && at % 16 == 0) return 8;
    return N % 2 == 0 && ld % 2 == 0 && at % 4 == 0 ? 2 : 1;
}

template <int DT, int MODE, int TM, int TN, int NS, bool SPLIT, bool ADD>
int launch_tiles(const A8Params &p, const A8Tiles &t, hipStream_t s) {
    constexpr int LDS = SPLIT ? NS * 64 * (TM + TN) * 128 : a8_lds(TM, TN, NS);
    auto kern = gemm_a8_kernel<DT, MODE, TM, TN, NS, SPLIT, ADD>;
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

template <int DT, int MODE, int TM, int TN, int NS>
int launch_a8(const A8Params &p, int splits, hipStream_t s) {
    constexpr int BM = 64 * TM, BN_OUT = MODE == MODE_SWIGLU ? 32 * TN : 64 * TN;
    A8Tiles t{};
    t.tiles_m = (p.M + BM - 1) / BM;
    t.tiles_n = (p.N + BN_OUT - 1) / BN_OUT;
    const int out = values_by(p.y, p.copy, p.ldy, p.N), in = p.addend == nullptr ? 8 : values_by(p.addend, 0, p.ldadd, p.N);
    t.store = out < in ? out : in;
    t.direct = t.store == 8 && (MODE == MODE_SWIGLU || p.act == TPAMD_ACT_NONE) && aligned(p.sw, 16) && aligned(p.sw2, 16) && aligned(p.bias, 8) &&
               (p.addend == nullptr || p.ldadd < (1ll << 21));
    const int kt = (p.K + A8_BK - 1) / A8_BK;
    int dev = 0, cus = 256;
    const size_t plane = static_cast<size_t>(t.tiles_m) * t.tiles_n * (BM * 64 * TN) * sizeof(int);  // a range's partial tiles
    if (splits > 1) {  // no more ranges than every stream's buffer has room for, whichever call allocated it
        TPAMD_HIP(hipGetDevice(&dev));
        if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
        const size_t most = scratch_reserve(cus) / plane;
        splits = most < 1 ? 1 : most < static_cast<size_t>(splits) ? static_cast<int>(most) : splits;
    }
    t.kt_per_split = (kt + splits - 1) / splits;
    t.splits = (kt + t.kt_per_split - 1) / t.kt_per_split;
    if (t.splits > 1) {
        const size_t need = t.splits * plane;
        std::lock_guard<std::mutex> hold(splitk_mutex(dev));
        void *ws = nullptr;
        if (int rc = splitk_scratch(dev, s, need, scratch_reserve(cus), &ws); rc != TPAMD_OK) return rc;
        if (ws != nullptr) {
            t.ws = static_cast<int *>(ws);
            if (int rc = launch_tiles<DT, MODE, TM, TN, NS, true, false>(p, t, s); rc != TPAMD_OK) return rc;
            const int64_t units = static_cast<int64_t>(t.tiles_m) * t.tiles_n * 4 * TM * TN;
            hipLaunchKernelGGL((finish_a8_kernel<DT, MODE, TM, TN>), dim3(static_cast<unsigned>((units + 3) / 4)), dim3(256), 0, s, p, t);
            TPAMD_HIP(hipGetLastError());
            return TPAMD_OK;
        }
        t.splits = 1;  // no scratch memory for the stream: all of K in a block
        t.kt_per_split = kt;
    }
    if constexpr (MODE == MODE_LINEAR)
        if (p.addend != nullptr) return launch_tiles<DT, MODE, TM, TN, NS, false, true>(p, t, s);
    return launch_tiles<DT, MODE, TM, TN, NS, false, false>(p, t, s);
}

template <int DT, int MODE>
int launch_a8_tile(const A8Params &p, int tm, int tn, int splits, hipStream_t s) {
#define A8_TILE(tm, tn, stages) case tm * 8 + tn: return launch_a8<DT, MODE, tm, tn, stages>(p, splits, s)
    switch (tm * 8 + tn) {
        A8_TILE(1, 2, 3);
        A8_TILE(2, 2, 3);
        A8_TILE(2, 3, 3);
        A8_TILE(3, 3, 3);
        A8_TILE(3, 4, 2);
        A8_TILE(4, 4, 2);
    }
#undef A8_TILE
    set_error("a8: no tile of %d x %d rows", 64 * tm, 64 * tn);
    return TPAMD_ERR_UNSUPPORTED;
}

}  // namespace

// K a multiple of 16, at least 16; ldx, ldw multiples of 16 below 2^22; x, w, w2 on 16-byte boundaries.
int gemm_a8(const A8Params &p, bool pair, int dtype, int tm, int tn, int splits, hipStream_t s) {
    if (dtype == TPAMD_BF16) return pair ? launch_a8_tile<TPAMD_BF16, MODE_SWIGLU>(p, tm, tn, splits, s) : launch_a8_tile<TPAMD_BF16, MODE_LINEAR>(p, tm, tn, splits, s);
    return pair ? launch_a8_tile<TPAMD_F16, MODE_SWIGLU>(p, tm, tn, splits, s) : launch_a8_tile<TPAMD_F16, MODE_LINEAR>(p, tm, tn, splits, s);
}

}  // namespace tpamd
