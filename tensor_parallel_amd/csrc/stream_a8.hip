#include "a8.h"
#include "gemm_tile.h"
#include "stream_model.h"

namespace tpamd {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int SA_NW = 4;        // wavefronts per block
constexpr int SA_LDS_KB = 160;  // one block per CU
// Most stages, by the loads of one. Three are enough but where a stage is small: three take 0.98 of the time of four at 16 x 16384 x 8192, 32 x 4096 x 5504 and the pair of 8 x 5504 x 4096, but 1.02 at
// 1 x 4096 x 5504 and 1.03 at 1 x 2048 x 4096; six or eight cost 1-6 % on small matrices and change nothing on large ones.
constexpr int sa_depth(int loads) { return loads <= 4 ? 4 : 3; }

// stream_a8_kernel: products of up to 64 rows of 8-bit codes on one block per CU, cut and staged as stream_kernel cuts and stages 16-bit ones (stream.hip): a block owns an even share of the
// columns and all of K, its wavefronts contiguous quarters of K, 128 elements (bytes) of NR weight rows (a pair: gate rows, then up rows) and XR rows of x at a time through rings of their own in
// LDS, filled by loads that go straight there; the wavefronts' sums meet in LDS. K ends in a multiple of 16: the pieces of x behind it are asked for outside the descriptor's range, which
// gives zeros, and so are rows that there are none of, which cost no memory traffic (reading the last row in their place takes 8 % longer at 16 x 16384 x 8192).
// The matrix pipe idles (a stage's MFMAs take 2-6 % of its time), so the half-rate 16 x 16 form serves, whose rows of 16 fit few columns a CU.
// Bound: memory, N K bytes of weights: 16 x 16384 x 8192 in 25.5 us, 5.3 TB/s where a large copy has 6.0; at smaller matrices its latency: a launch and the first loads are 3.4 us of 6.1 for
// 1 x 4096 x 5504 (22.5 MB), of 10.1 for the pair of 8 x 5504 x 4096 (45 MB; 17 rows 10.8, 32 rows 11.9, 48 13.7). From 33 rows on x, which every CU reads whole from the L2: 32 x 4096 x 5504 9.1, 64 rows 12.2.
// Two ranks' products are one launch with half the CUs each (blockIdx.y).
// Slower, tried: weights straight into registers in the order of the matrix instructions (16 rows x 64 bytes a load: 37 us for the first), two blocks of half the LDS to a CU, eight wavefronts.
__device__ __forceinline__ const float *by_bytes(const float *p, int64_t bytes) { return reinterpret_cast<const float *>(reinterpret_cast<const char *>(p) + bytes); }

template <int DT, bool PAIR, int NR, int XR, int D>
__global__ __launch_bounds__(SA_NW * 64) void stream_a8_kernel(A8Params p) {
    constexpr int NT = (NR + 15) / 16, MT = (XR + 15) / 16, KK = 2;
    constexpr int RP = 8, PITCH = 128;  // rows per load, bytes of a staged row
    constexpr int NB = NR / RP, XB = XR / RP, L = NB + XB, STAGE = L * 1024, RING = D * STAGE;
    constexpr int UP = PAIR ? NR / 2 : 0;
    static_assert(NR % RP == 0 && XR % RP == 0 && UP % RP == 0, "whole loads");
    static_assert(SA_NW * RING <= SA_LDS_KB * 1024 && D >= 2 && (D - 1) * L < 64, "LDS, and the count in s_waitcnt");
    static_assert(NT * MT * 1024 <= RING, "the partial sums take the place of the stages");
    constexpr int XLAST = XR - (MT - 1) * 16;  // staged rows of the last 16 of x: the lanes of the others read these again
    static_assert(NT * 16 * PITCH <= STAGE && NB * 1024 + ((MT - 1) * 16 + XLAST) * PITCH <= STAGE && (XLAST & (XLAST - 1)) == 0, "fragments are read inside their stage");
    extern __shared__ __align__(16) char smem[];
    if (blockIdx.y != 0) {
        p.x += p.to.x; p.w += p.to.w; p.w2 += p.to.w2; p.bias += p.to.bias; p.y += p.to.y;
        p.sx = by_bytes(p.sx, p.to.sx); p.sw = by_bytes(p.sw, p.to.sw); p.sw2 = by_bytes(p.sw2, p.to.sw2);
    }

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4, rb = lane >> 3;
    const int n0 = static_cast<int>(static_cast<int64_t>(p.N) * blockIdx.x / gridDim.x);
    const int cols = static_cast<int>(static_cast<int64_t>(p.N) * (blockIdx.x + 1) / gridDim.x) - n0;
    const int KU = (p.K + 127) / 128, pieces = (p.K - (KU - 1) * 128) / 16;
    const int first = KU * wave / SA_NW, units = KU * (wave + 1) / SA_NW - first;
    // blocks start at different places of long rows: they would otherwise ask for the same columns of all rows at one time, which the memory channels answer unevenly
    const int skew = units >= 32 ? static_cast<int>(((blockIdx.x >> 3) * 5 + (blockIdx.x & 7) * 3) % static_cast<unsigned>(units)) : 0;
    const uint32_t ldw = static_cast<uint32_t>(p.ldw), ldx = static_cast<uint32_t>(p.ldx);
    uint32_t w_off[NB], x_off[XB], behind[2];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int row = j * RP + rb, r = row - (PAIR && j >= NB / 2 ? UP : 0);
        w_off[j] = r < cols ? static_cast<uint32_t>(r) * ldw + ((lane & 7) ^ ((row >> 1) & 7)) * 16 : 0x80000000u;
    }
#pragma unroll
    for (int j = 0; j < XB; ++j) {
        const int row = j * RP + rb;
        x_off[j] = row < p.M ? static_cast<uint32_t>(row) * ldx + ((lane & 7) ^ ((row >> 1) & 7)) * 16 : 0x80000000u;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) behind[h] = static_cast<int>((lane & 7) ^ ((h * 4 + (rb >> 1)) & 7)) >= pieces ? 0x80000000u : 0u;
    const uint32_t w_extent = static_cast<uint32_t>(cols - 1) * ldw + static_cast<uint32_t>(p.K);
    const __amdgpu_buffer_rsrc_t w_rsrc = make_rsrc(p.w + static_cast<int64_t>(n0) * ldw, w_extent);
    const __amdgpu_buffer_rsrc_t w2_rsrc = PAIR ? make_rsrc(p.w2 + static_cast<int64_t>(n0) * ldw, w_extent) : w_rsrc;
    const __amdgpu_buffer_rsrc_t x_rsrc = make_rsrc(p.x, static_cast<uint32_t>(p.M - 1) * ldx + static_cast<uint32_t>(p.K));
    // Weights pass the caches by, unless rows begin inside 128-byte lines: the next unit then asks for the rest of a line (the pair of 8 x 5504 x 4112 takes 0.88 of the time so, 12.6 us, 16 x 16384 x 8208
    // 0.85, 33.8; whole lines kept in the caches cost 16 x 16384 x 8192 9 %)
    const bool whole_lines = ((reinterpret_cast<uintptr_t>(p.w) | reinterpret_cast<uintptr_t>(p.w2) | static_cast<uintptr_t>(p.ldw)) & 127) == 0;
    char *ring = smem + wave * RING;
    auto load = [&](int stage_off, int i) __attribute__((always_inline)) {  // unit number i of this wavefront; behind the last one the same count of loads from outside the descriptors
        const int t = i < units ? skew + i : 0;  // (the wavefront-uniform offset stays inside the extents)
        const int u = first + (t < units || t == 0 ? t : t - units);
        const uint32_t none = i < units ? 0u : 0x80000000u;
        unrolled<NB>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            const __amdgpu_buffer_rsrc_t rsrc = PAIR && j >= NB / 2 ? w2_rsrc : w_rsrc;
            lds_void *to = (lds_void *)(ring + stage_off + j * 1024);
            const int at = static_cast<int>(w_off[j] | none);
            if (whole_lines) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 16, at, u * PITCH, 0, 2);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 16, at, u * PITCH, 0, 0);
        });
        unrolled<XB>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            buffer_load16_to_lds(x_rsrc, x_off[j] | none | (u == KU - 1 ? behind[j & 1] : 0u), u * PITCH, ring + stage_off + (NB + j) * 1024);
        });
    };

    i32x4 acc[NT][MT];
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int a = 0; a < MT; ++a) acc[b][a] = i32x4{0, 0, 0, 0};

    unrolled<D>([&](auto sc) { load(decltype(sc)::value * STAGE, decltype(sc)::value); });
    const uint32_t rd = lds_addr_of(ring) + l16 * PITCH;
    const uint32_t rd_last = lds_addr_of(ring) + (l16 & (XLAST - 1)) * PITCH;
    uint32_t kk_off[KK];
#pragma unroll
    for (int k = 0; k < KK; ++k) kk_off[k] = static_cast<uint32_t>(((k * 4 + lq) ^ (l16 >> 1)) * 16);
    int stage_off = 0;
    for (int i = 0; i < units; ++i) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * L) : "memory");
        u32x4 wq[KK][NT], xq[KK][MT];
        unrolled<KK>([&](auto hc) {
            constexpr int h = decltype(hc)::value;
            const uint32_t at = rd + stage_off + kk_off[h], at_last = rd_last + stage_off + kk_off[h];
            unrolled<NT>([&](auto bc) { wq[h][decltype(bc)::value] = lds_read16<decltype(bc)::value * 16 * PITCH>(at); });
            unrolled<MT>([&](auto ac) { xq[h][decltype(ac)::value] = lds_read16<NB * 1024 + decltype(ac)::value * 16 * PITCH>(decltype(ac)::value == MT - 1 ? at_last : at); });
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        unrolled<KK>([&](auto hc) {
            constexpr int h = decltype(hc)::value;
            unrolled<NT>([&](auto bc) { already_landed(wq[h][decltype(bc)::value]); });
            unrolled<MT>([&](auto ac) { already_landed(xq[h][decltype(ac)::value]); });
        });
        load(stage_off, i + D);
#pragma unroll
        for (int h = 0; h < KK; ++h)
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int a = 0; a < MT; ++a)
                    acc[b][a] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wq[h][b]), __builtin_bit_cast(i32x4, xq[h][a]), acc[b][a], 0, 0, 0);
        stage_off = stage_off + STAGE == RING ? 0 : stage_off + STAGE;
    }
    // every load into the stages has landed before the partial sums take their place
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    i32x4 *red = reinterpret_cast<i32x4 *>(smem);
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int a = 0; a < MT; ++a) red[(wave * NT * MT + b * MT + a) * 64 + lane] = acc[b][a];
    __syncthreads();
    const int *sums = reinterpret_cast<const int *>(smem);
    auto total = [&](int row, int m) __attribute__((always_inline)) {
        const int at = (((row >> 4) * MT + (m >> 4)) * 64 + ((row & 15) >> 2) * 16 + (m & 15)) * 4 + (row & 3);
        int s = 0;
#pragma unroll
        for (int v = 0; v < SA_NW; ++v) s += sums[v * NT * MT * 256 + at];
        return s;
    };
    for (int e = tid; e < cols * p.M; e += SA_NW * 64) {
        const int m = e / cols, c = e - m * cols, n = n0 + c;
        const float sx = p.sx[m];
        uint16_t out;
        if constexpr (PAIR) {
            out = a8_round<DT>(a8_gated(a8_linear(total(c, m), sx, p.sw[n], 0.f), a8_linear(total(c + UP, m), sx, p.sw2[n], 0.f)));
        } else {
            out = a8_round<DT>(a8_act(a8_linear(total(c, m), sx, p.sw[n], p.bias != nullptr ? half_to_f32<DT>(reinterpret_cast<const uint16_t *>(p.bias)[n]) : 0.f), p.act));
            if (p.addend != nullptr) out = f32_to_half<DT>(half_to_f32<DT>(out) + half_to_f32<DT>(reinterpret_cast<const uint16_t *>(p.addend)[m * p.ldadd + n]));
        }
        uint16_t *y = reinterpret_cast<uint16_t *>(p.y) + m * p.ldy + n;
        *y = out;
        if (!PAIR && p.copy != 0) *reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(y) + p.copy) = out;
    }
}

template <int DT, bool PAIR, int NR, int XR>
int launch_nr(const A8Params &p, int blocks, int ranks, hipStream_t s) {
    constexpr int L = (NR + XR) / 8, DM = SA_LDS_KB / SA_NW / L, D = DM < sa_depth(L) ? DM : sa_depth(L);
    static_assert(D >= 2, "LDS");
    constexpr int LDS = SA_NW * D * L * 1024;
    auto kern = stream_a8_kernel<DT, PAIR, NR, XR, D>;
    static thread_local int configured_dev = -1;  // per instantiation and host thread
    int dev = 0;
    TPAMD_HIP(hipGetDevice(&dev));
    if (configured_dev != dev) {
        TPAMD_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
        configured_dev = dev;
    }
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(ranks)), dim3(SA_NW * 64), LDS, s, p);
    TPAMD_HIP(hipGetLastError());
    return TPAMD_OK;
}

template <int DT, bool PAIR, int XR>
int launch_xr(const A8Params &p, int nr, int blocks, int ranks, hipStream_t s) {
#define SA_ROWS(n) case n: return launch_nr<DT, PAIR, n, XR>(p, blocks, ranks, s)
    switch (nr) {
        SA_ROWS(32);
        SA_ROWS(48);
        SA_ROWS(64);
        SA_ROWS(80);
        SA_ROWS(96);
    }
    if constexpr (!PAIR) {
        switch (nr) {
            SA_ROWS(16);
            SA_ROWS(24);
        }
    }
#undef SA_ROWS
    set_error("a8: no kernel of %d rows", nr);
    return TPAMD_ERR_UNSUPPORTED;
}

template <int DT, bool PAIR>
int launch_m(const A8Params &p, int nr, int blocks, int ranks, hipStream_t s) {
    if (p.M <= 8) return launch_xr<DT, PAIR, 8>(p, nr, blocks, ranks, s);
    if (p.M <= 16) return launch_xr<DT, PAIR, 16>(p, nr, blocks, ranks, s);
    if (p.M <= 24) return launch_xr<DT, PAIR, 24>(p, nr, blocks, ranks, s);
    if (p.M <= 32) return launch_xr<DT, PAIR, 32>(p, nr, blocks, ranks, s);
    if (p.M <= 48) return launch_xr<DT, PAIR, 48>(p, nr, blocks, ranks, s);
    return launch_xr<DT, PAIR, 64>(p, nr, blocks, ranks, s);
}

}  // namespace

bool stream_a8_takes(const A8Params &p, bool pair, int ranks, int cus) { return p.M <= 64 && stream_cut(p.N, ranks, pair, false, cus).groups > 0; }

// Fitted to 300 shapes of 1-64 rows (within 8 % of them in the mean, and of 150 others): each turn of the blocks costs 3.4 us, what it stages of weight rows (padded ones too) 0.010 us per KB,
// of x 0.012, what it reads of memory 0.028 with every CU at it, and a thousand outputs 1.6.
float stream_a8_us(const A8Params &p, bool pair, int cus) {
    const StreamCut cut = stream_cut(p.N, 1, pair, false, cus);
    const int xr = p.M <= 32 ? (p.M + 7) / 8 * 8 : p.M <= 48 ? 48 : 64;
    const float k = static_cast<float>(p.K) * 1e-3f, columns = static_cast<float>((p.N + cut.blocks - 1) / cut.blocks * (pair ? 2 : 1));
    const float busy = cut.blocks < cus ? static_cast<float>(cut.blocks) / static_cast<float>(cus) : 1.f;
    return static_cast<float>(cut.groups) *
           (3.37f + k * (0.0101f * static_cast<float>(cut.rows) + 0.0118f * static_cast<float>(xr) + 0.028f * columns * busy) + 1.62e-3f * columns * static_cast<float>(p.M));
}

int stream_a8(const A8Params &p, bool pair, int dtype, int ranks, int cus, hipStream_t s) {
    const StreamCut cut = stream_cut(p.N, ranks, pair, false, cus);
    TPAMD_REQUIRE(cut.groups > 0, "a8: no cut of %d columns", p.N);
    if (dtype == TPAMD_BF16) return pair ? launch_m<TPAMD_BF16, true>(p, cut.rows, cut.blocks, ranks, s) : launch_m<TPAMD_BF16, false>(p, cut.rows, cut.blocks, ranks, s);
    return pair ? launch_m<TPAMD_F16, true>(p, cut.rows, cut.blocks, ranks, s) : launch_m<TPAMD_F16, false>(p, cut.rows, cut.blocks, ranks, s);
}

}  // namespace tpamd
