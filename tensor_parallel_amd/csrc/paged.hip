// Attention of new rows on keys and values that lie in pages: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the positions j <= length - count + i of the row's
// sequence. Sequences of one call differ in length and in how many new rows they have, and none of that is known to the host: lengths, starts and the page table are
// read by the kernels.
//
// A sequence whose rows (new rows times query heads of a key/value head) fill at most one MFMA tile of 16 goes to paged_few_kernel, which is bound by reading keys and
// values once; any other to paged_many_kernel, bound by its matrix products and exponentials. A call that may have both kinds runs both (with blocks of 4 wavefronts as one
// launch, paged_both_kernel); each leaves the other's sequences alone. What was cut is joined by paged_merge_kernel.
//
// Both load K and V straight into LDS, 16 positions by 16 positions: those lie in one page (pages have 16 positions or more, a power of two), so that a page is looked
// up once for them and the loads have one descriptor and fixed offsets. A piece (16 bytes) c of a staged row r is in slot c ^ turned(r): rows are read as MFMA operands
// (16 or 32 rows, one piece each) and through the transposing read (4 consecutive rows, 2 or 4 neighbouring pieces) without bank conflicts.
#include "gemm_tile.h"
#include "paged.h"

#include <math.h>

namespace tpamd {
namespace {

constexpr int FEW = 16;    // rows of a paged_few_kernel item
constexpr int GROUP = 16;  // positions that lie in one page
constexpr int UNIT = 64;   // positions of a piece of paged_few_kernel's work: a group for each of its wavefronts
constexpr int START = 3;   // units that the start and the end of an item cost about as much as; 200 sequences of 100 positions and 4 of 8000, 32 heads on 8 of 128: 60, 51, 48, 52 us with 0, 1, 3, 6

struct PagedParams {
    const char *q;
    char *o;
    int64_t q_row, q_head, o_row, o_head;  // elements
    float *many_part, *few_part;
    float scale_log2;  // scale * log2(e)
    int Hkv, G;
    int few, many;     // which of the kernels run
    int spread;        // paged_many_kernel: blocks that its work is spread over; 0: a row tile is never cut
    int least;         // paged_few_kernel: the least share of a block; 0: a block takes one item, whole
    PagesView pages;
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

template <int D>
__device__ __forceinline__ constexpr int turned(int r) {
    if constexpr (D == 64) return ((r >> 1) & 1) << 2 | ((r >> 3) & 1) << 1 | ((r >> 2) & 1);  // two rows share 256 bytes
    else if constexpr (D == 96) return (r >> 2) & 3;
    else return (r & 3) << 2 | ((r >> 2) & 3);
}

template <int OFFSET>
__device__ __forceinline__ u32x2 lds_transpose_read(uint32_t at) {  // ds_read_b64_tr_b16, unseen by the compiler (as lds_read16)
    static_assert(OFFSET >= 0 && OFFSET < 65536, "ds offset field is 16 bits");
    u32x2 v;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(at), "n"(OFFSET));
    return v;
}
__device__ __forceinline__ void half_landed(u32x2 &r) { asm volatile("" : "+v"(r)); }

template <int DT>
__device__ __forceinline__ f32x4 mfma16_k16(u32x2 a, u32x2 b, f32x4 c) {
    if constexpr (DT == TPAMD_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
    } else {
        typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
    }
}
template <int DT>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (DT == TPAMD_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Values that some rows of a tile do not see may be infinite or NaN, and zero times those would reach the rows through the matrix product. They go in as zeros. Where there are any, two more
// products, of the largest bf16 value in the place of every +inf and NaN (then of its negative in the place of -inf and NaN) and of every probability of a position that the row sees (which may be
// too small for the dtype, and is not zero for that), add what overflows to an infinity where it belongs: through the same sums, which are touched by nothing but matrix instructions.
template <int DT>
struct Beyond {
    static constexpr uint32_t E = DT == TPAMD_BF16 ? 0x7f80u : 0x7c00u, LAST = DT == TPAMD_BF16 ? 0x0080u : 0x0400u, HUGE_BF16 = 0x7f7fu;
    // a bit of 0x80008000 for either value whose exponent is all ones (adding the exponent's last bit carries out of it)
    static __device__ __forceinline__ uint32_t carries(uint32_t two) { return (two & (E << 16 | E)) + (LAST << 16 | LAST); }
    static __device__ __forceinline__ uint32_t finite(uint32_t two) {
        return two & (((two & E) == E ? 0u : 0xffffu) | ((two & (E << 16)) == (E << 16) ? 0u : 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t huge_one(uint32_t h, uint32_t sign) {  // of the low half: NaN and the infinity of this sign
        return (h & E) == E && ((h & 0x7fffu) != E || (h & 0x8000u) == sign) ? HUGE_BF16 | sign : 0u;
    }
    static __device__ __forceinline__ uint32_t huge(uint32_t two, uint32_t sign) { return huge_one(two & 0xffffu, sign) | huge_one(two >> 16, sign) << 16; }
    static __device__ __forceinline__ uint32_t seen(int most) { return (most >= 0 ? HUGE_BF16 : 0u) | (most >= 1 ? HUGE_BF16 << 16 : 0u); }  // of two positions, where those up to the most-th are seen
};

// The descriptor of 16 rows that begin at `base`: nothing (loads give zeros) where there is no page.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t group_rsrc(const char *pool, int page, int64_t page_step, int64_t head, int slot, int64_t pos_step, int D) {
    const char *base = pool + (static_cast<int64_t>(page < 0 ? 0 : page) * page_step + head + static_cast<int64_t>(slot) * pos_step) * 2;
    const uint32_t extent = page < 0 ? 0u : (15u * static_cast<uint32_t>(pos_step) + static_cast<uint32_t>(D)) * 2u;
    return make_rsrc(base, extent);
}

// A value that was loaded is here from now on: the compiler would otherwise wait for it inside the loop that uses it, and with it for loads that the loop has requested.
__device__ __forceinline__ void arrived(int &v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void arrived(u32x4 &v) { asm volatile("" : "+v"(v)); }

// What the sum of a row's products is multiplied by, l its probabilities' sum and `last` the last position it sees: nothing for a row in front of position 0. A row all of whose scores are -inf has no
// softmax: its sums are zeros, and zero times 1 / 0 the NaN that it is by definition.
__device__ __forceinline__ float factor_of(float l, int last) { return last >= 0 ? 1.0f / l : 0.f; }

// ---- which rows go where ---------------------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ bool is_few(const PagedParams &p, int count) { return p.few && count > 0 && count * p.G <= FEW; }
__device__ __forceinline__ int units_of(const PagedParams &p, const SeqRows &s) {
    return is_few(p, s.count) ? max((s.length + UNIT - 1) / UNIT, 1) : 0;  // one for a sequence without positions too: its rows are zeros
}
// What it costs a block of paged_few_kernel: its units, behind START for getting there.
__device__ __forceinline__ int cost_of(const PagedParams &p, const SeqRows &s) {
    const int n = units_of(p, s);
    return n == 0 ? 0 : n + START;
}
// paged_many_kernel's share of a sequence: tiles of ROWS rows (0 for the other kernel's sequences), and the tiles of KT positions that its first and its last row tile see.
struct Tiles {
    int rows, first, last;
};
template <int ROWS, int KT>
__device__ __forceinline__ Tiles tiles_of(const PagedParams &p, const SeqRows &s) {
    if (s.count <= 0 || is_few(p, s.count)) return {0, 0, 0};
    const int rows = s.count * p.G, before = s.length - s.count;
    return {(rows + ROWS - 1) / ROWS, (max(before + (min(rows, ROWS) - 1) / p.G + 1, 0) + KT - 1) / KT, (s.length + KT - 1) / KT};
}
// 64 sequences, one in a lane: lengths and counts of a batch are loaded once and asked for by lane from then on.
struct Lanes {
    SeqRows mine;
    int b0;
};
__device__ __forceinline__ Lanes lanes_from(const PagedParams &p, int b0) {
    Lanes l{{0, 0, 0}, b0};
    const int b = b0 + static_cast<int>(threadIdx.x & 63);
    if (b < p.pages.seqs) l.mine = rows_of(p.pages, b);
    return l;
}
__device__ __forceinline__ SeqRows pick(const PagedParams &p, Lanes &l, int b) {  // b: the same in all lanes
    if (b - l.b0 >= 64 || b < l.b0) l = lanes_from(p, b & ~63);
    const int at = b - l.b0;
    return {__builtin_amdgcn_readlane(l.mine.first, at), __builtin_amdgcn_readlane(l.mine.count, at), __builtin_amdgcn_readlane(l.mine.length, at)};
}
// v of the lanes that a DPP control names, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ int from_lanes(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lanes(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = from_lanes<CTRL, ROWS>(static_cast<int>(u)), hi = from_lanes<CTRL, ROWS>(static_cast<int>(u >> 32));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// The sum over this lane and those before it, by moves inside the vector unit (1, 2, 4, 8 lanes up in a row of 16, then the last lane of a row to the next, of 32 to the others): six trips through
// LDS are 0.3 us, and every block has two or three such sums in front of its first load.
template <class T>
__device__ __forceinline__ T sums_to_lane(T v) {
    v += from_lanes<0x111, 0xf>(v);
    v += from_lanes<0x112, 0xf>(v);
    v += from_lanes<0x114, 0xf>(v);
    v += from_lanes<0x118, 0xf>(v);
    v += from_lanes<0x142, 0xa>(v);
    v += from_lanes<0x143, 0xc>(v);
    return v;
}
// The sum over all sequences of what `of` gives; l holds the first 64.
template <class F>
__device__ __forceinline__ int sum_over(const PagedParams &p, const Lanes &l, F &&of) {
    int mine = of(l.mine);
    for (int b0 = 64; b0 < p.pages.seqs; b0 += 64) mine += of(lanes_from(p, b0).mine);
    return __builtin_amdgcn_readlane(sums_to_lane(mine), 63);
}
// The sequence that the at-th of these falls into (0 <= at < their sum), and how many come before that sequence's; l ends up with it among its 64.
template <class F>
__device__ __forceinline__ int find_in(const PagedParams &p, Lanes &l, int at, int &before, F &&of) {
    int done = 0;
    for (int b0 = 0; b0 < p.pages.seqs; b0 += 64) {
        if (b0 != l.b0) l = lanes_from(p, b0);
        const int mine = of(l.mine), sum = sums_to_lane(mine);
        const uint64_t hit = __ballot(done + sum > at);
        if (hit != 0) {
            const int lane = __ffsll(static_cast<unsigned long long>(hit)) - 1;
            before = done + __builtin_amdgcn_readlane(sum, lane) - __builtin_amdgcn_readlane(mine, lane);
            return b0 + lane;
        }
        done += __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}
// The positions of a sequence's row tiles are cut into ranges where the tiles have more of them than an equal share of all work (in tiles of KT positions) on `spread` blocks, so that a few long
// sequences in a batch do not keep a few blocks busy when all others have ended. Sums of whole numbers in 64 bits: exact. With R the share there are at most sum(1 + work / R) = row tiles +
// spread ranges, and fewer than 2 spread of tiles that are cut.
constexpr int LEAST_TILES = 4;  // of a range: with 8 512 rows of 16 heads of 128 take 22.7 us instead of 20.7, 32 rows on 500 14.4 instead of 13.2
template <int ROWS, int KT>
__device__ __forceinline__ int range_tiles(const PagedParams &p, const Lanes &l) {
    if (p.spread == 0) return 0;
    auto work = [&](const SeqRows &s) {
        const Tiles t = tiles_of<ROWS, KT>(p, s);
        return static_cast<double>(t.rows) * (t.first + t.last);
    };
    double mine = work(l.mine);
    for (int b0 = 64; b0 < p.pages.seqs; b0 += 64) mine += work(lanes_from(p, b0).mine);
    const double share = ceil(__shfl(sums_to_lane(mine), 63) * p.Hkv / (2.0 * p.spread));
    return __builtin_amdgcn_readfirstlane(share < 1.0e9 ? max(static_cast<int>(share), LEAST_TILES) : 1000000000);
}
__device__ __forceinline__ int ranges_of(const Tiles &t, int range) { return range == 0 ? 1 : max((t.first + t.last + 2 * range - 1) / (2 * range), 1); }

// What a block of paged_few_kernel takes: alike for all, but `least` at least.
__device__ __forceinline__ int share_of(const PagedParams &p, int cost, int blocks) { return max(p.least, (cost + blocks - 1) / blocks); }

// ---- few rows --------------------------------------------------------------------------------------------------------------------------------------------------------
// An item is one key/value head of one sequence, its work the sequence's positions in units of 64. The costs of all items (their units, and START units in front of them), one after
// another, are cut into equal shares, one for a block, so that a batch of sequences of very different lengths keeps all blocks busy to the end; where a cut falls inside an item, both sides
// leave (m, l, O) as partials, and few_merge joins them. A block has at most two such pieces (its first and its last), so the partials' memory does not
// grow with the batch. `least` == 0: a block takes an item whole and nothing is merged.
//
// Inside a block each of the 4 wavefronts (8: plan_of) takes every fourth 16 positions through LDS stages of their own and meet at the end of an item.
//
// Bound by HBM where there is enough to read: 100000 positions of 8 key/value heads of 128 elements 66 us and their merge 5 (410 MB, 5.7 TB/s of the whole call); 64 sequences of 81 to
// 7113 positions, 4 key/value heads of 64 elements: 27 and 6. Below that by the way to the first positions: 500 positions of 16 heads of 128 elements 8.0 us in a graph on three pools in turn,
// 8.8 on so many that they come from HBM.
template <int DT, int D, int WAVES, int NST>
__device__ __forceinline__ void few_rows(const PagedParams &p, const int share_index, const int blocks) {
    constexpr int PITCH = D * 2, LK = D / 32, LPS = 2 * LK, VAT = GROUP * PITCH, STAGE = 2 * VAT, RING = NST * STAGE;
    constexpr int DK = D / 32, DT16 = D / 16, PW = D + 4, PIECES = D / 8;
    static_assert(NST >= 2 && (NST - 1) * LPS < 64, "the count in s_waitcnt");
    static_assert(FEW * PW * 4 <= RING, "the partials take the place of the stages");
    extern __shared__ __align__(1024) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, lq = lane >> 4;
    char *ring = smem + wave * RING;

    // ---- this block's share
    int b, hkv, at, left;  // where it begins, inside an item's cost, and how much it has
    auto costs = [&](const SeqRows &s) { return cost_of(p, s); };
    Lanes seqs = lanes_from(p, p.least == 0 ? share_index / p.Hkv & ~63 : 0);
    int first_pages = -1;  // of a whole item, asked for together with its length
    if (p.least == 0) {
        b = share_index / p.Hkv;
        hkv = share_index - b * p.Hkv;
        at = 0;
        const int position = (wave + WAVES * lane) * GROUP;
        if (position < p.pages.room) first_pages = page_of(p.pages, b, position);
        left = cost_of(p, pick(p, seqs, b));
        if (left == 0) return;
    } else {
        const int all = sum_over(p, seqs, costs) * p.Hkv, share = share_of(p, all, blocks);
        const int64_t from = static_cast<int64_t>(share_index) * share;
        if (from >= all) return;
        left = min(share, all - static_cast<int>(from));
        // costs of a sequence before all heads': the scan counts a sequence once
        int before;
        b = find_in(p, seqs, static_cast<int>(from) / p.Hkv, before, costs);
        const int cost = cost_of(p, pick(p, seqs, b)), inside = static_cast<int>(from) - before * p.Hkv;
        hkv = inside / cost;
        at = inside - hkv * cost;
    }
    // pieces of 1024 bytes of a group: which row and piece this lane loads
    uint32_t k_off[LK], v_off[LK];
#pragma unroll
    for (int j = 0; j < LK; ++j) {
        const int at = j * 64 + lane, r = at / PIECES, piece = (at % PIECES) ^ turned<D>(r);
        k_off[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.pages.k_pos) * 2 + piece * 16;
        v_off[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.pages.v_pos) * 2 + piece * 16;
    }
    const int vkey = 4 * lq + (l16 >> 2);  // the row and 8-byte piece that this lane points the transposing read at
    const uint32_t k_rd = lds_addr_of(ring) + l16 * PITCH + (lq ^ turned<D>(l16)) * 16;
    const uint32_t v_rd = lds_addr_of(ring) + VAT + vkey * PITCH + (((l16 & 3) >> 1) ^ turned<D>(vkey)) * 16 + (l16 & 1) * 8;

    while (left > 0 && b < p.pages.seqs) {
        const SeqRows s = pick(p, seqs, b);
        const int n_units = units_of(p, s);
        if (n_units == 0) {  // the other kernel's, or empty
            ++b;
            continue;
        }
        const int take = min(left, n_units + START - at), unit = max(at - START, 0), unit_end = max(at + take - START, 0);
        const int item = hkv;
        left -= take;
        at = 0;
        if (++hkv == p.Hkv) {
            hkv = 0;
            ++b;
        }
        if (unit_end == unit) continue;  // the share ends in front of the item's units
        const int seq = item + 1 == p.Hkv ? b - 1 : b;
        const int k_begin = unit * UNIT, k_end = min(unit_end * UNIT, s.length);
        const bool from_start = unit == 0, to_end = unit_end == n_units;
        const int rows = s.count * p.G;
        const int groups = k_end > k_begin ? (k_end - k_begin + GROUP - 1) / GROUP : 0;
        const int n = (groups - wave + WAVES - 1) / WAVES;  // of this wavefront: wave, wave + WAVES, ...

        // ---- this lane's row (those past the last: row 0, never stored)
        const int row = l16 < rows ? l16 : 0, place = row / p.G;
        const int last = s.length - s.count + place;  // position that the row sees last
        const int seen_by_all = s.length - s.count;
        const char *qrow = p.q + (static_cast<int64_t>(s.first + place) * p.q_row + static_cast<int64_t>(item * p.G + row - place * p.G) * p.q_head) * 2;
        u32x4 qf[DK];
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) qf[kk] = *reinterpret_cast<const u32x4 *>(qrow + (32 * kk + 8 * lq) * 2);

        f32x4 acc[DT16];
        float m_run = -INFINITY, l_run = 0.f;  // l_run: of the positions that this lane saw
#pragma unroll
        for (int dt = 0; dt < DT16; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (n > 0) {
            const int group0 = k_begin / GROUP + wave;  // of the sequence
            const int64_t k_at = item * p.pages.k_head, v_at = item * p.pages.v_head;
            // the pages of this wavefront's next 64 groups, one in a lane
            auto pages_from = [&](int i) {
                const int g = group0 + WAVES * (i + lane);
                return g * GROUP < s.length ? page_of(p.pages, seq, g * GROUP) : -1;
            };
            int my_page = p.least == 0 ? first_pages : pages_from(0), base = 0;
            arrived(my_page);
            auto load = [&](int stage_off, int i) __attribute__((always_inline)) {
                if (i < n) {
                    if (i - base == 64) {
                        base = i;
                        my_page = pages_from(i);
                        arrived(my_page);
                    }
                    const int page = __builtin_amdgcn_readlane(my_page, i - base);
                    const int slot = ((group0 + WAVES * i) * GROUP) & ((1 << p.pages.shift) - 1);
                    const __amdgpu_buffer_rsrc_t kr = group_rsrc(p.pages.k, page, p.pages.k_page, k_at, slot, p.pages.k_pos, D);
                    const __amdgpu_buffer_rsrc_t vr = group_rsrc(p.pages.v, page, p.pages.v_page, v_at, slot, p.pages.v_pos, D);
#pragma unroll
                    for (int j = 0; j < LK; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void *)(ring + stage_off + j * 1024), 16, static_cast<int>(k_off[j]), 0, 0, 2);
#pragma unroll
                    for (int j = 0; j < LK; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void *)(ring + stage_off + VAT + j * 1024), 16, static_cast<int>(v_off[j]), 0, 0, 2);
                } else {  // as many loads, so that the waits can count: of nothing
                    const __amdgpu_buffer_rsrc_t none = make_rsrc(p.pages.k, 0);
#pragma unroll
                    for (int j = 0; j < LPS; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(none, (lds_void *)(ring + stage_off + j * 1024), 16, 0, 0, 0, 0);
                }
            };
            unrolled<NST>([&](auto sc) { load(decltype(sc)::value * STAGE, decltype(sc)::value); });
            int stage_off = 0;
            for (int i = 0; i < n; ++i) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * LPS) : "memory");
                u32x4 kf[DK];
                u32x2 vf[DT16];
                unrolled<DK>([&](auto kc) {
                    constexpr int kk = decltype(kc)::value;
                    kf[kk] = lds_read16<0>(D == 96 ? k_rd + stage_off + kk * 64 : (k_rd + stage_off) ^ (kk * 64));
                });
                unrolled<DT16>([&](auto dc) {
                    constexpr int dt = decltype(dc)::value;
                    vf[dt] = lds_transpose_read<0>(D == 96 ? ((v_rd + stage_off) ^ ((dt & 1) * 32)) + (dt >> 1) * 64 : (v_rd + stage_off) ^ (dt * 32));
                });
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                unrolled<DK>([&](auto kc) { already_landed(kf[decltype(kc)::value]); });
                unrolled<DT16>([&](auto dc) { half_landed(vf[decltype(dc)::value]); });
                load(stage_off, i + NST);
                stage_off = stage_off + STAGE == RING ? 0 : stage_off + STAGE;

                // S^T = K Q^T: sc[j] = score of position 4 lq + j of the group against this lane's row
                f32x4 sc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < DK; ++kk) sc = mfma16<DT>(kf[kk], qf[kk], sc);
                const int k0 = (group0 + WAVES * i) * GROUP;
                const bool partly = k0 + GROUP - 1 > seen_by_all;  // some row does not see all of them
                if (partly) {
                    // the values behind the sequence's end are whatever the page held
                    const int have = s.length - k0 - 4 * lq;
                    const uint32_t m0 = have >= 2 ? 0xffffffffu : have == 1 ? 0xffffu : 0u, m1 = have >= 4 ? 0xffffffffu : have == 3 ? 0xffffu : 0u;
#pragma unroll
                    for (int dt = 0; dt < DT16; ++dt) vf[dt] &= u32x2{m0, m1};
                }
                // online softmax: probabilities are taken against a maximum that is raised only when a score outgrows it by 2^LAZY
                constexpr float LAZY = 6.0f;
                const float neg_ref = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[j] = fmaf(sc[j], p.scale_log2, neg_ref);
                if (partly) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[j] = k0 + 4 * lq + j <= last ? sc[j] : -INFINITY;
                }
                float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                if (__any(mx > LAZY || m_run == -INFINITY)) {
                    mx = fmaxf(mx, __shfl_xor(mx, 16));
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float m_abs = mx - neg_ref;
                    const bool up = m_abs > m_run + LAZY;  // false for -inf on either side
                    const float m_new = up ? m_abs : m_run;
                    const float m_use = m_new == -INFINITY ? 0.f : m_new;
                    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
                    const float move = -neg_ref - m_use;
                    m_run = m_new;
                    l_run *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT16; ++dt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[dt][j] *= alpha;
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[j] += move;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[j] = __builtin_amdgcn_exp2f(sc[j]);
                l_run += (sc[0] + sc[1]) + (sc[2] + sc[3]);
                // probabilities are rounded to the dtype, as the matrix instruction takes them: half a step each, errors of either sign that the sum averages. Against 64 bits results of bf16 are off by
                // 0.0021 of their size on average and of fp16 by 0.00026, where the rounding of the result alone is 0.0016 and 0.00021.
                const u32x2 pf = {pack2_half<DT>(sc[0], sc[1]), pack2_half<DT>(sc[2], sc[3])};
                u32x2 all[DT16];
                uint32_t carried = 0;
                if (partly && s.count > 1) {
#pragma unroll
                    for (int dt = 0; dt < DT16; ++dt) {
                        carried |= Beyond<DT>::carries(vf[dt].x) | Beyond<DT>::carries(vf[dt].y);
                        all[dt] = vf[dt];
                        vf[dt] = u32x2{Beyond<DT>::finite(vf[dt].x), Beyond<DT>::finite(vf[dt].y)};
                    }
                }
#pragma unroll
                for (int dt = 0; dt < DT16; ++dt) acc[dt] = mfma16_k16<DT>(vf[dt], pf, acc[dt]);
                if (__any((carried & 0x80008000u) != 0)) {
                    const int most = last - k0 - 4 * lq;
                    const u32x2 seen = {Beyond<DT>::seen(most), Beyond<DT>::seen(most - 2)};
#pragma unroll
                    for (int dt = 0; dt < DT16; ++dt)
#pragma unroll
                        for (uint32_t sign : {0u, 0x8000u}) acc[dt] = mfma16_k16<TPAMD_BF16>(u32x2{Beyond<DT>::huge(all[dt].x, sign), Beyond<DT>::huge(all[dt].y, sign)}, seen, acc[dt]);
                }
            }
        }
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
        // ---- the wavefronts' results meet in the place of the stages, once every load into them has landed
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        float *mine = reinterpret_cast<float *>(smem) + (wave * FEW + l16) * PW;
        if (l16 < rows) {
#pragma unroll
            for (int dt = 0; dt < DT16; ++dt) *reinterpret_cast<f32x4 *>(mine + 16 * dt + 4 * lq) = acc[dt];
            if (lq == 0) *reinterpret_cast<float2 *>(mine + D) = make_float2(m_run, l_run);
        }
        __syncthreads();
        constexpr int per_row = D / 4;
        const float *parts = reinterpret_cast<const float *>(smem);
        const bool whole = from_start && to_end;
        // the block's first piece, where it continues an item, has its even slot, one that goes on behind the block its odd slot
        float *out_part = p.few_part + (static_cast<int64_t>(2 * share_index) + (from_start ? 1 : 0)) * FEW * PW;
        for (int e = tid; e < rows * per_row; e += WAVES * 64) {
            const int r = e / per_row, d4 = (e % per_row) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) M = fmaxf(M, parts[(v * FEW + r) * PW + D]);
            const float m_use = M == -INFINITY ? 0.f : M;
            float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                const float weight = exp2f(parts[(v * FEW + r) * PW + D] - m_use);
                const f32x4 ov = *reinterpret_cast<const f32x4 *>(parts + (v * FEW + r) * PW + d4);
                l += weight * parts[(v * FEW + r) * PW + D + 1];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] += weight * ov[j];
            }
            if (whole) {
                const int at = r / p.G;
                const float inv = factor_of(l, seen_by_all + at);
                *reinterpret_cast<uint2 *>(p.o + (static_cast<int64_t>(s.first + at) * p.o_row + static_cast<int64_t>(item * p.G + r - at * p.G) * p.o_head + d4) * 2) =
                    make_uint2(pack2_half<DT>(o[0] * inv, o[1] * inv), pack2_half<DT>(o[2] * inv, o[3] * inv));
            } else {
                *reinterpret_cast<f32x4 *>(out_part + r * PW + d4) = f32x4{o[0], o[1], o[2], o[3]};
                if (d4 == 0) *reinterpret_cast<float2 *>(out_part + r * PW + D) = make_float2(M, l);
            }
        }
        __syncthreads();  // read before the next item's loads
    }
}

template <int DT, int D, int WAVES, int NST>
__global__ __launch_bounds__(WAVES * 64) void paged_few_kernel(PagedParams p) {
    few_rows<DT, D, WAVES, NST>(p, blockIdx.x, gridDim.x);
}

// Joins the pieces of the items that paged_few_kernel's shares cut (ys blocks an item). D / 4 lanes hold a row; a block has as many such groups as there are threads for. Of an item in a few pieces each group
// takes a row; the pieces of a longer one (a single long sequence has one in every block: 64 of them, one after another, cost 13 us) are dealt out to the groups, row by row.
template <int DT, int D>
__device__ __forceinline__ void few_merge(const PagedParams &p, const int blocks, const int item, const int y, const int ys) {
    constexpr int PW = D + 4, LANES = D / 4, TAKERS = 256 / LANES;
    __shared__ __align__(16) f32x4 sums[TAKERS][LANES];
    __shared__ float2 weights[TAKERS];
    const int b = item / p.Hkv, hkv = item - b * p.Hkv;
    Lanes seqs = lanes_from(p, 0);
    int before = 0, done = 0;
    SeqRows s{0, 0, 0};
    for (int b0 = 0; b0 < p.pages.seqs; b0 += 64) {
        if (b0 != 0) seqs = lanes_from(p, b0);
        const int mine = cost_of(p, seqs.mine), sum = sums_to_lane(mine);
        if (b >= b0 && b < b0 + 64) {
            s = pick(p, seqs, b);
            before = done + __builtin_amdgcn_readlane(sum, b - b0) - __builtin_amdgcn_readlane(mine, b - b0);
        }
        done += __builtin_amdgcn_readlane(sum, 63);
    }
    const int n = units_of(p, s), rows = s.count * p.G;
    if (n == 0) return;
    const int share = share_of(p, done * p.Hkv, blocks);
    const int from = before * p.Hkv + hkv * (n + START) + START, first = from / share, last = (from + n - 1) / share;
    if (first == last) return;  // whole in one block, which has stored it
    const bool dealt = last - first >= TAKERS;
    const int taker = threadIdx.x / LANES, d4 = (threadIdx.x % LANES) * 4, at_once = dealt ? 1 : TAKERS;
    for (int r0 = y * at_once; r0 < rows; r0 += ys * at_once) {
        const int r = dealt ? r0 : r0 + taker, step = dealt ? TAKERS : 1;
        const bool mine = taker < TAKERS && r < rows;
        float M = -INFINITY, l = 0.f;
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
        if (mine) {
            for (int i0 = first + (dealt ? taker : 0); i0 <= last; i0 += 4 * step) {
                float2 ml[4];
                f32x4 ov[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = min(i0 + j * step, last);  // the piece of block i: its odd slot where the item begins in it
                    const float *piece = p.few_part + (static_cast<int64_t>(2 * i + (i == first ? 1 : 0)) * FEW + r) * PW;
                    ml[j] = *reinterpret_cast<const float2 *>(piece + D);
                    ov[j] = *reinterpret_cast<const f32x4 *>(piece + d4);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (i0 + j * step > last) continue;
                    const float m = fmaxf(M, ml[j].x), m_use = m == -INFINITY ? 0.f : m, old = exp2f(M - m_use), now = exp2f(ml[j].x - m_use);
                    M = m;
                    l = l * old + ml[j].y * now;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = o[e] * old + ov[j][e] * now;
                }
            }
        }
        if (dealt) {
            if (mine) {
                sums[taker][d4 / 4] = o;
                if (d4 == 0) weights[taker] = make_float2(M, l);
            }
            __syncthreads();
            M = -INFINITY;
            for (int t = 0; t < TAKERS; ++t) M = fmaxf(M, weights[t].x);
            const float m_use = M == -INFINITY ? 0.f : M;
            l = 0.f;
            o = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int t = 0; t < TAKERS; ++t) {
                const float weight = exp2f(weights[t].x - m_use);
                l += weight * weights[t].y;
                for (int e = 0; e < 4; ++e) o[e] += weight * sums[t][d4 / 4][e];
            }
            __syncthreads();
        }
        if (!mine || (dealt && taker != 0)) continue;
        const int place = r / p.G;
        const float inv = factor_of(l, s.length - s.count + place);
        *reinterpret_cast<uint2 *>(p.o + (static_cast<int64_t>(s.first + place) * p.o_row + static_cast<int64_t>(hkv * p.G + r - place * p.G) * p.o_head + d4) * 2) =
            make_uint2(pack2_half<DT>(o[0] * inv, o[1] * inv), pack2_half<DT>(o[2] * inv, o[3] * inv));
    }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------------------------------------------------
// A block has 32 rows of one key/value head of one sequence for each of its 8 or 4 wavefronts (plan_of says which); row = new row * G + query head, so that the heads of a group meet the
// same keys. It walks the positions in tiles of KT through NST stages in LDS, each wavefront loading 16 rows of K or V; one barrier a tile says that the tile is there
// and that the stage before it is free.
//   S^T = K Q^T   v_mfma_f32_32x32x16 with K rows as the first operand: a lane has, of ONE query row, 16 of 32 positions, and one exchange with lane ^ 32 finishes a row's maximum
//   O^T += V^T P^T  the lane's probabilities are the second operand as they are (8 positions of each 16, in an order that the transposing read of V follows)
// Blocks are given out with the last row tiles first; ranges of a tile whose positions were cut (range_tiles) leave (m, l, O) to many_merge.
//
// A tile of 256 rows and 64 positions reads 256 KiB of fragments from LDS and has 2048 cycles of matrix instructions (heads of 128 elements), and the two do not hide behind one another: 4096 new
// rows of 32 heads on themselves take 152 - 165 us (830 - 900 TFLOP/s of what is not masked, the library's product of 8192^3 reaches 1340), 149 without a softmax and 138 without loads and barriers.
// 500 rows on 30000 positions, 16 heads: 144 us (860 TFLOP/s) and 13 for the merge of 34 MB of partials.
template <int DT, int D, int WAVES, int KT, int NST>
__device__ __forceinline__ void many_rows(const PagedParams &p, const int block) {
    constexpr int MANY = WAVES * 32, PITCH = D * 2, PIECES = D / 8, KTILE = KT * PITCH, STAGE = 2 * KTILE, PW = D + 4;
    constexpr int NL = D / 32, KK = D / 16, DT32 = D / 32, T32 = KT / 32;
    static_assert(WAVES / 2 == KT / GROUP, "a wavefront loads 16 rows of K or V");
    static_assert(NST >= 3 && (NST - 2) * NL < 64, "the count in s_waitcnt");
    extern __shared__ __align__(1024) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, h = lane >> 5;

    // ---- which rows: the last sequence's last tile first
    const int hkv = block % p.Hkv, nth = block / p.Hkv;
    Lanes seqs = lanes_from(p, 0);
    const int range = range_tiles<MANY, KT>(p, seqs);
    auto pieces_in = [&](const SeqRows &s) {
        const Tiles t = tiles_of<MANY, KT>(p, s);
        return t.rows * ranges_of(t, range);
    };
    const int all = sum_over(p, seqs, pieces_in);
    if (nth >= all) return;
    int before;
    const int b = find_in(p, seqs, all - 1 - nth, before, pieces_in);
    const SeqRows s = pick(p, seqs, b);
    const int cut = ranges_of(tiles_of<MANY, KT>(p, s), range), piece = all - 1 - nth - before, row_tile = piece / cut, nth_range = piece - row_tile * cut;
    const int row0 = row_tile * MANY;
    const int rows = s.count * p.G, seen_before = s.length - s.count;
    // a wavefront's number fixes its SIMD: rows that end early share one with rows that end late
    const int wave_row0 = row0 + (wave < 4 ? wave : 11 - wave) * 32;
    const int row = wave_row0 + l32, safe = row < rows ? row : wave_row0 < rows ? wave_row0 : 0, place = safe / p.G;
    const int last = seen_before + place;
    const int wave_first = seen_before + (wave_row0 < rows ? wave_row0 : 0) / p.G;              // what every row of the wavefront sees ends here
    const int wave_last = wave_row0 < rows ? seen_before + min(wave_row0 + 31, rows - 1) / p.G : -1;  // and what some row sees here
    const int seen = max(seen_before + min(row0 + MANY - 1, rows - 1) / p.G + 1, 0);
    const int positions = ((seen + KT - 1) / KT + cut - 1) / cut * KT;
    const int k_begin = min(nth_range * positions, seen), k_end = min(k_begin + positions, seen);
    const int tiles = (k_end - k_begin + KT - 1) / KT;

    const char *qrow = p.q + (static_cast<int64_t>(s.first + place) * p.q_row + static_cast<int64_t>(hkv * p.G + safe - place * p.G) * p.q_head) * 2;
    u32x4 qf[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = *reinterpret_cast<const u32x4 *>(qrow + (16 * kk + 8 * h) * 2);

    // ---- this wavefront's loads: 16 rows of K or V
    const bool loads_v = wave >= WAVES / 2;
    const char *pool = loads_v ? p.pages.v : p.pages.k;
    const int64_t page_step = loads_v ? p.pages.v_page : p.pages.k_page, pos_step = loads_v ? p.pages.v_pos : p.pages.k_pos, head_at = hkv * (loads_v ? p.pages.v_head : p.pages.k_head);
    const int group = wave % (WAVES / 2);
    uint32_t off[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int at = j * 64 + lane, r = at / PIECES;
        off[j] = static_cast<uint32_t>(r) * static_cast<uint32_t>(pos_step) * 2 + ((at % PIECES) ^ turned<D>(r)) * 16;
    }
    char *to = smem + (loads_v ? KTILE : 0) + group * GROUP * PITCH;
    auto pages_from = [&](int i) {
        const int at = k_begin + (i + lane) * KT + group * GROUP;
        return at < s.length ? page_of(p.pages, b, at) : -1;
    };
    int my_page = pages_from(0), base = 0;
    arrived(my_page);
    unrolled<KK>([&](auto kc) { arrived(qf[decltype(kc)::value]); });
    auto load = [&](int stage_off, int i) __attribute__((always_inline)) {
        if (i < tiles && i - base == 64) {
            base = i;
            my_page = pages_from(i);
            arrived(my_page);
        }
        const int page = i < tiles ? __builtin_amdgcn_readlane(my_page, i - base) : -1;  // behind the last tile: as many loads, of nothing
        const int slot = (k_begin + i * KT + group * GROUP) & ((1 << p.pages.shift) - 1);
        const __amdgpu_buffer_rsrc_t rsrc = group_rsrc(pool, page, page_step, head_at, slot, pos_step, D);
#pragma unroll
        for (int j = 0; j < NL; ++j) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(to + stage_off + j * 1024), 16, static_cast<int>(off[j]), 0, 0, 0);
    };

    f32x16 acc[DT32];
    float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[dt][j] = 0.f;

    // fragment addresses: row l32 of 32, piece 2 kk + h of K; rows 4 h + (l16 / 4) of 16 (and 8 further), elements 16 (l32 / 16) + 4 (l16 % 4) of 32 of V
    const uint32_t lds0 = lds_addr_of(smem);
    const uint32_t k_rd = lds0 + l32 * PITCH + (h ^ turned<D>(l32 & 15)) * 16;
    const int vkey = 4 * h + ((lane & 15) >> 2), vpiece = 2 * (l32 >> 4) + ((lane & 3) >> 1);
    const uint32_t v_rd0 = lds0 + KTILE + vkey * PITCH + (vpiece ^ turned<D>(vkey)) * 16 + (lane & 1) * 8;
    const uint32_t v_rd1 = lds0 + KTILE + (vkey + 8) * PITCH + (vpiece ^ turned<D>(vkey + 8)) * 16 + (lane & 1) * 8;

    unrolled<NST - 1>([&](auto sc) { load(decltype(sc)::value * STAGE, decltype(sc)::value); });
    int stage_off = 0, next_off = (NST - 1) * STAGE;
    for (int i = 0; i < tiles; ++i) {
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NST - 2) * NL) : "memory");
        load(next_off, i + NST - 1);
        next_off = stage_off;
        const int k0 = k_begin + i * KT;
        const uint32_t at = stage_off;
        stage_off = stage_off + STAGE == NST * STAGE ? 0 : stage_off + STAGE;
        if (k0 > wave_last) continue;

        // ---- scores: sc[t][i] = position k0 + 32 t + 8 (i / 4) + 4 h + i % 4 against this lane's row
        f32x16 sc[T32];
        constexpr int AHEAD = KK < 4 ? KK : 4;  // fragments of K that are on their way
        u32x4 kf[T32][AHEAD];
        auto k_read = [&](auto kc) {
            constexpr int kk = decltype(kc)::value;
            unrolled<T32>([&](auto tc) {
                constexpr int t = decltype(tc)::value;
                // (piece 2 kk + h: of 12 pieces a row only the low two bits are turned)
                kf[t][kk % AHEAD] = lds_read16<t * 32 * PITCH>(D == 96 ? ((k_rd + at) ^ ((kk & 1) * 32)) + (kk >> 1) * 64 : (k_rd + at) ^ (kk * 32));
            });
        };
        unrolled<AHEAD>(k_read);
#pragma unroll
        for (int t = 0; t < T32; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[t][j] = 0.f;
        unrolled<KK>([&](auto kc) {
            constexpr int kk = decltype(kc)::value;
            constexpr int younger = (AHEAD - 1 < KK - 1 - kk ? AHEAD - 1 : KK - 1 - kk) * T32;
            unrolled<T32>([&](auto tc) {
                constexpr int t = decltype(tc)::value;
                reads_landed<younger + T32 - 1 - t>(kf[t][kk % AHEAD]);
                sc[t] = mfma32<DT>(kf[t][kk % AHEAD], qf[kk], sc[t]);
            });
            if constexpr (kk + AHEAD < KK) k_read(std::integral_constant<int, kk + AHEAD>{});
        });

        // ---- online softmax, as in paged_few_kernel
        constexpr float LAZY = 6.0f;
        const bool partly = k0 + KT - 1 > wave_first;
        const float neg_ref = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
        for (int t = 0; t < T32; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[t][j] = fmaf(sc[t][j], p.scale_log2, neg_ref);
        if (partly) {
            int vis = last - k0 - 4 * h;
            asm volatile("" : "+v"(vis));  // a branch: as selects the masks cost every tile 64 instructions
#pragma unroll
            for (int t = 0; t < T32; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) sc[t][j] = 32 * t + 8 * (j >> 2) + (j & 3) <= vis ? sc[t][j] : -INFINITY;
        }
        float mx = fmaxf(sc[0][0], sc[0][1]);
#pragma unroll
        for (int t = 0; t < T32; ++t)
#pragma unroll
            for (int j = (t == 0 ? 2 : 0); j < 16; j += 2) mx = fmaxf(fmaxf(mx, sc[t][j]), sc[t][j + 1]);
        if (__any(mx > LAZY || m_run == -INFINITY)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_abs = mx - neg_ref;
            const bool up = m_abs > m_run + LAZY;  // false for -inf on either side
            const float m_new = up ? m_abs : m_run;
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
            const float move = -neg_ref - m_use;
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[dt][j] *= alpha;
#pragma unroll
            for (int t = 0; t < T32; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) sc[t][j] += move;
        }
        u32x4 pf[2 * T32];
#pragma unroll
        for (int t = 0; t < T32; ++t) {
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[t][j] = __builtin_amdgcn_exp2f(sc[t][j]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {  // (rounded to the dtype, as there)
                pf[2 * t + u] = u32x4{pack2_half<DT>(sc[t][8 * u], sc[t][8 * u + 1]), pack2_half<DT>(sc[t][8 * u + 2], sc[t][8 * u + 3]), pack2_half<DT>(sc[t][8 * u + 4], sc[t][8 * u + 5]),
                                      pack2_half<DT>(sc[t][8 * u + 6], sc[t][8 * u + 7])};
            }
#pragma unroll
            for (int j = 0; j < 16; j += 4) l_run += (sc[t][j] + sc[t][j + 1]) + (sc[t][j + 2] + sc[t][j + 3]);
        }

        // ---- O^T += V^T P^T, 16 positions at a time
        auto v_reads = [&](auto uc, u32x2 (&lo)[DT32], u32x2 (&hi)[DT32]) {
            constexpr int u = decltype(uc)::value;
            unrolled<DT32>([&](auto dc) {
                constexpr int dt = decltype(dc)::value;
                const uint32_t a0 = D == 96 ? v_rd0 + at + dt * 64 : (v_rd0 + at) ^ (dt * 64), a1 = D == 96 ? v_rd1 + at + dt * 64 : (v_rd1 + at) ^ (dt * 64);
                lo[dt] = lds_transpose_read<u * GROUP * PITCH>(a0);
                hi[dt] = lds_transpose_read<u * GROUP * PITCH>(a1);
            });
        };
        unrolled<2 * T32>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            u32x2 lo[DT32], hi[DT32];
            v_reads(uc, lo, hi);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            unrolled<DT32>([&](auto dc) {
                half_landed(lo[decltype(dc)::value]);
                half_landed(hi[decltype(dc)::value]);
            });
            if (!partly) {
                unrolled<DT32>([&](auto dc) {
                    constexpr int dt = decltype(dc)::value;
                    acc[dt] = mfma32<DT>(u32x4{lo[dt].x, lo[dt].y, hi[dt].x, hi[dt].y}, pf[u], acc[dt]);
                });
                return;
            }
            // the values behind the sequence's end are whatever the page held
            const int have = s.length - (k0 + 16 * u + 4 * h), more = have - 8;
            const u32x2 m_lo = {have >= 2 ? 0xffffffffu : have == 1 ? 0xffffu : 0u, have >= 4 ? 0xffffffffu : have == 3 ? 0xffffu : 0u};
            const u32x2 m_hi = {more >= 2 ? 0xffffffffu : more == 1 ? 0xffffu : 0u, more >= 4 ? 0xffffffffu : more == 3 ? 0xffffu : 0u};
            unrolled<DT32>([&](auto dc) {
                constexpr int dt = decltype(dc)::value;
                u32x4 w = u32x4{lo[dt].x, lo[dt].y, hi[dt].x, hi[dt].y} & u32x4{m_lo.x, m_lo.y, m_hi.x, m_hi.y};
                if (__any(((Beyond<DT>::carries(w.x) | Beyond<DT>::carries(w.y) | Beyond<DT>::carries(w.z) | Beyond<DT>::carries(w.w)) & 0x80008000u) != 0)) {
                    const int most = last - k0 - 16 * u - 4 * h;
                    const u32x4 seen = {Beyond<DT>::seen(most), Beyond<DT>::seen(most - 2), Beyond<DT>::seen(most - 8), Beyond<DT>::seen(most - 10)};
#pragma unroll
                    for (uint32_t sign : {0u, 0x8000u}) {
                        const u32x4 huge = {Beyond<DT>::huge(w.x, sign), Beyond<DT>::huge(w.y, sign), Beyond<DT>::huge(w.z, sign), Beyond<DT>::huge(w.w, sign)};
                        acc[dt] = mfma32<TPAMD_BF16>(huge, seen, acc[dt]);
                    }
                    w = u32x4{Beyond<DT>::finite(w.x), Beyond<DT>::finite(w.y), Beyond<DT>::finite(w.z), Beyond<DT>::finite(w.w)};
                }
                acc[dt] = mfma32<DT>(w, pf[u], acc[dt]);
            });
        });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads into LDS end before the block does
    l_run += __shfl_xor(l_run, 32);

    // ---- acc[dt][i] = O[this lane's row][32 dt + 8 (i / 4) + 4 h + i % 4]
    // (the rows of a tile that was cut go to its range's place among the partials: those of the ranges of sequences before it, then its own)
    int64_t slot = 0;
    if (cut > 1) {
        int mine = 0;
        for (int b0 = 0; b0 <= b; b0 += 64) {
            const Lanes l = lanes_from(p, b0);
            const Tiles t = tiles_of<MANY, KT>(p, l.mine);
            const int ranges = ranges_of(t, range);
            mine += b0 + lane < b && ranges > 1 ? t.rows * ranges : 0;
        }
        slot = static_cast<int64_t>(__builtin_amdgcn_readlane(sums_to_lane(mine), 63) + piece) * p.Hkv + hkv;
    }
    if (row >= rows) return;
    const int64_t token = s.first + place;
    const int head = hkv * p.G + row - place * p.G;
    if (cut == 1) {
        const float inv = factor_of(l_run, last);
        char *orow = p.o + (token * p.o_row + head * p.o_head) * 2;
#pragma unroll
        for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<uint2 *>(orow + (32 * dt + 2 * j + 4 * h) * 2) =
                    make_uint2(pack2_half<DT>(acc[dt][j] * inv, acc[dt][j + 1] * inv), pack2_half<DT>(acc[dt][j + 2] * inv, acc[dt][j + 3] * inv));
        return;
    }
    float *pr = p.many_part + (slot * MANY + row - row0) * PW;
#pragma unroll
    for (int dt = 0; dt < DT32; ++dt)
#pragma unroll
        for (int j = 0; j < 16; j += 4) *reinterpret_cast<f32x4 *>(pr + 32 * dt + 2 * j + 4 * h) = f32x4{acc[dt][j], acc[dt][j + 1], acc[dt][j + 2], acc[dt][j + 3]};
    if (h == 0) *reinterpret_cast<float2 *>(pr + D) = make_float2(m_run, l_run);
}

constexpr int many_waves_per_eu(int D, int WAVES) { return D == 256 ? 1 : D == 64 && WAVES == 4 ? 3 : 2; }
constexpr int MANY_STAGES = 4, FEW_STAGES = 2;  // more stages of few rows are no faster: a block starts later with more LDS
template <int DT, int D, int WAVES, int KT>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(many_waves_per_eu(D, WAVES), many_waves_per_eu(D, WAVES)))) void paged_many_kernel(PagedParams p) {
    many_rows<DT, D, WAVES, KT, MANY_STAGES>(p, blockIdx.x);
}
// Both kinds of sequences in one launch: blocks that read run beside blocks that multiply, and in the places of those that have ended. The first `many` blocks are row tiles, which are the longer
// ones. 18 sequences with a row each and 6 with 85 to 293, up to 5800 positions, 32 heads on 8 of 128: 75 us with the merge, as two launches and two merges one after another 103; with the few rows' blocks
// first 93, with the kinds alternating 109.
template <int DT, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(many_waves_per_eu(D, 4), many_waves_per_eu(D, 4)))) void paged_both_kernel(PagedParams p, int many) {
    const int block = blockIdx.x;
    if (block < many) many_rows<DT, D, 4, 32, MANY_STAGES>(p, block);
    else few_rows<DT, D, 4, FEW_STAGES>(p, block - many, gridDim.x - many);
}

// Joins the ranges of paged_many_kernel's row tiles that were cut: ys blocks a row tile.
template <int DT, int D, int WAVES, int KT>
__device__ __forceinline__ void many_merge(const PagedParams &p, const int block, const int y, const int ys) {
    constexpr int MANY = WAVES * 32, PW = D + 4, per_row = D / 4;
    const int hkv = block % p.Hkv, nth = block / p.Hkv;
    Lanes seqs = lanes_from(p, 0);
    const int range = range_tiles<MANY, KT>(p, seqs);
    auto cut_tiles = [&](const SeqRows &s) {
        const Tiles t = tiles_of<MANY, KT>(p, s);
        return ranges_of(t, range) > 1 ? t.rows : 0;
    };
    auto slots_in = [&](const SeqRows &s) {
        const Tiles t = tiles_of<MANY, KT>(p, s);
        const int ranges = ranges_of(t, range);
        return ranges > 1 ? t.rows * ranges : 0;
    };
    if (nth >= sum_over(p, seqs, cut_tiles)) return;
    int before;
    const int b = find_in(p, seqs, nth, before, cut_tiles);
    const SeqRows s = pick(p, seqs, b);
    const int cut = ranges_of(tiles_of<MANY, KT>(p, s), range), tile = nth - before;
    int slots = 0;  // of the sequences before it
    for (int b0 = 0; b0 <= b; b0 += 64) {
        const Lanes l = lanes_from(p, b0);
        slots += b0 + static_cast<int>(threadIdx.x & 63) < b ? slots_in(l.mine) : 0;
    }
    slots = __builtin_amdgcn_readlane(sums_to_lane(slots), 63);
    const int rows = min(s.count * p.G - tile * MANY, MANY);
    const int64_t pitch = static_cast<int64_t>(p.Hkv) * MANY * PW;
    const float *base = p.many_part + ((static_cast<int64_t>(slots) + static_cast<int64_t>(tile) * cut) * p.Hkv + hkv) * MANY * PW;
    for (int e = y * 256 + threadIdx.x; e < rows * per_row; e += ys * 256) {
        const int r = e / per_row, d4 = (e % per_row) * 4;
        const float *pr = base + r * PW;
        float M = -INFINITY, l = 0.f;
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < cut; i0 += 4) {
            float2 ml[4];
            f32x4 ov[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float *from = pr + min(i0 + j, cut - 1) * pitch;
                ml[j] = *reinterpret_cast<const float2 *>(from + D);
                ov[j] = *reinterpret_cast<const f32x4 *>(from + d4);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i0 + j >= cut) continue;
                const float m = fmaxf(M, ml[j].x), m_use = m == -INFINITY ? 0.f : m, old = exp2f(M - m_use), now = exp2f(ml[j].x - m_use);
                M = m;
                l = l * old + ml[j].y * now;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = o[k] * old + ov[j][k] * now;
            }
        }
        const int row = tile * MANY + r, place = row / p.G;
        const float inv = factor_of(l, s.length - s.count + place);
        *reinterpret_cast<uint2 *>(p.o + (static_cast<int64_t>(s.first + place) * p.o_row + static_cast<int64_t>(hkv * p.G + row - place * p.G) * p.o_head + d4) * 2) =
            make_uint2(pack2_half<DT>(o[0] * inv, o[1] * inv), pack2_half<DT>(o[2] * inv, o[3] * inv));
    }
}

// The first WAVES * many blocks join row tiles, WAVES of them each, the others items of few rows, as many of them each as there are. Blocks of a tile lie `many` apart: with key/value heads a multiple
// of the 8 XCDs a tile is joined on the one that left its ranges (16 heads, 512 rows: 20.1 us with paged_many_kernel, 25.7 with a tile's blocks side by side).
template <int DT, int D, int WAVES>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedParams p, int many, int few_blocks, int few_y) {
    const int block = blockIdx.x, few = block - WAVES * many, items = p.pages.seqs * p.Hkv;
    if (few < 0) many_merge<DT, D, WAVES, WAVES * 8>(p, block % many, block / many, WAVES);
    else few_merge<DT, D>(p, few_blocks, few % items, few / items, few_y);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------------------------------------
// How a call is laid out, from what the host knows: the number of rows and sequences, and bounds of their new rows and lengths.
struct Plan {
    bool few, many;
    int few_blocks, least;  // paged_few_kernel: blocks, and the least share of one (0: a block an item)
    int few_waves;          // wavefronts of its blocks
    int merge_y;            // blocks of an item in its merge
    int waves;              // paged_many_kernel: wavefronts of a block
    int64_t tiles;          // row tiles of a key/value head, at most
    int spread;
    uint64_t bytes, many_bytes;  // of partials: all, and paged_many_kernel's, which come first
};

Plan plan_of(int64_t rows, int64_t seqs, int64_t Hq, int64_t Hkv, int64_t D, bool packed, bool counted, int64_t max_new, int64_t max_length, int64_t room, int cus) {
    const int64_t G = Hq / Hkv, each = packed ? 0 : rows / seqs;
    const int64_t most = packed ? (max_new < rows ? max_new : rows) : (max_new < each ? max_new : each);  // new rows of a sequence
    Plan p{};
    p.few = G <= FEW && (packed || counted || most * G <= FEW);
    p.many = most * G > FEW;
    if (p.few) {
        const int64_t items = seqs * Hkv;
        p.few_waves = 4;
        const int per_cu = D <= 64 ? 4 : D <= 96 ? 3 : D <= 128 ? 2 : 1;  // blocks that a CU holds (registers; 64 KiB of LDS a block of heads of 128)
        // Where every whole item has a CU to itself its block has 8 wavefronts: 500 positions of 16 heads of 128 take 8.9 us, with 4 wavefronts 10.0; 700 9.7 and 12.0; of 4 heads of 64 6.8 and 7.8.
        // Not for up to 4 units (128 positions 6.3 and 5.8), nor for items on most CUs (192: 500 12.7 and 12.4), nor beside row tiles, whose blocks have 4.
        const bool wide = items <= cus / 2 && D <= 128 && !p.many;
        // A whole item takes a time that grows with its units of 64 positions (in hundredths of a us each, 60 with 4 wavefronts and 48 with 8, up to 64 elements 43 and 28), cut ones the second launch:
        // whole up to 7 us. Whole with 4, with 8 and cut, us: one sequence, 16 heads of 128: 500 10.2, 8.9, 11.7; 1000 15.6, 12.2, 12.0; 2000 25.9, 21.5, 13.3. 4 heads of 64: 1000 11.8, 8.5, 9.7;
        // 2000 19.6, 12.5, 10.7. 16 of 96: 500 9.1, 8.0, 10.8; 1000 13.7, 10.2, 11.0; 2000 22.9, 17.1, 12.0. 16 of 256 (with 4, and cut): 500 15.2, 15.9; 700 18.9, 16.2; 1000 24.5, 16.4.
        // Of many sequences the longest says it, since how they differ is not known here. 24 of 32 heads on 8 of 96, 128 and 256 elements between 100 and 3000 positions, whole and cut: 30.1 and 21.9,
        // 33.7 and 25.0, 57.7 and 37.3; all of 1000: 16.9 and 21.0, 19.9 and 25.2, 35.6 and 39.9; 200 of 100 and 4 of 8000 108 and 49.
        const bool cut = max_length * (wide ? (D <= 64 ? 28 : 48) : (D <= 64 ? 43 : 60)) > 64 * 700;
        if (cut && items * (room / UNIT + 1 + START) < (1ll << 31)) {  // costs are counted in 32 bits
            p.few_blocks = per_cu * cus;
            p.least = START + 2;
            p.bytes = static_cast<uint64_t>(2) * p.few_blocks * FEW * (D + 4) * sizeof(float);
            const int few_rows = static_cast<int>(most * G < FEW ? most * G : FEW), at_once = static_cast<int>(1024 / D);
            p.merge_y = items * few_rows <= 2ll * cus ? few_rows : (few_rows + at_once - 1) / at_once;
        } else {
            p.few_blocks = static_cast<int>(items);
            p.few_waves = wide && max_length > 4 * UNIT ? 8 : 4;
        }
    }
    if (p.many) {
        // Blocks of 8 wavefronts load keys and values half as often, blocks of 4, two to a CU, leave less of the device idle at the end of a batch and have shorter tiles. With 4 and 8, heads of
        // 128: 4096 rows 164 and 154 us, 500 on 30000 203 and 151, 8 x 1024 (32 heads on 8) 120 and 131, 3 x 701 32 and 45; of 64: 4096 rows 103 and 114;
        // of 96: 250 rows 12.9 and 16.3, 512 17.8 and 22.1, 3 x 701 23.6 and 37.1, 4096 136 and 124, 500 on 30000 189 and 120.
        // tiles of 256 rows and 64 positions for a CU; of sequences that may differ, half of what the bounds allow
        const double per_cu = static_cast<double>(rows) * Hq * (max_length - most / 2) / (256.0 * 64.0) / cus * (packed || counted ? 0.5 : 1.0);
        const bool enough = rows * G / 256 * Hkv >= cus;  // row tiles of 256, none of which need be cut
        p.waves = D == 256 || per_cu < 40 || (D == 64 && enough) ? 4 : 8;
        const int64_t MANY = p.waves * 32;
        p.tiles = packed ? rows * G / MANY + seqs : seqs * ((each * G + MANY - 1) / MANY);
        // Nothing is cut, and there is no merge, of a single sequence with two row tiles and more for a CU (a share is at least as long as its last tile: the average one has half of that or more), of
        // sequences with a row tile for each CU that differ in length by twice at most (uncut and cut, us: 3 x 701 rows of 16 heads of 128 26.6 and 29.8, 8 x 1024 of 32 on 8 111 and 115, of 64 71
        // and 77), and of few tiles of positions (250 rows 14.7 and 18.5, 8 x 256 21.3 and 24.7; 512 rows 21.0 and 20.7).
        const bool alike = !packed && !counted && max_length <= 2 * each && p.tiles * Hkv >= cus;
        if (!alike && !(seqs == 1 && p.tiles * Hkv >= 2ll * cus) && max_length > 2 * LEAST_TILES * p.waves * 8) {
            p.spread = cus;
            p.many_bytes = static_cast<uint64_t>(2) * p.spread * MANY * (D + 4) * sizeof(float);
            p.bytes += p.many_bytes;
        }
    }
    return p;
}

template <auto KERNEL>
struct Kernel {
    static constexpr auto at = KERNEL;
};

template <int DT, int D, int WAVES>
int launch(PagedParams p, const Plan &plan, hipStream_t s) {
    constexpr int KT = WAVES * 8, MANY_LDS = MANY_STAGES * 2 * KT * D * 2, FEW_LDS = 4 * FEW_STAGES * 2 * GROUP * D * 2;
    static_assert(WAVES != 4 || MANY_LDS == FEW_LDS, "one launch of both");
    int dev = 0;
    TPAMD_HIP(hipGetDevice(&dev));
    p.spread = plan.spread;
    p.least = plan.least;
    const int64_t tiles = plan.many ? plan.tiles * p.Hkv : 0;
    // (a cut tile has two ranges and more, fewer than 2 spread in all)
    const int64_t cut = tiles < plan.spread ? tiles : plan.spread;
    const int64_t joins = (cut + p.Hkv - 1) / p.Hkv * p.Hkv, few_joins = plan.least > 0 ? static_cast<int64_t>(p.pages.seqs) * p.Hkv * plan.merge_y : 0;
    TPAMD_REQUIRE(tiles + plan.spread < (1ll << 22) && tiles + plan.spread + p.Hkv + (plan.few ? plan.few_blocks : 0) < (1ll << 24) && WAVES * joins + few_joins < (1ll << 24),
                  "tpamd_attention_paged: too many rows or sequences for one launch");
    const unsigned many = static_cast<unsigned>(plan.many ? (tiles + plan.spread + p.Hkv - 1) / p.Hkv * p.Hkv : 0), few = static_cast<unsigned>(plan.few ? plan.few_blocks : 0);
    auto run = [&](auto kernel, unsigned blocks, int threads, int lds, auto... more) -> int {
        static thread_local int configured = -1;  // (one for each kernel and its call)
        if (configured != dev) {
            TPAMD_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(decltype(kernel)::at), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
            configured = dev;
        }
        hipLaunchKernelGGL(decltype(kernel)::at, dim3(blocks), dim3(threads), lds, s, p, more...);
        TPAMD_HIP(hipGetLastError());
        return TPAMD_OK;
    };
    if (WAVES == 4 && many > 0 && few > 0) {
        if (int rc = run(Kernel<paged_both_kernel<DT, D>>{}, many + few, 256, FEW_LDS, static_cast<int>(many)); rc != TPAMD_OK) return rc;
    } else {
        if (many > 0) {
            if (int rc = run(Kernel<paged_many_kernel<DT, D, WAVES, KT>>{}, many, WAVES * 64, MANY_LDS); rc != TPAMD_OK) return rc;
        }
        if (few > 0) {
            int rc;
            if constexpr (D <= 128) rc = plan.few_waves == 8 ? run(Kernel<paged_few_kernel<DT, D, 8, FEW_STAGES>>{}, few, 512, 2 * FEW_LDS) : run(Kernel<paged_few_kernel<DT, D, 4, FEW_STAGES>>{}, few, 256, FEW_LDS);
            else rc = run(Kernel<paged_few_kernel<DT, D, 4, FEW_STAGES>>{}, few, 256, FEW_LDS);
            if (rc != TPAMD_OK) return rc;
        }
    }
    if (joins + few_joins > 0) {
        hipLaunchKernelGGL((paged_merge_kernel<DT, D, WAVES>), dim3(static_cast<unsigned>(WAVES * joins + few_joins)), dim3(256), 0, s, p, static_cast<int>(joins), plan.few_blocks, plan.merge_y);
        TPAMD_HIP(hipGetLastError());
    }
    return TPAMD_OK;
}

template <int DT, int D>
int launch(const PagedParams &p, const Plan &plan, hipStream_t s) {
    if constexpr (D != 256) {  // (two wavefronts of a SIMD do not have the registers)
        if (plan.waves == 8) return launch<DT, D, 8>(p, plan, s);
    }
    return launch<DT, D, 4>(p, plan, s);
}

}  // namespace

int take_pages(const char *who, const tpamd_pages *g, int64_t rows, PagesView *out) {
    TPAMD_REQUIRE(g->seqs >= 0 && g->seqs < (1ll << 24) && g->columns >= 0 && g->pages >= 0 && g->pages < (1ll << 31), "%s: bad dimension", who);
    TPAMD_REQUIRE(g->page >= GROUP && g->page < (1ll << 30) && (g->page & (g->page - 1)) == 0, "%s: a page has %lld positions: a power of two from %d on is needed", who, (long long)g->page, GROUP);
    // (positions are counted in 32 bits, and some behind a sequence's last: whole tiles, ranges of up to 512 x 64, the pages of the next 64 tiles of 128)
    TPAMD_REQUIRE(g->columns <= ((1ll << 31) - (1 << 16)) / g->page, "%s: %lld pages of %lld positions a sequence are too many", who, (long long)g->columns, (long long)g->page);
    TPAMD_REQUIRE(g->starts == nullptr || g->counts == nullptr, "%s: starts (packed rows) or counts (padded rows), not both", who);
    TPAMD_REQUIRE(g->seqs == 0 || g->starts != nullptr || rows % g->seqs == 0, "%s: %lld rows are not the same number for each of %lld sequences", who, (long long)rows, (long long)g->seqs);
    for (int64_t s : {g->k_page, g->k_head, g->k_pos, g->v_page, g->v_head, g->v_pos, g->table_row}) TPAMD_REQUIRE(s >= 0, "%s: a negative stride", who);
    PagesView v{};
    v.seqs = static_cast<int>(g->seqs);
    if (g->seqs > 0) {
        TPAMD_REQUIRE(g->lengths != nullptr && (g->columns == 0 || g->table != nullptr) && (g->pages == 0 || (g->k_pages && g->v_pages)), "%s: null pointer", who);
        v.each = g->starts != nullptr ? 0 : static_cast<int>(rows / g->seqs);
    }
    v.k = static_cast<char *>(g->k_pages); v.v = static_cast<char *>(g->v_pages);
    v.k_page = g->k_page; v.k_head = g->k_head; v.k_pos = g->k_pos; v.v_page = g->v_page; v.v_head = g->v_head; v.v_pos = g->v_pos;
    v.table = g->table; v.lengths = g->lengths; v.starts = g->starts; v.counts = g->counts; v.table_row = g->table_row;
    v.pages = static_cast<int>(g->pages);
    v.shift = __builtin_ctzll(static_cast<unsigned long long>(g->page));
    v.rows = static_cast<int>(rows);
    v.room = static_cast<int>(g->columns * g->page);
    *out = v;
    return TPAMD_OK;
}

namespace {
int check_sizes(const char *who, const tpamd_pages *g, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D) {
    TPAMD_REQUIRE(g != nullptr, "%s: null pointer", who);
    TPAMD_REQUIRE(rows >= 0 && rows < (1ll << 24) && Hq > 0 && Hkv > 0 && Hq < (1ll << 16), "%s: bad dimension", who);
    TPAMD_REQUIRE(Hq % Hkv == 0, "%s: %lld query heads are not a multiple of %lld key/value heads", who, (long long)Hq, (long long)Hkv);
    TPAMD_REQUIRE(rows * Hq < (1ll << 31) && g->seqs * Hkv < (1ll << 24), "%s: too many rows or sequences for one call", who);
    if (D != 64 && D != 96 && D != 128 && D != 256) {
        set_error("%s: head_dim must be 64, 96, 128 or 256", who);
        return TPAMD_ERR_UNSUPPORTED;
    }
    return TPAMD_OK;
}
}  // namespace

}  // namespace tpamd

using namespace tpamd;

extern "C" int tpamd_attention_paged_workspace(const tpamd_pages *pages, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, int64_t max_length, uint64_t *bytes_out) {
    const char *who = "tpamd_attention_paged_workspace";
    if (int rc = check_sizes(who, pages, rows, Hq, Hkv, D); rc != TPAMD_OK) return rc;
    TPAMD_REQUIRE(bytes_out != nullptr && max_new >= 0 && max_length >= 0, "%s: bad argument", who);
    *bytes_out = 0;
    PagesView view;
    if (int rc = take_pages(who, pages, rows, &view); rc != TPAMD_OK) return rc;
    if (rows == 0 || view.seqs == 0) return TPAMD_OK;
    int dev = 0, cus = 256;
    TPAMD_HIP(hipGetDevice(&dev));
    if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
    *bytes_out = plan_of(rows, view.seqs, Hq, Hkv, D, view.starts != nullptr, view.counts != nullptr, max_new, max_length < view.room ? max_length : view.room, view.room, cus).bytes;
    return TPAMD_OK;
}

extern "C" int tpamd_attention_paged(const void *q_dev, int64_t q_row, int64_t q_head, const tpamd_pages *pages, void *out_dev, int64_t o_row, int64_t o_head, int64_t rows, int64_t Hq,
                                     int64_t Hkv, int64_t D, int64_t max_new, int64_t max_length, float scale, int dtype, void *workspace_dev, uint64_t workspace_bytes, void *stream) {
    const char *who = "tpamd_attention_paged";
    TPAMD_REQUIRE(dtype == TPAMD_BF16 || dtype == TPAMD_F16, "%s: dtype must be BF16 or F16", who);
    if (int rc = check_sizes(who, pages, rows, Hq, Hkv, D); rc != TPAMD_OK) return rc;
    TPAMD_REQUIRE(max_new >= 0 && max_length >= 0 && q_row >= 0 && q_head >= 0 && o_row >= 0 && o_head >= 0, "%s: bad argument", who);
    PagedParams p{};
    if (int rc = take_pages(who, pages, rows, &p.pages); rc != TPAMD_OK) return rc;
    if (rows == 0 || p.pages.seqs == 0) return TPAMD_OK;
    TPAMD_REQUIRE(q_dev != nullptr && out_dev != nullptr, "%s: null pointer", who);
    bool ok = aligned(q_dev, 16) && q_row % 8 == 0 && q_head % 8 == 0 && aligned(out_dev, 8) && o_row % 4 == 0 && o_head % 4 == 0 && aligned(p.pages.k, 16) && aligned(p.pages.v, 16);
    for (int64_t s : {p.pages.k_page, p.pages.k_head, p.pages.k_pos, p.pages.v_page, p.pages.v_head, p.pages.v_pos}) ok = ok && s % 8 == 0;
    ok = ok && p.pages.k_pos < (1ll << 26) && p.pages.v_pos < (1ll << 26);  // 16 positions by 32-bit byte offsets
    if (!ok) {
        set_error("%s: rows of q, keys and values must lie on 16-byte boundaries (out: 8), positions of a page within 2^26 elements", who);
        return TPAMD_ERR_UNSUPPORTED;
    }
    int dev = 0, cus = 256;
    TPAMD_HIP(hipGetDevice(&dev));
    if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
    const Plan plan = plan_of(rows, p.pages.seqs, Hq, Hkv, D, p.pages.starts != nullptr, p.pages.counts != nullptr, max_new, max_length < p.pages.room ? max_length : p.pages.room, p.pages.room, cus);
    TPAMD_REQUIRE(workspace_bytes >= plan.bytes && (plan.bytes == 0 || (workspace_dev != nullptr && aligned(workspace_dev, 16))), "%s: %llu bytes of workspace on a 16-byte boundary are needed", who,
                  (unsigned long long)plan.bytes);
    p.q = static_cast<const char *>(q_dev);
    p.o = static_cast<char *>(out_dev);
    p.q_row = q_row; p.q_head = q_head; p.o_row = o_row; p.o_head = o_head;
    p.many_part = static_cast<float *>(workspace_dev);
    p.few_part = p.many_part + plan.many_bytes / sizeof(float);
    p.scale_log2 = scale * 1.4426950408889634f;
    p.Hkv = static_cast<int>(Hkv); p.G = static_cast<int>(Hq / Hkv);
    p.few = plan.few; p.many = plan.many;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool bf = dtype == TPAMD_BF16;
    switch (D) {
        case 64: return bf ? launch<TPAMD_BF16, 64>(p, plan, s) : launch<TPAMD_F16, 64>(p, plan, s);
        case 96: return bf ? launch<TPAMD_BF16, 96>(p, plan, s) : launch<TPAMD_F16, 96>(p, plan, s);
        case 128: return bf ? launch<TPAMD_BF16, 128>(p, plan, s) : launch<TPAMD_F16, 128>(p, plan, s);
        default: return bf ? launch<TPAMD_BF16, 256>(p, plan, s) : launch<TPAMD_F16, 256>(p, plan, s);
    }
}
