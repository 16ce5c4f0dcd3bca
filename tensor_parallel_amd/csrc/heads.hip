// Heads of queries and keys between their projection and attention: an RMS norm of each head, the rotation to its position, and (append) the hand-over of k and v to
// a paged cache, in one pass.
//
//   x' = x * rsqrt(mean(x^2) + eps) * w                                   (where there is a weight)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq, cos and sin times `scaling`,
// for the pairs of the first `part` elements of a head: neighbours (2 i, 2 i + 1), or (i, i + part / 2); the others stay. Everything in fp32 and rounded once, at the
// store. An angle is a product in 64 bits, reduced to one turn before it is 32 bits: at position 10^6 an angle in 32 bits is off by up to 0.03 (half of 2^-4).
//
// Bound: HBM (every byte once), or the launch: 4096 rows of 32 + 32 heads of 128, normed, 27 us (134 MB, 5.0 TB/s); 2103 rows of 64 + 4 heads of 64 10.8 (37 MB, 3.4 TB/s); one row 2.8. A block takes
// all heads of one row (or, of few rows, as many as its lanes hold), so that the row's angles are computed once, into LDS. A lane holds 2 VEC elements of a head: the VEC pairs, in either layout,
// whose cos and sin follow one another. With pieces of 4 elements the 4096 rows take 37 us, with single ones 101 (the 2103 rows 11.5 and 20). To ask for the next head's elements before this row's
// place and angles are known is 8 - 21 % slower: a head's address is worked out twice then, and other rows' blocks hide the way to memory already.
#include "paged.h"

#include <math.h>

namespace tpamd {
namespace {

struct HeadsParams {
    const char *q, *k, *v;
    char *q_out, *k_out;
    int64_t q_row, q_group, q_head, k_row, k_head, v_row, v_head, qo_row, qo_head, ko_row, ko_head;  // elements
    const char *q_norm, *k_norm;
    float eps, scaling;
    const float *inv_freq;
    const char *cos, *sin;  // tables instead of frequencies: a value a pair
    int64_t table_row;
    int table_dtype;
    const int64_t *positions;
    int Hq, Hkv, per, D, part, interleaved;
    int heads;   // that a row has: queries, keys and, with a cache, values
    int paged;
    PagesView pages;
};

template <int DT>
__device__ __forceinline__ void unpack8(uint4 u, float *x) {
    x[0] = lo_half_to_f32<DT>(u.x); x[1] = hi_half_to_f32<DT>(u.x); x[2] = lo_half_to_f32<DT>(u.y); x[3] = hi_half_to_f32<DT>(u.y);
    x[4] = lo_half_to_f32<DT>(u.z); x[5] = hi_half_to_f32<DT>(u.z); x[6] = lo_half_to_f32<DT>(u.w); x[7] = hi_half_to_f32<DT>(u.w);
}
// VEC elements: 16 bytes, 8, or one element
template <int DT, int VEC>
struct Piece {
    static __device__ __forceinline__ void load(const char *p, float *x) {
        if constexpr (VEC == 8) {
            unpack8<DT>(*reinterpret_cast<const uint4 *>(p), x);
        } else if constexpr (VEC == 4) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p);
            x[0] = lo_half_to_f32<DT>(u.x); x[1] = hi_half_to_f32<DT>(u.x); x[2] = lo_half_to_f32<DT>(u.y); x[3] = hi_half_to_f32<DT>(u.y);
        } else {
            x[0] = half_to_f32<DT>(*reinterpret_cast<const uint16_t *>(p));
        }
    }
    static __device__ __forceinline__ void store(char *p, const float *x) {
        if constexpr (VEC == 8)
            *reinterpret_cast<uint4 *>(p) = make_uint4(pack2_half<DT>(x[0], x[1]), pack2_half<DT>(x[2], x[3]), pack2_half<DT>(x[4], x[5]), pack2_half<DT>(x[6], x[7]));
        else if constexpr (VEC == 4)
            *reinterpret_cast<uint2 *>(p) = make_uint2(pack2_half<DT>(x[0], x[1]), pack2_half<DT>(x[2], x[3]));
        else
            *reinterpret_cast<uint16_t *>(p) = f32_to_half<DT>(x[0]);
    }
    static __device__ __forceinline__ void copy(char *to, const char *from) {
        if constexpr (VEC == 8) *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
        else if constexpr (VEC == 4) *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(from);
        else *reinterpret_cast<uint16_t *>(to) = *reinterpret_cast<const uint16_t *>(from);
    }
};

// cos and sin of position * inv_freq: the product is exact in 64 bits but for its last bits (31 and 24 significant ones), whole turns are taken off it there
__device__ __forceinline__ void turn(double position, float inv_freq, float &c, float &s) {
    const double angle = position * static_cast<double>(inv_freq);
    const double turns = rint(angle * 0.15915494309189533577);                    // 1 / (2 pi)
    const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586477, angle));  // 2 pi in two parts
    sincosf(static_cast<float>(rest), &s, &c);
}

__device__ __forceinline__ float table_value(const char *t, int dtype, int64_t i) {
    if (dtype == TPAMD_F32) return reinterpret_cast<const float *>(t)[i];
    const uint16_t h = reinterpret_cast<const uint16_t *>(t)[i];
    return dtype == TPAMD_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}

constexpr int MAX_HALF = 256;  // pairs of a head: heads of up to 512 elements

// lanes: of a head, a power of two (those beyond D / (2 VEC) idle); VEC = 1 walks a head in steps of its lanes, and reads it twice where it is normed.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void heads_kernel(HeadsParams p, int lanes) {
    __shared__ __align__(16) float cs[MAX_HALF], sn[MAX_HALF];
    const int row = blockIdx.x, tid = threadIdx.x;
    // ---- whose row it is
    int64_t position = row;
    char *k_to = nullptr, *v_to = nullptr;  // position of head 0 in the pools; NULL: none
    if (p.paged) {
        int place;
        const int b = seq_of_row(p.pages, row, place);
        if (b < 0) return;  // (the whole block)
        const SeqRows s = rows_of(p.pages, b);
        const int at = s.length - s.count + place;
        position = at;
        if (at >= 0 && at < s.length) {
            const int page = page_of(p.pages, b, at), slot = at & ((1 << p.pages.shift) - 1);
            if (page >= 0) {
                k_to = p.pages.k + (page * p.pages.k_page + slot * p.pages.k_pos) * 2;
                v_to = p.pages.v + (page * p.pages.v_page + slot * p.pages.v_pos) * 2;
            }
        }
    }
    if (p.positions != nullptr) position = p.positions[row];
    const int half = p.part >> 1;
    for (int i = tid; i < half; i += 256) {
        float c, s;
        if (p.inv_freq != nullptr) {
            turn(static_cast<double>(position), p.inv_freq[i], c, s);
        } else {
            c = table_value(p.cos, p.table_dtype, row * p.table_row + i);
            s = table_value(p.sin, p.table_dtype, row * p.table_row + i);
        }
        cs[i] = c * p.scaling;
        sn[i] = s * p.scaling;
    }
    __syncthreads();

    const int lane = tid & (lanes - 1), slots = 256 / lanes;
    const int first = blockIdx.y * slots + tid / lanes, step = gridDim.y * slots;
    const int pair_lanes = half / VEC, all_lanes = p.D / (2 * VEC);
    for (int head = first; head < p.heads; head += step) {
        const bool is_q = head < p.Hq, is_v = head >= p.Hq + p.Hkv;
        const int h = is_q ? head : is_v ? head - p.Hq - p.Hkv : head - p.Hq;
        const char *from;
        char *to;
        if (is_q) {
            from = p.q + (row * p.q_row + (h / p.per) * p.q_group + (h % p.per) * p.q_head) * 2;
            to = p.q_out + (row * p.qo_row + h * p.qo_head) * 2;
        } else if (is_v) {
            from = p.v + (row * p.v_row + h * p.v_head) * 2;
            to = v_to != nullptr ? v_to + h * p.pages.v_head * 2 : nullptr;
        } else {
            from = p.k + (row * p.k_row + h * p.k_head) * 2;
            to = !p.paged ? p.k_out + (row * p.ko_row + h * p.ko_head) * 2 : k_to != nullptr ? k_to + h * p.pages.k_head * 2 : nullptr;
        }
        if (to == nullptr) continue;  // (all lanes of the head)
        const char *norm = is_q ? p.q_norm : p.k_norm;
        // the first elements of a lane's two pieces, and its pairs
        auto pieces = [&](int l, int &a, int &b) {
            if (l >= pair_lanes) {
                a = p.part + (l - pair_lanes) * 2 * VEC;
                b = a + VEC;
            } else if (p.interleaved) {
                a = 2 * VEC * l;
                b = a + VEC;
            } else {
                a = VEC * l;
                b = a + half;
            }
        };
        if (is_v) {
            for (int l = lane; l < all_lanes; l += lanes) {
                Piece<DT, VEC>::copy(to + l * 4 * VEC, from + l * 4 * VEC);
                Piece<DT, VEC>::copy(to + l * 4 * VEC + 2 * VEC, from + l * 4 * VEC + 2 * VEC);
            }
            continue;
        }
        float factor = 1.f;
        float x[2 * VEC];
        if (norm != nullptr) {
            float sum = 0.f;
            for (int l = lane; l < all_lanes; l += lanes) {
                int a, b;
                pieces(l, a, b);
                Piece<DT, VEC>::load(from + a * 2, x);
                Piece<DT, VEC>::load(from + b * 2, x + VEC);
#pragma unroll
                for (int j = 0; j < 2 * VEC; ++j) sum = fmaf(x[j], x[j], sum);
            }
            for (int d = 1; d < lanes; d *= 2) sum += __shfl_xor(sum, d);
            factor = rsqrtf(sum / static_cast<float>(p.D) + p.eps);
        }
        for (int l = lane; l < all_lanes; l += lanes) {
            int a, b;
            pieces(l, a, b);
            if (VEC == 1 || norm == nullptr) {  // else they are here: one turn of this loop
                Piece<DT, VEC>::load(from + a * 2, x);
                Piece<DT, VEC>::load(from + b * 2, x + VEC);
            }
            if (norm != nullptr) {
                float w[2 * VEC];
                Piece<DT, VEC>::load(norm + a * 2, w);
                Piece<DT, VEC>::load(norm + b * 2, w + VEC);
#pragma unroll
                for (int j = 0; j < 2 * VEC; ++j) x[j] = x[j] * factor * w[j];
            }
            if (l < pair_lanes) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float c = cs[l * VEC + j], s = sn[l * VEC + j];
                    float &u = p.interleaved ? x[2 * j] : x[j], &w = p.interleaved ? x[2 * j + 1] : x[VEC + j];
                    const float turned = u * c - w * s;
                    w = w * c + u * s;
                    u = turned;
                }
            }
            Piece<DT, VEC>::store(to + a * 2, x);
            Piece<DT, VEC>::store(to + b * 2, x + VEC);
        }
    }
}

bool fits(const void *p, int vec) { return p == nullptr || aligned(p, 2 * vec); }

// How many elements a lane's pieces have: 8, or 4, as far as sizes, strides and addresses go, or 1.
int piece_of(const tpamd_heads *h, const tpamd_pages *pages, int64_t D) {
    for (int vec : {8, 4}) {
        if (D % (2 * vec) != 0 || h->part % (2 * vec) != 0) continue;
        bool ok = fits(h->q, vec) && fits(h->k, vec) && fits(h->v, vec) && fits(h->q_out, vec) && fits(h->k_out, vec) && fits(h->q_norm, vec) && fits(h->k_norm, vec);
        for (int64_t s : {h->q_row, h->q_group, h->q_head, h->k_row, h->k_head, h->v_row, h->v_head, h->qo_row, h->qo_head, h->ko_row, h->ko_head}) ok = ok && s % vec == 0;
        if (pages != nullptr) {
            ok = ok && fits(pages->k_pages, vec) && fits(pages->v_pages, vec);
            for (int64_t s : {pages->k_page, pages->k_head, pages->k_pos, pages->v_page, pages->v_head, pages->v_pos}) ok = ok && s % vec == 0;
        }
        if (ok) return vec;
    }
    return 1;
}

int heads_entry(const char *who, const tpamd_heads *h, const tpamd_pages *pages, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, int dtype, hipStream_t stream) {
    TPAMD_REQUIRE(h != nullptr, "%s: null pointer", who);
    TPAMD_REQUIRE(dtype == TPAMD_BF16 || dtype == TPAMD_F16, "%s: dtype must be BF16 or F16", who);
    TPAMD_REQUIRE(rows >= 0 && Hq > 0 && Hkv > 0 && D > 0 && rows < (1ll << 24) && Hq + 2 * Hkv < (1ll << 16), "%s: bad dimension", who);
    TPAMD_REQUIRE(Hq % Hkv == 0, "%s: %lld query heads are not a multiple of %lld key/value heads", who, (long long)Hq, (long long)Hkv);
    TPAMD_REQUIRE(D % 2 == 0 && D <= 2 * MAX_HALF, "%s: heads of %lld elements: an even number up to %d is needed", who, (long long)D, 2 * MAX_HALF);
    TPAMD_REQUIRE(h->part >= 0 && h->part % 2 == 0 && h->part <= D, "%s: %lld of %lld elements cannot be turned in pairs", who, (long long)h->part, (long long)D);
    if (rows == 0) return TPAMD_OK;
    TPAMD_REQUIRE(h->part == 0 || (h->inv_freq != nullptr) != (h->cos != nullptr && h->sin != nullptr), "%s: frequencies or tables are needed, and not both", who);
    TPAMD_REQUIRE(h->part == 0 || h->inv_freq == nullptr || h->positions != nullptr || pages != nullptr, "%s: positions are needed", who);
    TPAMD_REQUIRE(h->cos == nullptr || h->table_dtype == TPAMD_BF16 || h->table_dtype == TPAMD_F16 || h->table_dtype == TPAMD_F32, "%s: unknown dtype of tables", who);
    TPAMD_REQUIRE(h->part == 0 || h->cos == nullptr || h->positions == nullptr, "%s: tables have a row for each of the call's rows: positions go with frequencies", who);
    HeadsParams p{};
    p.paged = pages != nullptr;
    if (pages != nullptr) {
        if (int rc = take_pages(who, pages, rows, &p.pages); rc != TPAMD_OK) return rc;
        if (p.pages.seqs == 0) return TPAMD_OK;
    }
    TPAMD_REQUIRE(h->q && h->k && h->q_out && (pages != nullptr ? h->v != nullptr : h->k_out != nullptr), "%s: null pointer", who);
    p.q = static_cast<const char *>(h->q); p.k = static_cast<const char *>(h->k); p.v = static_cast<const char *>(h->v);
    p.q_out = static_cast<char *>(h->q_out); p.k_out = static_cast<char *>(h->k_out);
    p.q_row = h->q_row; p.q_group = h->q_group; p.q_head = h->q_head;
    p.k_row = h->k_row; p.k_head = h->k_head; p.v_row = h->v_row; p.v_head = h->v_head;
    p.qo_row = h->qo_row; p.qo_head = h->qo_head; p.ko_row = h->ko_row; p.ko_head = h->ko_head;
    p.q_norm = static_cast<const char *>(h->q_norm); p.k_norm = static_cast<const char *>(h->k_norm);
    p.eps = h->eps; p.scaling = h->scaling;
    p.inv_freq = static_cast<const float *>(h->inv_freq);
    p.cos = static_cast<const char *>(h->cos); p.sin = static_cast<const char *>(h->sin);
    p.table_row = h->table_row; p.table_dtype = h->table_dtype;
    p.positions = h->positions;
    p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv); p.per = static_cast<int>(Hq / Hkv);
    p.D = static_cast<int>(D); p.part = static_cast<int>(h->part); p.interleaved = h->interleaved;
    p.heads = static_cast<int>(Hq + (pages != nullptr ? 2 : 1) * Hkv);
    const int vec = piece_of(h, pages, D);
    int lanes = 1;  // of a head, within a wavefront
    while (lanes < 64 && lanes * 2 * vec < p.D) lanes *= 2;
    const int turns = (p.heads + 256 / lanes - 1) / (256 / lanes);
    int dev = 0, cus = 256;
    TPAMD_HIP(hipGetDevice(&dev));
    if (int rc = device_cus(dev, &cus); rc != TPAMD_OK) return rc;
    // few rows: a block for every 256 lanes' heads instead of one that takes them in turn (40 rows of 48 heads 4.1 and 5.4 us; always: 4096 rows 29.5 instead of 27.4)
    const unsigned y = rows * turns <= 4ll * cus ? turns : 1;
    const dim3 grid(static_cast<unsigned>(rows), y);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p, lanes); };
    const bool bf = dtype == TPAMD_BF16;
    if (vec == 8) bf ? run(heads_kernel<TPAMD_BF16, 8>) : run(heads_kernel<TPAMD_F16, 8>);
    else if (vec == 4) bf ? run(heads_kernel<TPAMD_BF16, 4>) : run(heads_kernel<TPAMD_F16, 4>);
    else bf ? run(heads_kernel<TPAMD_BF16, 1>) : run(heads_kernel<TPAMD_F16, 1>);
    TPAMD_HIP(hipGetLastError());
    return TPAMD_OK;
}

}  // namespace
}  // namespace tpamd

using namespace tpamd;

extern "C" int tpamd_rotate_heads(const tpamd_heads *heads, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, int dtype, void *stream) {
    return heads_entry("tpamd_rotate_heads", heads, nullptr, rows, Hq, Hkv, D, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int tpamd_append_paged(const tpamd_heads *heads, const tpamd_pages *pages, int64_t rows, int64_t Hq, int64_t Hkv, int64_t D, int dtype, void *stream) {
    TPAMD_REQUIRE(pages != nullptr, "tpamd_append_paged: null pointer");
    return heads_entry("tpamd_append_paged", heads, pages, rows, Hq, Hkv, D, dtype, static_cast<hipStream_t>(stream));
}
