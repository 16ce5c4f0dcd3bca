// Which tile and how many ranges of K the products of two 8-bit operands take (host code).
#pragma once
#include <stdint.h>

#include <initializer_list>

namespace tpamd {

// A launch on tiles of 64 tm x 64 tn (a pair: 32 tn columns): fixed + whole rounds of the CUs * (round + full * K tiles) + a last round that costs part + K tiles at a rate between
// few (one block) and full (every CU has one). `two`: two blocks fit a CU, the rates with up to one (at one block on every CU) and with the first CU that has two.
// Ranges of K add split + per_mb * MB of partial sums + per_range * ranges. All in us.
struct A8Tile {
    int tm, tn, blocks_per_cu;
    float fixed, round, full, few, part, one, two, split, per_mb, per_range;
};
// Fitted to 400 shapes at 65-6144 rows, 1024-16384 columns, K 1024-11008, each tile with 1-12 ranges timed inside HIP graphs on rotated weights; the choice is 1.2 % off the best of them in the
// geometric mean, 0.8 % on 200 others (worst 32 and 18 %). Without one of the tiles the best would be 1-4 % slower each.
constexpr A8Tile A8_TILES[2][6] = {
    {
        {1, 2, 2, 4.8, 0.9, 0.75, 0.25, 0.0, 0.44, 0.62, 2.1, 0.27, 0.22},
        {2, 2, 1, 5.6, 1.8, 0.60, 0.36, 0.0, 0, 0, 2.4, 0.20, 0.17},
        {2, 3, 1, 5.3, 2.6, 0.77, 0.45, 1.6, 0, 0, 1.9, 0.20, 0.20},
        {3, 3, 1, 5.7, 3.1, 1.03, 0.55, 2.8, 0, 0, 1.0, 0.20, 0.09},
        {3, 4, 1, 6.0, 2.1, 1.46, 0.86, 2.5, 0, 0, 0.7, 0.21, 0.08},
        {4, 4, 1, 0.5, 9.7, 1.59, 1.00, 9.9, 0, 0, 0.0, 0.22, 0.00},
    },
    {
        {1, 2, 2, 4.5, 1.4, 0.75, 0.25, 0.0, 0.46, 0.65, 2.5, 0.29, 0.00},
        {2, 2, 1, 4.7, 1.9, 0.59, 0.36, 0.8, 0, 0, 2.9, 0.22, 0.00},
        {2, 3, 1, 6.0, 3.0, 0.76, 0.45, 0.8, 0, 0, 2.6, 0.21, 0.00},
        {3, 3, 1, 3.2, 4.0, 1.02, 0.59, 4.4, 0, 0, 2.2, 0.20, 0.00},
        {3, 4, 1, 6.9, 2.3, 1.48, 0.93, 0.4, 0, 0, 2.0, 0.21, 0.00},
        {4, 4, 1, 3.4, 7.3, 1.64, 1.03, 6.0, 0, 0, 0.8, 0.21, 0.00},
    },
};
inline float a8_tile_us(const A8Tile &t, bool pair, uint32_t M, uint32_t N, uint32_t K, uint32_t ranges, int cus, float *mb) {
    // (divisions in 32 bits, sizes are below 2^30: a choice takes the host 0.5 us, 0.8 with 64)
    const uint32_t rows = static_cast<uint32_t>(64 * t.tm), columns = static_cast<uint32_t>((pair ? 32 : 64) * t.tn);
    const uint32_t all = (K + 127) / 128, kt = (all + ranges - 1) / ranges, splits = (all + kt - 1) / kt;
    const int64_t blocks = static_cast<int64_t>((M + rows - 1) / rows) * ((N + columns - 1) / columns) * splits;
    const int64_t round = static_cast<int64_t>(t.blocks_per_cu) * cus, rounds = blocks < round ? 0 : blocks / round, rest = blocks - rounds * round;
    const float k = static_cast<float>(kt), part = static_cast<float>(rest) / static_cast<float>(cus);
    float us = static_cast<float>(rounds) * (t.round + t.full * k);
    if (rest > 0) {
        float rate = t.few + (t.full - t.few) * part;
        if (t.blocks_per_cu == 2) rate = part <= 1.f ? t.few + (t.one - t.few) * part : t.two + (t.full - t.two) * (part - 1.f);
        us += t.part + rate * k;
    }
    const float weights = static_cast<float>(N) * static_cast<float>(K) * (pair ? 2.f : 1.f) * (1.f / 4.8e6f);  // from memory, at what tiles of few rows read
    us = t.fixed + (us > weights ? us : weights);
    *mb = static_cast<float>(blocks) * static_cast<float>(t.tm * t.tn) * (64 * 64 * 4 * 1e-6f);
    return splits > 1 ? us + t.split + t.per_mb * *mb + t.per_range * static_cast<float>(splits) : us;
}
struct A8Choice {
    int tm, tn, ranges;
    float us;
};
// The fastest by the model; partial sums of at most `scratch` bytes.
inline A8Choice a8_choose(bool pair, uint32_t M, uint32_t N, uint32_t K, int cus, int64_t scratch) {
    A8Choice best{4, 4, 1, 1e30f};
    for (const A8Tile &t : A8_TILES[pair])
        for (uint32_t ranges : {1, 2, 3, 4, 6, 8, 12}) {
            if (ranges > 1 && (K + 127) / 128 < 2 * ranges) break;
            float mb = 0.f;
            const float us = a8_tile_us(t, pair, M, N, K, ranges, cus, &mb);
            if (ranges > 1 && mb * 1e6f > static_cast<float>(scratch)) break;
            if (us < best.us) best = {t.tm, t.tn, static_cast<int>(ranges), us};
        }
    return best;
}

}  // namespace tpamd
