// Which tile and how many ranges of K the products of two 8-bit operands take (host code).
#pragma once
#include <stdint.h>

namespace tpamd {

// A launch on tiles of 64 tm x 64 tn (a pair: 32 tn columns): fixed + whole rounds of the CUs * (round + full * K tiles) + a last round that costs part + K tiles at a rate between
// few (one block) and full (every CU has one). `two`: two blocks fit a CU, the rates with up to one (at one block on every CU) and with the first CU that has two.
// Ranges of K add split + per_mb * MB of partial sums + per_range * ranges. All in us.
struct A8Tile {
    int tm, tn, blocks_per_cu;
    float fixed, round, full, few, part, one, two, split, per_mb, per_range;
};
// Fitted to 300 shapes at 65-6144 rows, 1024-16384 columns, K 1024-11008, each tile with 1-12 ranges timed inside HIP graphs on rotated weights; the choice is 0.8 % off the best of them in the
// geometric mean, 1.0 % on 200 others (worst 28 %). Without one of the tiles the best would be 1-4 % slower each.
constexpr A8Tile A8_TILES[2][6] = {
    {
        {1, 2, 2, 5.1, 1.3, 0.77, 0.21, 0.0, 0.42, 0.58, 2.4, 0.25, 0.13},
        {2, 2, 1, 4.6, 2.1, 0.60, 0.31, 1.1, 0, 0, 2.7, 0.18, 0.10},
        {2, 3, 1, 6.6, 2.8, 0.77, 0.39, 0.5, 0, 0, 2.1, 0.19, 0.12},
        {3, 3, 1, 5.7, 3.5, 1.02, 0.51, 2.7, 0, 0, 1.3, 0.19, 0.04},
        {3, 4, 1, 7.5, 1.7, 1.45, 0.80, 1.3, 0, 0, 0.7, 0.20, 0.02},
        {4, 4, 1, 2.2, 9.2, 1.61, 0.92, 8.6, 0, 0, 0.0, 0.21, 0.00},
    },
    {
        {1, 2, 2, 4.1, 1.3, 0.83, 0.19, 0.0, 0.49, 0.58, 3.3, 0.28, 0.00},
        {2, 2, 1, 4.7, 2.0, 0.63, 0.34, 0.0, 0, 0, 3.5, 0.20, 0.02},
        {2, 3, 1, 5.9, 2.3, 0.83, 0.44, 0.0, 0, 0, 3.4, 0.21, 0.02},
        {3, 3, 1, 7.1, 3.1, 1.06, 0.53, 0.5, 0, 0, 2.8, 0.17, 0.00},
        {3, 4, 1, 4.6, 2.6, 1.56, 0.84, 3.0, 0, 0, 2.5, 0.17, 0.00},
        {4, 4, 1, 1.5, 7.7, 1.70, 0.95, 8.2, 0, 0, 1.7, 0.18, 0.00},
    },
};
inline float a8_tile_us(const A8Tile &t, bool pair, int64_t M, int64_t N, int64_t K, int ranges, int cus, float *mb) {
    const int64_t columns = (pair ? 32 : 64) * t.tn, tiles = (M + 64 * t.tm - 1) / (64 * t.tm) * ((N + columns - 1) / columns);
    const int64_t all = (K + 127) / 128, kt = (all + ranges - 1) / ranges, splits = (all + kt - 1) / kt, blocks = tiles * splits;
    const int64_t round = static_cast<int64_t>(t.blocks_per_cu) * cus, rounds = blocks / round, rest = blocks % round;
    const float k = static_cast<float>(kt), part = static_cast<float>(rest) / static_cast<float>(cus);
    float us = t.fixed + static_cast<float>(rounds) * (t.round + t.full * k);
    if (rest > 0) {
        float rate = t.few + (t.full - t.few) * part;
        if (t.blocks_per_cu == 2) rate = part <= 1.f ? t.few + (t.one - t.few) * part : t.two + (t.full - t.two) * (part - 1.f);
        us += t.part + rate * k;
    }
    *mb = static_cast<float>(blocks) * static_cast<float>(t.tm * t.tn) * (64 * 64 * 4 * 1e-6f);
    return splits > 1 ? us + t.split + t.per_mb * *mb + t.per_range * static_cast<float>(splits) : us;
}
struct A8Choice {
    int tm, tn, ranges;
    float us;
};
// The fastest by the model; partial sums of at most `scratch` bytes.
inline A8Choice a8_choose(bool pair, int64_t M, int64_t N, int64_t K, int cus, int64_t scratch) {
    A8Choice best{4, 4, 1, 1e30f};
    for (const A8Tile &t : A8_TILES[pair])
        for (int ranges : {1, 2, 3, 4, 6, 8, 12}) {
            if (ranges > 1 && (K + 127) / 128 < 2 * ranges) break;
            float mb = 0.f;
            const float us = a8_tile_us(t, pair, M, N, K, ranges, cus, &mb);
            if (ranges > 1 && mb * 1e6f > static_cast<float>(scratch)) break;
            if (us < best.us) best = {t.tm, t.tn, ranges, us};
        }
    return best;
}

}  // namespace tpamd
