// How the tcgen05 kernel of the projections with 4-bit weights divides its work. Host arithmetic.
#pragma once

namespace efa {

constexpr int W4_MAX_PARTS = 8;

// Channels of a tile (a block has two) and blocks of a cluster that share k. at_once[p]: clusters of p blocks that the device holds at a time, 0: none, which is
// then no choice; a block by itself there always is. The fewest rounds, each 4 us and 0.6 us a unit of 128 k, and 1 us for the sums of several blocks. A
// block of fewer channels computes as long.
struct W4Division { int channels, parts; };
inline W4Division w4_division(int d_out, int row_tiles, int units, const int* at_once)
{
    W4Division to{128, 1};
    double best = 1e30;
    for (int p = 1; p <= W4_MAX_PARTS && p <= units; p++) {
        const int clusters_at_once = p == 1 && at_once[1] < 1 ? 1 : at_once[p];
        if (clusters_at_once < 1) continue;
        for (int c = 128; c >= 96; c -= 16) {
            const long long clusters = (long long)((d_out + 2 * c - 1) / (2 * c)) * row_tiles;
            const double time = (double)((clusters + clusters_at_once - 1) / clusters_at_once) * (4.0 + 0.6 * ((units + p - 1) / p) + (p > 1 ? 1.0 : 0.0));
            if (time < best * 0.999) { best = time; to = W4Division{c, p}; }
        }
    }
    return to;
}

}  // namespace efa
