// Which kernel the projections with 4-bit weights take for more than eight rows, and how the work is divided among blocks. Host arithmetic.
#pragma once

namespace efa {

constexpr int W4_MAX_PARTS = 8;

// tcgen05: channels of a tile (a block has two), blocks of a cluster that share k, and what that makes: rounds of clusters, units of 128 k to a block. at_once[p]: clusters of
// p blocks that the device holds at a time, 0: none, which is then no choice; a block by itself there always is. The fewest rounds, each 4 us and 0.6 us a unit, and
// 1 us for the sums of several blocks. A block of fewer channels computes as long.
struct W4Division { int channels, parts; long long rounds; int units; };
inline W4Division w4_division(int d_out, int row_tiles, int units, const int* at_once)
{
    W4Division to{128, 1, 1, units};
    double best = 1e30;
    for (int p = 1; p <= W4_MAX_PARTS && p <= units; p++) {
        const int clusters_at_once = p == 1 && at_once[1] < 1 ? 1 : at_once[p];
        if (clusters_at_once < 1) continue;
        const int share = (units + p - 1) / p;
        for (int c = 128; c >= 96; c -= 16) {
            const long long clusters = (long long)((d_out + 2 * c - 1) / (2 * c)) * row_tiles, rounds = (clusters + clusters_at_once - 1) / clusters_at_once;
            const double time = (double)rounds * (4.0 + 0.6 * share + (p > 1 ? 1.0 : 0.0));
            if (time < best * 0.999) { best = time; to = W4Division{c, p, rounds, share}; }
        }
    }
    return to;
}

// mma.sync: few tiles have clusters that share k, as long as every warp has a unit of 256 k and every block an SM. us in 1 / 2 / 4 parts: 16 rows, 8192 x 1024 10.0 / 7.0 / 5.6,
// 4096 x 4096 (one part) 6.8 / 7.2.
inline int w4_parts(long long tiles, int units, int warps, int sms)
{
    int parts = 1;
    while (parts < W4_MAX_PARTS && 2 * parts * warps <= units && tiles * 2 * parts <= sms) parts *= 2;
    return parts;
}

// us that a call of more than eight rows takes on either, as fitted to 1138 measurements of both (weights from memory, one launch behind another, groups of 32, 64 and 128, 9 to 512 rows,
// 2^20 to 2^28 weights): a standard deviation of 8 to 10 % for mma.sync, 4 to 10 for tcgen05. Taken by the smaller figure a call is 0.15 % above the better of the two on average, in
// 23 of the 1138 by more than 3 %, at most by 18 (16 rows, 2560 x 10240 in groups of 32: 14.3 / 12.0). By the number of weights alone it was 1.4 %, 93 of them and 81 %: 64 rows, 512 x 8192
// 15.5 / 8.5; 33 rows, 16384 x 1024 in groups of 32 21.1 / 33.9.
struct W4Mma { double start, block, unit, block_unit; };           // of an SM's blocks, of a block's units, of both
struct W4Tc { double round, round_unit, weights; };                // of rounds, of their units, of 2^24 weights for 16 rows
inline double w4_mma_time(int d_in, int d_out, int rows, int group, int sms)
{
    static const W4Mma costs[3] = {{1.52, 1.07, 0.09, 0.20}, {1.68, 1.03, 0.09, 0.17}, {1.46, 1.07, 0.13, 0.17}};
    const W4Mma& c = costs[group == 32 ? 0 : group == 64 ? 1 : 2];
    const long long tiles = (long long)((d_out + 31) / 32) * ((rows + 15) / 16);
    const int units = (d_in + 255) / 256, parts = w4_parts(tiles, units, 8, sms), share = (units + parts - 1) / parts;
    const double even = (double)tiles * parts / sms;
    double blocks = (double)((tiles * parts + sms - 1) / sms);
    if (blocks <= 2) {                                             // side by side: where some SMs have one and some two, in between
        blocks = 0.6 * blocks + 0.4 * even;
        blocks = blocks < 1 ? 1 : blocks;
    }
    return c.start + c.block * blocks + (c.unit + c.block_unit * blocks) * share;
}
inline double w4_tc_time(const W4Division& to, int d_in, int d_out, int rows, int group)
{
    static const W4Tc costs[3][3] = {{{5.35, 0.70, 0.90}, {6.03, 0.88, 0.47}, {7.23, 1.60, 0.22}},
                                     {{5.76, 0.41, 0.91}, {5.88, 0.52, 0.35}, {6.82, 0.92, 0.14}},
                                     {{5.49, 0.35, 0.95}, {5.95, 0.44, 0.33}, {7.17, 0.50, 0.15}}};
    const W4Tc& c = costs[group == 32 ? 0 : group == 64 ? 1 : 2][rows <= 16 ? 0 : rows <= 32 ? 1 : 2];
    return (double)to.rounds * (c.round + c.round_unit * to.units) + c.weights * ((rows + 15) / 16) * ((double)d_in * d_out / (1 << 24));
}
// However the device divides it: one round, k in as many parts as there can be.
inline double w4_tc_least(int d_in, int d_out, int rows, int group)
{
    return w4_tc_time(W4Division{128, W4_MAX_PARTS, 1, ((d_in + 127) / 128 + W4_MAX_PARTS - 1) / W4_MAX_PARTS}, d_in, d_out, rows, group);
}

}  // namespace efa
