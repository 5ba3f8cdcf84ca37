// The linear layer with 4-bit weights (linear_int4.hip): which kernel and work group a problem gets. Host code without HIP in it, so that a test can ask.
#pragma once
#include <cmath>

namespace mi {

enum Int4FormIndex { kFew16, kFew32, kFew64, kTile32x64, kTile32x128, kTile64x128, kTile64x256, kInt4Forms };      // features of 16 rows; tokens x features

// Rows and features that the tiles' 32-bit offsets do not span
inline bool int4_far_apart(int N, long ldx) { return ldx * 2 * 64 >= (1L << 31) || N > 1 << 24; }

// The form of a launch: the one with the smallest estimated time (us). W work groups on C compute units, R of which take one at a time, are ceil(W / C R) rounds
// that each wait for every step (a block of 128 contraction elements) and c = ceil(W / C) work groups on the busiest compute unit, which share what it issues:
//   time = launch + steps (rounds * wait + c * issue) + c * end
// fitted, least relative squares, to 1108 measured problems (1 to 4096 rows, eight pairs of contraction and features from 1280 x 10240 to 16384 x 6144, groups of 128, 64
// and 32, with and without zero points); the one taken is 1.2 % slower than the fastest on average.
struct Int4Cost { float launch, wait, issue, end; };
struct Int4FormRule { int rows, features, resident; Int4Cost cost[3]; };      // [groups of 128 and more, 64, 32]
inline constexpr Int4FormRule kInt4Rules[kInt4Forms] = {
    {16, 16, 2, {{1.14f, 0.0378f, 0.0577f, 1.24f}, {0.847f, 0.0f, 0.108f, 1.54f}, {0.805f, 0.0f, 0.127f, 1.65f}}},    // kFew16
    {16, 32, 1, {{0.549f, 0.128f, 0.0f, 2.2f}, {0.513f, 0.145f, 0.0f, 2.34f}, {0.536f, 0.18f, 0.0f, 2.52f}}},    // kFew32
    {16, 64, 1, {{0.458f, 0.183f, 0.0f, 3.19f}, {0.546f, 0.226f, 0.0f, 3.27f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kFew64
    {32, 64, 4, {{3.0f, 0.196f, 0.16f, 0.361f}, {3.17f, 0.213f, 0.193f, 0.28f}, {3.2f, 0.295f, 0.22f, 0.328f}}},    // kTile32x64
    {32, 128, 3, {{3.0f, 0.228f, 0.266f, 0.817f}, {3.7f, 0.291f, 0.306f, 0.656f}, {3.45f, 0.542f, 0.403f, 0.61f}}},    // kTile32x128
    {64, 128, 2, {{5.99f, 0.614f, 0.263f, 0.0f}, {4.84f, 0.864f, 0.265f, 0.583f}, {6.59f, 1.01f, 0.457f, 0.0f}}},    // kTile64x128
    {64, 256, 2, {{3.05f, 0.995f, 0.432f, 2.19f}, {5.52f, 1.06f, 0.849f, 1.05f}, {4.81f, 1.18f, 1.14f, 0.557f}}},    // kTile64x256
};
// A launch: its form, and the shares that the contraction is given in, each to work groups of its own (1: all in one). Shares cost a second launch, which
// adds them, and what it reads and writes: kJoin us and 1 us for kJoinBytes of sums, fitted with the rest.
struct Int4Launch { int form, shares; };
constexpr int kInt4Shares[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr float kJoin = 3.0f, kJoinBytes = 6.0e6f;
inline Int4Launch int4_launch(int M, int N, int KB, long ldx, int parts, int cu, unsigned long lent) {
    const int which = parts == 1 ? 0 : parts == 2 ? 1 : 2, forms = int4_far_apart(N, ldx) ? kTile32x64 : kInt4Forms;
    Int4Launch best{-1, 1};
    float least = 0.f;
    for (int i = 0; i < forms; ++i) {
        const Int4FormRule& f = kInt4Rules[i];
        if ((i == kFew64 && parts == 4) || (i < kTile32x64 && M > 65535L * 16)) continue;
        const float whole = static_cast<float>((static_cast<long>(M) + f.rows - 1) / f.rows * ((static_cast<long>(N) + f.features - 1) / f.features));
        for (const int shares : kInt4Shares) {
            const float bytes = 4.f * shares * M * N;
            if (shares > 1 && (KB < 4 * shares || whole * shares > 4 * cu || bytes > 1e9f || 4ul * shares * M * N > lent)) break;
            const float groups = whole * shares, c = std::ceil(groups / cu), rounds = std::ceil(groups / (cu * f.resident));
            const Int4Cost& t = f.cost[which];
            const float time = t.launch + static_cast<float>((KB + shares - 1) / shares) * (rounds * t.wait + c * t.issue) + c * t.end + (shares > 1 ? kJoin + bytes / kJoinBytes : 0.f);
            if (best.form < 0 || time < least) { best = {i, shares}; least = time; }
        }
    }
    return best;
}

}  // namespace mi
