// The linear layer with 4-bit weights (linear_int4.hip): which kernel and work group a problem gets. Host code without HIP in it, so that a test can ask.
#pragma once
#include <cmath>

namespace mi {

enum Int4FormIndex { kFew16, kFew32, kFew64, kTile32x64, kTile32x128, kTile64x128, kTile64x192, kTile96x192, kTile64x256, kInt4Forms };      // features of 16 rows; tokens x features

// Rows and features that the tiles' 32-bit offsets do not span
inline bool int4_far_apart(int N, long ldx) { return ldx * 2 * 96 >= (1L << 31) || N > 1 << 24; }

// The form of a launch: the one with the smallest estimated time (us). W work groups on C compute units, R of which take one at a time, are ceil(W / C R) rounds
// that each wait for every step (a block of 128 contraction elements) and c = ceil(W / C) work groups on the busiest compute unit, which share what it issues:
//   time = launch + steps (rounds * wait + c * issue) + c * end
// fitted, least relative squares, to 495 measured problems (1 to 4608 rows, nine pairs of contraction and features from 2560 x 640 to 16384 x 6144, groups of 128, 64
// with zero points and 32, whole and in shares), the ones within 1.15 of a problem's fastest weighing ten times those beyond 1.5; the one taken is 0.9 % slower than the
// fastest on average, 16 % at most. Without a form the fastest of the rest is slower on average by 2.4 % (kFew16), 1.4, 0.7, 3.2, 0.8 and less (the tiles of 64 and 96 tokens, of
// which any one can be replaced within 0.4 %, 64 x 256, kept for groups of 128 and more alone, by up to 28 % where it leaves no compute unit idle and 96 x 192 does).
struct Int4Cost { float launch, wait, issue, end; };
struct Int4FormRule { int rows, features, resident; Int4Cost cost[3]; };      // [groups of 128 and more, 64, 32]
inline constexpr Int4FormRule kInt4Rules[kInt4Forms] = {
    {16, 16, 2, {{1.52f, 0.0485f, 0.0471f, 0.936f}, {0.735f, 0.0f, 0.109f, 1.78f}, {0.752f, 0.0f, 0.128f, 1.71f}}},    // kFew16
    {16, 32, 1, {{0.504f, 0.124f, 0.0f, 2.4f}, {0.59f, 0.145f, 0.0f, 2.48f}, {0.791f, 0.182f, 0.0f, 2.29f}}},    // kFew32
    {16, 64, 1, {{0.282f, 0.184f, 0.0f, 3.54f}, {0.833f, 0.24f, 0.0f, 3.09f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kFew64
    {32, 64, 4, {{2.95f, 0.212f, 0.164f, 0.273f}, {2.92f, 0.249f, 0.205f, 0.247f}, {2.87f, 0.349f, 0.206f, 0.279f}}},    // kTile32x64
    {32, 128, 3, {{3.42f, 0.218f, 0.281f, 0.233f}, {3.77f, 0.314f, 0.348f, 0.0716f}, {4.57f, 0.547f, 0.381f, 0.0f}}},    // kTile32x128
    {64, 128, 3, {{4.15f, 0.838f, 0.285f, 0.0f}, {4.53f, 0.815f, 0.526f, 0.0f}, {5.08f, 1.29f, 0.484f, 0.0f}}},    // kTile64x128
    {64, 192, 2, {{4.19f, 0.891f, 0.34f, 0.0f}, {4.44f, 1.01f, 0.537f, 0.0f}, {5.18f, 1.72f, 0.553f, 0.0f}}},    // kTile64x192
    {96, 192, 2, {{4.23f, 1.11f, 0.472f, 0.0f}, {4.34f, 1.29f, 0.663f, 0.0f}, {4.71f, 2.45f, 0.819f, 0.0f}}},    // kTile96x192
    {64, 256, 2, {{4.64f, 1.05f, 0.432f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kTile64x256
};
// A launch: its form, and the shares that the contraction is given in, each to work groups of its own (1: all in one). Shares cost a second launch, which
// adds them, and what it reads and writes: kJoin us, fitted with the rest, and 1 us for kJoinBytes of sums, half of what a copy moves, as they are written and read
// (4096 x 4608 x 1152 in two shares of 64 x 192, 38 MB: 74 + 12 us, in one 72)
struct Int4Launch { int form, shares; };
constexpr int kInt4Shares[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr float kJoin = 3.0f, kJoinBytes = 3.0e6f;
inline Int4Launch int4_launch(int M, int N, int KB, long ldx, int parts, int cu, unsigned long lent) {
    const int which = parts == 1 ? 0 : parts == 2 ? 1 : 2, forms = int4_far_apart(N, ldx) ? kTile32x64 : kInt4Forms;
    Int4Launch best{-1, 1};
    float least = 0.f;
    for (int i = 0; i < forms; ++i) {
        const Int4FormRule& f = kInt4Rules[i];
        if ((parts == 4 && i == kFew64) || (parts > 1 && i == kTile64x256) || (i < kTile32x64 && M > 65535L * 16)) continue;
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
