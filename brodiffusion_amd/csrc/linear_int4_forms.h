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
// with zero points and 32, whole and in shares), the ones within 1.15 of a problem's fastest weighing ten times those beyond 1.5; the one taken is 0.8 % slower than the
// fastest on average, 16 % at most. Without a form the fastest of the rest is slower on average by 2.4 % (kFew16), 1.4, 0.7, 3.2, 0.8 and less (the tiles of 64 and 96 tokens, of
// which any one can be replaced within 0.4 %, 64 x 256 by up to 28 % where 64 x 256 leaves no compute unit idle and 96 x 192 does).
struct Int4Cost { float launch, wait, issue, end; };
struct Int4FormRule { int rows, features, resident; Int4Cost cost[3]; };      // [groups of 128 and more, 64, 32]
inline constexpr Int4FormRule kInt4Rules[kInt4Forms] = {
    {16, 16, 2, {{1.09f, 0.0514f, 0.0482f, 0.98f}, {0.335f, 0.0f, 0.114f, 1.76f}, {0.321f, 0.0f, 0.134f, 1.7f}}},    // kFew16
    {16, 32, 1, {{0.11f, 0.128f, 0.0f, 2.44f}, {0.136f, 0.148f, 0.0f, 2.55f}, {0.317f, 0.187f, 0.0f, 2.36f}}},    // kFew32
    {16, 64, 1, {{0.0f, 0.187f, 0.0f, 3.5f}, {0.443f, 0.243f, 0.0f, 3.13f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kFew64
    {32, 64, 4, {{2.36f, 0.225f, 0.157f, 0.548f}, {2.37f, 0.262f, 0.198f, 0.511f}, {2.34f, 0.362f, 0.198f, 0.542f}}},    // kTile32x64
    {32, 128, 3, {{2.95f, 0.216f, 0.279f, 0.621f}, {3.33f, 0.315f, 0.343f, 0.489f}, {4.36f, 0.528f, 0.385f, 0.331f}}},    // kTile32x128
    {64, 128, 3, {{4.28f, 0.785f, 0.298f, 0.621f}, {5.45f, 0.7f, 0.585f, 0.151f}, {6.84f, 1.17f, 0.535f, 0.0f}}},    // kTile64x128
    {64, 192, 2, {{3.93f, 0.871f, 0.339f, 1.06f}, {5.11f, 0.923f, 0.596f, 0.48f}, {7.2f, 1.57f, 0.65f, 0.0f}}},    // kTile64x192
    {96, 192, 2, {{4.32f, 1.05f, 0.479f, 1.58f}, {6.01f, 1.12f, 0.759f, 0.69f}, {7.95f, 2.24f, 0.945f, 0.054f}}},    // kTile96x192
    {64, 256, 2, {{5.09f, 0.962f, 0.471f, 1.06f}, {7.56f, 1.18f, 0.965f, 0.0441f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kTile64x256
};
// A launch: its form, and the shares that the contraction is given in, each to work groups of its own (1: all in one). Shares cost a second launch, which
// adds them, and what it reads and writes: kJoin us and 1 us for kJoinBytes of sums, fitted with the rest.
struct Int4Launch { int form, shares; };
constexpr int kInt4Shares[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr float kJoin = 3.5f, kJoinBytes = 6.0e6f;
inline Int4Launch int4_launch(int M, int N, int KB, long ldx, int parts, int cu, unsigned long lent) {
    const int which = parts == 1 ? 0 : parts == 2 ? 1 : 2, forms = int4_far_apart(N, ldx) ? kTile32x64 : kInt4Forms;
    Int4Launch best{-1, 1};
    float least = 0.f;
    for (int i = 0; i < forms; ++i) {
        const Int4FormRule& f = kInt4Rules[i];
        if ((parts == 4 && (i == kFew64 || i == kTile64x256)) || (i < kTile32x64 && M > 65535L * 16)) continue;
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
