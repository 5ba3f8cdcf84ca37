// The linear layer with 4-bit weights (linear_int4.hip): which kernel and work group a problem gets. Host code without HIP in it, so that a test can ask.
#pragma once
#include <cmath>

namespace mi {

enum Int4FormIndex { kFew16, kFew32, kFew64, kTile32x64, kTile32x128, kTile64x128, kTile64x192, kTile96x192, kTile64x256, kInt4Forms };      // features of 16 rows; tokens x features

// Rows and features that the tiles' 32-bit offsets do not span
inline bool int4_far_apart(int N, long ldx) { return ldx * 2 * 96 >= (1L << 31) || N > 1 << 24; }

// The form of a launch: the one with the smallest estimated time (us). W work groups on C compute units, each of which takes R at a time, are ceil(W / C R) rounds
// (beyond two, W / C R + 1/2: they no longer begin and end together) that each wait for every step (a block of 128 contraction elements) and c = ceil(W / C) work
// groups on the busiest compute unit, which share what it issues:
//   time = launch + steps (rounds * wait + c * issue) + c * end
// fitted, least relative squares, to 495 measured problems (1 to 4608 rows, nine pairs of contraction and features from 2560 x 640 to 16384 x 6144, groups of 128, 64
// with zero points and 32, whole and in shares), the ones within 1.15 of a problem's fastest weighing ten times those beyond 1.5, long ones more; the one taken is
// 0.9 % slower than the fastest on average, 16 % at most. Without a form the fastest of the rest is slower on average by 2.4 % (kFew16), 1.4, 0.7, 3.2, 0.8 and less (any
// one of the tiles of 64 and 96 tokens can be replaced within 0.4 %; 64 x 256, kept for groups of 128 and more alone, by up to 28 % where it leaves no compute unit idle
// and 96 x 192 does).
struct Int4Cost { float launch, wait, issue, end; };
struct Int4FormRule { int rows, features, resident; Int4Cost cost[3]; };      // [groups of 128 and more, 64, 32]
inline constexpr Int4FormRule kInt4Rules[kInt4Forms] = {
    {16, 16, 2, {{1.09f, 0.0516f, 0.0484f, 0.965f}, {0.344f, 0.0f, 0.114f, 1.74f}, {0.326f, 0.0f, 0.134f, 1.69f}}},    // kFew16
    {16, 32, 1, {{0.129f, 0.0f, 0.128f, 2.4f}, {0.16f, 0.0143f, 0.134f, 2.5f}, {0.338f, 0.0216f, 0.165f, 2.32f}}},    // kFew32
    {16, 64, 1, {{0.00451f, 0.0779f, 0.109f, 3.43f}, {0.551f, 0.0839f, 0.16f, 2.98f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kFew64
    {32, 64, 4, {{2.4f, 0.225f, 0.164f, 0.282f}, {2.32f, 0.271f, 0.2f, 0.293f}, {2.19f, 0.378f, 0.194f, 0.396f}}},    // kTile32x64
    {32, 128, 3, {{2.93f, 0.222f, 0.285f, 0.216f}, {3.14f, 0.334f, 0.337f, 0.188f}, {4.21f, 0.53f, 0.375f, 0.101f}}},    // kTile32x128
    {64, 128, 3, {{3.54f, 0.851f, 0.281f, 0.08f}, {4.38f, 0.744f, 0.55f, 0.0f}, {5.07f, 1.16f, 0.527f, 0.0f}}},    // kTile64x128
    {64, 192, 2, {{3.34f, 0.911f, 0.348f, 0.0484f}, {3.9f, 1.02f, 0.54f, 0.0f}, {5.45f, 1.5f, 0.65f, 0.0f}}},    // kTile64x192
    {96, 192, 2, {{2.57f, 1.14f, 0.454f, 0.714f}, {4.03f, 1.17f, 0.738f, 0.0f}, {6.13f, 1.81f, 1.1f, 0.0f}}},    // kTile96x192
    {64, 256, 2, {{3.81f, 1.07f, 0.435f, 0.0598f}, {0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kTile64x256
};
// A launch: its form (-1: none, every grid would have 2^32 work-items across or 2^16 work groups down and more), and the shares that the contraction is given in, each
// to work groups of its own (1: all in one). Shares cost a second launch, which adds them, and what it reads and writes: kJoin us, fitted with the rest, and 1 us for
// kJoinBytes of sums, half of what a copy moves, as they are written and read (4096 x 4608 x 1152, operands from memory, groups of 128: in three shares, 57 MB,
// which the rule would take if sums cost nothing, 78 us, in one 68; groups of 64: 84 and 75)
struct Int4Launch { int form, shares; };
constexpr int kInt4Shares[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr long kMostItems = 0xffffffffL;      // work-items of a grid across: 512 for a run of features (few rows), 256 for a tile of a multiple of 8
constexpr float kJoin = 3.5f, kJoinBytes = 3.0e6f;
inline Int4Launch int4_launch(int M, int N, int KB, long ldx, int parts, int cu, unsigned long lent) {
    const int which = parts == 1 ? 0 : parts == 2 ? 1 : 2, forms = int4_far_apart(N, ldx) ? kTile32x64 : kInt4Forms;
    Int4Launch best{-1, 1};
    float least = 0.f;
    for (int i = 0; i < forms; ++i) {
        const Int4FormRule& f = kInt4Rules[i];
        const long down = (static_cast<long>(M) + f.rows - 1) / f.rows, across = (static_cast<long>(N) + f.features - 1) / f.features;
        if ((parts == 4 && i == kFew64) || (parts > 1 && i == kTile64x256)) continue;
        if (i < kTile32x64 ? down > 65535 || across > kMostItems / 512 : down * across > kMostItems / 256 - 7) continue;
        const float whole = static_cast<float>(down * across);
        for (const int shares : kInt4Shares) {
            const float bytes = 4.f * shares * M * N;
            if (shares > 1 && (KB < 4 * shares || whole * shares > 4 * cu || bytes > 1e9f || 4ul * shares * M * N > lent)) break;
            const float groups = whole * shares, c = std::ceil(groups / cu), full = groups / (cu * f.resident), rounds = full <= 2.f ? std::ceil(full) : full + 0.5f;
            const Int4Cost& t = f.cost[which];
            const float time = t.launch + static_cast<float>((KB + shares - 1) / shares) * (rounds * t.wait + c * t.issue) + c * t.end + (shares > 1 ? kJoin + bytes / kJoinBytes : 0.f);
            if (best.form < 0 || time < least) { best = {i, shares}; least = time; }
        }
    }
    return best;
}

}  // namespace mi
