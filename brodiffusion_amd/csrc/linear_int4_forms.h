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
// fitted, least relative squares, to 796 measured problems (1 to 4096 rows, eight pairs of contraction and features from 1280 x 10240 to 16384 x 6144, groups of 128, 64
// and 32, with and without zero points); the one taken is 0.6 % slower than the fastest on average.
struct Int4Cost { float launch, wait, issue, end; };
struct Int4FormRule { int rows, features, resident; Int4Cost cost[3]; };      // [groups of 128 and more, 64, 32]
inline constexpr Int4FormRule kInt4Rules[kInt4Forms] = {
    {16, 16, 2, {{0.691f, 0.0f, 0.106f, 1.39f}, {0.603f, 0.0f, 0.115f, 1.45f}, {0.614f, 0.0f, 0.133f, 1.63f}}},    // kFew16
    {16, 32, 1, {{0.545f, 0.135f, 0.0f, 2.02f}, {0.484f, 0.148f, 0.0f, 2.2f}, {0.467f, 0.182f, 0.0f, 2.48f}}},    // kFew32
    {16, 64, 1, {{0.513f, 0.183f, 0.0f, 2.92f}, {0.87f, 0.231f, 0.0f, 2.76f}, {0.0f, 0.0f, 0.0f, 0.0f}}},    // kFew64
    {32, 64, 4, {{2.59f, 0.205f, 0.161f, 0.228f}, {2.56f, 0.224f, 0.187f, 0.226f}, {2.93f, 0.294f, 0.225f, 0.194f}}},    // kTile32x64
    {32, 128, 3, {{2.85f, 0.276f, 0.26f, 0.511f}, {2.83f, 0.302f, 0.296f, 0.526f}, {3.62f, 0.595f, 0.405f, 0.482f}}},    // kTile32x128
    {64, 128, 2, {{6.11f, 0.582f, 0.264f, 0.0f}, {5.39f, 0.795f, 0.271f, 0.0f}, {8.23f, 0.665f, 0.645f, 0.0f}}},    // kTile64x128
    {64, 256, 2, {{3.21f, 1.07f, 0.395f, 1.65f}, {5.89f, 0.963f, 0.825f, 0.504f}, {6.84f, 1.14f, 1.24f, 0.618f}}},    // kTile64x256
};
inline int int4_form(int M, int N, int KB, long ldx, int parts, int cu) {
    const int which = parts == 1 ? 0 : parts == 2 ? 1 : 2, forms = int4_far_apart(N, ldx) ? kTile32x64 : kInt4Forms;
    int best = -1;
    float least = 0.f;
    for (int i = 0; i < forms; ++i) {
        const Int4FormRule& f = kInt4Rules[i];
        if ((i == kFew64 && parts == 4) || (i < kTile32x64 && M > 65535L * 16)) continue;
        const float groups = static_cast<float>((static_cast<long>(M) + f.rows - 1) / f.rows * ((static_cast<long>(N) + f.features - 1) / f.features));
        const float c = std::ceil(groups / cu), rounds = std::ceil(groups / (cu * f.resident));
        const Int4Cost& t = f.cost[which];
        const float time = t.launch + KB * (rounds * t.wait + c * t.issue) + c * t.end;
        if (best < 0 || time < least) { best = i; least = time; }
    }
    return best;
}

}  // namespace mi
