// The linear layer with an epilogue for few rows (linear_few.hip): which problems that kernel takes and with which work groups. Host code without HIP in it, so
// that a test can ask.
#pragma once
#include <algorithm>

#include "linear_forms.h"

namespace mi {
namespace gemm {

enum FewKind { kSixteen, kWeights8, kBoth8 };      // operands of 16 bits, INT8 weights, both INT8 (then K and strides in pairs of elements)
inline FewKind few_kind(const LinearProblem& p) { return p.x_scale ? kBoth8 : p.w_scale ? kWeights8 : kSixteen; }

// How a problem stands to the GPU. narrow: up to 8 features per compute unit, so that work groups of 8 features are what there is to spread;
// wide: over 32; brief: not narrow, with a contraction of at most 4 KB of W's row, of which a wavefront gets a step or two.
struct FewShape {
    int cu;
    bool narrow, wide, brief;
    FewShape(const LinearProblem& p, FewKind kind, int n_cu) : cu(n_cu) {
        narrow = p.N <= 8 * cu;
        wide = p.N > 32 * cu;
        brief = !narrow && p.K * (kind == kWeights8 ? 1L : 2L) <= 4096;
    }
};

// Which problems this kernel is the faster one for, by both sides' times (us, this kernel / the rings of linear_pipe.h, with parts where those are
// taken; bf16, weights of up to 500 MB in turn; features x contraction). Its time goes with the rows and the contraction, that of the rings hardly:
//   narrow      368 x 15984: 16-bit 8 rows 8.2 / 8.1, 16 11.0 / 8.1; W8A16 12 9.8 / 10.1, 20 16.4 / 10.0; W8A8 16 6.9 / 7.5, 20 9.3 / 7.9;
//               1152 x 4616: 16-bit 16 5.7 / 7.1, 32 7.9 / 7.4; W8A16 32 8.4 / 8.5; W8A8 32 5.4 / 6.8; 1792 x 10488 W8A16 16 8.8 / 11.5, 20 13.0 / 11.7
//   up to 16 features per compute unit
//               2240 x 6728: 16-bit 16 9.3 / 9.7, 20 11.3 / 9.9; W8A16 32 10.7 / 11.2; 4096 x 8192: 16-bit 24 17.6 / 18.5, 32 19.3 / 18.7
//   brief       4608 x 1152: 16-bit 4 rows 4.2 / 4.4, 8 5.1 / 4.4; W8A16 24 5.8 / 5.9, 32 6.3 / 5.9; W8A8 1 5.0 / 4.0;
//               8192 x 2048: 16-bit 1 row 7.6 / 6.9; W8A16 24 7.3 / 8.6; W8A8 1 5.3 / 5.2
//   otherwise   7168 x 4096: 16-bit 8 12.9 / 13.5, 16 16.5 / 13.5; 6144 x 16384: 16-bit 24 41.9 / 43.2, 32 44.9 / 44.8; W8A16 32 32.6 / 37.8; W8A8 16 20.5 / 26.0
//   wide        16384 x 6144: 16-bit 16 39.3 / 43.0, 24 42.6 / 44.7, rows off lines (6152) 4 36.1 / 35.9, 8 38.4 / 36.0; 9968 x 12808: 16-bit 4
//               46.0 / 52.7, 8 55.3 / 52.8; W8A16 8 37.2 / 42.1; 16384 x 6144 W8A16 4 21.2 / 24.0, W8A8 16 19.8 / 19.8
inline bool few_takes(const LinearProblem& p, int n_cu) {
    const FewKind kind = few_kind(p);
    const FewShape s(p, kind, n_cu);
    if (p.M > 32) return false;
    const long work = static_cast<long>(p.M) * p.K;
    if (kind == kSixteen) {
        if (s.brief) return p.M <= 4 && p.N <= 24 * s.cu;
        if (s.wide) return p.M <= (off_lines(p) ? 4 : 24);
        if (p.N <= 16 * s.cu) return work <= std::max(130000, 60 * p.N);
        return p.M <= 8 || (p.M <= 24 && p.K >= 5000);
    }
    if (kind == kWeights8) {
        if (s.narrow) return work <= (p.M <= 16 ? 240000 : 170000);
        return p.M <= (s.wide ? 8 : s.brief ? 24 : 32);
    }
    if (s.narrow) return work <= 150000;
    return !s.brief && (p.M <= 16 || p.N <= 16 * s.cu);
}

// A work group: operands of 16 / G rows, FB of them for features and TB for rows of X, U steps on their way per wavefront.
struct FewForm {
    int G, FB, TB, U, wavefronts;
    constexpr bool operator==(const FewForm&) const = default;
};
inline constexpr FewForm kFew16[] = {{4, 4, 1, 1, 8}, {4, 2, 1, 2, 8}, {4, 2, 2, 2, 8}, {4, 2, 4, 2, 8}, {4, 2, 8, 1, 8}, {4, 3, 2, 2, 8}, {4, 4, 2, 2, 8}, {4, 3, 2, 2, 4},
                                     {4, 4, 2, 2, 4}, {2, 2, 2, 2, 8}, {2, 3, 2, 2, 4}, {2, 4, 2, 2, 4}, {2, 2, 3, 1, 8}, {2, 2, 4, 1, 8}, {2, 3, 3, 2, 4}, {2, 4, 3, 2, 4}};
inline constexpr FewForm kFewW8[] = {{4, 4, 1, 1, 8}, {4, 2, 1, 2, 8}, {4, 2, 2, 2, 8}, {4, 2, 4, 2, 8}, {4, 2, 8, 1, 4}, {4, 3, 2, 2, 8}, {4, 4, 2, 2, 8}, {4, 3, 2, 2, 4},
                                     {4, 4, 2, 2, 4}, {2, 2, 2, 2, 8}, {2, 3, 2, 2, 4}, {2, 4, 2, 2, 4}, {2, 2, 3, 1, 8}, {2, 2, 4, 1, 8}, {2, 3, 3, 2, 4}, {2, 4, 3, 2, 4},
                                     {2, 3, 4, 2, 4}, {2, 4, 4, 2, 4}};
inline constexpr FewForm kFewBoth8[] = {{4, 2, 1, 2, 8}, {4, 2, 2, 2, 8}, {4, 2, 4, 2, 8}, {4, 2, 8, 1, 8}, {4, 3, 2, 2, 8}, {4, 4, 2, 2, 8}, {4, 3, 2, 2, 4},
                                        {4, 4, 2, 2, 4}, {2, 2, 2, 2, 8}, {2, 3, 2, 2, 4}, {2, 4, 2, 2, 4}, {2, 2, 3, 1, 8}, {2, 2, 4, 1, 8}};
// The form of a problem that few_takes: one of the table of its kind
inline FewForm few_form(const LinearProblem& p, int n_cu) {
    const FewKind kind = few_kind(p);
    const FewShape s(p, kind, n_cu);
    if (p.M <= 4) return s.brief && kind != kBoth8 ? FewForm{4, 4, 1, 1, 8} : FewForm{4, 2, 1, 2, 8};
    if (s.narrow) {
        if (p.M <= 8) return {4, 2, 2, 2, 8};
        if (p.M <= 16) return {4, 2, 4, 2, 8};
        return {4, 2, 8, 1, kind == kWeights8 ? 4 : 8};
    }
    // Three or four blocks of R features, by which of them the busiest compute unit has less: 6144 features are 256 work groups of 24 or
    // 192 of 32 (us, three / four blocks, 6144 x 16384: 16-bit 16 rows 39.2 / 42.8, W8A16 20 rows 26.7 / 30.7, W8A8 16 rows 20.4 / 24.3).
    auto blocks = [&](int R) {
        auto share = [&](int n) { return (p.N + R * n * s.cu - 1) / (R * n * s.cu) * n; };
        return share(3) <= share(4) ? 3 : 4;
    };
    // four wavefronts with two steps on their way each where there are work groups enough, else eight (with one, where a step is many loads)
    const bool many = p.N > 16 * s.cu;
    if (p.M <= 8) return {4, blocks(4), 2, 2, many ? 4 : 8};
    if (!many) return p.M <= 16 ? FewForm{2, 2, 2, 2, 8} : FewForm{2, 2, p.M <= 24 ? 3 : 4, 1, 8};
    return {2, blocks(8), (p.M + 7) / 8, 2, 4};
}

}  // namespace gemm
}  // namespace mi
