// Which tile a projection takes: the forms of linear_pipe.h (and the 256 x 256 tiles of linear_dma.h) with what a launch on each is
// expected to cost. Host code without HIP in it, so that a test can ask which form a problem gets.
#pragma once
#include <algorithm>

#include "internal.h"

namespace mi {
namespace gemm {

// ── which form a launch takes ──
// A launch of n tiles on a GPU of C compute units costs about
//     phi + steps lam + (m - 1) (steps tau + eps),   m = ceil(n / C) tiles on the busiest compute unit,
// with steps = K / 64: phi what a launch of one tile per compute unit costs beyond its steps (start, first loads, write-out), lam
// a step when the compute unit has one tile, tau and eps a step and the rest of every further tile. The constants (us) are fitted
// on MI355X to 350 problems (32 to 16384 rows, eleven layers of the supported models, one or three of a launch; 16-bit: jointly with a
// term for the bytes of the operands, the same for every form), with all products v_mfma_f32_32x32x16. As built now steps of the large
// tiles are 6 to 12 % shorter and the others much as they were, and the constants still rank the forms: every form timed on 452 such
// problems (profiles/linear_form_times.txt), the form taken is 0.7 (INT8 0.5 to 0.8, GEGLU 1.2 to 1.7, GEGLU of INT8 0.6 to 0.7) % slower
// than the fastest one on average, where the same form timed twice differs by 0.8 %; at worst 16 % (GEGLU 6144 x 640 -> 2 x 2560 56.5 us on
// 192 x 128 tiles, 48.5 on 128 x 64). Large tiles
// need fewer bytes per FLOP: a compute unit takes 1 KB from its L2 in 16 to 24 clocks, so a step of 128 x 128 (32 KB) took 600 to 700 where its products take 512, one of 128 x 64 (24 KB) 450 to 650 where they take
// 256 (with products of 32 x 32 x 16). Small ones fill the GPU: 128 x 1280 x 1280 takes 4.8 us with 160 tiles of 32 x 32, 5.1 with 80 of 64 x 32, 7.0 with 20 of
// 128 x 64; 1024 x 2240 x 2240 takes 15.6 us with 192 tiles of 128 x 96, 23 with 280 of 128 x 64, 46 with 36 of 256 x 256.
// The tiles 96 features wide and the GEGLU tile of 192 x 128 (constants set by hand from 17 problems of their own) are for
// the counts between (us, best other form / theirs, profiles/linear_form_times.txt): 1024 x 2240 x 2240 16.8 / 15.6 on
// 192 tiles of 128 x 96, 2048 x 1152 x 1152 10.5 / 9.9, 2048 x 640 x 2560 15.0 / 13.2 on 224 of 64 x 96; GEGLU 2048 x 640 ->
// 2 x 2560 21.6 / 21.1 and 1024 x 1280 -> 2 x 5120 35.5 / 33.8 (INT8 22.9 / 21.3, 38.2 / 33.1) on 220 and 240 of 192 x 128; INT8
// 1024 x 1280 x 1280 8.7 (128 x 64) / 8.8, 4096 x 640 x 640 8.4 / 7.8. Wavefronts that own 128 x 64
// or 96 x 64 instead of 64 x 64 (a quarter fewer LDS reads) gave nothing with products of 32 x 32 x 16: 1024 x 6720 x 2240 32.8 -> 32.9.
// Loading wavefronts (see the top) pay where the products of a step are short. They are no help where a compute unit holds two work
// groups of large register use (products of 32 x 32 x 16): GEGLU 3072 x 640 -> 2 x 2560 29 -> 37 us, three of 16384 x 512 x 512 37 -> 42.
struct Form {
    int bm, bn_out;
    float phi, lam, tau, eps;
};
enum { k32x32, k64x32, k64x64, k64x96, k128x64_load, k128x64, k128x96, k128x128, k128x128_2, k192x128, k256x128, k256x256, kPlainForms };
inline constexpr Form kPlain[kPlainForms] = {{32, 32, 2.46f, 0.091f, 0.058f, 0.22f},   {64, 32, 2.60f, 0.111f, 0.126f, 0.34f},   {64, 64, 2.52f, 0.154f, 0.190f, 0.42f},
                                      {64, 96, 3.10f, 0.225f, 0.240f, 1.50f},   {128, 64, 2.53f, 0.250f, 0.322f, 0.76f},  {128, 64, 2.57f, 0.274f, 0.322f, 0.59f},
                                      {128, 96, 3.50f, 0.318f, 0.360f, 2.30f},  {128, 128, 3.95f, 0.356f, 0.529f, 3.18f}, {128, 128, 3.19f, 0.515f, 0.465f, 1.20f},
                                      {192, 128, 4.67f, 0.511f, 0.727f, 4.11f}, {256, 128, 5.03f, 0.656f, 0.839f, 6.17f}, {256, 256, 8.05f, 1.379f, 1.789f, 6.40f}};
// INT8 weights: the widening makes small steps dearer and the large tiles no better (those above 128 x 128 are not built)
enum { k8_32x32, k8_64x64, k8_64x96, k8_128x64, k8_128x96, k8_128x128, k8_128x128_2, kPlainW8Forms };
inline constexpr Form kPlainW8[kPlainW8Forms] = {{32, 32, 2.47f, 0.155f, 0.049f, 0.33f},
                                          {64, 64, 2.75f, 0.209f, 0.187f, 0.80f},
                                          {64, 96, 3.30f, 0.245f, 0.235f, 0.90f},
                                          {128, 64, 3.03f, 0.325f, 0.286f, 1.43f},
                                          {128, 96, 4.00f, 0.350f, 0.360f, 1.50f},
                                          {128, 128, 4.03f, 0.420f, 0.562f, 3.98f},
                                          {128, 128, 2.89f, 0.658f, 0.382f, 3.13f}};
enum { kG64x64, kG128x64_2, kG128x64, kG256x64, kG192x128, kGegluForms };   // output features; the W tile holds twice as many rows
inline constexpr Form kGeglu[kGegluForms] = {{64, 64, 2.65f, 0.377f, 0.330f, 1.20f}, {128, 64, 3.66f, 0.648f, 0.496f, 2.09f}, {128, 64, 4.41f, 0.442f, 0.588f, 4.08f},
                                      {256, 64, 5.99f, 0.800f, 0.834f, 8.98f}, {192, 128, 7.00f, 1.200f, 1.250f, 7.00f}};
enum { kG8_64x64, kG8_128x64_2, kG8_256x64, kG8_192x128, kGegluW8Forms };
inline constexpr Form kGegluW8[kGegluW8Forms] = {{64, 64, 3.92f, 0.315f, 0.302f, 1.17f}, {128, 64, 3.92f, 0.653f, 0.429f, 2.93f}, {256, 64, 7.90f, 0.816f, 1.031f, 6.53f},
                                          {192, 128, 9.30f, 1.290f, 1.500f, 5.50f}};

// 256 x 256 tiles take contractions from 512 on (below, their prologue is most of the launch).
inline int pick_form(const Form* forms, int n_forms, const LinearBatch& batch, int n_problems, int n_cu) {
    int best = 0;
    double best_cost = 1e30;
    for (int f = 0; f < n_forms; ++f) {
        long tiles = 0;
        int k = 0;
        for (int i = 0; i < n_problems; ++i) {
            const LinearProblem& p = batch.p[i];
            tiles += static_cast<long>((p.M + forms[f].bm - 1) / forms[f].bm) * ((p.N + forms[f].bn_out - 1) / forms[f].bn_out);
            k = std::max(k, p.K);
        }
        if (forms[f].bn_out == 256 && k < 512) continue;
        const double steps = k / 64, m = static_cast<double>((tiles + n_cu - 1) / n_cu);
        const double cost = forms[f].phi + steps * forms[f].lam + (m - 1) * (steps * forms[f].tau + forms[f].eps);
        if (cost < best_cost) { best_cost = cost; best = f; }
    }
    return best;
}

// The form of a launch: an index into the table of its kind.
inline int pick_form(const LinearBatch& batch, int n_problems, bool geglu, int n_cu) {
    if (batch.p[0].w_scale != nullptr)
        return geglu ? pick_form(kGegluW8, kGegluW8Forms, batch, n_problems, n_cu) : pick_form(kPlainW8, kPlainW8Forms, batch, n_problems, n_cu);
    return geglu ? pick_form(kGeglu, kGegluForms, batch, n_problems, n_cu) : pick_form(kPlain, kPlainForms, batch, n_problems, n_cu);
}

// ── the layer with an epilogue, rows that do not begin on 128-byte lines ──
// The tiles that load by lines (linear_pipe.h, OFF; here _row) and, where a launch is short or very large, some that do not. Constants fitted to 216
// such problems of 16-bit operands (33 to 4608 rows, contractions of 328 to 15976 elements, fp16) and 336 of INT8 weights, with launches of one
// form for 10 ms, as the power limit moves the large ones: the form taken is 0.4 (INT8 weights: 1.7) % slower than the fastest of 13 (18) on
// average, 13 (23) % at worst. Against the forms and constants of rows on lines 0.89 (0.98) of the time.
enum { kOff32x32, kOff64x32, kOff128x128_2, kOff256x256, kOff64x32_row, kOff64x64_row, kOff64x96_row, kOff128x64_row, kOff128x96_row, kOff128x128_row, kOff192x128_row, kOffForms };
inline constexpr Form kOff[kOffForms] = {{32, 32, 3.09f, 0.108f, 0.097f, 0.46f},   {64, 32, 3.07f, 0.154f, 0.149f, 0.80f},   {128, 128, 6.25f, 0.494f, 0.622f, 1.07f},
                                         {256, 256, 13.89f, 1.368f, 1.751f, 11.05f}, {64, 32, 3.70f, 0.140f, 0.123f, 0.88f}, {64, 64, 4.02f, 0.161f, 0.175f, 0.89f},
                                         {64, 96, 4.49f, 0.206f, 0.242f, 3.05f},   {128, 64, 4.70f, 0.268f, 0.322f, 3.01f},  {128, 96, 6.21f, 0.314f, 0.400f, 4.20f},
                                         {128, 128, 6.77f, 0.360f, 0.484f, 4.72f}, {192, 128, 7.53f, 0.511f, 0.694f, 5.33f}};
enum { kOff8_32x32, kOff8_64x64, kOff8_64x96, kOff8_128x96, kOff8_128x64_row, kOff8_128x96_row, kOff8_128x128_2_row, kOff8_128x128_row, kOff8Forms };
inline constexpr Form kOff8[kOff8Forms] = {{32, 32, 3.05f, 0.166f, 0.058f, 0.62f},  {64, 64, 3.80f, 0.215f, 0.208f, 0.93f},  {64, 96, 4.34f, 0.260f, 0.299f, 1.36f},   {128, 96, 5.37f, 0.388f, 0.444f, 2.10f},
                                           {128, 64, 5.38f, 0.263f, 0.261f, 1.93f}, {128, 96, 6.74f, 0.349f, 0.409f, 5.10f}, {128, 128, 6.50f, 0.611f, 0.407f, 3.38f}, {128, 128, 6.72f, 0.442f, 0.517f, 5.50f}};
// (INT8 weights: lines of 64 bytes of them; and the last row ends where a piece does, as pieces are loaded whole)
inline bool off_lines(const LinearProblem& p) {
    const auto x = reinterpret_cast<uintptr_t>(p.x) | static_cast<uintptr_t>(p.ldx * 2), w = reinterpret_cast<uintptr_t>(p.w);
    if (p.w_scale && !p.x_scale) return ((x & 127) || ((w | static_cast<uintptr_t>(p.ldw)) & 63)) && (p.ldw - p.K) % 16 == 0;
    return ((x | w | static_cast<uintptr_t>(p.ldw * 2)) & 127) != 0;
}

// ── several work groups for a tile's contraction (the layer with an epilogue, where the caller lends memory for their sums) ──
// Parts leave FP32 or INT32 sums, a second launch adds them and finishes the layer: 2 us and the bytes of the parts, written and read at
// 5 TB/s. Paid where few tiles have a long contraction (us, one part / several; rows x features x contraction): 46 x 368 x 15984 29.5 / 8.2
// (8 parts of 32 x 32 tiles), 224 x 1320 x 16320 35.3 / 22.3, with INT8 weights 55.4 / 21.4; not for 40 x 320 x 1280 5.7 / 6.4 or 1031 x 1152 x 4608
// 19.8 / 22.0. Over 150 problems of 16-bit rows off lines, each in every form and number of parts, what the rule takes is 1.1 % slower than the
// fastest on average (one part: 22 %), over 130 of INT8 weights 1.9 %. Over 280 others of 33 to 1500 rows that it gives parts the time was 0.71 (16-bit),
// 0.52 (W8A16) and 0.78 (W8A8) of one part's on average, at worst 1.14 (96 x 10144 x 6016 26.9 -> 30.5).
struct Parts { int form, splits; };
inline constexpr int kSplitPlain[] = {k32x32, k64x64, k128x64_load, k128x128};
inline constexpr int kSplitW8[] = {k8_32x32, k8_64x64, k8_128x64, k8_128x96};
inline constexpr int kSplitOff[] = {kOff32x32, kOff64x64_row, kOff128x64_row, kOff128x128_row};
inline constexpr int kSplitOff8[] = {kOff8_32x32, kOff8_64x64, kOff8_128x64_row, kOff8_128x96_row};
// The forms of a problem of the layer with an epilogue, and those with parts
struct FormTable { const Form* forms; int n; const int* split; };
inline constexpr FormTable kTables[] = {{kPlain, kPlainForms, kSplitPlain}, {kOff, kOffForms, kSplitOff}, {kPlainW8, kPlainW8Forms, kSplitW8}, {kOff8, kOff8Forms, kSplitOff8}};
inline const FormTable& table_of(const LinearProblem& p) { return kTables[(p.w_scale && !p.x_scale ? 2 : 0) + (off_lines(p) ? 1 : 0)]; }
inline long tiles_of(const Form& f, const LinearProblem& p) { return static_cast<long>((p.M + f.bm - 1) / f.bm) * ((p.N + f.bn_out - 1) / f.bn_out); }
inline long part_bytes(const Form& f, const LinearProblem& p, int splits) { return tiles_of(f, p) * splits * f.bm * f.bn_out * 4; }
inline Parts pick_parts(const LinearProblem& p, int n_cu) {
    const FormTable& table = table_of(p);
    const double steps = p.K / 64;
    auto cost = [&](const Form& f, int splits) {
        const double m = static_cast<double>((tiles_of(f, p) * splits + n_cu - 1) / n_cu), s = steps / splits;
        return f.phi + s * f.lam + (m - 1) * (s * f.tau + f.eps) + (splits > 1 ? 2.0 + 2.0 * part_bytes(f, p, splits) / 5e6 : 0.0);
    };
    LinearBatch b{};
    b.p[0] = p;
    const int whole = pick_form(table.forms, table.n, b, 1, n_cu);
    Parts best{whole, 1};
    double best_cost = 0.97 * cost(table.forms[whole], 1);
    for (int i = 0; i < 4; ++i)
        for (int splits : {2, 3, 4, 6, 8, 12, 16}) {
            // (at most two work groups per compute unit: with more, small tiles of large weights, what bounds a launch is the memory, which the
            //  costs leave out: 16 x 16384 x 6144 W8A16 24.5 us in one part, 33.9 in 3 of 32 x 32 tiles)
            if (splits * 4 > p.K / 64 || tiles_of(table.forms[table.split[i]], p) * splits > 2 * n_cu) break;
            if (const double c = cost(table.forms[table.split[i]], splits); c < best_cost) { best_cost = c; best = {table.split[i], splits}; }
        }
    return best;
}
// What a call is launched as: in parts where the caller lent the memory for them
struct ActLaunch { int form, splits; bool off; };
inline ActLaunch act_launch(const LinearProblem& p, size_t lent_bytes, int n_cu) {
    const FormTable& table = table_of(p);
    const Parts s = pick_parts(p, n_cu);
    const bool off = off_lines(p);
    if (s.splits == 1 || lent_bytes >= static_cast<size_t>(part_bytes(table.forms[s.form], p, s.splits))) return {s.form, s.splits, off};
    LinearBatch b{};
    b.p[0] = p;
    return {pick_form(table.forms, table.n, b, 1, n_cu), 1, off};
}

}  // namespace gemm
}  // namespace mi
