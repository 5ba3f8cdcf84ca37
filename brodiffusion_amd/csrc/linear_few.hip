// The linear layer with an epilogue for few rows (a token of a serving step, a draft, a short prompt).
//
// Bound: the bytes of W, each used once. There is nothing to share, so W goes from memory straight to the registers of the wavefront that
// multiplies it, as operand pieces, and so does X, which comes from the L2. A work group owns F features; its wavefronts take chunks of
// the contraction in turn, each with its next chunk on its way while it multiplies, and their sums meet in LDS, added in the order of the
// wavefronts: no result depends on timing. One launch, no workspace, no atomics.
//
// What costs next to those bytes is how a load's 64 lanes lie in memory. An operand of v_mfma_f32_16x16x32 wants 16 rows and four
// pieces of 8 contraction elements, row = lane % 16: as a load that is 64 lanes of which no two neighbours touch, and one such load of 1 KB
// kept a compute unit's memory path for 56 clocks, whatever rows it was of (measured: time goes with the number of loads, 1152 features
// x 4608 10 us at 16 rows, 22 at 64). So an operand here holds 16 / G rows and G groups of pieces, the groups as neighbouring lanes: G 16 bytes
// in a run. Row (r, h) of W meets column (t, h') of X, and of the 16 x 16 results those with h = h' are wanted, G partial sums of each
// of 16 / G x 16 / G results; the others are waste, and the matrix pipes have it to spare: at G = 4 and 16 rows they take 64 bytes of
// W per clock and compute unit, memory brings 10. (us, G = 1 / 4, bf16, 1152 x 4608: 1 row 7.0 / 3.9, 16 rows 10.0 / 5.3, 32 rows 13.9 / 7.3.)
// Weights of 100 MB (INT8, 6144 x 16384), one token: 18.5 to 19.9 us = 5.1 to 5.4 TB/s, what a large copy reaches here.
#include <algorithm>
#include <type_traits>

#include "linear_forms.h"
#include "linear_math.h"

namespace mi {
namespace gemm {
namespace {

enum { kSixteen, kWeights8, kBoth8 };      // operands of 16 bits, INT8 weights, both INT8 (then K and strides in pairs of elements)

// a 16-byte piece of a row whose rows are 8-byte aligned (INT8 weights of a contraction that is no multiple of 16)
typedef unsigned u32x4_a8 __attribute__((ext_vector_type(4), aligned(8)));

template <typename T, int KIND, int G, int FB, int TB, int U, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) linear_few_kernel(const LinearProblem p) {
    using M = Mma<std::conditional_t<KIND == kBoth8, Int8, T>>;
    using V8 = typename M::v8;
    using Sum = typename M::sum4;
    using Scalar = std::conditional_t<KIND == kBoth8, int, float>;
    constexpr int R = 16 / G;                                // rows of an operand
    constexpr int XP = KIND == kWeights8 ? 2 : 1;            // pieces of X that go with one of W
    constexpr int PIECE = 8 * XP;                            // contraction elements of a piece of W
    constexpr int STEP = 4 * G * PIECE;                      // ... of a step
    constexpr int WB = KIND == kWeights8 ? 1 : 2;            // bytes of an element of W
    constexpr int F = R * FB, NT = 64 * WAVES;               // features of the work group, threads
    constexpr int OUT = (F * R * TB + NT - 1) / NT;          // results per thread
    __shared__ __attribute__((aligned(16))) Scalar sums[WAVES][FB * TB][G * R * R];   // [group][column][row] of the G squares of a block

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = static_cast<int>(blockIdx.x) * F;

    // What the epilogue needs, requested ahead of everything: result i of a thread is number i NT + tid, features running fastest.
    float bias[OUT], res[OUT], scale[OUT], xs[KIND == kBoth8 ? OUT : 1];
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
        const int o = i * NT + tid, feat = n0 + o % F, row = o / F;
        bias[i] = res[i] = 0.f;
        scale[i] = 1.f;
        if constexpr (KIND == kBoth8) xs[i] = 1.f;
        if (row < p.M && feat < p.N) {
            if (p.bias) bias[i] = static_cast<float>(static_cast<const T*>(p.bias)[feat]);
            if (p.residual) res[i] = static_cast<float>(static_cast<const T*>(p.residual)[static_cast<long>(row) * p.ldr + feat]);
            if constexpr (KIND != kSixteen) scale[i] = p.w_scale[feat];
            if constexpr (KIND == kBoth8) xs[i] = p.x_scale[row];
        }
    }

    // this lane's piece of a step, and its rows of either operand
    const int piece = lg * G + lr % G;
    const unsigned char* wrow[FB];
    const unsigned char* xrow[TB];
#pragma unroll
    for (int a = 0; a < FB; ++a) wrow[a] = static_cast<const unsigned char*>(p.w) + static_cast<long>(min(n0 + R * a + lr / G, p.N - 1)) * p.ldw * WB + piece * PIECE * WB;
#pragma unroll
    for (int b = 0; b < TB; ++b) xrow[b] = static_cast<const unsigned char*>(p.x) + static_cast<long>(min(R * b + lr / G, p.M - 1)) * p.ldx * 2 + piece * PIECE * 2;

    Sum acc[FB][TB];
#pragma unroll
    for (int a = 0; a < FB; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = Sum{0, 0, 0, 0};

    struct Chunk { u32x4 w[U][FB]; V8 x[U][TB * XP]; };
    auto load = [&](Chunk& c, int step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long at = static_cast<long>(step + u) * STEP;
#pragma unroll
            for (int a = 0; a < FB; ++a) c.w[u][a] = *reinterpret_cast<const u32x4_a8*>(wrow[a] + at * WB);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long at = static_cast<long>(step + u) * STEP;
#pragma unroll
            for (int b = 0; b < TB; ++b)
#pragma unroll
                for (int j = 0; j < XP; ++j) c.x[u][b * XP + j] = *reinterpret_cast<const V8*>(xrow[b] + at * 2 + j * 16);
        }
    };
    auto products = [&](u32x4 w, const V8* x, Sum (&sum)[TB]) {
        if constexpr (KIND == kWeights8) {
            const V8 lo = widen<T>(u32x2{w[0], w[1]}), hi = widen<T>(u32x2{w[2], w[3]});
#pragma unroll
            for (int b = 0; b < TB; ++b) sum[b] = M::run16(hi, x[2 * b + 1], M::run16(lo, x[2 * b], sum[b]));
        } else {
#pragma unroll
            for (int b = 0; b < TB; ++b) sum[b] = M::run16(__builtin_bit_cast(V8, w), x[b], sum[b]);
        }
    };
    auto multiply = [&](const Chunk& c) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < FB; ++a) products(c.w[u][a], c.x[u], acc[a]);
    };

    const int whole = p.K / (STEP * U);                      // chunks
    if (wave < whole) {
        Chunk c[2];
        load(c[0], wave * U);
        int i = wave;
        for (; i + WAVES < whole; i += 2 * WAVES) {
            load(c[1], (i + WAVES) * U);
            multiply(c[0]);
            if (i + 2 * WAVES < whole) load(c[0], (i + 2 * WAVES) * U);
            multiply(c[1]);
        }
        if (i < whole) multiply(c[0]);
    }
    // the steps behind the whole chunks, one per wavefront at a time; pieces past the end count as zeros (of INT8 weights: halves of pieces)
    for (int s = whole * U + wave; s * STEP < p.K; s += WAVES) {
        const int left = p.K - s * STEP - piece * PIECE;     // elements from this lane's first on
        const bool there = left > 0, there2 = left > 8;
        const long at = there ? static_cast<long>(s) * STEP : -static_cast<long>(piece) * PIECE;      // (else the row's first piece, blanked)
        V8 x[TB * XP];
#pragma unroll
        for (int b = 0; b < TB; ++b)
#pragma unroll
            for (int j = 0; j < XP; ++j) {
                const bool ok = j == 0 ? there : there2;
                const V8 v = *reinterpret_cast<const V8*>(xrow[b] + (ok ? at * 2 + j * 16 : at * 2));
                x[b * XP + j] = ok ? v : V8{};
            }
#pragma unroll
        for (int a = 0; a < FB; ++a) {
            u32x4 w = {0u, 0u, 0u, 0u};
            if constexpr (KIND == kWeights8) {
                const u32x2 lo = *reinterpret_cast<const u32x2*>(wrow[a] + at), hi = *reinterpret_cast<const u32x2*>(wrow[a] + (there2 ? at + 8 : at));
                if (there) { w[0] = lo[0]; w[1] = lo[1]; }
                if (there2) { w[2] = hi[0]; w[3] = hi[1]; }
            } else {
                const u32x4 v = *reinterpret_cast<const u32x4*>(wrow[a] + at * WB);
                if (there) w = v;
            }
            products(w, x, acc[a]);
        }
    }

#pragma unroll
    for (int a = 0; a < FB; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            // rows 4 lg + e of column lr: those of the column's group are valid
            Scalar* const to = &sums[wave][a * TB + b][((lr % G) * R + lr / G) * R];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((4 * lg + e) % G == lr % G) to[(4 * lg + e) / G] = acc[a][b][e];
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
        const int o = i * NT + tid, f = o % F, row = o / F;
        if (row >= p.M || n0 + f >= p.N) continue;
        Scalar total = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int h = 0; h < G; ++h) total += sums[w][f / R * TB + row / R][(h * R + row % R) * R + f % R];
        const float sum = static_cast<float>(total);
        float v;
        if constexpr (KIND == kSixteen) v = sum + bias[i];
        else if constexpr (KIND == kWeights8) v = scaled_acc(sum, scale[i], bias[i]);
        else v = scaled_acc(sum * scale[i], xs[i], bias[i]);
        with_activation(p.act, [&](auto act) { v = act(v); });
        static_cast<T*>(p.y)[static_cast<long>(row) * p.ldy + n0 + f] = static_cast<T>(v + res[i]);
    }
}

template <typename T, int KIND, int G, int FB, int TB, int U, int WAVES>
int launch(const LinearProblem& p, hipStream_t st) {
    constexpr int F = 16 / G * FB;
    hipLaunchKernelGGL((linear_few_kernel<T, KIND, G, FB, TB, U, WAVES>), dim3((p.N + F - 1) / F), dim3(64 * WAVES), 0, st, p);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

// How a problem stands to the GPU. narrow: up to 8 features per compute unit, so that work groups of 8 features are what there is to spread;
// wide: over 32; brief: not narrow, with a contraction of at most 4 KB of W's row, of which a wavefront gets a step or two.
struct Shape {
    int cu;
    bool narrow, wide, brief;
    Shape(const LinearProblem& p, int kind) {
        cu = device_cu_count();
        narrow = p.N <= 8 * cu;
        wide = p.N > 32 * cu;
        brief = !narrow && p.K * (kind == kWeights8 ? 1L : 2L) <= 4096;
    }
};
int kind_of(const LinearProblem& p) { return p.x_scale ? kBoth8 : p.w_scale ? kWeights8 : kSixteen; }

// Three or four blocks of R features per work group, by which of them the busiest compute unit has less: 6144 features are 256 work groups of 24 or
// 192 of 32 (us, three / four blocks, 6144 x 16384: 16-bit 16 rows 39.2 / 42.8, W8A16 20 rows 26.7 / 30.7, W8A8 16 rows 20.4 / 24.3).
template <int R> bool three_blocks(const LinearProblem& p, int cu) {
    auto share = [&](int blocks) { return (p.N + R * blocks * cu - 1) / (R * blocks * cu) * blocks; };
    return share(3) <= share(4);
}

template <typename T, int KIND>
int launch_rows(const LinearProblem& p, hipStream_t st) {
    const Shape s(p, KIND);
    // four wavefronts with two steps on their way each where there are work groups enough, else eight (with one, where a step is many loads)
    const bool many = p.N > 16 * s.cu;
    if (p.M <= 4) {
        if constexpr (KIND != kBoth8) if (s.brief) return launch<T, KIND, 4, 4, 1, 1, 8>(p, st);
        return launch<T, KIND, 4, 2, 1, 2, 8>(p, st);
    }
    if (s.narrow) {
        if (p.M <= 8) return launch<T, KIND, 4, 2, 2, 2, 8>(p, st);
        if (p.M <= 16) return launch<T, KIND, 4, 2, 4, 2, 8>(p, st);
        return launch<T, KIND, 4, 2, 8, 1, KIND == kWeights8 ? 4 : 8>(p, st);
    }
    if (p.M <= 8) {
        if (!many) return three_blocks<4>(p, s.cu) ? launch<T, KIND, 4, 3, 2, 2, 8>(p, st) : launch<T, KIND, 4, 4, 2, 2, 8>(p, st);
        return three_blocks<4>(p, s.cu) ? launch<T, KIND, 4, 3, 2, 2, 4>(p, st) : launch<T, KIND, 4, 4, 2, 2, 4>(p, st);
    }
    if (p.M <= 16) {
        if (!many) return launch<T, KIND, 2, 2, 2, 2, 8>(p, st);
        return three_blocks<8>(p, s.cu) ? launch<T, KIND, 2, 3, 2, 2, 4>(p, st) : launch<T, KIND, 2, 4, 2, 2, 4>(p, st);
    }
    if (!many) return p.M <= 24 ? launch<T, KIND, 2, 2, 3, 1, 8>(p, st) : launch<T, KIND, 2, 2, 4, 1, 8>(p, st);
    if constexpr (KIND != kBoth8) {
        if (p.M <= 24) return three_blocks<8>(p, s.cu) ? launch<T, KIND, 2, 3, 3, 2, 4>(p, st) : launch<T, KIND, 2, 4, 3, 2, 4>(p, st);
    }
    if constexpr (KIND == kWeights8) {
        return three_blocks<8>(p, s.cu) ? launch<T, KIND, 2, 3, 4, 2, 4>(p, st) : launch<T, KIND, 2, 4, 4, 2, 4>(p, st);
    }
    return fail("linear: no kernel for %d rows", p.M);      // (linear_few_takes leaves these to others)
}

template <typename T>
int launch_kind(const LinearProblem& p, hipStream_t st) {
    switch (kind_of(p)) {
        case kBoth8: return launch_rows<T, kBoth8>(p, st);
        case kWeights8: return launch_rows<T, kWeights8>(p, st);
        default: return launch_rows<T, kSixteen>(p, st);
    }
}

}  // namespace
}  // namespace gemm

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
bool linear_few_takes(const LinearProblem& p) {
    const int kind = gemm::kind_of(p);
    const gemm::Shape s(p, kind);
    if (p.M > 32) return false;
    const long work = static_cast<long>(p.M) * p.K;
    if (kind == gemm::kSixteen) {
        if (s.brief) return p.M <= 4 && p.N <= 24 * s.cu;
        if (s.wide) return p.M <= (gemm::off_lines(p) ? 4 : 24);
        if (p.N <= 16 * s.cu) return work <= std::max(130000, 60 * p.N);
        return p.M <= 8 || (p.M <= 24 && p.K >= 5000);
    }
    if (kind == gemm::kWeights8) {
        if (s.narrow) return work <= (p.M <= 16 ? 240000 : 170000);
        return p.M <= (s.wide ? 8 : s.brief ? 24 : 32);
    }
    if (s.narrow) return work <= 150000;
    return !s.brief && (p.M <= 16 || p.N <= 16 * s.cu);
}

int launch_linear_few(const LinearProblem& p, int dtype, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_kind<__bf16>(p, st) : gemm::launch_kind<_Float16>(p, st);
}

}  // namespace mi
