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
// W per clock and compute unit, memory brings 10. (us, G = 1 / 4, bf16, 1152 x 4608 in the last-level
// cache: 1 row 7.0 / 3.9, 16 rows 10.0 / 5.3, 32 rows 13.9 / 7.3.)
// Weights of 100 MB (INT8, 6144 x 16384), several in turn, one token: 18.5 to 19.9 us = 5.1 to 5.4 TB/s, what a large copy reaches here.
// Which problems come here and with which work groups: linear_few_forms.h.
#include <iterator>
#include <type_traits>
#include <utility>

#include "linear_few_forms.h"
#include "linear_math.h"

namespace mi {
namespace gemm {
namespace {

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

// the instance of a form: one of the N of the table FORMS
template <typename T, int KIND, const auto& FORMS, int... I>
int launch_form(const LinearProblem& p, const FewForm& form, std::integer_sequence<int, I...>, hipStream_t st) {
    int rc = 1;
    (void)((form == FORMS[I] ? (rc = launch<T, KIND, FORMS[I].G, FORMS[I].FB, FORMS[I].TB, FORMS[I].U, FORMS[I].wavefronts>(p, st), true) : false) || ...);
    return rc <= 0 ? rc : fail("linear: no kernel for %d rows", p.M);
}
template <typename T, int KIND, const auto& FORMS>
int launch_table(const LinearProblem& p, hipStream_t st) {
    return launch_form<T, KIND, FORMS>(p, few_form(p, device_cu_count()), std::make_integer_sequence<int, std::size(FORMS)>{}, st);
}

template <typename T>
int launch_kind(const LinearProblem& p, hipStream_t st) {
    switch (few_kind(p)) {
        case kBoth8: return launch_table<T, kBoth8, kFewBoth8>(p, st);
        case kWeights8: return launch_table<T, kWeights8, kFewW8>(p, st);
        default: return launch_table<T, kSixteen, kFew16>(p, st);
    }
}

}  // namespace
}  // namespace gemm

bool linear_few_takes(const LinearProblem& p) { return gemm::few_takes(p, device_cu_count()); }

int launch_linear_few(const LinearProblem& p, int dtype, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_kind<__bf16>(p, st) : gemm::launch_kind<_Float16>(p, st);
}

}  // namespace mi
