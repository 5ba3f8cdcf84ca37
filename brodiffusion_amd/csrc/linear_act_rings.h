// The linear layer with an epilogue on operands of one kind, both of 16 bits (A = T) or both INT8 (A = Int8, in pairs): which instance of linear_pipe.h or
// linear_dma.h a launch takes. The forms and their rule are those of the layer without an epilogue and, for rows off 128-byte lines, kOff (linear_forms.h).
#pragma once
#include "linear_dma.h"
#include "linear_pipe.h"

namespace mi {
namespace gemm {
namespace {

template <typename T, typename A>
int launch_form(const LinearBatch& b, int form, hipStream_t st) {
    switch (form) {
        case k32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2, A, true>(b, 1, st);
        case k64x32: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2, A, true>(b, 1, st);
        case k64x64: return launch_pipe<T, false, false, 2, 2, 1, 1, 4, 4, A, true>(b, 1, st);
        case k64x96: return launch_pipe<T, false, false, 2, 3, 1, 1, 5, 4, A, true>(b, 1, st);
        case k128x64_load: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 4, A, true>(b, 1, st);
        case k128x96: return launch_pipe<T, false, false, 2, 3, 2, 1, 4, 4, A, true>(b, 1, st);
        case k128x64: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 0, A, true>(b, 1, st);
        case k128x128: return launch_pipe<T, false, false, 2, 2, 2, 2, 3, 4, A, true>(b, 1, st);
        case k128x128_2: return launch_pipe<T, false, false, 2, 2, 2, 2, 2, 0, A, true>(b, 1, st);
        case k192x128: return launch_pipe<T, false, false, 2, 4, 3, 1, 4, 0, A, true>(b, 1, st);
        case k256x128: return launch_pipe<T, false, false, 4, 2, 2, 2, 3, 0, A, true>(b, 1, st);
        default: return gemm_dma::launch_t<T, A, true>(b, 1, st);
    }
}
// ... in several parts (the forms of kSplitPlain)
template <typename T, typename A>
int launch_split(const LinearBatch& b, const ActLaunch& s, void* parts, hipStream_t st) {
    switch (s.form) {
        case k32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2, A, true, 16, true>(b, 1, st, s.splits, parts);
        case k64x64: return launch_pipe<T, false, false, 2, 2, 1, 1, 4, 4, A, true, 16, true>(b, 1, st, s.splits, parts);
        case k128x64_load: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 4, A, true, 16, true>(b, 1, st, s.splits, parts);
        default: return launch_pipe<T, false, false, 2, 2, 2, 2, 3, 4, A, true, 16, true>(b, 1, st, s.splits, parts);
    }
}
// ... of rows that do not begin on lines (kOff), in one part or, with memory for them, several
template <typename T, typename A, bool JOIN>
int launch_off(const LinearBatch& b, const ActLaunch& s, void* parts, hipStream_t st) {
    switch (s.form) {
        case kOff32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2, A, true, 16, JOIN>(b, 1, st, s.splits, parts);
        case kOff64x64_row: return launch_pipe<T, false, false, 2, 2, 1, 1, 5, 4, A, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
        case kOff128x64_row: return launch_pipe<T, false, false, 2, 2, 2, 1, 4, 4, A, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
        case kOff128x128_row: return launch_pipe<T, false, false, 2, 2, 2, 2, 4, 4, A, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
    }
    if constexpr (!JOIN) switch (s.form) {
        case kOff64x32: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2, A, true>(b, 1, st);
        case kOff64x32_row: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2, A, true, 16, false, true>(b, 1, st);
        case kOff64x96_row: return launch_pipe<T, false, false, 2, 3, 1, 1, 5, 4, A, true, 16, false, true>(b, 1, st);
        case kOff128x96_row: return launch_pipe<T, false, false, 2, 3, 2, 1, 4, 4, A, true, 16, false, true>(b, 1, st);
        case kOff192x128_row: return launch_pipe<T, false, false, 2, 4, 3, 1, 4, 0, A, true, 16, false, true>(b, 1, st);
        case kOff128x128_2: return launch_pipe<T, false, false, 2, 2, 2, 2, 2, 0, A, true>(b, 1, st);
        case kOff256x256: return gemm_dma::launch_t<T, A, true>(b, 1, st);
    }
    return fail("linear: no kernel for form %d", s.form);      // (not asked for)
}
template <typename T, typename A>
int launch_rings(const LinearProblem& p, const LinearScratch& lent, hipStream_t st) {
    LinearBatch b{};
    b.p[0] = p;
    const ActLaunch s = act_launch(p, lent.bytes, device_cu_count());
    if (s.splits > 1) return s.off ? launch_off<T, A, true>(b, s, lent.p, st) : launch_split<T, A>(b, s, lent.p, st);
    return s.off ? launch_off<T, A, false>(b, s, nullptr, st) : launch_form<T, A>(b, s.form, st);
}

}  // namespace
}  // namespace gemm
}  // namespace mi
