// The linear layer with an epilogue, INT8 operands (W8A8): which instance of linear_pipe.h or linear_dma.h a launch takes (the forms and their
// rule are those of the layer without one, linear_forms.h).
#include "linear_dma.h"
#include "linear_pipe.h"

namespace mi {
namespace gemm {
namespace {

template <typename T>
int launch_form(const LinearBatch& b, int form, hipStream_t st) {
    switch (form) {
        case k32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2, Int8, true>(b, 1, st);
        case k64x32: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2, Int8, true>(b, 1, st);
        case k64x64: return launch_pipe<T, false, false, 2, 2, 1, 1, 4, 4, Int8, true>(b, 1, st);
        case k64x96: return launch_pipe<T, false, false, 2, 3, 1, 1, 5, 4, Int8, true>(b, 1, st);
        case k128x64_load: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 4, Int8, true>(b, 1, st);
        case k128x96: return launch_pipe<T, false, false, 2, 3, 2, 1, 4, 4, Int8, true>(b, 1, st);
        case k128x64: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 0, Int8, true>(b, 1, st);
        case k128x128: return launch_pipe<T, false, false, 2, 2, 2, 2, 3, 4, Int8, true>(b, 1, st);
        case k128x128_2: return launch_pipe<T, false, false, 2, 2, 2, 2, 2, 0, Int8, true>(b, 1, st);
        case k192x128: return launch_pipe<T, false, false, 2, 4, 3, 1, 4, 0, Int8, true>(b, 1, st);
        case k256x128: return launch_pipe<T, false, false, 4, 2, 2, 2, 3, 0, Int8, true>(b, 1, st);
        default: return gemm_dma::launch_t<T, gemm::Int8, true>(b, 1, st);
    }
}
// ... in several parts (the forms of kSplitPlain)
template <typename T>
int launch_split(const LinearBatch& b, Parts s, void* parts, hipStream_t st) {
    switch (s.form) {
        case k32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2, Int8, true, 16, true>(b, 1, st, s.splits, parts);
        case k64x64: return launch_pipe<T, false, false, 2, 2, 1, 1, 4, 4, Int8, true, 16, true>(b, 1, st, s.splits, parts);
        case k128x64_load: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 4, Int8, true, 16, true>(b, 1, st, s.splits, parts);
        default: return launch_pipe<T, false, false, 2, 2, 2, 2, 3, 4, Int8, true, 16, true>(b, 1, st, s.splits, parts);
    }
}
// ... of rows that do not begin on lines (kOff), in one part or, with memory for them, several
template <typename T, bool JOIN>
int launch_off(const LinearBatch& b, Parts s, void* parts, hipStream_t st) {
    switch (s.form) {
        case kOff32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2, Int8, true, 16, JOIN>(b, 1, st, s.splits, parts);
        case kOff64x64_row: return launch_pipe<T, false, false, 2, 2, 1, 1, 5, 4, Int8, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
        case kOff128x64_row: return launch_pipe<T, false, false, 2, 2, 2, 1, 4, 4, Int8, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
        case kOff128x128_row: return launch_pipe<T, false, false, 2, 2, 2, 2, 4, 4, Int8, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
    }
    if constexpr (!JOIN) switch (s.form) {
        case kOff64x32: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2, Int8, true>(b, 1, st);
        case kOff64x32_row: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2, Int8, true, 16, false, true>(b, 1, st);
        case kOff64x96_row: return launch_pipe<T, false, false, 2, 3, 1, 1, 5, 4, Int8, true, 16, false, true>(b, 1, st);
        case kOff128x96_row: return launch_pipe<T, false, false, 2, 3, 2, 1, 4, 4, Int8, true, 16, false, true>(b, 1, st);
        case kOff192x128_row: return launch_pipe<T, false, false, 2, 4, 3, 1, 4, 0, Int8, true, 16, false, true>(b, 1, st);
        case kOff128x128_2: return launch_pipe<T, false, false, 2, 2, 2, 2, 2, 0, Int8, true>(b, 1, st);
        case kOff256x256: return gemm_dma::launch_t<T, gemm::Int8, true>(b, 1, st);
    }
    return fail("linear: no kernel for form %d", s.form);      // (not asked for)
}
template <typename T>
int launch_any(const LinearBatch& b, const LinearScratch& lent, hipStream_t st) {
    const LinearProblem& p = b.p[0];
    const FormTable& table = table_of(p);
    const bool off = off_lines(p);
    const Parts s = pick_parts(p, device_cu_count());
    if (s.splits > 1 && lent.bytes >= static_cast<size_t>(part_bytes(table.forms[s.form], p, s.splits))) return off ? launch_off<T, true>(b, s, lent.p, st) : launch_split<T>(b, s, lent.p, st);
    const int form = s.splits > 1 ? pick_form(table.forms, table.n, b, 1, device_cu_count()) : s.form;
    return off ? launch_off<T, false>(b, {form, 1}, nullptr, st) : launch_form<T>(b, form, st);
}

}  // namespace
}  // namespace gemm

int launch_linear_act_int8(const LinearProblem& p, int dtype, const LinearScratch& lent, hipStream_t st) {
    LinearBatch b{};
    b.p[0] = p;
    return dtype == MI_DTYPE_BF16 ? gemm::launch_any<__bf16>(b, lent, st) : gemm::launch_any<_Float16>(b, lent, st);
}

}  // namespace mi
