// The linear layer with an epilogue, INT8 weights and 16-bit rows (W8A16): which instance of linear_pipe.h a launch takes (linear_forms.h).
#include "linear_pipe.h"

namespace mi {
namespace gemm {
namespace {

// WL: linear_pipe.h. Words are four times the load instructions of W: one stage fewer of the tiles of 64 x 96 keeps their count within the
// counter of loads in flight.
template <typename T, int WL>
int launch_form(const LinearBatch& b, int form, hipStream_t st) {
    switch (form) {
        case k8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2, T, true, WL>(b, 1, st);
        case k8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4, T, true, WL>(b, 1, st);
        case k8_64x96: return launch_pipe<T, true, false, 2, 3, 1, 1, WL == 16 ? 5 : 4, 2, T, true, WL>(b, 1, st);
        case k8_128x64: return launch_pipe<T, true, false, 2, 2, 2, 1, 3, 4, T, true, WL>(b, 1, st);
        case k8_128x96: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2, T, true, WL>(b, 1, st);
        case k8_128x128: return launch_pipe<T, true, false, 2, 4, 2, 1, 4, 0, T, true, WL>(b, 1, st);
        default: return launch_pipe<T, true, false, 2, 2, 2, 2, 2, 0, T, true, WL>(b, 1, st);
    }
}
// ... in several parts (the forms of kSplitW8)
template <typename T, int WL>
int launch_split(const LinearBatch& b, const ActLaunch& s, void* parts, hipStream_t st) {
    switch (s.form) {
        case k8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2, T, true, WL, true>(b, 1, st, s.splits, parts);
        case k8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4, T, true, WL, true>(b, 1, st, s.splits, parts);
        case k8_128x64: return launch_pipe<T, true, false, 2, 2, 2, 1, 3, 4, T, true, WL, true>(b, 1, st, s.splits, parts);
        default: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2, T, true, WL, true>(b, 1, st, s.splits, parts);
    }
}
// ... of rows that do not begin on lines (kOff8), in one part or, with memory for them, several
template <typename T, int WL, bool JOIN>
int launch_off(const LinearBatch& b, const ActLaunch& s, void* parts, hipStream_t st) {
    switch (s.form) {
        case kOff8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2, T, true, WL, JOIN>(b, 1, st, s.splits, parts);
        case kOff8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4, T, true, WL, JOIN>(b, 1, st, s.splits, parts);
        case kOff8_128x64_row: return launch_pipe<T, true, false, 2, 2, 2, 1, 4, 4, T, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
        case kOff8_128x96_row: return launch_pipe<T, true, false, 2, 3, 2, 1, 4, 2, T, true, 16, JOIN, true>(b, 1, st, s.splits, parts);
    }
    if constexpr (!JOIN) switch (s.form) {
        case kOff8_64x96: return launch_pipe<T, true, false, 2, 3, 1, 1, WL == 16 ? 5 : 4, 2, T, true, WL>(b, 1, st);
        case kOff8_128x96: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2, T, true, WL>(b, 1, st);
        case kOff8_128x128_2_row: return launch_pipe<T, true, false, 2, 2, 2, 2, 3, 0, T, true, 16, false, true>(b, 1, st);
        case kOff8_128x128_row: return launch_pipe<T, true, false, 2, 4, 2, 1, 5, 0, T, true, 16, false, true>(b, 1, st);
    }
    return fail("linear: no kernel for form %d", s.form);      // (not asked for)
}
template <typename T, int WL>
int launch_words(const LinearBatch& b, const LinearScratch& lent, hipStream_t st) {
    const ActLaunch s = act_launch(b.p[0], lent.bytes, device_cu_count());
    if (s.splits > 1) return s.off ? launch_off<T, WL, true>(b, s, lent.p, st) : launch_split<T, WL>(b, s, lent.p, st);
    return s.off ? launch_off<T, WL, false>(b, s, nullptr, st) : launch_form<T, WL>(b, s.form, st);
}
template <typename T>
int launch_any(const LinearBatch& b, const LinearScratch& lent, hipStream_t st) {
    return b.p[0].ldw % 16 == 0 && b.p[0].K % 16 == 0 ? launch_words<T, 16>(b, lent, st) : launch_words<T, 4>(b, lent, st);
}

}  // namespace
}  // namespace gemm

int launch_linear_act_w8(const LinearProblem& p, int dtype, const LinearScratch& lent, hipStream_t st) {
    LinearBatch b{};
    b.p[0] = p;
    return dtype == MI_DTYPE_BF16 ? gemm::launch_any<__bf16>(b, lent, st) : gemm::launch_any<_Float16>(b, lent, st);
}

}  // namespace mi
