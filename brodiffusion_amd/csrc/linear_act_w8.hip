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
int launch_split(const LinearBatch& b, Parts s, void* parts, hipStream_t st) {
    switch (s.form) {
        case k8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2, T, true, WL, true>(b, 1, st, s.splits, parts);
        case k8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4, T, true, WL, true>(b, 1, st, s.splits, parts);
        case k8_128x64: return launch_pipe<T, true, false, 2, 2, 2, 1, 3, 4, T, true, WL, true>(b, 1, st, s.splits, parts);
        default: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2, T, true, WL, true>(b, 1, st, s.splits, parts);
    }
}
template <typename T, int WL>
int launch_words(const LinearBatch& b, const LinearScratch& lent, hipStream_t st) {
    const Parts s = pick_parts(b.p[0], device_cu_count());
    if (s.splits > 1 && lent.bytes >= static_cast<size_t>(part_bytes(kPlainW8[s.form], b.p[0], s.splits))) return launch_split<T, WL>(b, s, lent.p, st);
    return launch_form<T, WL>(b, s.splits > 1 ? pick_form(kPlainW8, kPlainW8Forms, b, 1, device_cu_count()) : s.form, st);
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
