// The linear layer with an epilogue, INT8 weights and 16-bit rows (W8A16): which instance of linear_pipe.h a launch takes (linear_forms.h).
#include "linear_pipe.h"

namespace mi {
namespace gemm {
namespace {

// WL: linear_pipe.h. Words are four times the load instructions of W: one stage fewer of the tiles of 64 x 96 keeps their count within the
// counter of loads in flight.
template <typename T, int WL>
int launch_form(const LinearBatch& b, hipStream_t st) {
    switch (pick_form(kPlainW8, kPlainW8Forms, b, 1, device_cu_count())) {
        case k8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2, T, true, WL>(b, 1, st);
        case k8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4, T, true, WL>(b, 1, st);
        case k8_64x96: return launch_pipe<T, true, false, 2, 3, 1, 1, WL == 16 ? 5 : 4, 2, T, true, WL>(b, 1, st);
        case k8_128x64: return launch_pipe<T, true, false, 2, 2, 2, 1, 3, 4, T, true, WL>(b, 1, st);
        case k8_128x96: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2, T, true, WL>(b, 1, st);
        case k8_128x128: return launch_pipe<T, true, false, 2, 4, 2, 1, 4, 0, T, true, WL>(b, 1, st);
        default: return launch_pipe<T, true, false, 2, 2, 2, 2, 2, 0, T, true, WL>(b, 1, st);
    }
}
template <typename T>
int launch_words(const LinearBatch& b, hipStream_t st) {
    return b.p[0].ldw % 16 == 0 && b.p[0].K % 16 == 0 ? launch_form<T, 16>(b, st) : launch_form<T, 4>(b, st);
}

}  // namespace
}  // namespace gemm

int launch_linear_act_w8(const LinearProblem& p, int dtype, hipStream_t st) {
    LinearBatch b{};
    b.p[0] = p;
    return dtype == MI_DTYPE_BF16 ? gemm::launch_words<__bf16>(b, st) : gemm::launch_words<_Float16>(b, st);
}

}  // namespace mi
