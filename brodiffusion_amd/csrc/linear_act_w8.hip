// The linear layer with an epilogue, INT8 weights and 16-bit rows (W8A16): which instance of linear_pipe.h a launch takes (linear_forms.h).
#include "linear_pipe.h"

namespace mi {
namespace gemm {
namespace {

template <typename T>
int launch_form(const LinearBatch& b, hipStream_t st) {
    switch (pick_form(kPlainW8, kPlainW8Forms, b, 1, device_cu_count())) {
        case k8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2, T, true>(b, 1, st);
        case k8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4, T, true>(b, 1, st);
        case k8_64x96: return launch_pipe<T, true, false, 2, 3, 1, 1, 5, 2, T, true>(b, 1, st);
        case k8_128x64: return launch_pipe<T, true, false, 2, 2, 2, 1, 3, 4, T, true>(b, 1, st);
        case k8_128x96: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2, T, true>(b, 1, st);
        case k8_128x128: return launch_pipe<T, true, false, 2, 4, 2, 1, 4, 0, T, true>(b, 1, st);
        default: return launch_pipe<T, true, false, 2, 2, 2, 2, 2, 0, T, true>(b, 1, st);
    }
}

}  // namespace
}  // namespace gemm

int launch_linear_act_w8(const LinearProblem& p, int dtype, hipStream_t st) {
    LinearBatch b{};
    b.p[0] = p;
    return dtype == MI_DTYPE_BF16 ? gemm::launch_form<__bf16>(b, st) : gemm::launch_form<_Float16>(b, st);
}

}  // namespace mi
