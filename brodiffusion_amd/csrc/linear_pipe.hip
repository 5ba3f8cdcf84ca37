// The linear layers without an activation or residual on the kernel of linear_pipe.h: which instance a launch takes.
#include "linear_pipe.h"

namespace mi {
namespace gemm {
namespace {

template <typename T>
int launch_form(const LinearBatch& b, int n, bool geglu, int dtype, hipStream_t st) {
    const bool w8 = b.p[0].w_scale != nullptr;
    const int form = pick_form(b, n, geglu, device_cu_count());
    if (geglu && w8) {
        switch (form) {
            case kG8_64x64: return launch_pipe<T, true, true, 2, 2, 1, 2, 3, 0>(b, n, st);
            case kG8_128x64_2: return launch_pipe<T, true, true, 2, 2, 2, 2, 2, 0>(b, n, st);
            case kG8_192x128: return launch_pipe<T, true, true, 2, 4, 3, 2, 3, 0>(b, n, st);
            default: return launch_pipe<T, true, true, 4, 2, 2, 2, 3, 0>(b, n, st);
        }
    }
    if (geglu) {
        switch (form) {
            case kG64x64: return launch_pipe<T, false, true, 2, 2, 1, 2, 3, 4>(b, n, st);
            case kG128x64_2: return launch_pipe<T, false, true, 2, 2, 2, 2, 2, 0>(b, n, st);
            case kG128x64: return launch_pipe<T, false, true, 2, 2, 2, 2, 3, 4>(b, n, st);
            case kG192x128: return launch_pipe<T, false, true, 2, 4, 3, 2, 2, 0>(b, n, st);
            default: return launch_pipe<T, false, true, 4, 2, 2, 2, 3, 0>(b, n, st);
        }
    }
    if (w8) {
        switch (form) {
            case k8_32x32: return launch_pipe<T, true, false, 1, 1, 1, 1, 6, 2>(b, n, st);
            case k8_64x64: return launch_pipe<T, true, false, 2, 2, 1, 1, 4, 4>(b, n, st);
            case k8_64x96: return launch_pipe<T, true, false, 2, 3, 1, 1, 5, 2>(b, n, st);
            case k8_128x64: return launch_pipe<T, true, false, 2, 2, 2, 1, 3, 4>(b, n, st);
            case k8_128x96: return launch_pipe<T, true, false, 2, 3, 2, 1, 3, 2>(b, n, st);
            case k8_128x128: return launch_pipe<T, true, false, 2, 4, 2, 1, 4, 0>(b, n, st);
            default: return launch_pipe<T, true, false, 2, 2, 2, 2, 2, 0>(b, n, st);
        }
    }
    switch (form) {
        case k32x32: return launch_pipe<T, false, false, 1, 1, 1, 1, 6, 2>(b, n, st);
        case k64x32: return launch_pipe<T, false, false, 2, 1, 1, 1, 6, 2>(b, n, st);
        case k64x64: return launch_pipe<T, false, false, 2, 2, 1, 1, 4, 4>(b, n, st);
        case k64x96: return launch_pipe<T, false, false, 2, 3, 1, 1, 5, 4>(b, n, st);
        case k128x64_load: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 4>(b, n, st);
        case k128x96: return launch_pipe<T, false, false, 2, 3, 2, 1, 4, 4>(b, n, st);
        case k128x64: return launch_pipe<T, false, false, 2, 2, 2, 1, 3, 0>(b, n, st);
        case k128x128: return launch_pipe<T, false, false, 2, 2, 2, 2, 3, 4>(b, n, st);
        case k128x128_2: return launch_pipe<T, false, false, 2, 2, 2, 2, 2, 0>(b, n, st);
        case k192x128: return launch_pipe<T, false, false, 2, 4, 3, 1, 4, 0>(b, n, st);
        case k256x128: return launch_pipe<T, false, false, 4, 2, 2, 2, 3, 0>(b, n, st);
        default: return launch_linear_dma(b, n, dtype, st);
    }
}

}  // namespace
}  // namespace gemm

// Contractions of whole stages; operands whose tiles (GEGLU: whose whole W) are addressable with 32-bit byte offsets.
bool linear_pipe_takes(const LinearBatch& batch, int n_problems, bool geglu) {
    for (int i = 0; i < n_problems; ++i) {
        const LinearProblem& p = batch.p[i];
        if (p.K % gemm::kBK != 0) return false;
        if (p.w_scale != nullptr && (p.ldw % 16 != 0)) return false;   // (rows of 16-byte pieces)
        if (static_cast<long>(p.ldx) * 2 * 256 >= (1L << 31) || static_cast<long>(p.ldw) * 2 * 256 >= (1L << 31)) return false;
        if (geglu && static_cast<long>(p.N) * 2 * p.ldw * 2 >= (1L << 32)) return false;
    }
    return true;
}

int launch_linear_pipe(const LinearBatch& batch, int n_problems, int dtype, bool geglu, hipStream_t st) {
    if (dtype == MI_DTYPE_BF16) return gemm::launch_form<__bf16>(batch, n_problems, geglu, dtype, st);
    return gemm::launch_form<_Float16>(batch, n_problems, geglu, dtype, st);
}

}  // namespace mi
