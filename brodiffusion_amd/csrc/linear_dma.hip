// The linear layers without an activation or residual on the kernel of linear_dma.h.
#include "linear_dma.h"

namespace mi {

int launch_linear_dma(const LinearBatch& batch, int n_problems, int dtype, hipStream_t st) {
    if (dtype == MI_DTYPE_BF16) return gemm_dma::launch_t<__bf16>(batch, n_problems, st);
    if (dtype == MI_DTYPE_F16) return gemm_dma::launch_t<_Float16>(batch, n_problems, st);
    return fail("linear: dtype %d is neither MI_DTYPE_F16 nor MI_DTYPE_BF16", dtype);
}

}  // namespace mi
