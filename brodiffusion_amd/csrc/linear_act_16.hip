// The linear layer with an epilogue, 16-bit operands.
#include "linear_act_rings.h"

namespace mi {

int launch_linear_act_16(const LinearProblem& p, int dtype, const LinearScratch& lent, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_rings<__bf16, __bf16>(p, lent, st) : gemm::launch_rings<_Float16, _Float16>(p, lent, st);
}

}  // namespace mi
