// The linear layer with an epilogue, INT8 operands (W8A8).
#include "linear_act_rings.h"

namespace mi {

int launch_linear_act_int8(const LinearProblem& p, int dtype, const LinearScratch& lent, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_rings<__bf16, gemm::Int8>(p, lent, st) : gemm::launch_rings<_Float16, gemm::Int8>(p, lent, st);
}

}  // namespace mi
