// Whether a linear layer with an epilogue gives its tiles to several work groups (csrc/linear_forms.h), for tests that mean it: the form, by its place in
// the table of its kind, and how many parts. int8_weights: W8A16; INT8 operands of both kinds count as 16-bit ones of half the contraction.
#include "linear_forms.h"

extern "C" int linear_parts(int m, int n, int k, int int8_weights, int compute_units, int* splits) {
    mi::LinearBatch b{};
    b.p[0].M = m;
    b.p[0].N = n;
    b.p[0].K = k;
    b.p[0].ldx = b.p[0].ldw = k;
    static const float scale = 1.f;
    b.p[0].w_scale = int8_weights ? &scale : nullptr;
    const mi::gemm::Parts s = int8_weights ? mi::gemm::pick_parts(mi::gemm::kPlainW8, mi::gemm::kPlainW8Forms, mi::gemm::kSplitW8, b, compute_units)
                                           : mi::gemm::pick_parts(mi::gemm::kPlain, mi::gemm::kPlainForms, mi::gemm::kSplitPlain, b, compute_units);
    *splits = s.splits;
    return s.form;
}
