// Which form a linear layer with an epilogue takes and whether it gives its tiles to several work groups (csrc/linear_forms.h), for tests that mean
// one: the form, by its place in the table of its kind, and how many parts. row: the stride of both operands' rows, in elements like the contraction.
// int8_weights: W8A16; INT8 operands of both kinds count as 16-bit ones of half the contraction and half the stride.
#include "linear_forms.h"

extern "C" int linear_parts(int m, int n, int k, int row, int int8_weights, int compute_units, int* splits) {
    mi::LinearProblem p{};
    p.M = m;
    p.N = n;
    p.K = k;
    p.ldx = p.ldw = row;
    static const float scale = 1.f;
    p.w_scale = int8_weights ? &scale : nullptr;
    const mi::gemm::Parts s = mi::gemm::pick_parts(p, compute_units);
    *splits = s.splits;
    return s.form;
}
