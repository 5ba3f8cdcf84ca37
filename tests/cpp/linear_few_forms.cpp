// Whether the kernel for few rows takes a linear layer with an epilogue, and with which work groups (csrc/linear_few_forms.h), for tests that mean a certain
// one. kind: 0 operands of 16 bits, 1 INT8 weights, 2 both INT8. row: the stride of both operands' rows, in elements like k; their first bytes are on lines.
// Returns whether it does; form: blocks' groups, features, rows, steps, wavefronts.
#include "linear_few_forms.h"

extern "C" {

int linear_few(int m, int n, int k, int row, int kind, int compute_units, int* form) {
    static const float scale = 1.f;
    const int pair = kind == 2 ? 2 : 1;
    mi::LinearProblem p{};
    p.M = m; p.N = n; p.K = k / pair;
    p.ldx = p.ldw = row / pair;
    p.w_scale = kind >= 1 ? &scale : nullptr;
    p.x_scale = kind == 2 ? &scale : nullptr;
    if (!mi::gemm::few_takes(p, compute_units)) return 0;
    const mi::gemm::FewForm f = mi::gemm::few_form(p, compute_units);
    const int all[] = {f.G, f.FB, f.TB, f.U, f.wavefronts};
    for (int i = 0; i < 5; ++i) form[i] = all[i];
    return 1;
}

// The table of a kind; returns how many forms it has (at most 32 are written)
int linear_few_table(int kind, int* forms) {
    int n = 0;
    auto add = [&](const auto& table) {
        for (const mi::gemm::FewForm& f : table) {
            const int all[] = {f.G, f.FB, f.TB, f.U, f.wavefronts};
            for (int i = 0; i < 5 && n < 32; ++i) forms[5 * n + i] = all[i];
            ++n;
        }
    };
    if (kind == 0) add(mi::gemm::kFew16);
    else if (kind == 1) add(mi::gemm::kFewW8);
    else add(mi::gemm::kFewBoth8);
    return n;
}

}  // extern "C"
