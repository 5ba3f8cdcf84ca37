// What int4_launch (csrc/linear_int4_forms.h) gives a problem, for tests: the form, and the shares of the contraction with so many bytes lent
#include "linear_int4_forms.h"

extern "C" __attribute__((visibility("default"))) int int4_form_test(int rows, int features, int contraction, long row_stride, int group, int compute_units, unsigned long lent, int* shares) {
    const mi::Int4Launch l = mi::int4_launch(rows, features, (contraction + 127) / 128, row_stride, group >= 128 ? 1 : 128 / group, compute_units, lent);
    *shares = l.shares;
    return l.form;
}
