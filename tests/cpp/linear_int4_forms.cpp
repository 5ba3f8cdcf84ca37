// What int4_form (csrc/linear_int4_forms.h) gives a problem, for tests
#include "linear_int4_forms.h"

extern "C" __attribute__((visibility("default"))) int int4_form_test(int rows, int features, int contraction, long row_stride, int group, int compute_units) {
    return mi::int4_form(rows, features, (contraction + 127) / 128, row_stride, group >= 128 ? 1 : 128 / group, compute_units);
}
