// What the entry points of row kernels (rows_int8.hip, gate_norm.hip) check of their operands.
#pragma once
#include "internal.h"

namespace mi {

constexpr int kMostCols = 65536;

struct Operand { const char* name; const void* p; long rs, len; };      // bytes

inline int check_rows(const char* op, int dtype, int rows, int cols) {
    if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_F16) return fail("%s: dtype %d is neither MI_DTYPE_F16 nor MI_DTYPE_BF16", op, dtype);
    if (rows < 0 || cols <= 0 || cols % 8 != 0) return fail("%s: cols must be a positive multiple of 8, rows >= 0", op);
    if (cols > kMostCols) return fail("%s: rows of more than %d columns are not supported", op, kMostCols);
    return 0;
}
// Strides and alignment; then no output shares memory with another operand, but that a 16-bit output may be an input itself.
inline int check_operands(const char* op, int rows, int cols, const Operand* ins, int n_in, const Operand* outs, int n_out) {
    for (const Operand* list : {ins, outs})
        for (int i = 0; i < (list == ins ? n_in : n_out); ++i) {
            const Operand& o = list[i];
            const long bytes = o.len / cols;
            if (o.p == nullptr || bytes == 0) continue;
            if (o.rs % (8 * bytes) != 0 || o.rs < o.len) return fail("%s: the row stride of %s must be a multiple of 8 elements and at least cols", op, o.name);
            if (o.rs > bytes * kMostStride) return fail("%s: the row stride of %s exceeds 2^40 elements", op, o.name);
            if (reach_too_far(rows, o.rs / bytes)) return fail("%s: the rows of %s reach over more than 2^56 elements", op, o.name);
            if (reinterpret_cast<uintptr_t>(o.p) % (8 * bytes) != 0) return fail("%s: %s must be %ld-byte aligned", op, o.name, 8 * bytes);
        }
    for (int i = 0; i < n_out; ++i) {
        const Operand& o = outs[i];
        if (o.p == nullptr) continue;
        for (int j = 0; j < n_in; ++j)
            if (ins[j].p != nullptr && !(o.p == ins[j].p && o.rs == ins[j].rs && o.len == ins[j].len) && rows_share(o.p, o.rs, o.len, ins[j].p, ins[j].rs, ins[j].len, rows))
                return fail("%s: %s overlaps %s", op, o.name, ins[j].name);
        for (int j = 0; j < i; ++j)
            if (outs[j].p != nullptr && rows_share(o.p, o.rs, o.len, outs[j].p, outs[j].rs, outs[j].len, rows)) return fail("%s: %s overlaps %s", op, o.name, outs[j].name);
    }
    return 0;
}

}  // namespace mi
