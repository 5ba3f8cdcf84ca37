// Y = act(X W^T [* w_scales] [* x_scales] + bias) + residual: the linear layer with its epilogue, for 16-bit operands, INT8 weights
// (W8A16) and INT8 operands (W8A8).
//
// Few rows (linear_few.hip): bound by the bytes of W, which go to registers once. Otherwise the rings of linear_pipe.h and the 256 x 256 tiles of
// linear_dma.h with this epilogue, bound by the matrix pipes under the power limit. Rows so far apart that 32-bit offsets do not span a tile: tiles
// through registers (linear.hip). Measured (us; kernel, epilogue included, operands of 1 GiB in turn; rows x contraction x features): 1 x 1152 x 4608 bf16 5.2
// (weights in the last-level cache: 3.5 to 3.9); 1 x 6144 x 16384 W8A8 19.2 = 5.2 TB/s; 20 x 16384 x 6144 W8A16 27.5; 1031 x 1160 x 4608 fp16 22.9;
// 4608 x 6144 x 16384 bf16 767 = 1.21 PFLOP/s, W8A8 423 = 2.19 PTOP/s.
#include "linear_forms.h"

namespace mi {

namespace {
// what the rings take: tiles that 32-bit byte offsets reach
bool rings_take(const LinearProblem& p) { return p.ldx * 2 * 256 < (1L << 31) && p.ldw * 2 * 256 < (1L << 31); }
}  // namespace

int launch_linear_act(const LinearProblem& p, int dtype, const LinearScratch& lent, hipStream_t st) {
    if (linear_few_takes(p)) return launch_linear_few(p, dtype, st);
    if (!rings_take(p)) return launch_linear_act_tiles(p, dtype, st);
    if (p.x_scale) return launch_linear_act_int8(p, dtype, lent, st);
    return p.w_scale ? launch_linear_act_w8(p, dtype, lent, st) : launch_linear_act_16(p, dtype, lent, st);
}

namespace {

// The problem of a call, checked. 1: there is one, 0: no rows, -1: refused.
int problem_of(const mi_linear_act_args& a, const char* op, LinearProblem& p) {
    if (a.dtype != MI_DTYPE_BF16 && a.dtype != MI_DTYPE_F16) return fail("%s: dtype %d is neither MI_DTYPE_F16 nor MI_DTYPE_BF16", op, a.dtype);
    if (a.rows < 0 || a.in_features <= 0 || a.out_features <= 0) return fail("%s: %d rows, %d x %d features", op, a.rows, a.in_features, a.out_features);
    if (a.activation < MI_ACT_NONE || a.activation > MI_ACT_SILU) return fail("%s: activation %d is none of MI_ACT_*", op, a.activation);
    const bool a8 = a.x_scales != nullptr;
    if (a8 && !a.w_scales) return fail("%s: INT8 rows need INT8 weights (w_scales)", op);
    // (tile and step indices are 32-bit)
    if (a.rows > 1 << 30 || a.in_features > 1 << 30 || a.out_features > 1 << 30) return fail("%s: more than 2^30 rows or features are not supported", op);
    const int step = a8 ? 16 : 8;
    if (a.in_features % step || a.out_features % 8) return fail("%s: in_features %d must be a multiple of %d, out_features %d of 8", op, a.in_features, step, a.out_features);
    // 128 * 128 * in_features stays below 2^31
    if (a8 && a.in_features > 131056) return fail("%s: in_features %d exceed the 131056 whose INT32 sums are exact", op, a.in_features);
    if (a.rows == 0) return 0;
    if (!a.x || !a.w || !a.y) return fail("%s: null operand", op);
    p.x = a.x; p.w = a.w; p.bias = a.bias; p.y = a.y; p.residual = a.residual;
    p.w_scale = a.w_scales; p.x_scale = a.x_scales; p.act = a.activation;
    p.M = a.rows; p.N = a.out_features; p.K = a.in_features;
    p.ldx = a.x_row_stride ? a.x_row_stride : a.in_features;
    p.ldw = a.w_row_stride ? a.w_row_stride : a.in_features;
    p.ldy = a.y_row_stride ? a.y_row_stride : a.out_features;
    p.ldr = a.residual_row_stride ? a.residual_row_stride : a.out_features;
    if (p.ldx % step || p.ldw % step || p.ldy % 8 || p.ldr % 8) return fail("%s: row strides must be multiples of 8 elements (INT8 rows and their weights: of 16)", op);
    if (p.ldx < p.K || p.ldw < p.K || p.ldy < p.N || (p.residual && p.ldr < p.N)) return fail("%s: a row stride is smaller than the row", op);
    for (long s : {p.ldx, p.ldw, p.ldy, p.ldr})
        if (s > kMostStride) return fail("%s: a row stride exceeds 2^40 elements", op);
    if (reach_too_far(p.M, p.ldx) || reach_too_far(p.N, p.ldw) || reach_too_far(p.M, p.ldy) || reach_too_far(p.M, p.ldr))
        return fail("%s: rows reach over more than 2^56 elements", op);
    uintptr_t al = 0;
    for (const void* q : {p.x, p.w, p.bias, p.residual, static_cast<const void*>(p.y)}) al |= reinterpret_cast<uintptr_t>(q);
    if (al & 15u) return fail("%s: operands must be 16-byte aligned", op);
    if ((reinterpret_cast<uintptr_t>(p.x_scale) | reinterpret_cast<uintptr_t>(p.w_scale)) & 3u) return fail("%s: scales must be 4-byte aligned", op);
    if (p.residual && !(p.residual == p.y && p.ldr == p.ldy) && operands_overlap(p.residual, p.ldr, 0, p.y, p.ldy, 0, 1, p.M, p.N))
        return fail("%s: y overlaps the residual", op);
    const long x_bytes = a8 ? 1 : 2, w_bytes = a.w_scales ? 1 : 2;
    if (rows_share(p.y, 2 * p.ldy, 2L * p.N, p.x, x_bytes * p.ldx, x_bytes * p.K, p.M)) return fail("%s: y overlaps x", op);
    const long y_run = 2 * ((p.M - 1) * p.ldy + p.N);      // (from the first byte to the last: what is no rows of y's number is held against all of it)
    if (runs_share(p.y, y_run, p.w, w_bytes * ((p.N - 1) * p.ldw + p.K))) return fail("%s: y overlaps w", op);
    if (runs_share(p.y, y_run, p.bias, 2L * p.N)) return fail("%s: y overlaps the bias", op);
    if (runs_share(p.y, y_run, p.w_scale, 4L * p.N) || runs_share(p.y, y_run, p.x_scale, 4L * p.M)) return fail("%s: y overlaps scales", op);
    if (static_cast<long>((p.M + 31) / 32) * ((p.N + 31) / 32) > 0x7ffffff0L) return fail("%s: problem too large for one launch", op);
    if (a8) { p.K /= 2; p.ldx /= 2; p.ldw /= 2; }      // rows of pairs (LinearProblem::x_scale)
    return 1;
}

// Lent memory is none of the operands': parts of sums would go over them. (INT8 rows: K and their strides are in pairs by now)
int check_scratch(const LinearProblem& p, const char* op, const void* scratch, size_t bytes) {
    if (!scratch || bytes == 0) return 0;
    const long run = static_cast<long>(bytes < (1ul << 60) ? bytes : 1ul << 60), w_bytes = p.w_scale && !p.x_scale ? 1 : 2, rows = p.M - 1;
    const struct { const char* name; const void* first; long len; } operands[] = {
        {"x", p.x, 2 * (rows * p.ldx + p.K)}, {"w", p.w, w_bytes * ((p.N - 1) * p.ldw + p.K)}, {"bias", p.bias, 2L * p.N}, {"residual", p.residual, 2 * (rows * p.ldr + p.N)},
        {"y", p.y, 2 * (rows * p.ldy + p.N)}, {"w_scales", p.w_scale, 4L * p.N}, {"x_scales", p.x_scale, 4L * p.M}};
    for (const auto& o : operands)
        if (runs_share(scratch, run, o.first, o.len)) return fail("%s: scratch overlaps %s", op, o.name);
    return 0;
}

size_t scratch_bytes(const LinearProblem& p) {
    if (linear_few_takes(p) || !rings_take(p)) return 0;
    const gemm::Parts s = gemm::pick_parts(p, device_cu_count());
    return s.splits > 1 ? static_cast<size_t>(gemm::part_bytes(gemm::table_of(p).forms[s.form], p, s.splits)) : 0;
}

}  // namespace
}  // namespace mi

extern "C" {

int mi_linear_act_forward(const mi_linear_act_args* a) {
    const char* op = "mi_linear_act_forward";
    mi::clear_error();
    if (!a) return mi::fail("%s: null args", op);
    if (a->struct_size != sizeof(*a)) return mi::fail("%s: struct_size %u != %zu (header mismatch)", op, a->struct_size, sizeof(*a));
    if (reinterpret_cast<uintptr_t>(a->scratch) & 15u) return mi::fail("%s: scratch must be 16-byte aligned", op);
    mi::LinearProblem p{};
    const int rc = mi::problem_of(*a, op, p);
    if (rc <= 0) return rc;
    if (mi::check_scratch(p, op, a->scratch, a->scratch_bytes)) return -1;
    return mi::launch_linear_act(p, a->dtype, {a->scratch, a->scratch ? a->scratch_bytes : 0}, mi::resolve_stream(a->stream));
}

size_t mi_linear_act_scratch_bytes(const mi_linear_act_args* a) {
    mi::LinearProblem p{};
    if (!a || a->struct_size != sizeof(*a) || mi::problem_of(*a, "mi_linear_act_scratch_bytes", p) != 1) return 0;
    return mi::scratch_bytes(p);
}

}  // extern "C"
