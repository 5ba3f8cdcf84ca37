// Y = act(X W^T + bias) + residual with 4-bit weights: the entries, the packing of weights and the choice between the kernels of linear_int4_few.hip and
// linear_int4_tile.hip (linear_int4_forms.h). Formulas and layout: linear_int4.h.
#include "linear_int4.h"

namespace mi {
namespace {

// One word of packed weights per thread: 8 elements of a row, as the matrix instructions take them
__global__ void __launch_bounds__(256) pack_int4_kernel(const unsigned char* q, unsigned* out, int N, int K, int KB, long q_rs, long words) {
    for (long i = blockIdx.x * 256L + threadIdx.x; i < words; i += gridDim.x * 256L) {
        const int j = static_cast<int>(i & 3), lane = static_cast<int>(i >> 2) & 63;
        const long block = i >> 8;
        const long n = block / KB * 16 + (lane & 15);
        const int k = static_cast<int>(block % KB) * 128 + 32 * j + 8 * (lane >> 4);
        unsigned w = 0;                           // (features and elements that are not there: any 0 .. 15, they meet zeros of x or are not stored)
        if (n < N && k < K) w = *reinterpret_cast<const unsigned*>(q + n * q_rs + k / 2);
        unsigned r = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) r |= ((w >> (4 * e)) & 15u) << (e < 4 ? 8 * e : 8 * (e - 4) + 4);
        out[i] = r;
    }
}

// The sums of the shares of a contraction, added in their order, and what follows them: 4 features per thread. Shares put compute units to work that one work group for
// each piece of Y would leave idle: 20 x 16384 x 6144 (rows x contraction x features, operands from memory) 28.7 -> 21.9 us, 128 x 16384 x 6144 70.5 -> 43.6,
// 1 x 16384 x 128 11.8 -> 6.5; this launch is 3.5 to 4.5 us of that. The rule for them is int4_launch's.
template <typename T>
__global__ void __launch_bounds__(256) join_int4_kernel(const Int4Problem p) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int quads = p.N / 4;
    const long all = static_cast<long>(p.M) * quads;
    for (long i = blockIdx.x * 256L + threadIdx.x; i < all; i += gridDim.x * 256L) {
        const long m = i / quads;
        const int f = static_cast<int>(i - m * quads) * 4;
        const float* at = p.parts + 4 * i;
        gemm::f32x4 v = *reinterpret_cast<const gemm::f32x4*>(at);
#pragma unroll 4
        for (int s = 1; s < p.shares; ++s) v += *reinterpret_cast<const gemm::f32x4*>(at + s * 4 * all);
        if (p.bias) {
            const t4 b = *reinterpret_cast<const t4*>(static_cast<const T*>(p.bias) + f);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(b[e]);
        }
        gemm::with_activation(p.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = act(v[e]);
        });
        if (p.residual) {
            const t4 r = *reinterpret_cast<const t4*>(static_cast<const T*>(p.residual) + m * p.ldr + f);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(r[e]);
        }
        t4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(v[e]);
        *reinterpret_cast<t4*>(static_cast<T*>(p.y) + m * p.ldy + f) = o;
    }
}

long packed_bytes(long n, long k) { return (n + 15) / 16 * ((k + 127) / 128) * 1024; }

// Features and contraction of a call
int check_sizes(const char* op, int n, int k) {
    if (n <= 0 || k <= 0) return fail("%s: %d x %d features", op, k, n);
    if (n > 1 << 30 || k > 1 << 30) return fail("%s: more than 2^30 features are not supported", op);
    if (k % 8 || n % 8) return fail("%s: in_features %d and out_features %d must be multiples of 8", op, k, n);
    return 0;
}

// The problem of a call, checked. 1: there is one, 0: no rows, -1: refused.
int problem_of(const mi_linear_int4_args& a, const char* op, Int4Problem& p) {
    if (a.dtype != MI_DTYPE_BF16 && a.dtype != MI_DTYPE_F16) return fail("%s: dtype %d is neither MI_DTYPE_F16 nor MI_DTYPE_BF16", op, a.dtype);
    if (a.rows < 0 || a.rows > 1 << 30) return fail("%s: %d rows", op, a.rows);
    if (check_sizes(op, a.out_features, a.in_features)) return -1;
    if (a.activation < MI_ACT_NONE || a.activation > MI_ACT_SILU) return fail("%s: activation %d is none of MI_ACT_*", op, a.activation);
    if (a.group != 32 && a.group != 64 && (a.group <= 0 || a.group % 128)) return fail("%s: group %d is neither 32, 64 nor a multiple of 128", op, a.group);
    if (a.rows == 0) return 0;
    if (!a.x || !a.w || !a.scales || !a.y) return fail("%s: null operand", op);
    p.x = a.x; p.w = a.w; p.scales = a.scales; p.zeros = static_cast<const unsigned char*>(a.zeros); p.bias = a.bias; p.residual = a.residual; p.y = a.y;
    p.M = a.rows; p.N = a.out_features; p.K = a.in_features; p.act = a.activation;
    p.KB = (p.K + 127) / 128; p.groups = static_cast<int>((p.K - 1L + a.group) / a.group); p.span = a.group > 128 ? a.group / 128 : 1;
    p.ldx = a.x_row_stride ? a.x_row_stride : p.K;
    p.ldy = a.y_row_stride ? a.y_row_stride : p.N;
    p.ldr = a.residual_row_stride ? a.residual_row_stride : p.N;
    if (p.ldx % 8 || p.ldy % 8 || p.ldr % 8) return fail("%s: row strides must be multiples of 8 elements", op);
    if (p.ldx < p.K || p.ldy < p.N || (p.residual && p.ldr < p.N)) return fail("%s: a row stride is smaller than the row", op);
    for (long s : {p.ldx, p.ldy, p.ldr})
        if (s > kMostStride) return fail("%s: a row stride exceeds 2^40 elements", op);
    if (reach_too_far(p.M, p.ldx) || reach_too_far(p.M, p.ldy) || (p.residual && reach_too_far(p.M, p.ldr))) return fail("%s: rows reach over more than 2^56 elements", op);
    uintptr_t al = 0;
    for (const void* q : {p.x, p.w, p.scales, p.bias, p.residual, static_cast<const void*>(p.y)}) al |= reinterpret_cast<uintptr_t>(q);
    if (al & 15u) return fail("%s: operands must be 16-byte aligned", op);
    if (reinterpret_cast<uintptr_t>(p.zeros) & 7u) return fail("%s: zeros must be 8-byte aligned", op);
    if (p.residual && !(p.residual == p.y && p.ldr == p.ldy) && operands_overlap(p.residual, p.ldr, 0, p.y, p.ldy, 0, 1, p.M, p.N)) return fail("%s: y overlaps the residual", op);
    if (rows_share(p.y, 2 * p.ldy, 2L * p.N, p.x, 2 * p.ldx, 2L * p.K, p.M)) return fail("%s: y overlaps x", op);
    const long y_run = 2 * ((p.M - 1) * p.ldy + p.N), per_group = static_cast<long>(p.groups) * p.N;
    if (runs_share(p.y, y_run, p.w, packed_bytes(p.N, p.K))) return fail("%s: y overlaps w", op);
    if (runs_share(p.y, y_run, p.scales, 2 * per_group)) return fail("%s: y overlaps scales", op);
    if (runs_share(p.y, y_run, p.zeros, per_group)) return fail("%s: y overlaps zeros", op);
    if (runs_share(p.y, y_run, p.bias, 2L * p.N)) return fail("%s: y overlaps the bias", op);
    return 1;
}

// Lent memory is none of the operands'
int check_scratch(const Int4Problem& p, const char* op, const void* scratch, size_t bytes) {
    if (!scratch || bytes == 0) return 0;
    const long run = static_cast<long>(bytes < (1ul << 60) ? bytes : 1ul << 60), per_group = static_cast<long>(p.groups) * p.N, rows = p.M - 1;
    const struct { const char* name; const void* first; long len; } operands[] = {
        {"x", p.x, 2 * (rows * p.ldx + p.K)}, {"w", p.w, packed_bytes(p.N, p.K)}, {"scales", p.scales, 2 * per_group}, {"zeros", p.zeros, per_group}, {"bias", p.bias, 2L * p.N},
        {"residual", p.residual, 2 * (rows * p.ldr + p.N)}, {"y", p.y, 2 * (rows * p.ldy + p.N)}};
    for (const auto& o : operands)
        if (runs_share(scratch, run, o.first, o.len)) return fail("%s: scratch overlaps %s", op, o.name);
    return 0;
}

Int4Launch launch_of(const Int4Problem& p, int group, size_t lent) { return int4_launch(p.M, p.N, p.KB, p.ldx, int4_parts(group), device_cu_count(), lent); }
size_t parts_bytes(const Int4Problem& p, int shares) { return shares > 1 ? sizeof(float) * static_cast<size_t>(shares) * p.M * p.N : 0; }

}  // namespace
}  // namespace mi

extern "C" {

size_t mi_int4_packed_bytes(int32_t out_features, int32_t in_features) {
    return out_features > 0 && in_features > 0 ? static_cast<size_t>(mi::packed_bytes(out_features, in_features)) : 0;
}

int mi_pack_int4(const mi_pack_int4_args* a) {
    const char* op = "mi_pack_int4";
    mi::clear_error();
    if (!a) return mi::fail("%s: null args", op);
    if (a->struct_size != sizeof(*a)) return mi::fail("%s: struct_size %u != %zu (header mismatch)", op, a->struct_size, sizeof(*a));
    if (mi::check_sizes(op, a->out_features, a->in_features)) return -1;
    if (!a->q || !a->packed) return mi::fail("%s: null operand", op);
    const long n = a->out_features, k = a->in_features, rs = a->q_row_stride ? a->q_row_stride : k / 2;
    if (rs < k / 2 || rs % 4) return mi::fail("%s: the row stride of q must be a multiple of 4 bytes and at least in_features / 2", op);
    if (rs > mi::kMostStride || mi::reach_too_far(n, rs)) return mi::fail("%s: rows of q reach over more than 2^56 bytes", op);
    if (reinterpret_cast<uintptr_t>(a->q) & 3u) return mi::fail("%s: q must be 4-byte aligned", op);
    if (reinterpret_cast<uintptr_t>(a->packed) & 15u) return mi::fail("%s: packed must be 16-byte aligned", op);
    const long bytes = mi::packed_bytes(n, k), words = bytes / 4;
    if (mi::runs_share(a->packed, bytes, a->q, (n - 1) * rs + k / 2)) return mi::fail("%s: packed overlaps q", op);
    const long groups = (words + 255) / 256;
    hipLaunchKernelGGL(mi::pack_int4_kernel, dim3(static_cast<unsigned>(groups < (1L << 20) ? groups : 1L << 20)), dim3(256), 0, mi::resolve_stream(a->stream),
                       static_cast<const unsigned char*>(a->q), static_cast<unsigned*>(a->packed), a->out_features, a->in_features, static_cast<int>((k + 127) / 128), rs, words);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

int mi_linear_int4_forward(const mi_linear_int4_args* a) {
    const char* op = "mi_linear_int4_forward";
    mi::clear_error();
    if (!a) return mi::fail("%s: null args", op);
    if (a->struct_size != sizeof(*a)) return mi::fail("%s: struct_size %u != %zu (header mismatch)", op, a->struct_size, sizeof(*a));
    if (reinterpret_cast<uintptr_t>(a->scratch) & 15u) return mi::fail("%s: scratch must be 16-byte aligned", op);
    mi::Int4Problem p{};
    const int rc = mi::problem_of(*a, op, p);
    if (rc <= 0) return rc;
    if (mi::check_scratch(p, op, a->scratch, a->scratch_bytes)) return -1;
    const int parts = mi::int4_parts(a->group);
    const mi::Int4Launch launch = mi::launch_of(p, a->group, a->scratch ? a->scratch_bytes : 0);
    if (launch.form < 0) return mi::fail("%s: problem too large for one launch", op);
    p.shares = launch.shares;
    p.parts = launch.shares > 1 ? static_cast<float*>(a->scratch) : nullptr;
    const hipStream_t st = mi::resolve_stream(a->stream);
    if (launch.form < mi::kTile32x64 ? mi::launch_int4_few(p, a->dtype, parts, launch.form, st) : mi::launch_int4_tile(p, a->dtype, parts, launch.form, st)) return -1;
    if (launch.shares == 1) return 0;
    const long groups = (static_cast<long>(p.M) * (p.N / 4) + 255) / 256;
    const dim3 grid(static_cast<unsigned>(groups < (1L << 20) ? groups : 1L << 20));
    if (a->dtype == MI_DTYPE_BF16) hipLaunchKernelGGL(mi::join_int4_kernel<__bf16>, grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(mi::join_int4_kernel<_Float16>, grid, dim3(256), 0, st, p);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

size_t mi_linear_int4_scratch_bytes(const mi_linear_int4_args* a) {
    mi::Int4Problem p{};
    if (!a || a->struct_size != sizeof(*a) || mi::problem_of(*a, "mi_linear_int4_scratch_bytes", p) != 1) return 0;
    return mi::parts_bytes(p, mi::launch_of(p, a->group, ~static_cast<size_t>(0)).shares);
}

}  // extern "C"
