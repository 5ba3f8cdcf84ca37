// Rows in front of a projection: h = x + residual with the RMS normalisation of h behind it, and rows as 8-bit integers with one
// FP32 scale each (of the normalised rows, or of rows as they are).
//
//   h = T(x + residual)                       stored if asked for; everything below is of the stored value
//   inv = 1 / sqrt(mean h^2 + eps)            FP32
//   y = T(h inv gain)                         one rounding
//   z = h gain (FP32: a product of two 16-bit values has at most 22 significant bits), a = max |z|
//   q = 127 z / a rounded to the nearest integer, ties to even; scale = a inv / 127
// inv is a factor of the whole row, so it goes into the scale and the integers do not depend on it: they are the exactly rounded
// quotients whatever the order of the sum of squares. A row of zeros has q = 0 and scale 0, one with a value that is not finite q = 0
// and scale NaN.
//
// Bound: HBM. Each row is read once, held in registers between its sums and what is written, and nothing else passes through memory but the gain.
// A lane holds N 16-byte chunks; a row belongs to W wavefronts (one: sums by lane exchanges alone, four rows in a work group; more:
// one exchange through LDS behind a barrier). 4608 rows of 6144, several sets in turn: 41.9 us = 5.4 TB/s, a large copy's rate here (5.1 to 5.4);
// to 8 bits 37.9 us (5.2 TB/s).
#include "internal.h"

namespace mi {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

struct RowsArgs {
    const void* x; const void* residual; const void* gain;
    void* sum; void* out; void* q; float* scales;      // each null: not asked for
    int rows, cols;
    long x_rs, r_rs, s_rs, o_rs, q_rs;                 // elements
    float eps;
};

// 127 z / a to the nearest integer, exactly; inv_step = 127 / a to a few units. The quotient by multiplication is within 2.3e-5 of the
// true one (127 times 3 roundings of 2^-24); only where it lies that near to the middle of two integers the question is asked again
// in 64 bits, where both sides of the comparison are exact (7 + 24 and 8 + 24 bits).
__device__ __forceinline__ int to_step(float z, float a, float inv_step) {
    const float t = z * inv_step, n = __builtin_rintf(t);
    int q = static_cast<int>(n);
    if (__builtin_expect(__builtin_fabsf(t - n) > 0.49995f, 0)) {
        const float lo = __builtin_floorf(t);
        const double num = 127.0 * static_cast<double>(z), mid = (static_cast<double>(lo) + 0.5) * static_cast<double>(a);
        const int l = static_cast<int>(lo);
        q = num > mid ? l + 1 : num < mid ? l : l + (l & 1);
    }
    return q;
}

// NORM: with gain and inv (otherwise z = x, inv = 1).
template <typename T, int N, int W, bool NORM>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) rows_kernel(const RowsArgs a) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    constexpr int LANES = 64 * W;                 // of a row
    __shared__ float red_sum[W];
    __shared__ unsigned red_max[W];
    const int cpr = a.cols / 8, lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const long first = W == 1 ? blockIdx.x * 4L + (threadIdx.x >> 6) : blockIdx.x, step = gridDim.x * (W == 1 ? 4L : 1L);
    const T* const x = static_cast<const T*>(a.x);
    const T* const res = static_cast<const T*>(a.residual);
    const T* const gain = static_cast<const T*>(a.gain);
    auto mine = [&](int i) { return lane + LANES * i < cpr; };      // (lanes past the end load the last chunk and leave it out of everything)
    auto at = [&](int i) { return min(lane + LANES * i, cpr - 1) * 8; };
    // The gain waits in registers for the sums, but of a lane with more than 4 chunks (sixteen wavefronts have 128 registers): 8 chunks of both put 68 to
    // 72 bytes a lane into memory. There it is read again, from the L2.
    constexpr bool KEEP = NORM && N <= 4;
    for (long r = first; r < a.rows; r += step) {
        u32x4 v[N], g[KEEP ? N : 1];
        auto gain_of = [&](int i) { if constexpr (KEEP) return g[i]; else return *reinterpret_cast<const u32x4*>(gain + at(i)); };
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = *reinterpret_cast<const u32x4*>(x + r * a.x_rs + at(i));
        if constexpr (NORM) {
            if (res != nullptr) {
                u32x4 b[N];
#pragma unroll
                for (int i = 0; i < N; ++i) b[i] = *reinterpret_cast<const u32x4*>(res + r * a.r_rs + at(i));
                if constexpr (KEEP) {
#pragma unroll
                    for (int i = 0; i < N; ++i) g[i] = *reinterpret_cast<const u32x4*>(gain + at(i));
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const t8 p = __builtin_bit_cast(t8, v[i]), s = __builtin_bit_cast(t8, b[i]);
                    t8 h;
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[e] = static_cast<T>(static_cast<float>(p[e]) + static_cast<float>(s[e]));
                    v[i] = __builtin_bit_cast(u32x4, h);
                    if (a.sum != nullptr && mine(i)) *reinterpret_cast<u32x4*>(static_cast<T*>(a.sum) + r * a.s_rs + at(i)) = v[i];
                }
            } else {
                if constexpr (KEEP) {
#pragma unroll
                    for (int i = 0; i < N; ++i) g[i] = *reinterpret_cast<const u32x4*>(gain + at(i));
                }
            }
        }
        // (the largest magnitude as an integer: of FP32 bit patterns without sign a NaN is the largest)
        float ss = 0.f;
        unsigned most = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const t8 h = __builtin_bit_cast(t8, v[i]);
            t8 w{};
            if constexpr (NORM) w = __builtin_bit_cast(t8, gain_of(i));
            float s = 0.f;
            unsigned m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = static_cast<float>(h[e]);
                if constexpr (NORM) s = __builtin_fmaf(f, f, s);
                m = max(m, __builtin_bit_cast(unsigned, NORM ? f * static_cast<float>(w[e]) : f) & 0x7fffffffu);
            }
            if (mine(i)) { ss += s; most = max(most, m); }
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            if constexpr (NORM) ss += __shfl_xor(ss, off);
            most = max(most, static_cast<unsigned>(__shfl_xor(static_cast<int>(most), off)));
        }
        if constexpr (W > 1) {
            __syncthreads();                      // the previous row's readers are done
            if ((lane & 63) == 0) { red_sum[lane >> 6] = ss; red_max[lane >> 6] = most; }
            __syncthreads();
            ss = 0.f;
            most = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) { ss += red_sum[i]; most = max(most, red_max[i]); }
        }
        // (the products are made again below: kept, the 8 of a chunk would hold more registers than the chunk and the gain they come from)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            asm volatile("" : "+v"(v[i]));
            if constexpr (KEEP) asm volatile("" : "+v"(g[i]));
        }
        const float inv = NORM ? inverse_root(ss / static_cast<float>(a.cols) + a.eps) : 1.f;
        if (NORM && a.out != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const t8 h = __builtin_bit_cast(t8, v[i]), w = __builtin_bit_cast(t8, gain_of(i));
                t8 o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(static_cast<float>(h[e]) * inv * static_cast<float>(w[e]));
                if (mine(i)) *reinterpret_cast<u32x4*>(static_cast<T*>(a.out) + r * a.o_rs + at(i)) = __builtin_bit_cast(u32x4, o);
            }
        }
        if (a.q == nullptr) continue;
        const bool finite = most < 0x7f800000u, some = finite && most != 0;
        // (a small row is lifted by a power of two, which changes no quotient: 127 / a would overflow below 2^-121)
        const float top = __builtin_bit_cast(float, most), lift = top < 0x1p-60f ? 0x1p80f : 1.f;
        const float most_z = some ? top * lift : 1.f, inv_step = 127.f / most_z, factor = some ? lift : 0.f;
        if (lane == 0) {
            const float scale = some ? top * inv / 127.f : 0.f;
            reinterpret_cast<unsigned*>(a.scales)[r] = finite ? __builtin_bit_cast(unsigned, scale) : 0x7fc00000u;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const t8 h = __builtin_bit_cast(t8, v[i]);
            t8 w{};
            if constexpr (NORM) w = __builtin_bit_cast(t8, gain_of(i));
            u32x2 o = {0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = static_cast<float>(h[e]), z = NORM ? f * static_cast<float>(w[e]) : f;
                o[e / 4] |= (static_cast<unsigned>(to_step(z * factor, most_z, inv_step)) & 0xffu) << (8 * (e % 4));
            }
            if (!some) o = u32x2{0u, 0u};         // (values that are not finite times 0)
            if (mine(i)) *reinterpret_cast<u32x2*>(static_cast<signed char*>(a.q) + r * a.q_rs + at(i)) = o;
        }
    }
}

constexpr int kMostCols = 65536;

template <typename T, int N, int W, bool NORM>
int launch_rows(const RowsArgs& a, hipStream_t st) {
    const long groups = W == 1 ? (a.rows + 3L) / 4 : a.rows;
    hipLaunchKernelGGL((rows_kernel<T, N, W, NORM>), dim3(static_cast<unsigned>(groups < (1L << 20) ? groups : 1L << 20)), dim3(W == 1 ? 256 : 64 * W), 0, st, a);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

// (launch_width asks for one chunk with one wavefront only, for four with eight and sixteen, for more with sixteen)
template <typename T, int W, bool NORM>
int launch_chunks(const RowsArgs& a, hipStream_t st) {
    const int n = (a.cols / 8 + 64 * W - 1) / (64 * W);
    if constexpr (W == 1) if (n == 1) return launch_rows<T, 1, W, NORM>(a, st);
    if (n == 2) return launch_rows<T, 2, W, NORM>(a, st);
    if (n == 3) return launch_rows<T, 3, W, NORM>(a, st);
    if constexpr (W >= 8) if (n == 4) return launch_rows<T, 4, W, NORM>(a, st);
    if constexpr (W == 16) if (n > 4) return launch_rows<T, 8, W, NORM>(a, st);
    return fail("rows: no kernel for %d columns", a.cols);
}

// Wavefronts per row. Where rows fill the GPU (4 for each compute unit) up to 3 chunks per lane: fewer lanes have none, fewer meet at the barrier;
// where they do not, a row is a chain of latencies and 2 chunks per lane shorten it. Measured (us, 8-bit norm, 1 / 2 / 4 / 8 / 16 wavefronts):
//   4608 rows of 2240 19.9 / 17.6 / 20.1 / 21.9 / -, of 6144 - / 41.7 / 37.9 / 40.1 / 52.1; 2048 of 16384 - / - / 51.9 / 53.4 / 59.7
//   333 rows of 2240 5.9 / 5.0 / 4.5 / 4.4 / -; 1 row of 6144 - / 5.3 / 3.9 / 3.8 / 4.0, of 16384 - / - / 6.7 / 5.6 / 5.3
template <typename T, bool NORM>
int launch_width(const RowsArgs& a, hipStream_t st) {
    const int chunks = a.cols / 8, each = a.rows >= 4 * device_cu_count() ? 3 : 2;
    if (chunks <= 64 * each) return launch_chunks<T, 1, NORM>(a, st);
    if (chunks <= 128 * each) return launch_chunks<T, 2, NORM>(a, st);
    if (chunks <= 256 * each) return launch_chunks<T, 4, NORM>(a, st);
    if (chunks <= 512 * (each == 3 ? 4 : 2)) return launch_chunks<T, 8, NORM>(a, st);
    return launch_chunks<T, 16, NORM>(a, st);
}

int launch(const RowsArgs& a, int dtype, bool norm, hipStream_t st) {
    if (dtype == MI_DTYPE_BF16) return norm ? launch_width<__bf16, true>(a, st) : launch_width<__bf16, false>(a, st);
    return norm ? launch_width<_Float16, true>(a, st) : launch_width<_Float16, false>(a, st);
}

struct Operand { const char* name; const void* p; long rs, len; };      // bytes

int check_rows(const char* op, int dtype, int rows, int cols) {
    if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_F16) return fail("%s: dtype %d is neither MI_DTYPE_F16 nor MI_DTYPE_BF16", op, dtype);
    if (rows < 0 || cols <= 0 || cols % 8 != 0) return fail("%s: cols must be a positive multiple of 8, rows >= 0", op);
    if (cols > kMostCols) return fail("%s: rows of more than %d columns are not supported", op, kMostCols);
    return 0;
}
// Strides and alignment; then no output shares memory with another operand, but that a 16-bit output may be an input itself.
int check_operands(const char* op, int rows, int cols, const Operand* ins, int n_in, const Operand* outs, int n_out) {
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

}  // namespace
}  // namespace mi

using mi::fail;

extern "C" {

int mi_add_rms_norm_forward(const mi_add_rms_norm_args* a) {
    const char* op = "mi_add_rms_norm_forward";
    mi::clear_error();
    if (!a) return fail("%s: null args", op);
    if (a->struct_size != sizeof(*a)) return fail("%s: struct_size %u != %zu (header mismatch)", op, a->struct_size, sizeof(*a));
    if (mi::check_rows(op, a->dtype, a->rows, a->cols)) return -1;
    // (by its bits: this library is compiled without NaN in comparisons)
    if (a->eps < 0.f || (__builtin_bit_cast(unsigned, a->eps) & 0x7fffffffu) >= 0x7f800000u) return fail("%s: eps must be >= 0 and finite", op);
    if (a->rows == 0) return 0;
    if (!a->out && !a->out_q) return fail("%s: neither out nor out_q is given", op);
    if ((a->out_q != nullptr) != (a->out_scales != nullptr)) return fail("%s: out_q and out_scales must be given together", op);
    if (a->sum_out && !a->residual) return fail("%s: sum_out without a residual", op);
    if (!a->x || !a->gain) return fail("%s: null tensor", op);
    if (reinterpret_cast<uintptr_t>(a->gain) & 15u) return fail("%s: gain must be 16-byte aligned", op);
    if (reinterpret_cast<uintptr_t>(a->out_scales) & 3u) return fail("%s: out_scales must be 4-byte aligned", op);
    const long n = a->cols;
    auto stride = [&](int64_t s) { return s ? static_cast<long>(s) : n; };
    mi::RowsArgs r{a->x, a->residual, a->gain, a->sum_out, a->out, a->out_q, a->out_scales, a->rows, a->cols,
                   stride(a->x_row_stride), stride(a->residual_row_stride), stride(a->sum_row_stride), stride(a->out_row_stride), stride(a->q_row_stride), a->eps};
    // (scales: rows of nothing but themselves, one behind the other)
    const mi::Operand ins[] = {{"x", r.x, 2 * r.x_rs, 2 * n}, {"residual", r.residual, 2 * r.r_rs, 2 * n}};
    const mi::Operand outs[] = {{"sum_out", r.sum, 2 * r.s_rs, 2 * n}, {"out", r.out, 2 * r.o_rs, 2 * n}, {"out_q", r.q, r.q_rs, n}, {"out_scales", r.scales, 4, 4}};
    if (mi::check_operands(op, a->rows, a->cols, ins, 2, outs, 4)) return -1;
    for (const mi::Operand& o : outs)
        if (mi::runs_share(o.p, (a->rows - 1) * o.rs + o.len, r.gain, 2 * n)) return fail("%s: %s overlaps gain", op, o.name);
    return mi::launch(r, a->dtype, true, mi::resolve_stream(a->stream));
}

int mi_quantize_rows_forward(const mi_quantize_rows_args* a) {
    const char* op = "mi_quantize_rows_forward";
    mi::clear_error();
    if (!a) return fail("%s: null args", op);
    if (a->struct_size != sizeof(*a)) return fail("%s: struct_size %u != %zu (header mismatch)", op, a->struct_size, sizeof(*a));
    if (mi::check_rows(op, a->dtype, a->rows, a->cols)) return -1;
    if (a->rows == 0) return 0;
    if (!a->x || !a->out_q || !a->out_scales) return fail("%s: null tensor", op);
    if (reinterpret_cast<uintptr_t>(a->out_scales) & 3u) return fail("%s: out_scales must be 4-byte aligned", op);
    const long n = a->cols;
    mi::RowsArgs r{};
    r.x = a->x; r.q = a->out_q; r.scales = a->out_scales;
    r.rows = a->rows; r.cols = a->cols;
    r.x_rs = a->x_row_stride ? a->x_row_stride : n;
    r.q_rs = a->q_row_stride ? a->q_row_stride : n;
    const mi::Operand ins[] = {{"x", r.x, 2 * r.x_rs, 2 * n}};
    const mi::Operand outs[] = {{"out_q", r.q, r.q_rs, n}, {"out_scales", r.scales, 4, 4}};
    if (mi::check_operands(op, a->rows, a->cols, ins, 1, outs, 2)) return -1;
    return mi::launch(r, a->dtype, false, mi::resolve_stream(a->stream));
}

}  // extern "C"
