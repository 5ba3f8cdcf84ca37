// The step between two blocks of a transformer: a block's output, normalised if the model does that, times its gate onto the residual stream, and the norm in
// front of the next block with that block's modulation, in one pass.
//
//   b = post(branch) post_gain                    post: nothing, RMS or layer norm, FP32
//   h = T(residual_scale x + gate b)              one rounding; everything below is of the stored value
//   y = T(pre(h) gain (1 + scale) + shift)        FP32 in between, one rounding
// RMS: v / sqrt(mean v^2 + eps); layer: (v - mean) / sqrt(mean (v - mean)^2 + eps), the squares summed of the differences, in registers, not as a difference of
// sums. gate, scale and shift are vectors of all rows or one for each run of rows (an image of a batch, a token).
//
// Bound: HBM. x and the branch are read once, h and y written once, the row stays in registers between its sums. The vectors come from the caches, which
// they have to themselves: the rows of x, of the branch and of h are marked as passing through. y, which the next product reads, is not: with it 4608 rows of 6144
// are 0.7 us faster, a block's norm, two products and norm 19 slower. Measured (us, gate, scale and shift, operands of 1 GiB in turn; without the marks): 4608 rows of 6144
// 42.7 = 5.3 TB/s, a large copy's rate (51.6), 4608 of 2240 19.6 (24.0), 16384 of 1152 31.5 (38.0), 1000 of 6144 14.4 (16.4), one of 6144 4.1. 4608 of 6144 without a branch
// 25.6 = 4.4 TB/s, beside 84 % of the vector instruction slots; the sum alone 28.9 = 5.9 TB/s.
#include "rows_checks.h"

namespace mi {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// A vector of the columns for each `each` rows
struct RowVectors {
    const void* p;       // null: not there
    long rs;             // elements
    int each;
};
struct GateNorm {
    const void* x; const void* branch; const void* post_gain; const void* gain;
    void* sum; void* out;                         // each null: not asked for
    RowVectors gate, scale, shift;
    int rows, cols, post, pre;                    // MI_NORM_*
    long x_rs, b_rs, s_rs, o_rs;                  // elements
    float alpha, post_eps, eps;
};

// W wavefronts per row (one: four rows to a work group), N 16-byte chunks per lane, as in rows_int8.hip. (Work groups that stay, with the vectors in registers from row
// to row and the next row on its way: 46 to 49 us instead of 44.6, their registers leave three wavefronts a SIMD. Three chunks by
// themselves take 97 registers, four wavefronts a SIMD; held to five, 4608 rows of 6144 take 42.7 us instead of 43.8, 4608 of 2240 19.6 for 20.9, 16384 of 1152 31.5 for 33.9,
// but rows that are four wavefronts a SIMD or one round of them lose: 4096 of 1152 10.9 for 10.2, 2048 of 2240 10.8 for 10.2, 1024 of 6144 12.9 for 12.4. Two chunks, held to
// seven for six, were 4 % slower.)
template <typename T, int N, int W>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W, N == 3 ? 5 : 1) gate_norm_kernel(const GateNorm a) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    constexpr int LANES = 64 * W;
    // (a chunk at a time where a lane has several: the FP32 values of all would cost wavefronts, of sixteen with 128 registers some would go to memory)
    constexpr bool TIGHT = N >= 2;
    __shared__ float red[2][4][W];                // [parity of the row][sum of it]: a slot is written again two rows on, a barrier after its last reader
    const int cpr = a.cols / 8;
    int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const long first = W == 1 ? blockIdx.x * 4L + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x, step = gridDim.x * (W == 1 ? 4L : 1L);
    const float inv_cols = 1.f / static_cast<float>(a.cols);
    auto mine = [&](int i) { return lane + LANES * i < cpr; };      // (lanes past the end load the last chunk and leave it out of everything)
    auto at = [&](int i) { return static_cast<unsigned>(min(lane + LANES * i, cpr - 1)) * 16u; };      // bytes
    auto store = [&](void* p, long row, int i, u32x4 v) { *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(static_cast<T*>(p) + row) + at(i)) = v; };
    auto load = [&](const void* p, long row) {
        const char* const base = reinterpret_cast<const char*>(static_cast<const T*>(p) + row);
        return [=](unsigned byte) { return __builtin_bit_cast(t8, *reinterpret_cast<const u32x4*>(base + byte)); };
    };
    // what passes through once: x, the branch, h (which is read again behind a block's products)
    auto load_once = [&](const void* p, long row) {
        const char* const base = reinterpret_cast<const char*>(static_cast<const T*>(p) + row);
        return [=](unsigned byte) { return __builtin_bit_cast(t8, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(base + byte))); };
    };
    auto store_once = [&](void* p, long row, int i, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(reinterpret_cast<char*>(static_cast<T*>(p) + row) + at(i))); };
    // (a chunk is made FP32 anew for each pass over the row: kept, its 8 values would hold twice the registers)
    auto anew = [](t8 (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u32x4 bits = __builtin_bit_cast(u32x4, v[i]);
            asm volatile("" : "+v"(bits));
            v[i] = __builtin_bit_cast(t8, bits);
        }
    };
    int parity = 0;
    for (long r = first; r < a.rows; r += step, parity ^= 1) {
        if constexpr (TIGHT) asm volatile("" : "+v"(lane));      // (nor offsets kept from row to row)
        int slot = 0;
        auto total = [&](float s) {
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off);
            if constexpr (W > 1) {
                float* const part = red[parity][slot++];
                if ((lane & 63) == 0) part[lane >> 6] = s;
                __syncthreads();
                s = 0.f;
#pragma unroll
                for (int i = 0; i < W; ++i) s += part[i];
            }
            return s;
        };
        // mean (0 for RMS) and factor of a row
        auto statistics = [&](t8 (&row)[N], int kind, float eps, float& mean, float& inv) {
            mean = 0.f;
            if (kind == MI_NORM_LAYER) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const t8 v = row[i];
                    float c = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) c += static_cast<float>(v[e]);
                    if (mine(i)) s += c;
                }
                mean = total(s) * inv_cols;
                anew(row);
            }
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const t8 v = row[i];
                float c = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float d = static_cast<float>(v[e]) - mean;
                    c = __builtin_fmaf(d, d, c);
                }
                if (mine(i)) s += c;
            }
            inv = inverse_root(total(s) / static_cast<float>(a.cols) + eps);
            anew(row);
        };
        auto vectors = [&](const RowVectors& v) { return load(v.p, (v.each == a.rows ? 0u : static_cast<unsigned>(r) / static_cast<unsigned>(v.each)) * v.rs); };

        // The vectors wait in registers for the sums, but of a lane with more than 3 chunks; there they are read behind the sums, from the L2, a latency that every
        // row then waits for.
        constexpr bool KEEP = N <= 3;
        const auto pg_at = load(a.post_gain, 0), gate_at = vectors(a.gate), gain_at = load(a.gain, 0), scale_at = vectors(a.scale), shift_at = vectors(a.shift);
        t8 pg[KEEP ? N : 1], gate[KEEP ? N : 1], gain[KEEP ? N : 1], scale[KEEP ? N : 1], shift[KEEP ? N : 1];
        auto keep = [&](t8* to, const void* p, auto from) {
            // (defined where there is none too: left undefined they cost 36 registers more)
            if constexpr (KEEP) {
#pragma unroll
                for (int i = 0; i < N; ++i) to[i] = p != nullptr ? from(at(i)) : t8{};
            }
        };
        auto kept = [&](const t8* v, auto from, int i) {
            if constexpr (KEEP) return v[i];
            else return from(at(i));
        };
        t8 h[N];
        const auto x_at = load_once(a.x, r * a.x_rs);
        constexpr bool LATE = N == 8;                 // (x behind the branch's sums: both together leave no registers for them)
        if (!LATE || a.branch == nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = x_at(at(i));
        }
        if (a.branch != nullptr) {
            t8 b[N];
            const auto b_at = load_once(a.branch, r * a.b_rs);
#pragma unroll
            for (int i = 0; i < N; ++i) b[i] = b_at(at(i));
            keep(pg, a.post_gain, pg_at);
            keep(gate, a.gate.p, gate_at);
            float mean = 0.f, inv = 1.f;
            if (a.post != MI_NORM_NONE) statistics(b, a.post, a.post_eps, mean, inv);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (static_cast<float>(b[i][e]) - mean) * inv;
                if constexpr (LATE) h[i] = x_at(at(i));
                if (a.post_gain != nullptr) {
                    const t8 g = kept(pg, pg_at, i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= static_cast<float>(g[e]);
                }
                if (a.gate.p != nullptr) {
                    const t8 g = kept(gate, gate_at, i);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= static_cast<float>(g[e]);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) h[i][e] = static_cast<T>(__builtin_fmaf(a.alpha, static_cast<float>(h[i][e]), f[e]));
                if (a.sum != nullptr && mine(i)) store_once(a.sum, r * a.s_rs, i, __builtin_bit_cast(u32x4, h[i]));
                if constexpr (TIGHT) asm volatile("" ::: "memory");
            }
        }
        if (a.out == nullptr) continue;
        asm volatile("" ::: "memory");                // (not earlier: all vectors at once would cost wavefronts)
        keep(gain, a.gain, gain_at);
        keep(scale, a.scale.p, scale_at);
        keep(shift, a.shift.p, shift_at);
        float mean, inv;
        statistics(h, a.pre, a.eps, mean, inv);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (static_cast<float>(h[i][e]) - mean) * inv;
            if (a.gain != nullptr) {
                const t8 g = kept(gain, gain_at, i);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= static_cast<float>(g[e]);
            }
            if (a.scale.p != nullptr) {
                const t8 g = kept(scale, scale_at, i);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= 1.f + static_cast<float>(g[e]);
            }
            if (a.shift.p != nullptr) {
                const t8 g = kept(shift, shift_at, i);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] += static_cast<float>(g[e]);
            }
            t8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(f[e]);
            if (mine(i)) store(a.out, r * a.o_rs, i, __builtin_bit_cast(u32x4, o));
            if constexpr (TIGHT) asm volatile("" ::: "memory");
        }
    }
}

template <typename T, int N, int W>
int launch_rows(const GateNorm& a, hipStream_t st) {
    const long groups = W == 1 ? (a.rows + 3L) / 4 : a.rows;
    hipLaunchKernelGGL((gate_norm_kernel<T, N, W>), dim3(static_cast<unsigned>(groups < (1L << 20) ? groups : 1L << 20)), dim3(W == 1 ? 256 : 64 * W), 0, st, a);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, int W>
int launch_chunks(const GateNorm& a, hipStream_t st) {
    const int n = (a.cols / 8 + 64 * W - 1) / (64 * W);
    if constexpr (W == 1) if (n == 1) return launch_rows<T, 1, W>(a, st);
    if (n <= 2) return launch_rows<T, 2, W>(a, st);
    if constexpr (W < 16) if (n == 3) return launch_rows<T, 3, W>(a, st);
    if constexpr (W >= 8) if (n <= 4) return launch_rows<T, 4, W>(a, st);
    if constexpr (W == 16) return launch_rows<T, 8, W>(a, st);
    return fail("gate_norm: no kernel for %d columns", a.cols);
}

// Wavefronts of a row: many for few rows, whose latency a chunk more adds to, few where rows fill the card. Measured (us, 2 / 4 / 8 / 16 wavefronts, three vectors): one row
// of 2240 4.0 / 3.8 / 4.0, 4608 rows 19.6 / 22.6 / 34.8; one of 6144 - / 4.2 / 4.1 / 5.2, 4608 rows - / 42.7 / 47.2 / 88.5. Over 64 sizes (1 to 16384 rows of 320 to 16384
// columns) the rule's choice is 0.5 % slower than the fastest on average, 12 % at most (1000 rows of 6144: 14.4, four wavefronts 12.8).
template <typename T>
int launch_width(const GateNorm& a, hipStream_t st) {
    const int chunks = a.cols / 8, each = a.rows >= 4 * device_cu_count() ? 3 : 2;
    if (chunks <= 64 * each) return launch_chunks<T, 1>(a, st);
    if (chunks <= 128 * each) return launch_chunks<T, 2>(a, st);
    if (chunks <= 256 * each) return launch_chunks<T, 4>(a, st);
    if (chunks <= 512 * (each == 3 ? 4 : 2)) return launch_chunks<T, 8>(a, st);
    return launch_chunks<T, 16>(a, st);
}

bool bad_eps(float e) { return e < 0.f || (__builtin_bit_cast(unsigned, e) & 0x7fffffffu) >= 0x7f800000u; }      // (by its bits: compiled without NaN in comparisons)

}  // namespace
}  // namespace mi

using mi::fail;

extern "C" int mi_gate_add_norm_forward(const mi_gate_add_norm_args* a) {
    const char* op = "mi_gate_add_norm_forward";
    mi::clear_error();
    if (!a) return fail("%s: null args", op);
    if (a->struct_size != sizeof(*a)) return fail("%s: struct_size %u != %zu (header mismatch)", op, a->struct_size, sizeof(*a));
    if (mi::check_rows(op, a->dtype, a->rows, a->cols)) return -1;
    for (const int32_t kind : {a->post_norm, a->norm})
        if (kind < MI_NORM_NONE || kind > MI_NORM_LAYER) return fail("%s: norm %d is none of MI_NORM_*", op, kind);
    if (mi::bad_eps(a->eps) || mi::bad_eps(a->post_eps)) return fail("%s: eps must be >= 0 and finite", op);
    if ((__builtin_bit_cast(unsigned, a->residual_scale) & 0x7fffffffu) >= 0x7f800000u) return fail("%s: residual_scale must be finite", op);
    if (a->rows == 0) return 0;
    if (!a->x) return fail("%s: null tensor", op);
    if (!a->out && !a->sum_out) return fail("%s: neither sum_out nor out is given", op);
    if ((a->out != nullptr) != (a->norm != MI_NORM_NONE)) return fail("%s: out and a norm must be given together", op);
    if (!a->out && (a->gain || a->scale || a->shift)) return fail("%s: gain, scale or shift without a norm", op);
    if (!a->branch && (a->gate || a->post_gain || a->sum_out || a->post_norm != MI_NORM_NONE)) return fail("%s: gate, post norm or sum_out without a branch", op);
    if (a->post_gain && a->post_norm == MI_NORM_NONE) return fail("%s: post_gain without a post norm", op);
    const long n = a->cols;
    auto stride = [&](int64_t s) { return s ? static_cast<long>(s) : n; };
    mi::GateNorm g{};
    g.x = a->x; g.branch = a->branch; g.post_gain = a->post_gain; g.gain = a->gain; g.sum = a->sum_out; g.out = a->out;
    g.rows = a->rows; g.cols = a->cols; g.post = a->post_norm; g.pre = a->norm;
    g.x_rs = stride(a->x_row_stride); g.b_rs = stride(a->branch_row_stride); g.s_rs = stride(a->sum_row_stride); g.o_rs = stride(a->out_row_stride);
    g.alpha = a->residual_scale; g.post_eps = a->post_eps; g.eps = a->eps;
    const mi::Operand ins[] = {{"x", g.x, 2 * g.x_rs, 2 * n}, {"branch", g.branch, 2 * g.b_rs, 2 * n}};
    const mi::Operand outs[] = {{"sum_out", g.sum, 2 * g.s_rs, 2 * n}, {"out", g.out, 2 * g.o_rs, 2 * n}};
    const struct { const char* name; const void* p; long rs; int32_t each; mi::RowVectors* to; } vectors[] = {
        {"gate", a->gate, stride(a->gate_row_stride), a->gate_rows, &g.gate}, {"scale", a->scale, stride(a->scale_row_stride), a->scale_rows, &g.scale},
        {"shift", a->shift, stride(a->shift_row_stride), a->shift_rows, &g.shift},
        {"post_gain", a->post_gain, n, 0, nullptr}, {"gain", a->gain, n, 0, nullptr}};
    auto items = [&](int each) { return each ? (a->rows - 1) / each + 1L : 1L; };
    for (const auto& v : vectors) {
        if (v.to) *v.to = {v.p, v.rs, v.each ? v.each : a->rows};
        if (!v.p) continue;
        if (v.each < 0) return fail("%s: %s_rows must not be negative", op, v.name);
        const mi::Operand rows{v.name, v.p, 2 * v.rs, 2 * n};
        if (mi::check_operands(op, items(v.each), a->cols, &rows, 1, nullptr, 0)) return -1;
    }
    if (mi::check_operands(op, a->rows, a->cols, ins, 2, outs, 2)) return -1;
    for (const auto& v : vectors)
        for (const mi::Operand& o : outs)
            if (mi::runs_share(o.p, (a->rows - 1) * o.rs + o.len, v.p, (items(v.each) - 1) * 2 * v.rs + 2 * n)) return fail("%s: %s overlaps %s", op, o.name, v.name);
    return a->dtype == MI_DTYPE_BF16 ? mi::launch_width<__bf16>(g, mi::resolve_stream(a->stream)) : mi::launch_width<_Float16>(g, mi::resolve_stream(a->stream));
}
