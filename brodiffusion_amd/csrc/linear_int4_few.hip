// The linear layer with 4-bit weights for few rows (linear_int4.h): a token of a serving step, a draft, a short prompt.
//
// Bound: the bytes of the packed weights, each used once per 16 rows of X. They go from memory straight to the registers of the wavefront that multiplies
// them, in whole kilobytes. A work group owns 16 FB features and 16 rows; its 8 wavefronts take the blocks of 128 contraction elements in turn, each with its
// next block on its way while it multiplies, and their sums meet in LDS, added in the order of the wavefronts: no result depends on timing, there are
// no atomics. Measured (rows x contraction x features, groups; operands from memory, in parentheses from the last-level cache): 1 x 6144 x 16384, 128, 14.4 us = 3.6 TB/s
// (12.8); 1 x 1152 x 4608, 64, 5.3; 77 x 4608 x 1152, 32, 11.3 (9.5). (32 and 64 rows to a work group were slower than two and four of them, or than tiles, at every size; so
// were two blocks on their way.)
#include "linear_int4.h"

namespace mi {
namespace gemm {
namespace {

constexpr int WAVES = 8;

template <typename T, int P, int FB>
__global__ void __launch_bounds__(64 * WAVES) linear_int4_few_kernel(const Int4Problem p) {
    using M = Mma<T>;
    using V8 = typename M::v8;
    typedef T t4 __attribute__((ext_vector_type(4)));
    constexpr int F = 16 * FB, NT = 64 * WAVES, OUT = (F * 16 + NT - 1) / NT;
    constexpr int kTokens = 16 * 256, kSums = FB * 1024;      // bytes of a wavefront: a block's rows of X, its sums
    __shared__ __attribute__((aligned(16))) unsigned char lds[WAVES * (kTokens > kSums ? kTokens : kSums)];

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = static_cast<int>(blockIdx.x) * F, m0 = static_cast<int>(blockIdx.y) * 16;
    const int last_block = (p.N + 15) / 16 - 1;

    // (addresses as a uniform base and an offset of the lane)
    const unsigned char* wrow[FB];
    unsigned foff[FB];
#pragma unroll
    for (int a = 0; a < FB; ++a) {
        wrow[a] = static_cast<const unsigned char*>(p.w) + static_cast<long>(min(n0 / 16 + a, last_block)) * p.KB * 1024;
        foff[a] = static_cast<unsigned>(min(n0 + 16 * a + 4 * lg, p.N - 4));      // (features come in eights)
    }
    // X comes in loads of 4 rows of 256 bytes, piece `lr` of row 4 u + lg, and goes through this wavefront's part of LDS: as operands are wanted, a row per
    // lane, a load's neighbouring lanes would lie in 4 rows, and such loads were the time of more than a few rows (20 x 16384 x 6144: 48 us)
    constexpr int XU = 4;
    const T* xrow[XU];
#pragma unroll
    for (int u = 0; u < XU; ++u) xrow[u] = static_cast<const T*>(p.x) + static_cast<long>(min(m0 + 4 * u + lg, p.M - 1)) * p.ldx;
    const int rows = p.M - m0;                              // (loads of rows that are all past the end are left out: their columns of the product are not stored)

    struct Block { u32x4 w[FB]; V8 x[XU]; t4 s[FB][P]; unsigned z[FB][P]; };
    auto load = [&](Block& c, int kb) {
#pragma unroll
        for (int a = 0; a < FB; ++a) c.w[a] = *reinterpret_cast<const u32x4*>(wrow[a] + static_cast<long>(kb) * 1024 + lane * 16u);
#pragma unroll
        for (int g = 0; g < P; ++g) {
            const long row = static_cast<long>(min(P == 1 ? kb / p.span : kb * P + g, p.groups - 1)) * p.N;
#pragma unroll
            for (int a = 0; a < FB; ++a) {
                c.s[a][g] = *reinterpret_cast<const t4*>(reinterpret_cast<const unsigned char*>(static_cast<const T*>(p.scales) + row) + foff[a] * 2u);
                c.z[a][g] = p.zeros ? *reinterpret_cast<const unsigned*>(p.zeros + row + foff[a]) : 0x08080808u;
            }
        }
        const int k0 = kb * 128 + 8 * lr;
        const bool there = k0 < p.K;                        // (pieces past the end: the row's first one, as zeros)
#pragma unroll
        for (int u = 0; u < XU; ++u)
            if (4 * u < rows) {
                const V8 v = *reinterpret_cast<const V8*>(xrow[u] + (there ? k0 : 0));
                c.x[u] = there ? v : V8{};
            }
    };
    unsigned char* const tokens = lds + wave * kTokens;
    auto stage = [&](const Block& c) {
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < XU; ++u)
            if (4 * u < rows) *reinterpret_cast<V8*>(tokens + (4 * u + lg) * 256 + ((lr ^ ((4 * u + lg) & 15)) << 4)) = c.x[u];
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
    };
    f32x4 acc[FB];
#pragma unroll
    for (int a = 0; a < FB; ++a) acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Block& c) {
        V8 x[4];
        f32x4 sx[P];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const V8*>(tokens + lr * 256 + (((4 * j + lg) ^ lr) << 4));
#pragma unroll
        for (int g = 0; g < P; ++g) {
            sx[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) sx[g] = M::run16(ones<T>(), x[j], sx[g]);
        }
#pragma unroll
        for (int a = 0; a < FB; ++a) {
            V8 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = nibbles<T>(c.w[a][j]);
#pragma unroll
            for (int g = 0; g < P; ++g) {
                f32x4 t;
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = -zero_point(c.z[a][g], e) * sx[g][e];
#pragma unroll
                for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) t = M::run16(w[j], x[j], t);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[a][e] = __builtin_fmaf(t[e], static_cast<float>(c.s[a][g][e]), acc[a][e]);
            }
        }
    };

    const int share = static_cast<int>(blockIdx.z), end = int4_share(p, share + 1);
    int i = int4_share(p, share) + wave;
    if (i < end) {
        Block c[2];
        load(c[0], i);
        for (; i + WAVES < end; i += 2 * WAVES) {
            stage(c[0]);
            load(c[1], i + WAVES);
            multiply(c[0]);
            stage(c[1]);
            if (i + 2 * WAVES < end) load(c[0], i + 2 * WAVES);
            multiply(c[1]);
        }
        if (i < end) {
            stage(c[0]);
            multiply(c[0]);
        }
    }

    __syncthreads();                                        // (the sums go where rows of X were)
    float* const sums = reinterpret_cast<float*>(lds);      // [wavefront][block of features][row][feature]
#pragma unroll
    for (int a = 0; a < FB; ++a) *reinterpret_cast<f32x4*>(sums + (wave * FB + a) * 256 + lr * 16 + 4 * lg) = acc[a];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
        const int o = i * NT + tid, f = o % F, row = o / F;
        if (row >= 16 || m0 + row >= p.M || n0 + f >= p.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += sums[(w * FB + f / 16) * 256 + row * 16 + f % 16];
        if (p.parts) {
            p.parts[(static_cast<long>(share) * p.M + m0 + row) * p.N + n0 + f] = v;
            continue;
        }
        if (p.bias) v += static_cast<float>(static_cast<const T*>(p.bias)[n0 + f]);
        with_activation(p.act, [&](auto act) { v = act(v); });
        if (p.residual) v += static_cast<float>(static_cast<const T*>(p.residual)[static_cast<long>(m0 + row) * p.ldr + n0 + f]);
        static_cast<T*>(p.y)[static_cast<long>(m0 + row) * p.ldy + n0 + f] = static_cast<T>(v);
    }
}

template <typename T, int P, int FB>
int launch(const Int4Problem& p, hipStream_t st) {
    hipLaunchKernelGGL((linear_int4_few_kernel<T, P, FB>), dim3((p.N + 16 * FB - 1) / (16 * FB), (p.M + 15) / 16, p.shares), dim3(64 * WAVES), 0, st, p);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, int P>
int launch_form(const Int4Problem& p, int form, hipStream_t st) {
    switch (form) {
        case kFew16: return launch<T, P, 1>(p, st);
        case kFew32: return launch<T, P, 2>(p, st);
        default: return launch<T, P, P == 4 ? 2 : 4>(p, st);      // (kFew64; not asked for with groups of 32)
    }
}
template <typename T>
int launch_parts(const Int4Problem& p, int parts, int form, hipStream_t st) {
    return parts == 1 ? launch_form<T, 1>(p, form, st) : parts == 2 ? launch_form<T, 2>(p, form, st) : launch_form<T, 4>(p, form, st);
}

}  // namespace
}  // namespace gemm

int launch_int4_few(const Int4Problem& p, int dtype, int parts, int form, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_parts<__bf16>(p, parts, form, st) : gemm::launch_parts<_Float16>(p, parts, form, st);
}

}  // namespace mi
