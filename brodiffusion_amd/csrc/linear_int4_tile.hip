// The linear layer with 4-bit weights for many rows (linear_int4.h).
//
// A work group owns a tile of tokens x features, 16 TB WM x 16 FB WN, of WM x WN wavefronts with TB x FB blocks of v_mfma_f32_16x16x32 each. X comes by LDS DMA in
// steps of 128 contraction elements (a block of packed weights) into a ring of three stages: rows of 256 bytes, the piece of 16 bytes at position c of row r is
// piece c ^ (r % 16), so that the 16 rows of an operand read lie in 16 different bank groups. Packed weights are operands already: every wavefront loads
// its own, 16 bytes a lane and block, a step ahead, and makes them 16-bit in registers. The sums of x that meet the zero points are formed a step
// ahead too, each 16 tokens by one wavefront, and shared through LDS.
#include "linear_int4.h"

namespace mi {
namespace gemm {
namespace {

constexpr int kStages = 3;

template <typename T, int P, bool ZEROS, int TB, int FB, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) linear_int4_tile_kernel(const Int4Problem p) {
    using M = Mma<T>;
    using V8 = typename M::v8;
    typedef T t4 __attribute__((ext_vector_type(4)));
    constexpr int NW = WM * WN, TM = 16 * TB * WM, TN = 16 * FB * WN;
    constexpr int kStage = TM * 256;
    constexpr int DI = TM / 4 / NW;                 // DMA instructions of a wavefront per stage, 4 rows each
    static_assert(TM % (4 * NW) == 0, "the rows of a stage are dealt out evenly");
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    float* const sums = reinterpret_cast<float*>(lds + kStages * kStage);      // [2][P][TM]

    const int tiles_n = (p.N + TN - 1) / TN, tiles_m = (p.M + TM - 1) / TM, n_tiles = tiles_m * tiles_n;
    // (every XCD takes a contiguous run of tiles, which share rows of X)
    const int chunk = (n_tiles + 7) >> 3, in_run = static_cast<int>(blockIdx.x) >> 3;
    const int logical = (static_cast<int>(blockIdx.x) & 7) * chunk + in_run;
    if (in_run >= chunk || logical >= n_tiles) return;
    const int m0 = (logical / tiles_n) * TM, n0 = (logical % tiles_n) * TN;

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
    const int nw = n0 + wn * 16 * FB, last_block = (p.N + 15) / 16 - 1;

    const unsigned char* xg = static_cast<const unsigned char*>(p.x) + static_cast<long>(m0) * p.ldx * 2;
    unsigned xoff[DI];
    int piece[DI];
#pragma unroll
    for (int u = 0; u < DI; ++u) {
        const int r = 4 * (wave * DI + u) + (lane >> 4);
        piece[u] = (lane & 15) ^ (r & 15);
        xoff[u] = static_cast<unsigned>(min(r, p.M - 1 - m0)) * (static_cast<unsigned>(p.ldx) * 2u);
    }
    const unsigned lds_base = static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) unsigned char*)lds));
    const int left = (p.K - (p.KB - 1) * 128) / 8;      // pieces of the last block's rows
    auto dma = [&](int kb) {
        const int most = kb == p.KB - 1 ? left - 1 : 15;      // (pieces past the end: the last one, left out of the products)
        const unsigned char* const base = xg + static_cast<long>(kb) * 256;
#pragma unroll
        for (int u = 0; u < DI; ++u) {
            const unsigned off = xoff[u] + static_cast<unsigned>(min(piece[u], most)) * 16u;
            asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(lds_base + (kb % kStages) * kStage + (wave * DI + u) * 1024) : "memory");
        }
    };
    // operands of 16 tokens, block `row16` of the tile, from the stage of kb
    auto tokens = [&](V8 (&x)[4], int kb, int row16) {
        const unsigned char* const at = lds + (kb % kStages) * kStage + row16 * 4096 + lr * 256;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const V8*>(at + (((4 * j + lg) ^ lr) << 4));
        if (kb == p.KB - 1 && left < 16) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * j + lg >= left) x[j] = V8{};
        }
    };
    // the sums of x of step kb, 16 tokens a wavefront
    auto sum_tokens = [&](int kb) {
        for (int b = wave; b < TM / 16; b += NW) {
            V8 x[4];
            tokens(x, kb, b);
#pragma unroll
            for (int g = 0; g < P; ++g) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) s = M::run16(ones<T>(), x[j], s);
                if (lg == 0) sums[((kb & 1) * P + g) * TM + 16 * b + lr] = s[0];
            }
        }
    };

    const unsigned char* wrow[FB];
    const T* scale[FB];
    const unsigned char* zero[FB];
#pragma unroll
    for (int a = 0; a < FB; ++a) {
        wrow[a] = static_cast<const unsigned char*>(p.w) + static_cast<long>(min(nw / 16 + a, last_block)) * p.KB * 1024 + lane * 16;
        const int f = min(nw + 16 * a + 4 * lg, p.N - 4);
        scale[a] = static_cast<const T*>(p.scales) + f;
        zero[a] = p.zeros + f;
    }
    struct Weights { u32x4 w[FB]; t4 s[FB][P]; unsigned z[FB][ZEROS ? P : 1]; };
    auto load = [&](Weights& c, int kb) {
#pragma unroll
        for (int a = 0; a < FB; ++a) c.w[a] = *reinterpret_cast<const u32x4*>(wrow[a] + static_cast<long>(kb) * 1024);
#pragma unroll
        for (int g = 0; g < P; ++g) {
            const long row = static_cast<long>(min(P == 1 ? kb / p.span : kb * P + g, p.groups - 1)) * p.N;
#pragma unroll
            for (int a = 0; a < FB; ++a) {
                c.s[a][g] = *reinterpret_cast<const t4*>(scale[a] + row);
                if constexpr (ZEROS) c.z[a][g] = *reinterpret_cast<const unsigned*>(zero[a] + row);
            }
        }
    };

    f32x4 acc[FB][TB];
#pragma unroll
    for (int a = 0; a < FB; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    // (all of this wavefront's loads have landed, DMA among them; said to the compiler, which counts the others)
    auto landed = [] {
        __builtin_amdgcn_s_waitcnt(0x0070);
        asm volatile("s_barrier" ::: "memory");
    };
    Weights c, next;
    load(next, 0);
    dma(0);
    if (p.KB > 1) dma(1);
    landed();
    sum_tokens(0);
    landed();
    for (int kb = 0; kb < p.KB; ++kb) {
        // the stages of kb and kb + 1 have landed, the sums of kb are there
        c = next;
        if (kb + 1 < p.KB) load(next, kb + 1);
        asm volatile("" ::: "memory");
        if (kb + 2 < p.KB) dma(kb + 2);
        V8 w[FB][4];
#pragma unroll
        for (int a = 0; a < FB; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[a][j] = nibbles<T>(c.w[a][j]);
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            V8 x[4];
            tokens(x, kb, wm * TB + b);
#pragma unroll
            for (int g = 0; g < P; ++g) {
                const float sx = sums[((kb & 1) * P + g) * TM + 16 * (wm * TB + b) + lr];
#pragma unroll
                for (int a = 0; a < FB; ++a) {
                    f32x4 t;
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = -(ZEROS ? zero_point(c.z[a][g], e) : 8.f) * sx;
#pragma unroll
                    for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) t = M::run16(w[a][j], x[j], t);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][b][e] = __builtin_fmaf(t[e], static_cast<float>(c.s[a][g][e]), acc[a][b][e]);
                }
            }
        }
        if (kb + 1 < p.KB) sum_tokens(kb + 1);
        landed();
    }

#pragma unroll
    for (int a = 0; a < FB; ++a) {
        const int f = nw + 16 * a + 4 * lg;
        if (f >= p.N) continue;
        f32x4 bias = {0.f, 0.f, 0.f, 0.f};
        if (p.bias) {
            const t4 v = *reinterpret_cast<const t4*>(static_cast<const T*>(p.bias) + f);
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[e] = static_cast<float>(v[e]);
        }
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            const int m = m0 + 16 * (wm * TB + b) + lr;
            if (m >= p.M) continue;
            f32x4 v = acc[a][b] + bias;
            with_activation(p.act, [&](auto act) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = act(v[e]);
            });
            if (p.residual) {
                const t4 r = *reinterpret_cast<const t4*>(static_cast<const T*>(p.residual) + static_cast<long>(m) * p.ldr + f);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(r[e]);
            }
            t4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(v[e]);
            *reinterpret_cast<t4*>(static_cast<T*>(p.y) + static_cast<long>(m) * p.ldy + f) = o;
        }
    }
}

template <typename T, int P, bool ZEROS, int TB, int FB, int WM, int WN>
int launch(const Int4Problem& p, hipStream_t st) {
    constexpr int TM = 16 * TB * WM, TN = 16 * FB * WN, bytes = kStages * TM * 256 + 2 * P * TM * 4;
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    const auto kernel = &linear_int4_tile_kernel<T, P, ZEROS, TB, FB, WM, WN>;
    if constexpr (bytes > 64 * 1024) {
        int device = 0;
        MI_HIP_CHECK(hipGetDevice(&device));
        static thread_local unsigned long raised = 0;      // devices
        if (device >= 64 || !(raised >> device & 1)) {
            MI_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
            if (device < 64) raised |= 1ul << device;
        }
    }
    const long tiles = static_cast<long>((p.M + TM - 1) / TM) * ((p.N + TN - 1) / TN);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((tiles + 7) / 8 * 8)), dim3(64 * WM * WN), bytes, st, p);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, int P, bool ZEROS>
int launch_form(const Int4Problem& p, hipStream_t st) {
    const long big = static_cast<long>((p.M + 127) / 128) * ((p.N + 255) / 256);
    if (big >= device_cu_count()) return launch<T, P, ZEROS, 4, 4, 2, 4>(p, st);      // 128 x 256
    return launch<T, P, ZEROS, 2, 2, 2, 2>(p, st);                                    // 64 x 64
}
template <typename T, int P>
int launch_zeros(const Int4Problem& p, hipStream_t st) { return p.zeros ? launch_form<T, P, true>(p, st) : launch_form<T, P, false>(p, st); }
template <typename T>
int launch_parts(const Int4Problem& p, int parts, hipStream_t st) {
    return parts == 1 ? launch_zeros<T, 1>(p, st) : parts == 2 ? launch_zeros<T, 2>(p, st) : launch_zeros<T, 4>(p, st);
}

}  // namespace
}  // namespace gemm

int launch_int4_tile(const Int4Problem& p, int dtype, int parts, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_parts<__bf16>(p, parts, st) : gemm::launch_parts<_Float16>(p, parts, st);
}

}  // namespace mi
