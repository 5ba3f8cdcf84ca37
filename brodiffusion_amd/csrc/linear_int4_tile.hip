// The linear layer with 4-bit weights for many rows (linear_int4.h).
//
// A work group owns a tile of tokens x features, 16 TB WM x 16 FB WN, of WM x WN wavefronts with TB x FB blocks of v_mfma_f32_16x16x32 each. All operands
// come by LDS DMA in steps of 128 contraction elements (a block of packed weights) into a ring of S stages: X in rows of 256 bytes, the piece of 16 bytes at
// position c of row r being piece c ^ (r % 16), so that the 16 rows of an operand read lie in 16 different bank groups; packed weights, operands already, a kilobyte
// each; scales and zero points. A step:
//   1. wait until all but the youngest S - 2 steps' loads of this wavefront have landed; barrier (and the stage before the ring's next is free)
//   2. request step + S - 1
//   3. the sums of x of the step, each 16 tokens by one wavefront, into LDS; the wavefront's weights to 16 bits, in registers for all its tokens; barrier
//   4. products: 16 tokens at a time against all the wavefront's features, a chain of matrix instructions per group from -z times the sum of x, scaled into the
//      accumulators
#include "linear_int4.h"

namespace mi {
namespace gemm {
namespace {

constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Sizes of a form: bytes of a stage's parts in LDS, DMA instructions of a wavefront for each (all wavefronts issue the same number: the wait counts them)
template <int P, bool ZEROS, int TB, int FB, int WM, int WN, int S>
struct TileForm {
    static constexpr int NW = WM * WN, TM = 16 * TB * WM, TN = 16 * FB * WN;
    static constexpr int XI = TM / 4 / NW, WI = ceil_div(TN / 16, NW);
    static constexpr int SD = ceil_div(TN * P, 128), ZD = ZEROS ? ceil_div(TN * P, 256) : 0;      // instructions of 256 bytes
    static constexpr int SI = ceil_div(SD, NW), ZI = ceil_div(ZD, NW), NI = XI + WI + SI + ZI;
    static constexpr int kW = TM * 256, kS = kW + TN / 16 * 1024, kZ = kS + SD * 256, kStage = kZ + ZD * 256;
    static constexpr int kSums = S * kStage, kBytes = kSums + P * TM * 4;
    static_assert(TM % (4 * NW) == 0, "the rows of a stage are dealt out evenly");
    static_assert(kBytes <= 160 * 1024, "LDS of a compute unit");
};

template <typename T, int P, bool ZEROS, int TB, int FB, int WM, int WN, int S, bool TURNS>
__global__ void __launch_bounds__(64 * WM * WN) linear_int4_tile_kernel(const Int4Problem p) {
    using M = Mma<T>;
    using V8 = typename M::v8;
    using L = TileForm<P, ZEROS, TB, FB, WM, WN, S>;
    typedef T t4 __attribute__((ext_vector_type(4)));
    constexpr int TM = L::TM, TN = L::TN;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    float* const sums = reinterpret_cast<float*>(lds + L::kSums);      // [P][TM]

    const int tiles_n = (p.N + TN - 1) / TN, tiles_m = (p.M + TM - 1) / TM, n_tiles = tiles_m * tiles_n;
    // (every XCD takes a contiguous run of tiles, which share rows of X)
    const int chunk = (n_tiles + 7) >> 3, in_run = static_cast<int>(blockIdx.x) >> 3;
    const int logical = (static_cast<int>(blockIdx.x) & 7) * chunk + in_run;
    if (in_run >= chunk || logical >= n_tiles) return;
    const int m0 = (logical / tiles_n) * TM, n0 = (logical % tiles_n) * TN;

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = TURNS ? wave / WN : wave % WM, wn = TURNS ? wave % WN : wave / WM;      // (wavefronts w and w + 4 share a SIMD)
    const int nw = n0 + wn * 16 * FB, last_block = (p.N + 15) / 16 - 1;

    // ── DMA: addresses as a uniform base and an offset per lane ──
    const unsigned char* const xg = static_cast<const unsigned char*>(p.x) + static_cast<long>(m0) * p.ldx * 2;
    unsigned xoff[L::XI];
    int piece[L::XI];
#pragma unroll
    for (int u = 0; u < L::XI; ++u) {
        const int r = 4 * (wave * L::XI + u) + lg;
        piece[u] = lr ^ (r & 15);
        xoff[u] = static_cast<unsigned>(min(r, p.M - 1 - m0)) * (static_cast<unsigned>(p.ldx) * 2u);
    }
    const unsigned char* wg[L::WI];
    int wi[L::WI], si[L::SI];
#pragma unroll
    for (int u = 0; u < L::WI; ++u) {
        wi[u] = min(wave * L::WI + u, TN / 16 - 1);
        wg[u] = static_cast<const unsigned char*>(p.w) + static_cast<long>(min(n0 / 16 + wi[u], last_block)) * p.KB * 1024;
    }
    // a lane's word of scales is 2 features of a group, of zero points 4 (words past a step's last are that one again)
    int sg[L::SI], zg[L::ZI ? L::ZI : 1], zi[L::ZI ? L::ZI : 1];
    unsigned soff[L::SI], zoff[L::ZI ? L::ZI : 1];
#pragma unroll
    for (int u = 0; u < L::SI; ++u) {
        si[u] = min(wave * L::SI + u, L::SD - 1);
        const int d = min(si[u] * 64 + lane, P * TN / 2 - 1);
        sg[u] = d / (TN / 2);
        soff[u] = static_cast<unsigned>(min(n0 + d % (TN / 2) * 2, p.N - 2)) * 2u;
    }
#pragma unroll
    for (int u = 0; u < L::ZI; ++u) {
        zi[u] = min(wave * L::ZI + u, L::ZD - 1);
        const int d = min(zi[u] * 64 + lane, P * TN / 4 - 1);
        zg[u] = d / (TN / 4);
        zoff[u] = static_cast<unsigned>(min(n0 + d % (TN / 4) * 4, p.N - 4));
    }
    const unsigned lds_base = static_cast<unsigned>(reinterpret_cast<size_t>((__attribute__((address_space(3))) unsigned char*)lds));
    const int left = (p.K - (p.KB - 1) * 128) / 8;      // pieces of the last block's rows
    // (the LDS destination travels in m0; the s_nop is the wait state an LDS-DMA instruction needs behind a write of m0)
    auto dma16 = [](unsigned off, const unsigned char* base, unsigned dst) { asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(dst) : "memory"); };
    auto dma4 = [](unsigned off, const unsigned char* base, unsigned dst) { asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "{m0}"(dst) : "memory"); };
    int filling = 0;                                    // the stage that the next request fills
    auto request = [&](int step) {
        const int kb = min(step, p.KB - 1);             // (past the end the last step again, into a stage that nobody reads: the wait counts instructions)
        const unsigned at = lds_base + filling * L::kStage;
        filling = filling + 1 == S ? 0 : filling + 1;
        const int most = kb == p.KB - 1 ? left - 1 : 15;      // (pieces past the end: the last one, left out of the products)
        const unsigned char* const base = xg + static_cast<long>(kb) * 256;
#pragma unroll
        for (int u = 0; u < L::WI; ++u) dma16(lane * 16u, wg[u] + static_cast<long>(kb) * 1024, at + L::kW + wi[u] * 1024);
        const int g0 = P == 1 ? kb / p.span : kb * P, most_g = p.groups - 1 - g0;
        const unsigned char* const sbase = static_cast<const unsigned char*>(p.scales) + static_cast<long>(g0) * p.N * 2;
#pragma unroll
        for (int u = 0; u < L::SI; ++u) dma4(soff[u] + (P == 1 ? 0u : static_cast<unsigned>(min(sg[u], most_g)) * (static_cast<unsigned>(p.N) * 2u)), sbase, at + L::kS + si[u] * 256);
#pragma unroll
        for (int u = 0; u < L::ZI; ++u)
            dma4(zoff[u] + (P == 1 ? 0u : static_cast<unsigned>(min(zg[u], most_g)) * static_cast<unsigned>(p.N)), p.zeros + static_cast<long>(g0) * p.N, at + L::kZ + zi[u] * 256);
#pragma unroll
        for (int u = 0; u < L::XI; ++u) dma16(xoff[u] + static_cast<unsigned>(min(piece[u], most)) * 16u, base, at + (wave * L::XI + u) * 1024);
    };

    f32x4 acc[FB][TB];
#pragma unroll
    for (int a = 0; a < FB; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (int i = 0; i < S - 1; ++i) request(i);
    int reading = 0;
    bool short_block = false;
    const unsigned char* stage = lds;
    V8 w[FB][4];
    // scales and zero points of a wavefront's features wait in registers, but for groups of 32, whose 16 FB values a lane would put others into memory:
    // those are read again for each 16 tokens
    constexpr bool AGAIN = P == 4;
    float scale[FB][P][4];
    unsigned zero[FB][P];
    auto factors = [&](int g) {
#pragma unroll
        for (int a = 0; a < FB; ++a) {
            const int f = g * TN + (wn * FB + a) * 16 + 4 * lg;
            const t4 v = *reinterpret_cast<const t4*>(stage + L::kS + f * 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) scale[a][g][e] = static_cast<float>(v[e]);
            if constexpr (ZEROS) zero[a][g] = *reinterpret_cast<const unsigned*>(stage + L::kZ + f);
        }
    };
    auto tokens = [&](V8 (&x)[4], int row16) {      // operands of 16 tokens, block `row16` of the tile
        const unsigned char* const at = stage + row16 * 4096 + lr * 256;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const V8*>(at + (((4 * j + lg) ^ lr) << 4));
        if (short_block) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * j + lg >= left) x[j] = V8{};
        }
    };
    // part 3 of a step: the sums of the 16-token blocks that the WN wavefronts of these tokens share out
    auto prepare = [&](int kb) {
        stage = lds + reading * L::kStage;
        reading = reading + 1 == S ? 0 : reading + 1;
        short_block = kb == p.KB - 1 && left < 16;
#pragma unroll
        for (int i = 0; i < ceil_div(TB, WN); ++i) {
            const int b = i * WN + wn;
            if (TB % WN != 0 && b >= TB) break;
            V8 x[4];
            tokens(x, wm * TB + b);
#pragma unroll
            for (int g = 0; g < P; ++g) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) s = M::run16(ones<T>(), x[j], s);
                if (lg == 0) sums[g * TM + 16 * (wm * TB + b) + lr] = s[0];
            }
        }
#pragma unroll
        for (int a = 0; a < FB; ++a) {
            const u32x4 packed = *reinterpret_cast<const u32x4*>(stage + L::kW + (wn * FB + a) * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[a][j] = nibbles<T>(packed[j]);
        }
        if constexpr (!AGAIN) {
#pragma unroll
            for (int g = 0; g < P; ++g) factors(g);
        }
    };
    auto products = [&] {
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            V8 x[4];
            tokens(x, wm * TB + b);
#pragma unroll
            for (int g = 0; g < P; ++g) {
                const float sx = sums[g * TM + 16 * (wm * TB + b) + lr];
                if constexpr (AGAIN) {
                    asm volatile("" ::: "memory");
                    factors(g);
                }
#pragma unroll
                for (int a = 0; a < FB; ++a) {
                    f32x4 t;
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = -(ZEROS ? zero_point(zero[a][g], e) : 8.f) * sx;
#pragma unroll
                    for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) t = M::run16(w[a][j], x[j], t);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][b][e] = __builtin_fmaf(t[e], scale[a][g][e], acc[a][b][e]);
                }
            }
        }
    };
    if constexpr (TURNS) {
        // The two wavefronts of a SIMD take turns: while one multiplies the other makes its weights. Wavefronts of wm = 1 are a part of a step behind; a step's
        // loads are requested where the first of them multiply and the others prepare, and waited for at the end of that.
        static_assert(WM == 2 && WN == 4);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((S - 2) * L::NI) : "memory");
        if (wm == 1) asm volatile("s_barrier" ::: "memory");
        for (int kb = 0; kb < p.KB; ++kb) {
            if (wm == 1) request(kb + S - 1);
            prepare(kb);
            if (wm == 1) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((S - 2) * L::NI) : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (wm == 0) request(kb + S - 1);
            products();
            if (wm == 0) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((S - 2) * L::NI) : "memory");
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (wm == 0) asm volatile("s_barrier" ::: "memory");
    } else {
        for (int kb = 0; kb < p.KB; ++kb) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((S - 2) * L::NI) : "memory");
            request(kb + S - 1);
            prepare(kb);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            products();
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (no DMA into LDS that is given back)

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

template <typename T, int P, bool ZEROS, int TB, int FB, int WM, int WN, int S, bool TURNS>
int launch(const Int4Problem& p, hipStream_t st) {
    using L = TileForm<P, ZEROS, TB, FB, WM, WN, S>;
    constexpr int TM = L::TM, TN = L::TN, bytes = L::kBytes;
    const auto kernel = &linear_int4_tile_kernel<T, P, ZEROS, TB, FB, WM, WN, S, TURNS>;
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
    if (big >= device_cu_count()) return launch<T, P, ZEROS, 4, 4, 2, 4, 3, true>(p, st);      // 128 x 256
    return launch<T, P, ZEROS, 2, 2, 2, 2, 3, false>(p, st);                                    // 64 x 64
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
