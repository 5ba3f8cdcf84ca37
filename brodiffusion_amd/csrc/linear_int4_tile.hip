// The linear layer with 4-bit weights for many rows (linear_int4.h).
//
// A work group of 4 wavefronts owns a tile of 16 TB tokens x 64 FB features, each wavefront all the tokens and 16 FB features: TB x FB blocks of
// v_mfma_f32_16x16x32. All operands come by LDS DMA in steps of 128 contraction elements (a block of packed weights) into a ring of S stages: X in rows of 256
// bytes, the piece of 16 bytes at position c of row r being piece c ^ (r % 16), so that the 16 rows of an operand read lie in 16 different bank groups; packed
// weights, operands already, a kilobyte for 16 features; scales and zero points. A step:
//   1. wait until all but the youngest S - 2 steps' loads of this wavefront have landed; barrier (and the stage before the ring's next is free)
//   2. the sums of x of the step, each 16 tokens by one wavefront, into LDS; the wavefront's weights to 16 bits, in registers for all tokens; barrier. With OWN a
//      wavefront sums for itself, along with its products, and the second barrier is gone: faster where a step is short
//   3. products: 16 tokens at a time against all the wavefront's features, a chain of matrix instructions per group from -z times the sum of x, scaled into the
//      accumulators; between them the loads of step + S - 1, dealt out: a request waits for those ahead of it (60 bytes a clock and compute unit)
// Bound: what a SIMD issues. 64 tokens x 64 features x 128 elements are 64 products and beside them 112 instructions of the weights, 64 that scale sums and about 60
// others; a 16 x 16 product takes the issue 12 of its 16 clocks, another vector instruction 4 (measured: one product and 1 to 4 others, two wavefronts, 17, 19.5,
// 24.4, 27.9 clocks). Tiles of 96 tokens spread the weights' instructions over half as many tokens more. 4608 x 6144 x 16384 bf16 (tokens, contraction, features) takes
// 0.89 to 0.93 ms from one GPU to the next, 1.0 PFLOP/s, the matrix pipes busy half of the time; groups of 64 with zero points 1.15 ms; this library's 16-bit layer of that size
// 0.77 to 0.80. It reads 2570 MiB where operands are 105: the tiles that an XCD has at one time are a strip of 96 tokens, and all weights pass for each strip. Few tiles are
// bound by latency instead: 4096 x 4608 x 1152, groups of 64, 75 to 83 us from memory (the 16-bit layer 57), one round of 64 x 192 with one step in flight, matrix pipes
// busy 28 %, vector instructions 43 %.
// Other ways: 32 x 32 products leave more room (32.3 clocks with 1, 33.5 with 6 others), but their accumulators came out slower at every size (970 us instead of 870 then), and
// so did wavefronts that take turns at products and weights (890), products, scaling and weights kept apart by scheduling barriers (0 to 3 % slower), and 6-bit conversions of
// 32 weights at once (as long as 28 instructions); without the sums of x and their barrier it would be 4 % faster, less than a launch that makes the sums ahead costs
// at most sizes. Neither built nor measured: a launch that writes q - z as 16-bit integers, which are exact, for tiles without conversions and sums of x.
#include <utility>

#include "linear_int4.h"

namespace mi {
namespace gemm {
namespace {

constexpr int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Sizes of a form: bytes of a stage's parts in LDS, DMA instructions of a wavefront for each (all wavefronts issue the same number: the wait counts them)
constexpr int kWaves = 4;
template <int P, bool ZEROS, int TB, int FB, int S>
struct TileForm {
    static constexpr int NW = kWaves, TM = 16 * TB, TN = 16 * FB * NW;
    static constexpr int XI = TM / 4 / NW, WI = ceil_div(TN / 16, NW);
    static constexpr int SD = ceil_div(TN * P, 128), ZD = ZEROS ? ceil_div(TN * P, 256) : 0;      // instructions of 256 bytes
    static constexpr int SI = ceil_div(SD, NW), ZI = ceil_div(ZD, NW), NI = XI + WI + SI + ZI;
    static constexpr int kW = TM * 256, kS = kW + TN / 16 * 1024, kZ = kS + SD * 256, kStage = kZ + ZD * 256;
    static constexpr int kSums = S * kStage, kBytes = kSums + P * TM * 4;
    static_assert(TM % (4 * NW) == 0, "the rows of a stage are dealt out evenly");
    static_assert(kBytes <= 160 * 1024, "LDS of a compute unit");
};

template <typename T, int P, bool ZEROS, int TB, int FB, int S, int SIMD, bool OWN>
__global__ void __launch_bounds__(64 * kWaves, SIMD) linear_int4_tile_kernel(const Int4Problem p) {
    using M = Mma<T>;
    using V8 = typename M::v8;
    using L = TileForm<P, ZEROS, TB, FB, S>;
    typedef T t4 __attribute__((ext_vector_type(4)));
    constexpr int NW = L::NW, TM = L::TM, TN = L::TN;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    float* const sums = reinterpret_cast<float*>(lds + L::kSums);      // [P][TM]

    const int tiles_n = (p.N + TN - 1) / TN, tiles_m = (p.M + TM - 1) / TM, n_tiles = tiles_m * tiles_n;
    // (every XCD takes a contiguous run of tiles, which share rows of X)
    const int chunk = (n_tiles + 7) >> 3, in_run = static_cast<int>(blockIdx.x) >> 3;
    const int logical = (static_cast<int>(blockIdx.x) & 7) * chunk + in_run;
    if (in_run >= chunk || logical >= n_tiles) return;
    const int m0 = (logical / tiles_n) * TM, n0 = (logical % tiles_n) * TN;

    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int last_block = (p.N + 15) / 16 - 1;

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
    // (the LDS destination travels in m0; the s_nop is the wait state an LDS-DMA instruction needs behind a write of m0. No memory clobber: what is read of
    // LDS between two barriers is another stage, and the barriers have one)
    auto dma16 = [](unsigned off, const unsigned char* base, unsigned dst) { asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(dst)); };
    auto dma4 = [](unsigned off, const unsigned char* base, unsigned dst) { asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "{m0}"(dst)); };
    const int share = static_cast<int>(blockIdx.y), begin = int4_share(p, share), end = int4_share(p, share + 1);
    int filling = 0, group = P == 1 ? begin / p.span : 0, of_group = P == 1 ? begin % p.span : 0;      // the stage that the next request fills; its group, of blocks and more, and which block of it
    // requests FROM .. TO - 1 of a step's L::NI
    auto request = [&]<int FROM, int TO>(int step, std::integer_sequence<int, FROM, TO>) {
        const int kb = min(step, end - 1);              // (past the end the last step again, into a stage that nobody reads: the wait counts instructions)
        const unsigned at = lds_base + filling * L::kStage;
        const int most = kb == p.KB - 1 ? left - 1 : 15;      // (pieces past the end: the last one, left out of the products)
        const int g0 = P == 1 ? min(group, p.groups - 1) : kb * P, most_g = p.groups - 1 - g0;
        [&]<int... I>(std::integer_sequence<int, I...>) {
            ([&] {
                constexpr int i = FROM + I;
                if constexpr (i < L::WI) dma16(lane * 16u, wg[i] + static_cast<long>(kb) * 1024, at + L::kW + wi[i] * 1024);
                else if constexpr (i < L::WI + L::SI) {
                    constexpr int u = i - L::WI;
                    dma4(soff[u] + (P == 1 ? 0u : static_cast<unsigned>(min(sg[u], most_g)) * (static_cast<unsigned>(p.N) * 2u)), static_cast<const unsigned char*>(p.scales) + static_cast<long>(g0) * p.N * 2,
                         at + L::kS + si[u] * 256);
                } else if constexpr (i < L::WI + L::SI + L::ZI) {
                    constexpr int u = i - L::WI - L::SI;
                    dma4(zoff[u] + (P == 1 ? 0u : static_cast<unsigned>(min(zg[u], most_g)) * static_cast<unsigned>(p.N)), p.zeros + static_cast<long>(g0) * p.N, at + L::kZ + zi[u] * 256);
                } else {
                    constexpr int u = i - L::WI - L::SI - L::ZI;
                    dma16(xoff[u] + static_cast<unsigned>(min(piece[u], most)) * 16u, xg + static_cast<long>(kb) * 256, at + (wave * L::XI + u) * 1024);
                }
            }(), ...);
        }(std::make_integer_sequence<int, TO - FROM>{});
        if constexpr (TO == L::NI && FROM < TO) {
            filling = filling + 1 == S ? 0 : filling + 1;
            if (++of_group == p.span) { of_group = 0; ++group; }
        }
    };

    f32x4 acc[FB][TB];
#pragma unroll
    for (int a = 0; a < FB; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
    for (int i = 0; i < S - 1; ++i) request(begin + i, std::integer_sequence<int, 0, L::NI>{});
    int reading = 0;
    for (int kb = begin; kb < end; ++kb) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((S - 2) * L::NI) : "memory");
        unsigned char* const stage = lds + reading * L::kStage;
        reading = reading + 1 == S ? 0 : reading + 1;
        auto tokens = [&](V8 (&x)[4], int row16) {      // operands of 16 tokens, block `row16` of the tile
            const unsigned char* const at = stage + row16 * 4096 + lr * 256;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const V8*>(at + (((4 * j + lg) ^ lr) << 4));
        };
        if (__builtin_expect(kb == p.KB - 1 && left < 16, 0)) {      // zeros behind the end of the rows: every wavefront those of the tokens that it sums
#pragma unroll
            for (int i = 0; i < ceil_div(TM / 16, NW); ++i) {
                const int b = i * NW + wave;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (b < TM / 16 && lr >= left) *reinterpret_cast<u32x4*>(stage + (16 * b + 4 * u + lg) * 256 + ((lr ^ (4 * u + lg)) << 4)) = u32x4{0u, 0u, 0u, 0u};
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
            if constexpr (OWN) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
#pragma unroll
        for (int i = 0; i < (OWN ? 0 : ceil_div(TM / 16, NW)); ++i) {
            const int b = i * NW + wave;
            if (TM / 16 % NW != 0 && b >= TM / 16) break;
            V8 x[4];
            tokens(x, b);
#pragma unroll
            for (int g = 0; g < P; ++g) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) s = M::run16(ones<T>(), x[j], s);
                if (lg == 0) sums[g * TM + 16 * b + lr] = s[0];
            }
        }
        V8 w[FB][4];
#pragma unroll
        for (int a = 0; a < FB; ++a) {
            const u32x4 packed = *reinterpret_cast<const u32x4*>(stage + L::kW + (wave * FB + a) * 1024 + lane * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[a][j] = nibbles<T>(packed[j]);
        }
        // scales and zero points of a wavefront's features wait in registers; where they would be 32 a lane and more they are read again for each 16 tokens,
        // one group at a time (the scheduling barrier: gathered ahead they do not fit the 256 registers)
        constexpr bool AGAIN = P * FB >= (SIMD == 3 && !OWN ? 4 : 8);
        float scale[FB][P][4];
        unsigned zero[FB][P];
        auto factors = [&](int g) {
#pragma unroll
            for (int a = 0; a < FB; ++a) {
                const int f = g * TN + (wave * FB + a) * 16 + 4 * lg;
                const t4 v = *reinterpret_cast<const t4*>(stage + L::kS + f * 2);
#pragma unroll
                for (int e = 0; e < 4; ++e) scale[a][g][e] = static_cast<float>(v[e]);
                if constexpr (ZEROS) zero[a][g] = *reinterpret_cast<const unsigned*>(stage + L::kZ + f);
            }
        };
        if constexpr (!AGAIN) {
#pragma unroll
            for (int g = 0; g < P; ++g) factors(g);
        }
        if constexpr (!OWN) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        V8 x[2][4];
        float sx[2][P];
        auto fetch = [&](int b) {
            tokens(x[b & 1], b);
#pragma unroll
            for (int g = 0; g < (OWN || AGAIN ? 0 : P); ++g) sx[b & 1][g] = sums[g * TM + 16 * b + lr];
        };
        fetch(0);
        [&]<int... B>(std::integer_sequence<int, B...>) {
            ([&] {
                constexpr int b = B;
                if constexpr (b + 1 < TB) fetch(b + 1);
                request(kb + S - 1, std::integer_sequence<int, b * L::NI / TB, (b + 1) * L::NI / TB>{});
#pragma unroll
                for (int g = 0; g < P; ++g) {
                    if constexpr (AGAIN) {
                        __builtin_amdgcn_sched_barrier(0);
                        asm volatile("" ::: "memory");
                        factors(g);
                        if constexpr (!OWN) sx[b & 1][g] = sums[g * TM + 16 * b + lr];
                    }
                    f32x4 t[FB];
#pragma unroll
                    for (int a = 0; a < FB; ++a)
#pragma unroll
                        for (int e = 0; e < 4; ++e) t[a][e] = OWN ? 0.f : -(ZEROS ? zero_point(zero[a][g], e) : 8.f) * sx[b & 1][g];
                    f32x4 total = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (OWN) {
#pragma unroll
                        for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j) total = M::run16(ones<T>(), x[b & 1][j], total);
                    }
#pragma unroll
                    for (int j = g * 4 / P; j < (g + 1) * 4 / P; ++j)
#pragma unroll
                        for (int a = 0; a < FB; ++a) t[a] = M::run16(w[a][j], x[b & 1][j], t[a]);
#pragma unroll
                    for (int a = 0; a < FB; ++a)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if constexpr (OWN) t[a][e] = __builtin_fmaf(ZEROS ? -zero_point(zero[a][g], e) : -8.f, total[e], t[a][e]);
                            acc[a][b][e] = __builtin_fmaf(t[a][e], scale[a][g][e], acc[a][b][e]);
                        }
                }
            }(), ...);
        }(std::make_integer_sequence<int, TB>{});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (no DMA into LDS that is given back)

    if (p.parts) {
        float* const to = p.parts + static_cast<long>(share) * p.M * p.N;
#pragma unroll
        for (int a = 0; a < FB; ++a)
#pragma unroll
            for (int b = 0; b < TB; ++b) {
                const int f = n0 + (wave * FB + a) * 16 + 4 * lg, m = m0 + 16 * b + lr;
                if (f < p.N && m < p.M) *reinterpret_cast<f32x4*>(to + static_cast<long>(m) * p.N + f) = acc[a][b];
            }
        return;
    }
    // (all of the bias and the residual on their way before the first is used: their latency once, not for each block)
    t4 bias[FB], res[FB][TB];
    if (p.bias) {
#pragma unroll
        for (int a = 0; a < FB; ++a) bias[a] = *reinterpret_cast<const t4*>(static_cast<const T*>(p.bias) + min(n0 + (wave * FB + a) * 16 + 4 * lg, p.N - 4));
    }
    if (p.residual) {
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            const T* const row = static_cast<const T*>(p.residual) + static_cast<long>(min(m0 + 16 * b + lr, p.M - 1)) * p.ldr;
#pragma unroll
            for (int a = 0; a < FB; ++a) res[a][b] = *reinterpret_cast<const t4*>(row + min(n0 + (wave * FB + a) * 16 + 4 * lg, p.N - 4));
        }
    }
    auto finish = [&](auto act) {
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            const int m = m0 + 16 * b + lr;
            T* const row = static_cast<T*>(p.y) + static_cast<long>(m) * p.ldy;
#pragma unroll
            for (int a = 0; a < FB; ++a) {
                const int f = n0 + (wave * FB + a) * 16 + 4 * lg;
                f32x4 v = acc[a][b];
                if (p.bias) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(bias[a][e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = act(v[e]);
                if (p.residual) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += static_cast<float>(res[a][b][e]);
                }
                t4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(v[e]);
                if (m < p.M && f < p.N) *reinterpret_cast<t4*>(row + f) = o;
            }
        }
    };
    if (p.act == MI_ACT_NONE) finish([](float v) { return v; });
    else with_activation(p.act, finish);
}

template <typename T, int P, bool ZEROS, int TB, int FB, int S, int SIMD, bool OWN>
int launch(const Int4Problem& p, hipStream_t st) {
    using L = TileForm<P, ZEROS, TB, FB, S>;
    constexpr int TM = L::TM, TN = L::TN, bytes = L::kBytes;
    const auto kernel = &linear_int4_tile_kernel<T, P, ZEROS, TB, FB, S, SIMD, OWN>;
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
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((tiles + 7) / 8 * 8), p.shares), dim3(64 * kWaves), bytes, st, p);
    MI_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, int P, bool ZEROS>
int launch_form(const Int4Problem& p, int form, hipStream_t st) {
    // Stages, wavefronts a SIMD and who sums x, by measurement. 32 tokens, a step is short: 3 stages and own sums (333 x 2240 x 6720, groups of 64: 29 us;
    // 2 stages 33, shared sums 36, 4 stages and 2 wavefronts 36; 128 x 4608 x 4608: 23, 29, 30, 24). More tokens: 2 stages and shared sums, so that three work groups of
    // 64 x 128 fit a compute unit (4096 x 4608 x 1152 from the last-level cache: 70 us; two of 3 stages 87 to 94, own sums as many) and two of the others.
    switch (form) {
        case kTile32x64: return launch<T, P, ZEROS, 2, 1, 3, 4, true>(p, st);
        case kTile32x128: return launch<T, P, ZEROS, 2, 2, 3, 3, true>(p, st);
        case kTile64x128: return launch<T, P, ZEROS, 4, 2, 2, 3, false>(p, st);
        case kTile64x192: return launch<T, P, ZEROS, 4, 3, 2, 2, false>(p, st);
        case kTile64x256:
            if constexpr (P == 1) return launch<T, P, ZEROS, 4, 4, 2, 2, false>(p, st);
        default: return launch<T, P, ZEROS, 6, 3, 2, 2, false>(p, st);
    }
}
template <typename T, int P>
int launch_zeros(const Int4Problem& p, int form, hipStream_t st) { return p.zeros ? launch_form<T, P, true>(p, form, st) : launch_form<T, P, false>(p, form, st); }
template <typename T>
int launch_parts(const Int4Problem& p, int parts, int form, hipStream_t st) {
    return parts == 1 ? launch_zeros<T, 1>(p, form, st) : parts == 2 ? launch_zeros<T, 2>(p, form, st) : launch_zeros<T, 4>(p, form, st);
}

}  // namespace
}  // namespace gemm

int launch_int4_tile(const Int4Problem& p, int dtype, int parts, int form, hipStream_t st) {
    return dtype == MI_DTYPE_BF16 ? gemm::launch_parts<__bf16>(p, parts, form, st) : gemm::launch_parts<_Float16>(p, parts, form, st);
}

}  // namespace mi
