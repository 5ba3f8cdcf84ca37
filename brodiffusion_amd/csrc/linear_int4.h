// The linear layer with 4-bit weights: what its kernels share (linear_int4.hip: entries and choice; linear_int4_few.hip, linear_int4_tile.hip).
//
//   Y[m][n] = act(sum over groups g of s[g][n] (sum over k in g of q[n][k] x[m][k] - z[g][n] sum over k in g of x[m][k]) + bias[n]) + residual[m][n]
// q is 0 .. 15 and becomes 16-bit operands of the matrix instructions exactly; a group's product is summed in FP32, starting at -z times the sum of its x (a
// product of x with ones, by the same instructions), and meets its scale in FP32. No weight is rounded. Subtracting z from the operands instead would take four
// more instructions for 8 weights of fp16 and far more of bf16, which has no packed subtraction.
//
// Packed weights: blocks of 16 features x 128 contraction elements, 1024 bytes, those of 16 features behind one another. Lane l of a wavefront holds bytes
// [16 l, 16 l + 16) of a block: row l % 16, in word j the elements k = 32 j + 8 (l / 16) .. + 8: the operand of v_mfma_f32_16x16x32 number j. Element i < 4 of a
// word lies in bits [8 i, 8 i + 4), element 4 + i above it: two ANDs and a shift leave bytes 0 .. 15, which as FP8 (E4M3) are multiples of 2^-9, the smallest
// subnormal numbers and the first binade behind them, and v_cvt_scalef32_pk_*_fp8 makes two of them 16-bit at 2^9 each: 7 instructions for 8 weights.
#pragma once
#include "linear_int4_forms.h"
#include "linear_math.h"

namespace mi {

struct Int4Problem {
    const void* x; const void* w;
    const void* scales;            // (groups, N) of T
    const unsigned char* zeros;    // (groups, N) or null: 8
    const void* bias; const void* residual; void* y;      // bias and residual may be null
    int M, N, K;
    int KB, groups, span;          // blocks of 128 contraction elements, groups, blocks that share a group (groups of 128 and more)
    long ldx, ldy, ldr;            // elements
    int act;                       // MI_ACT_*
    float* parts;                  // null, or (shares, M, N): the contraction in shares, whose sums go here
    int shares;
};
// the blocks of a share of the contraction
__device__ __forceinline__ int int4_share(const Int4Problem& p, int share) { return static_cast<int>(static_cast<long>(share) * p.KB / p.shares); }
// scale groups in a block: 4, 2, 1 (of 32, 64, 128 and more elements)
inline int int4_parts(int group) { return group >= 128 ? 1 : 128 / group; }

int launch_int4_few(const Int4Problem& p, int dtype, int parts, int form, hipStream_t st);
int launch_int4_tile(const Int4Problem& p, int dtype, int parts, int form, hipStream_t st);

namespace gemm {

template <typename T> struct Nibbles;
template <> struct Nibbles<__bf16> {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    template <bool HIGH> static __device__ __forceinline__ unsigned two(unsigned bytes) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.f, HIGH));
    }
    static constexpr unsigned kOnes = 0x3f803f80u;
};
template <> struct Nibbles<_Float16> {
    template <bool HIGH> static __device__ __forceinline__ unsigned two(unsigned bytes) {
        return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, HIGH));
    }
    static constexpr unsigned kOnes = 0x3c003c00u;
};
// a word of packed weights -> 8 values of T, exactly
template <typename T> __device__ __forceinline__ typename Mma<T>::v8 nibbles(unsigned w) {
    unsigned mask = 0x0f0f0f0fu;
    asm("" : "+s"(mask));                         // (a literal would double the instruction's length)
    const unsigned lo = w & mask, hi = (w >> 4) & mask;
    using N = Nibbles<T>;
    const u32x4 r = {N::template two<false>(lo), N::template two<true>(lo), N::template two<false>(hi), N::template two<true>(hi)};
    return __builtin_bit_cast(typename Mma<T>::v8, r);
}
template <typename T> __device__ __forceinline__ typename Mma<T>::v8 ones() {
    using N = Nibbles<T>;
    return __builtin_bit_cast(typename Mma<T>::v8, u32x4{N::kOnes, N::kOnes, N::kOnes, N::kOnes});
}
// byte e of z as FP32
__device__ __forceinline__ float zero_point(unsigned z, int e) { return static_cast<float>((z >> (8 * e)) & 0xffu); }

}  // namespace gemm
}  // namespace mi
