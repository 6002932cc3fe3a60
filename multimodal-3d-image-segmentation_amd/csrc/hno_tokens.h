// Operand fragments, conversions and activations shared by the token kernels (hno_attention.hip, hno_linear.hip, hno_gncl.hip).
//
// Matrix products run on the 32 x 32 tile of one wave.  A fragment is 8 contraction elements of one operand row per lane:
//   lane l holds row (or column) l & 31; its elements are the contraction indices the instruction assigns to half h = l >> 5
//   result    lane l, register r holds row 8 (r / 4) + 4 h + r % 4 of column l & 31
// on v_mfma_f32_32x32x16_bf16.  fp32 values are three bf16 terms: the leading 8 bits, the next 8 and the last 8 (cut, not rounded: their sum is the value); a product
// is the six products of terms down to 2^-16, smallest first -- the two dropped ones are at most 2^-22, on average 2^-25, of it.  The fp32 matrix instruction takes
// 2.7 times as long for the same work.  (An infinity becomes inf + NaN + NaN: products with it are NaN, which linear forms again in fp32 and attention leaves.)
// A sum does not depend on which index sits in which slot as long as both operands agree; the attention kernels use this to feed
// a result back as an operand without moving it between lanes: registers 8 t .. 8 t + 7 of a result are the fragment whose
// slots stand for rows 16 t + 4 h + {0..3} and 16 t + 8 + 4 h + {0..3}.
#pragma once
#include "hno_common.h"

namespace hno {

typedef unsigned short tkh;                                          // bf16 in memory
typedef __bf16 tkb8 __attribute__((ext_vector_type(8)));
typedef short tks4 __attribute__((ext_vector_type(4)));
typedef float tk16 __attribute__((ext_vector_type(16)));
typedef float tkf4 __attribute__((ext_vector_type(4)));
typedef unsigned tku4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float tk_up(float v) { return v; }
__device__ __forceinline__ float tk_up(tkh v) { return __uint_as_float((unsigned)v << 16); }
template <typename T> __device__ __forceinline__ T tk_down(float v);
template <> __device__ __forceinline__ float tk_down<float>(float v) { return v; }
template <> __device__ __forceinline__ tkh tk_down<tkh>(float v) { return __builtin_bit_cast(tkh, (__bf16)v); }   // to nearest even

// 8 values of a type as they lie in memory
template <typename T> struct TkFrag;
template <> struct TkFrag<tkh> {
    tkb8 v;
    __device__ __forceinline__ void set(int j, float x) { v[j] = (__bf16)x; }
};
template <> struct TkFrag<float> {
    float v[8];
    __device__ __forceinline__ void set(int j, float x) { v[j] = x; }
};
// the same as an operand: its bf16 terms
template <typename T> constexpr int tk_planes() { return sizeof(T) == 2 ? 1 : 3; }
template <typename T> struct TkOp { TkFrag<tkh> p[tk_planes<T>()]; };
__device__ __forceinline__ TkOp<tkh> tk_op(const TkFrag<tkh> &f) { return {{f}}; }
__device__ __forceinline__ TkOp<float> tk_op(const TkFrag<float> &f) {
    TkOp<float> o;
    tku4 h[3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned a = __float_as_uint(f.v[2 * j]), b = __float_as_uint(f.v[2 * j + 1]);
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            h[t][j] = __builtin_amdgcn_perm(b, a, 0x07060302);
            a = __float_as_uint(__uint_as_float(a) - __uint_as_float(a & 0xffff0000u));
            b = __float_as_uint(__uint_as_float(b) - __uint_as_float(b & 0xffff0000u));
        }
    }
#pragma unroll
    for (int t = 0; t < 3; ++t) o.p[t].v = __builtin_bit_cast(tkb8, h[t]);
    return o;
}
template <typename T>
__device__ __forceinline__ tk16 tk_mma(const TkOp<T> &a, const TkOp<T> &b, tk16 c) {
    constexpr int P = tk_planes<T>();
#pragma unroll
    for (int t = P - 1; t >= 0; --t)
#pragma unroll
        for (int p = 0; p <= t; ++p) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[p].v, b.p[t - p].v, c, 0, 0, 0);
    return c;
}

// 8 consecutive elements from LDS or memory, 16-byte aligned
__device__ __forceinline__ TkFrag<tkh> tk_row(const tkh *p) { return {__builtin_bit_cast(tkb8, *reinterpret_cast<const tku4 *>(p))}; }
__device__ __forceinline__ TkFrag<float> tk_row(const float *p) {
    TkFrag<float> f;
    const tkf4 a = *reinterpret_cast<const tkf4 *>(p), b = *reinterpret_cast<const tkf4 *>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = a[j], f.v[4 + j] = b[j];
    return f;
}
__device__ __forceinline__ void tk_store8(tkh *p, const TkFrag<tkh> &f) { *reinterpret_cast<tku4 *>(p) = __builtin_bit_cast(tku4, f.v); }
__device__ __forceinline__ void tk_store8(float *p, const TkFrag<float> &f) {
    *reinterpret_cast<tkf4 *>(p) = tkf4{f.v[0], f.v[1], f.v[2], f.v[3]};
    *reinterpret_cast<tkf4 *>(p + 4) = tkf4{f.v[4], f.v[5], f.v[6], f.v[7]};
}
// LDS-DMA: 64 lanes x 16 bytes from (wave-uniform base + per-lane byte offset) to 1024 consecutive LDS bytes at `dst` (wave-uniform).  No registers; retired by
// dma_wait (hno_common.h).  M0 holds the destination.
__device__ __forceinline__ void tk_dma16(const tkh *src, unsigned off, unsigned dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(src), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
}

// ------------------------------------------------------------------ activations (ids: hno.h)
// 1 - Phi(|z|) = erfc(|z| / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (five terms, absolute error of erf 1.5e-7); e2 = exp(-z^2 / 2).  libm's erfcf
// took longer than the product itself in the epilogue of an 8192 x 8192 x 2048 product.
__device__ __forceinline__ float tk_phi_tail(float z, float &e2) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
    float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    p = fmaf(p, t, 0.5f * 1.421413741f);
    p = fmaf(p, t, 0.5f * -0.284496736f);
    p = fmaf(p, t, 0.5f * 0.254829592f);
    e2 = __builtin_amdgcn_exp2f(z * z * (-0.5f * 1.4426950408889634f));
    return p * t * e2;
}
// act(z); the derivative is a function of z, which the backward passes recompute or keep.  Infinite arguments give the limits and NaN stays NaN without
// comparisons: where a factor is 0 the other one is bounded, and at a NaN the factor beside the bounded one is NaN.
__device__ __forceinline__ float tk_act(float z, int act) {
    switch (act) {
        case HNO_ACT_SELU: return z > 0.f ? HNO_SELU_SCALE * z : (HNO_SELU_SCALE * HNO_SELU_ALPHA) * neg_expm1(z);
        case HNO_ACT_ELU: return z > 0.f ? z : neg_expm1(z);
        case HNO_ACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);
        case HNO_ACT_GELU: {
            float e2;
            const float q = tk_phi_tail(z, e2);
            return fmaf(-fminf(fabsf(z), 20.f), q, fmaxf(z, 0.f));          // z > 0: z (1 - q), else z q
        }
        case HNO_ACT_SILU: return fmaxf(z, -200.f) * __builtin_amdgcn_rcpf(1.f + __expf(-z));
        default: return z;
    }
}
__device__ __forceinline__ float tk_act_grad(float z, int act) {
    switch (act) {
        case HNO_ACT_SELU: return z > 0.f ? HNO_SELU_SCALE : (HNO_SELU_SCALE * HNO_SELU_ALPHA) * __expf(z);
        case HNO_ACT_ELU: return z > 0.f ? 1.f : __expf(z);
        case HNO_ACT_RELU: return z > 0.f ? 1.f : (z == z ? 0.f : z);
        case HNO_ACT_GELU: {
            float e2;
            const float q = tk_phi_tail(z, e2);
            return fmaf(fminf(fmaxf(z, -20.f), 20.f) * 0.39894228040143268f, e2, z > 0.f ? 1.f - q : q);
        }
        case HNO_ACT_SILU: {
            const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
            return s * fmaf(fminf(fmaxf(z, -200.f), 200.f), 1.f - s, 1.f);
        }
        default: return 1.f;
    }
}

}  // namespace hno
