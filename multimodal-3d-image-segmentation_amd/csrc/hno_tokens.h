// Operand fragments, conversions and activations shared by the token kernels (hno_attention.hip, hno_linear.hip, hno_gncl.hip).
//
// Matrix products run on the 32 x 32 tile of one wave.  A fragment is 8 contraction elements of one operand row per lane:
//   lane l holds row (or column) l & 31; its elements are the contraction indices the instruction assigns to half h = l >> 5
//   result    lane l, register r holds row 8 (r / 4) + 4 h + r % 4 of column l & 31
// bf16: ONE v_mfma_f32_32x32x16_bf16 per fragment pair.  fp32: eight v_mfma_f32_32x32x2_f32 (element j of both halves per instruction).
// The sum does not depend on which index sits in which slot as long as both operands agree; the attention kernels use this to feed
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

struct TkF8 { float v[8]; };
template <typename T> struct TkFrag;
template <> struct TkFrag<tkh> {
    tkb8 v;
    __device__ __forceinline__ void set(int j, float x) { v[j] = (__bf16)x; }
};
template <> struct TkFrag<float> {
    float v[8];
    __device__ __forceinline__ void set(int j, float x) { v[j] = x; }
};

__device__ __forceinline__ tk16 tk_mma(const TkFrag<tkh> &a, const TkFrag<tkh> &b, tk16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ tk16 tk_mma(const TkFrag<float> &a, const TkFrag<float> &b, tk16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
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
// 8 elements of one tensor row starting at element d of D; `vec`: every row is 16-byte aligned and D % 8 == 0
template <typename T>
__device__ __forceinline__ TkFrag<T> tk_load8(const T *row, int d, int D, bool vec) {
    if (vec && d < D) return tk_row(row + d);
    TkFrag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.set(j, 0.f);
    if (!vec)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (d + j < D) f.set(j, tk_up(row[d + j]));
    return f;
}
// the fragment of the TRANSPOSE of a row-major LDS tile: column `col0 + (lane & 31)`, rows r0 .. r0 + 3 and r1 .. r1 + 3.
// bf16: ds_read_b64_tr_b16, which hands lane i of a group of 16 the column i of the 4 x 16 block whose rows the group's lanes address
__device__ __forceinline__ TkFrag<tkh> tk_col(const tkh *tile, int stride, int col0, int r0, int r1, int lane) {
    typedef __attribute__((address_space(3))) tks4 *lds4;
    const tkh *p = tile + ((lane & 15) >> 2) * stride + col0 + (lane & 16) + 4 * (lane & 3);
    const tks4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + r0 * stride));
    const tks4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + r1 * stride));
    return {__builtin_bit_cast(tkb8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7))};
}
__device__ __forceinline__ TkFrag<float> tk_col(const float *tile, int stride, int col0, int r0, int r1, int lane) {
    TkFrag<float> f;
    const float *p = tile + col0 + (lane & 31);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = p[(r0 + j) * stride], f.v[4 + j] = p[(r1 + j) * stride];
    return f;
}

// LDS-DMA: 64 lanes x 16 bytes from (wave-uniform base + per-lane byte offset) to 1024 consecutive LDS bytes at `dst` (wave-uniform).  No registers; retired by
// dma_wait (hno_common.h).  M0 holds the destination and is put back: the compiler owns it.
__device__ __forceinline__ void tk_dma16(const tkh *src, unsigned off, unsigned dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(src), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory");
}

// 16 bytes of padding behind each row of a tile: the row stride in 16-byte units is odd, so 8 lanes that read 16 bytes of 8
// consecutive rows cover all 64 banks' width once
template <typename T> constexpr int tk_pad() { return 16 / (int)sizeof(T); }

// ------------------------------------------------------------------ activations (ids: hno.h)
// 1 - Phi(|z|) = erfc(|z| / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (five terms, absolute error of erf 1.5e-7); e2 = exp(-z^2 / 2).  libm's erfcf
// took longer than the product itself in the epilogue of an 8192 x 8192 x 2048 product.
__device__ __forceinline__ float tk_phi_tail(float z, float &e2) {
    const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    e2 = __expf(-x * x);
    return 0.5f * p * t * e2;
}
// act(z); the derivative is a function of z, which the backward passes recompute or keep
__device__ __forceinline__ float tk_act(float z, int act) {
    switch (act) {
        case HNO_ACT_SELU: return z > 0.f ? HNO_SELU_SCALE * z : (HNO_SELU_SCALE * HNO_SELU_ALPHA) * neg_expm1(z);
        case HNO_ACT_ELU: return z > 0.f ? z : neg_expm1(z);
        case HNO_ACT_RELU: return z > 0.f ? z : (z == z ? 0.f : z);
        case HNO_ACT_GELU: {
            float e2;
            const float q = tk_phi_tail(z, e2);
            return fabsf(z) < 20.f ? z * (z > 0.f ? 1.f - q : q) : (z > 0.f ? z : (z == z ? 0.f : z));
        }
        case HNO_ACT_SILU: return z > -80.f ? z / (1.f + __expf(-z)) : (z == z ? 0.f : z);
        default: return z;
    }
}
__device__ __forceinline__ float tk_act_grad(float z, int act) {
    switch (act) {
        case HNO_ACT_SELU: return z > 0.f ? HNO_SELU_SCALE : (HNO_SELU_SCALE * HNO_SELU_ALPHA) * __expf(z);
        case HNO_ACT_ELU: return z > 0.f ? 1.f : __expf(z);
        case HNO_ACT_RELU: return z > 0.f ? 1.f : (z == z ? 0.f : z);
        case HNO_ACT_GELU: {
            if (!(fabsf(z) < 20.f)) return z > 0.f ? 1.f : (z == z ? 0.f : z);
            float e2;
            const float q = tk_phi_tail(z, e2);
            return (z > 0.f ? 1.f - q : q) + z * e2 * 0.39894228040143268f;
        }
        case HNO_ACT_SILU: {
            if (!(fabsf(z) < 80.f)) return z > 0.f ? 1.f : (z == z ? 0.f : z);
            const float s = 1.f / (1.f + __expf(-z));
            return s * (1.f + z * (1.f - s));
        }
        default: return 1.f;
    }
}

}  // namespace hno
