/*  p2hip_elem.h – what the kernels of a decoder's step share: element types, matrix products, transposing LDS reads,
 *  exchanges between lanes, values that are not finite, and the weights of a softmax.
 */
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace p2k {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

enum { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };
constexpr float kLog2e = 1.44269504088896340736f;

/* ── element types ─────────────────────────────────────────────────────────────────────────────────────────── */

template <int DT> struct Elem;
template <> struct Elem<T_F32> {
    typedef float type;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<T_F16> {
    typedef _Float16 type;
    static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <> struct Elem<T_BF16> {
    typedef __bf16 type;
    static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

/* 16 bytes of elements as floats, and back (each rounded to nearest even) */
template <int DT> constexpr int kPer16 = DT == T_F32 ? 4 : 8;

template <int DT> __device__ __forceinline__ void unpack(u4 r, float (&v)[kPer16<DT>])
{
    if constexpr (DT == T_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __uint_as_float(r[i]);
    } else if constexpr (DT == T_F16) {
        const h8 x = __builtin_bit_cast(h8, r);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(r[i] << 16);
            v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
}

template <int DT> __device__ __forceinline__ u4 pack(const float (&v)[kPer16<DT>])
{
    if constexpr (DT == T_F32) {
        return u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    } else if constexpr (DT == T_F16) {
        h8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (_Float16)v[i];
        return __builtin_bit_cast(u4, x);
    } else {
        b8 x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (__bf16)v[i];
        return __builtin_bit_cast(u4, x);
    }
}

/* the matrix products of 16-bit operands, bits as u4 */
template <int DT> __device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c)
{
    if constexpr (DT == T_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

template <int DT> __device__ __forceinline__ f16v mfma32(u4 a, u4 b, f16v c)
{
    if constexpr (DT == T_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

/* Transposing LDS read of 16-bit values: of the 4 × 16 values that the 16 lanes of a group address (lane i: 4 values,
 * row i / 4, columns 4·(i % 4) ..), lane i gets column i's four. */
__device__ __forceinline__ u2 lds_tr(uint32_t at)   /* an LDS byte address */
{
    typedef __attribute__((address_space(3))) s4 *lds4;
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at)));
}
__device__ __forceinline__ u2 lds_tr(const uint16_t *p)
{
    return lds_tr((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint16_t *)(p));
}

/* max and sum over lanes l, l ^ 16, l ^ 32, l ^ 48, and over l, l ^ 32 */
__device__ __forceinline__ float max_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_quarters(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_quarters(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

/* A sum to which 16 bytes of elements add 0, or a NaN if one of them is an infinity or a NaN: their products with zeros */
template <int DT> __device__ __forceinline__ float odd_sum(u4 v, float sum)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = v[i];   /* a bit cast of v[i] itself takes element 0, whatever i */
        if constexpr (DT == T_F32) sum = __builtin_fmaf(__uint_as_float(w), 0.0f, sum);
        else if constexpr (DT == T_F16) sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), h2{0, 0}, sum, false);
        else sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), b2{0, 0}, sum, false);
    }
    return sum;
}
template <int DT> __device__ __forceinline__ bool odd_values(u4 v)
{
    const float z = odd_sum<DT>(v, 0.0f);
    return z != z;
}

/* the infinities and NaN among 16 bytes of elements replaced by zeros */
template <int DT> __device__ __forceinline__ u4 only_finite(u4 v)
{
    constexpr uint32_t E = DT == T_F32 ? 0x7f800000u : DT == T_F16 ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t H = E & 0xffff0000u, L = E & 0xffffu;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t keep = 0xffffffffu;
        if ((v[i] & H) == H) keep = DT == T_F32 ? 0u : keep & 0xffffu;
        if (DT != T_F32 && (v[i] & L) == L) keep &= 0xffff0000u;
        v[i] &= keep;
    }
    return v;
}

/* Weights enter their product with V in the rows' type. fp16 keeps nothing under 2^-25, which many keys together, or one
 * with a large value beside values near 0, can make felt; so the reference that weights are taken from stands kLift powers
 * of two under the largest score (weights up to 2^kLift, and what is under 2^-(25 + kLift) of the largest is lost: 2^-40; kernels whose
 * sums of weights have to stay within the type lift by less and say so). Sums carry the same factor, so that it leaves with the division. bf16 ends where fp32 does and needs none. */
template <int DT> constexpr float kLift = DT == T_F16 ? 15.0f : 0.0f;

/* A score's place less the lift. In two instructions: as one, the constant or c would take a register of its own, which
 * attention_page of fp16 heads of 128 does not have (8 bytes a lane in scratch). */
__device__ __forceinline__ float lifted(float score, float c, float lift)
{
    float x = score * c;
    if (lift != 0.0f) {
        asm("" : "+v"(x));
        x -= lift;
    }
    return x;
}

}  // namespace p2k
