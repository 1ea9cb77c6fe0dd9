// ifa_fp8.h -- device helpers of the operators over 8-bit floating point (e4m3: four significant bits, largest value 448, one NaN a sign,
// no infinities) with a 32-bit scale for each block of 128 columns (activations) or 128 x 128 values (matrices).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/inferflow_amd.h"
#include "ifa_f32_common.h"

namespace ifa8 {

using ifa32::bf16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int BLOCK = 128;
constexpr float SCALE_MIN = 1.1754943508222875e-38f;      // 2^-126: its reciprocal is finite, and a block of zeros has it

__host__ __device__ constexpr size_t blocks_of(size_t n) { return (n + BLOCK - 1) / BLOCK; }

// ---- values of the three activation types
template <int DT> struct Elem;
template <> struct Elem<IFA_F32> { typedef float type; };
template <> struct Elem<IFA_F16> { typedef _Float16 type; };
template <> struct Elem<IFA_BF16> { typedef __bf16 type; };
inline size_t elem_bytes(int dt) { return dt == IFA_F32 ? 4 : 2; }
inline bool elem_known(int dt) { return dt == IFA_F32 || dt == IFA_F16 || dt == IFA_BF16; }

// 16 bytes: four 32-bit values or eight 16-bit ones
template <int DT> constexpr int VEC = DT == IFA_F32 ? 4 : 8;
template <int DT> __device__ __forceinline__ void unpack(const u32x4 v, float *f)
{
    if constexpr (DT == IFA_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(v[i]);
    } else if constexpr (DT == IFA_BF16) {
#pragma unroll
        for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(v[i] << 16); f[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u); }
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; i++) { const uint32_t u = v[i]; const h2 h = __builtin_bit_cast(h2, u); f[2 * i] = (float)h[0]; f[2 * i + 1] = (float)h[1]; }
    }
}
// one rounding, to the nearest even; what was rounded comes back in f
template <int DT> __device__ __forceinline__ u32x4 pack(float *f)
{
    u32x4 v;
    if constexpr (DT == IFA_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __float_as_uint(f[i]);
    } else {
        typedef typename Elem<DT>::type e2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            e2 h;
            h[0] = (typename Elem<DT>::type)f[2 * i]; h[1] = (typename Elem<DT>::type)f[2 * i + 1];
            v[i] = __builtin_bit_cast(uint32_t, h);
            f[2 * i] = (float)h[0]; f[2 * i + 1] = (float)h[1];
        }
    }
    return v;
}

// ---- quantisation.  |v| as bits orders like the values, and an infinity or a NaN comes out on top of every number: a block that holds one gets it as
// its scale, and every value of the block then stands for NaN instead of something that looks like a result.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ float scale_of(uint32_t most)
{
    const float s = __uint_as_float(most) / 448.0f;
    return s < SCALE_MIN ? SCALE_MIN : s;      // (false for a NaN)
}
// four values times 1 / scale, rounded to the nearest e4m3 (ties to even).  |v| / scale is 448 (1 + 2^-23) at most, which rounds to 448.
__device__ __forceinline__ uint32_t quantise4(const float *v, float inv)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
}
// ---- gated activations f(a, u): kind 0 a sigmoid(a) u, 1 gelu's tanh form (= a sigmoid(2 sqrt(2 / pi) (a + 0.044715 a^3))) u, 2 max(a, 0) u, 3 a' sigmoid(1.702 a') (u' + 1) with a' = min(a, limit),
// u' = u within +- limit; a NaN stays one.  sigmoid(x) = 1 / (1 + 2^t), t = -x log2(e): its rounding put right through the exponential's derivative, one instruction for the power of two and one
// for the reciprocal (1 unit in the last place each).  t goes no further than the largest power, where the reciprocal is 0.  (With the library's exponential and a correctly rounded
// quotient, 40 instructions a value instead of 17, the row kernel waits for instructions and not for memory: 2051 x 11008 bf16 28.0 us, so 22.3.)
__device__ __forceinline__ float sigmoid(float x)
{
    constexpr float L = 1.44269504f, L_REST = 1.92596303e-08f, LN2 = 0.69314718f;      // log2(e) = L + L_REST
    const float y = __builtin_amdgcn_fmed3f(-x, -88.0f, 88.7f), t = y * L;
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_amdgcn_rcpf(1.0f + fmaf(e, LN2 * fmaf(y, L_REST, fmaf(y, L, -t)), e));
}
template <int KIND> __device__ __forceinline__ float gated(float limit, float a, float u)
{
    if constexpr (KIND == 0) return a * sigmoid(a) * u;
    else if constexpr (KIND == 1) return a * sigmoid(a * fmaf(a * a, 0.0713548163f, 1.59576912f)) * u;
    else if constexpr (KIND == 2) return (a < 0.0f ? 0.0f : a) * u;
    else {
        const float ac = a > limit ? limit : a, uc = u > limit ? limit : u < -limit ? -limit : u;
        return ac * sigmoid(1.702f * ac) * (uc + 1.0f);
    }
}
// a[i] = f(a[i], u[i]): one look at the kind for all of them, so that their exponentials run beside each other
template <int N> __device__ __forceinline__ void gated_all(int kind, float limit, float (&a)[N], const float (&u)[N])
{
#define IFA_GATED(K) { _Pragma("unroll") for (int i = 0; i < N; i++) a[i] = gated<K>(limit, a[i], u[i]); }
    if (kind == 0) IFA_GATED(0) else if (kind == 1) IFA_GATED(1) else if (kind == 2) IFA_GATED(2) else IFA_GATED(3)
#undef IFA_GATED
}
// maximum over aligned groups of LANES lanes (16 or 32); every lane gets it
__device__ __forceinline__ uint32_t dpp_max(uint32_t v, uint32_t o) { return v > o ? v : o; }
template <int LANES> __device__ __forceinline__ uint32_t group_max(uint32_t v)
{
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));       // lanes ^ 1
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));       // lanes ^ 2
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));      // the other quad of eight lanes
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true));      // the other eight of sixteen
    if constexpr (LANES == 32) v = dpp_max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
    return v;
}

// ---- products over one block of 128 columns.  Lane l holds 32 values of row l % 16 of either operand; which 32 of the block is free as long as both operands have the same (the sum does not
// know their order); here columns 16 (l / 16) .. + 15 and those 64 further on.  The result: column l % 16 (an activation row), rows 4 (l / 16) .. + 3 (matrix rows).
// Two forms.  v_mfma_f32_16x16x128_f8f6f4 adds eight products after shifting them to the exponent of the largest one, and what falls below 2^-13 of it is cut off (measured with pairs of products;
// sums of unlike terms come out 1.5e-5 off, rms): enough in front of a rounding to 16 bits, not for a 32-bit result, nor for sums that choose an e4m3 value each (experts' gate and up; v_mfma_f32_16x16x32_fp8_fp8
// is off by as much).  WIDE: the values as halves (exact: e4m3 fits) through four
// v_mfma_f32_16x16x32_f16, which keep 32-bit sums; half the rate, and a conversion for each two values.
__device__ __forceinline__ i32x8 both_halves(u32x4 lo, u32x4 hi)
{
    i32x8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) { v[i] = (int)lo[i]; v[4 + i] = (int)hi[i]; }
    return v;
}
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f16x8 halves_of(int lo, int hi)      // eight e4m3 values
{
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <bool WIDE> struct Operand;
template <> struct Operand<false> {
    i32x8 v;
    __device__ __forceinline__ void set(u32x4 lo, u32x4 hi) { v = both_halves(lo, hi); }
};
template <> struct Operand<true> {
    f16x8 v[4];
    __device__ __forceinline__ void set(u32x4 lo, u32x4 hi)
    {
        v[0] = halves_of((int)lo[0], (int)lo[1]); v[1] = halves_of((int)lo[2], (int)lo[3]);
        v[2] = halves_of((int)hi[0], (int)hi[1]); v[3] = halves_of((int)hi[2], (int)hi[3]);
    }
};
__device__ __forceinline__ f32x4 mfma128(const Operand<false> &a, const Operand<false> &b)
{
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, zero, 0, 0, 0, 0, 0, 0);      // (scales 0: the form without)
}
__device__ __forceinline__ f32x4 mfma128(const Operand<true> &a, const Operand<true> &b)
{
    f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}

} // namespace ifa8
