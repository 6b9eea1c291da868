// Block-scaled (MX) operands: element formats, layouts and the block quantiser shared by the sdmi_mx kernels.
//
// A block is 32 consecutive values of a row with one power-of-two scale, held as its exponent + 127 in a byte (255: the
// block is NaN).  Elements are e4m3 (MX8) or e2m1 (MX4).  K is padded to whole k-steps of 128 = 4 blocks - the depth of
// v_mfma_scale_f32_16x16x128_f8f6f4 - with zero codes and scale bytes 0.
//   activations: codes in planes of 64 bytes a row, [Kp / 64][rows][64] (MX8) or [Kp / 128][rows][64] (MX4, even k in the
//                low nibble), scales [Kp / 128][rows][4].  What 16 rows give to one operand register quad is then 1 KB in one
//                piece: with the rows behind each other a 4-bit row's k-step is half a cache line, and the product fetches
//                every line twice (8192 x 10240 x 5120 on 128 x 128 tiles: 312 -> 275 us from this order alone)
//   weights:     in the order the matrix instruction reads them, see sdmi_mx_gemm.hip
#pragma once
#include "sdmi_common.h"

constexpr int MX_BLOCK = 32, MX_KSTEP = 128;

__host__ __device__ __forceinline__ int64_t mx_ksteps(int64_t K) { return (K + MX_KSTEP - 1) / MX_KSTEP; }
__host__ __device__ __forceinline__ int64_t mx_row_bytes(int64_t K, int fmt) { return mx_ksteps(K) * (fmt == SDMI_MX_FP8 ? 128 : 64); }

// What the operators take, and what their size queries answer for: -1 beyond.
constexpr int64_t MX_MAX_DIM = (int64_t)1 << 24, MX_MAX_ROWS = ((int64_t)1 << 31) - 1;      // K (and N of weights); rows
static inline bool mx_sizes_ok(int64_t rows, int64_t K) { return rows >= 0 && rows <= MX_MAX_ROWS && K > 0 && K <= MX_MAX_DIM; }

// A launch holds fewer than 2^32 threads: the most workgroups of `threads` that it may have.
constexpr int64_t mx_grid_blocks(int threads) { return (((int64_t)1 << 32) - 1) / threads; }

// Source types of the element-wise kernels: 0 bf16, 1 f16, 2 fp32 (sdmi_dtype mapped by mx_src_type on the host).
static inline int mx_src_type(int32_t dtype) {
    return dtype == SDMI_DTYPE_BF16 ? 0 : dtype == SDMI_DTYPE_F16 ? 1 : dtype == SDMI_DTYPE_F32 ? 2 : -1;
}
template <int T> struct MxElem { typedef unsigned short type; };
template <> struct MxElem<2> { typedef float type; };

template <int T> __device__ __forceinline__ float mx_to_f32(typename MxElem<T>::type v) {
    if constexpr (T == 2) return v;
    else return elem_to_f32<T>(v);
}

// 8 consecutive values from p[0..], of which `n` exist (the others read as 0).  Vector memory instructions take any address
// that the element's own alignment allows, so rows that are not 16-byte aligned - an odd width, a column slice - are read in
// vectors like others.
typedef uint4 __attribute__((aligned(2))) mx_u128_a2;
typedef uint2 __attribute__((aligned(2))) mx_u64_a2;
typedef f32x4 __attribute__((aligned(4))) mx_f128_a4;
template <int T> __device__ __forceinline__ void mx_load8(const typename MxElem<T>::type* p, int n, float* f) {
    if (n >= 8) {
        if constexpr (T == 2) {
            const f32x4 a = reinterpret_cast<const mx_f128_a4*>(p)[0], b = reinterpret_cast<const mx_f128_a4*>(p)[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) { f[j] = a[j]; f[4 + j] = b[j]; }
        } else {
            elem_unpack8<T>(*reinterpret_cast<const mx_u128_a2*>(p), f);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = j < n ? mx_to_f32<T>(p[j]) : 0.0f;
    }
}
// 8 consecutive values to p[0..], of which `n` exist.
template <int T> __device__ __forceinline__ void mx_store8(typename MxElem<T>::type* p, int n, const float* f) {
    if (n >= 8) {
        if constexpr (T == 2) {
            reinterpret_cast<mx_f128_a4*>(p)[0] = (f32x4){f[0], f[1], f[2], f[3]};
            reinterpret_cast<mx_f128_a4*>(p)[1] = (f32x4){f[4], f[5], f[6], f[7]};
        } else {
            *reinterpret_cast<mx_u128_a2*>(p) = elem_pack8<T>(f);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j < n) {
                if constexpr (T == 2) p[j] = f[j];
                else p[j] = elem_from_f32<T>(f[j]);
            }
        }
    }
}

// Lane exchanges inside a row of 16 lanes, without LDS.
template <int CTRL> __device__ __forceinline__ unsigned mx_dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}

// The shared exponent of a block from the bits of its largest magnitude: floor(log2 max) is the exponent field (0 for
// subnormals, whose byte is 0 in any case), the scale lies FMT's largest exponent below it.  255 marks NaN and infinity:
// their bits are the largest, so the integer maximum finds them.
template <int FMT> __device__ __forceinline__ unsigned mx_scale_byte(unsigned amax_bits) {
    const unsigned e = amax_bits >> 23, emax = FMT == SDMI_MX_FP8 ? 8u : 2u;
    return e == 255u ? 255u : (e > emax ? e - emax : 0u);
}
// The reciprocal of the scale: 2^(127 - byte), exact and normal for every byte <= 252, so that x * it is x / scale.
__device__ __forceinline__ float mx_inv_scale(unsigned byte) { return __uint_as_float((254u - byte) << 23); }

// 8 scaled values -> codes: 8 bytes (MX8) or 4 bytes (MX4, in .x).  Round to nearest even, saturating: the 8-bit convert
// would turn what rounds past 448 into NaN, so it is clamped first; the 4-bit one saturates by itself.
template <int FMT> __device__ __forceinline__ uint2 mx_codes8(const float* f, float inv) {
    uint2 r = {0u, 0u};
    if constexpr (FMT == SDMI_MX_FP8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __builtin_amdgcn_fmed3f(f[j] * inv, -448.0f, 448.0f);
        int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], a, true);
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], b, true);
        r.x = (unsigned)a;
        r.y = (unsigned)b;
    } else {
        unsigned a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0] * inv, f[1] * inv, 1.0f, 0);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[2] * inv, f[3] * inv, 1.0f, 1);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[4] * inv, f[5] * inv, 1.0f, 2);
        a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[6] * inv, f[7] * inv, 1.0f, 3);
        r.x = a;
    }
    return r;
}

__device__ __forceinline__ unsigned mx_amax8(const float* f) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
    return m;
}

// One k-step of one row, held by 16 consecutive lanes with 8 values each (4 lanes a block): `codes` gets this lane's codes,
// the return value is the row's scale dword (the same in the 16 lanes).  All 16 lanes have to take part.
template <int FMT> __device__ __forceinline__ unsigned mx_quantise8(const float* f, int lane, uint2& codes) {
    unsigned m = mx_amax8(f);
    m = max(m, mx_dpp<0xB1>(m));                          // quad_perm 1 0 3 2
    m = max(m, mx_dpp<0x4E>(m));                          // quad_perm 2 3 0 1
    const unsigned byte = mx_scale_byte<FMT>(m);
    codes = mx_codes8<FMT>(f, mx_inv_scale(min(byte, 252u)));
    if (byte == 255u) codes = (uint2){0u, 0u};            // the scale alone says NaN
    unsigned dw = byte << (8 * ((lane & 15) >> 2));
    dw |= mx_dpp<0x124>(dw);                              // row_ror 4
    dw |= mx_dpp<0x128>(dw);                              // row_ror 8
    return dw;
}

// The gates.  Both are taken in hardware approximations of exp2 and 1 / x (one step of fp32 each), as 16-bit and block-scaled
// results show their errors next to rounding borders alone (half a step is 2^-12 of a value at least); F32, the form for fp32
// results, takes out the one error that grows with |x|, the rounding of the exponential's argument.

// 2^-(c m) for finite m >= 0: c m as a rounded product and its remainder, c in two parts; exact but for exp2's own step.
__device__ __forceinline__ float mx_exp2_neg(float m, float c, float c_low) {
    const float t = m * c, low = fmaf(m, c_low, fmaf(m, c, -t));
    const float e = __builtin_amdgcn_exp2f(-t);
    return fmaf(e, -0.69314718055994531f * low, e);
}
constexpr float MX_HALF_LOG2E = 0.72134752044448170f, MX_HALF_LOG2E_LOW = (float)(0.72134752044448170368 - (double)MX_HALF_LOG2E);

// GELU by the error function, x Phi(x) = max(x, 0) - |x| Phi(-|x|), for any magnitude: Phi(-|x|) = erfc(z) / 2 with
// z = |x| / sqrt 2, and erfc(z) = exp(-z^2) t P(t), t = 1 / (1 + z / 2), P a degree-8 polynomial fitted to exp(z^2) erfc(z)
// on [0, 10] (relative error 0.72 x 2^-24; its halves stand below).  Written from the small side, so that the tail of negative
// x keeps its relative precision, and in 16 plain and two transcendental instructions.  Of 16.8 million products of standard
// normal fp16 values, as e4m3 with their scales, 13 lie on another side of a rounding border than the exact ones, and 12 of those
// that an fp32 erfc gives (degree 7 with t = 1 / (1 + 0.425 z), fitted to 2.4 x 2^-24: 26, in the same time).
template <bool F32> __device__ __forceinline__ float mx_gelu(float x) {
    const float d = fmaf(0.5f * 0.70710678118654752f, fabsf(x), 1.0f);
    float t = __builtin_amdgcn_rcpf(d);
    if constexpr (F32) t = fmaf(t, fmaf(-t, fminf(d, 3e38f), 1.0f), t);                    // (a Newton step: the reciprocal's own step)
    float p = fmaf(0.5f * -5.906898556e-02f, t, 0.5f * 2.845750810e-01f);
    p = fmaf(p, t, 0.5f * -4.872001292e-01f);
    p = fmaf(p, t, 0.5f * 2.780674087e-01f);
    p = fmaf(p, t, 0.5f * -2.662582689e-02f);
    p = fmaf(p, t, 0.5f * 2.026869332e-01f);
    p = fmaf(p, t, 0.5f * 2.431037475e-01f);
    p = fmaf(p, t, 0.5f * 2.823753105e-01f);
    p = fmaf(p, t, 0.5f * 2.820864178e-01f);
    if constexpr (F32) {
        // exp(-z^2) = 2^-(c x^2) with x^2 as a rounded square and its remainder (nothing is left of it from 30 on)
        const float m = fminf(fabsf(x), 30.0f), s = m * m, low = fmaf(fmaf(m, m, -s), -0.5f, 1.0f);
        return fmaf(-(fminf(fabsf(x), 3e38f) * p * t), mx_exp2_neg(s, MX_HALF_LOG2E, MX_HALF_LOG2E_LOW) * low, fmaxf(x, 0.0f));
    } else {
        const float half = p * t * __builtin_amdgcn_exp2f(x * x * -MX_HALF_LOG2E);         // Phi(-|x|)
        return fmaf(-fminf(fabsf(x), 3e38f), half, fmaxf(x, 0.0f));                       // (infinity times 0 would be NaN)
    }
}

// SiLU, x / (1 + exp(-x)).  The result is a normal fp32 number down to x = -91.6, exp(-x) only up to 88.7 and its reciprocal to
// 87.3.  The form for fp32 results is therefore written from exp(-|x|) = h^2, whose root goes into the product twice; the
// others take it for eight values at a time where one of them is below -87, and the plain form for all the rest (16384 x 5120
// bf16 with 4-bit results: 83 us, the plain form alone 88, the other one alone 92).
template <bool F32> __device__ __forceinline__ float mx_silu(float x) {
    if constexpr (F32) {
        const float h = mx_exp2_neg(fminf(fabsf(x), 200.0f), MX_HALF_LOG2E, MX_HALF_LOG2E_LOW);       // exp(-|x| / 2)
        const float w = x < 0.0f ? h : 1.0f;
        return x * w * w * __builtin_amdgcn_rcpf(fmaf(h, h, 1.0f));
    } else {
        return silu_f(x);
    }
}

// f[j] *= gate(g[j]), OP 1 GELU, 2 SiLU
template <int OP, bool F32> __device__ __forceinline__ void mx_gate8(float* f, const float* g) {
    if constexpr (OP == 2 && !F32) {
        unsigned most = 0u;                       // of the bits: -87 and further down, and negative NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(g[j]));
        if (most > __builtin_bit_cast(unsigned, -87.0f)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= mx_silu<true>(g[j]);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= OP == 1 ? mx_gelu<F32>(g[j]) : mx_silu<F32>(g[j]);
}
