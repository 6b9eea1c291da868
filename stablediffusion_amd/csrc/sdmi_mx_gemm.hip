// sdmi_mx_gemm: out[m, n] = sum_k x[m, k] w[n, k] + bias[n] + res[m, n] with 4-bit block-scaled weights and 8- or 4-bit
// block-scaled activations, on v_mfma_scale_f32_16x16x128_f8f6f4: sums in fp32, one rounding at the end.
//
// What the sums hold: 4-bit x 4-bit products span 2^6, and the instruction adds them without loss.  With 8-bit activations it
// first adds the products of 8 consecutive k on a grid 2^-13 below the power of two of the largest of them and cuts off what
// lies below, so that such a sum is off by up to 7 x 2^-13 of its group's largest product.  Over 5120 and 10240 k an fp32
// output is then 1.1e-5 from the exact sum of the same codes (2-norm; an fp32 product of them 3e-8), a bf16 output as far as
// its rounding alone (1.691e-3 either way), with 0.8 % of the values on the other side of a rounding border.  Taken as it is:
// the elements' own rounding is 2^-4 of a value, and keeping the products apart - the large codes in one instruction, the
// small ones in a second - would double the matrix work.
//
// The instruction's first operand is the weights, so that an accumulator register quad is 4 consecutive rows of the WEIGHT
// fragment at one token.  Lane l of an operand holds row l % 16; a 4-bit lane the 32 values of k-block l / 16 (16 bytes),
// an 8-bit lane the values [16 (l / 16), + 16) and 64 further on; the lane's scale is that of block l / 16 either way.
//
// Packed weights: per group of 64 output columns and k-step of 128, four fragments of 64 lanes x 16 bytes, then (in a second
// buffer) 64 lanes x 4 scale bytes, one for each fragment (the instruction selects the byte).  Fragment f, row 4 g + r holds
// column 32 (f / 2) + 8 g + 4 (f % 2) + r of its group: the accumulator quads of fragments 0 and 1 (2 and 3) are then 8
// CONSECUTIVE columns of a lane, 16 bytes of a 16-bit output, and the four lanes of a token have 64 bytes in one piece.
#include "sdmi_mx.h"
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) int i32x8;

// ---- packing -----------------------------------------------------------------------------------------------------------
template <int T>
__global__ __launch_bounds__(256) void sdmi_mx_pack_kernel(const typename MxElem<T>::type* w, int64_t ldw, int64_t N, int64_t K,
                                                           unsigned char* codes, unsigned char* scales) {
    const int64_t ksteps = mx_ksteps(K), kblocks = ksteps * 4, np = (N + 63) / 64 * 64;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= np * kblocks) return;
    const int64_t n = i / kblocks, kb = i - n * kblocks;
    float f[4][8];
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t k0 = kb * 32 + j * 8;
        const int have = n < N ? (int)max((int64_t)0, min((int64_t)8, K - k0)) : 0;
        mx_load8<T>(w + (n < N ? n : 0) * ldw + k0, have, f[j]);
        m = max(m, mx_amax8(f[j]));
    }
    const unsigned byte = mx_scale_byte<SDMI_MX_FP4>(m);
    const float inv = mx_inv_scale(min(byte, 252u));
    uint4 c;
    c.x = mx_codes8<SDMI_MX_FP4>(f[0], inv).x;
    c.y = mx_codes8<SDMI_MX_FP4>(f[1], inv).x;
    c.z = mx_codes8<SDMI_MX_FP4>(f[2], inv).x;
    c.w = mx_codes8<SDMI_MX_FP4>(f[3], inv).x;
    if (byte == 255u) c = (uint4){0u, 0u, 0u, 0u};
    const int nl = (int)(n & 63), frag = (nl >> 5) * 2 + (nl >> 2 & 1), lane = (int)(kb & 3) * 16 + (nl >> 3 & 3) * 4 + (nl & 3);      // (the map above, inverted)
    const int64_t at = (n >> 6) * ksteps + (kb >> 2);
    *reinterpret_cast<uint4*>(codes + at * 4096 + frag * 1024 + lane * 16) = c;
    scales[at * 256 + lane * 4 + frag] = (unsigned char)byte;
}

// ---- the product -------------------------------------------------------------------------------------------------------
struct MxGemmDev {
    const unsigned char* xc;
    const unsigned char* xs;
    const unsigned char* wc;
    const unsigned char* ws;
    const float* bias;
    const void* res;
    void* out;
    const void* x;             // the direct form that quantises: plain activations
    int64_t M, N, K, ksteps, ldx, ld_res, ld_out;
    int type;                  // of out and res: 0 bf16, 1 f16, 2 fp32
};

__device__ __forceinline__ i32x8 mx_op4(const uint4& a) { return (i32x8){(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}; }
__device__ __forceinline__ i32x8 mx_op8(const uint4& a, const uint4& b) {
    return (i32x8){(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
// weights (fragment byte F of ws) x activations (byte 0 of xs); FMT is the activations' format
template <int FMT, int F> __device__ __forceinline__ f32x4 mx_mfma(const i32x8& w, const i32x8& x, f32x4 c, int ws, int xs) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, FMT == SDMI_MX_FP8 ? 0 : 4, F, ws, 0, xs);
}
template <int FMT> __device__ __forceinline__ f32x4 mx_mfma_f(int f, const i32x8& w, const i32x8& x, f32x4 c, int ws, int xs) {
    switch (f) {               // (f is a constant after unrolling)
        case 0: return mx_mfma<FMT, 0>(w, x, c, ws, xs);
        case 1: return mx_mfma<FMT, 1>(w, x, c, ws, xs);
        case 2: return mx_mfma<FMT, 2>(w, x, c, ws, xs);
        default: return mx_mfma<FMT, 3>(w, x, c, ws, xs);
    }
}

// The quad at element `at` of a matrix of a type as it lies in memory (n of its 4 elements exist), and its values.
__device__ __forceinline__ uint4 mx_quad_load(const void* p, int64_t at, int type, int64_t n) {
    uint4 v = {0u, 0u, 0u, 0u};
    if (type == 2) {
        const float* const f = reinterpret_cast<const float*>(p) + at;
        if (n >= 4) v = __builtin_bit_cast(uint4, *reinterpret_cast<const mx_f128_a4*>(f));
        else v = (uint4){__float_as_uint(f[0]), n > 1 ? __float_as_uint(f[1]) : 0u, n > 2 ? __float_as_uint(f[2]) : 0u, 0u};
    } else {
        const unsigned short* const h = reinterpret_cast<const unsigned short*>(p) + at;
        if (n >= 4) {
            const uint2 w = *reinterpret_cast<const mx_u64_a2*>(h);
            v.x = w.x;
            v.y = w.y;
        } else {
            v.x = h[0] | (n > 1 ? (unsigned)h[1] << 16 : 0u);
            v.y = n > 2 ? h[2] : 0u;
        }
    }
    return v;
}
__device__ __forceinline__ f32x4 mx_quad_values(const uint4& v, int type) {
    if (type == 2) return __builtin_bit_cast(f32x4, v);
    const unsigned short h[4] = {(unsigned short)v.x, (unsigned short)(v.x >> 16), (unsigned short)v.y, (unsigned short)(v.y >> 16)};
    f32x4 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = type == 0 ? elem_to_f32<0>(h[r]) : elem_to_f32<1>(h[r]);
    return f;
}
__device__ __forceinline__ void mx_quad_store(const MxGemmDev& p, int64_t m, int64_t n, const f32x4& v) {
    const int64_t at = m * p.ld_out + n;
    if (p.type == 2) {
        float* const o = reinterpret_cast<float*>(p.out) + at;
        if (n + 4 <= p.N) *reinterpret_cast<mx_f128_a4*>(o) = v;
        else for (int r = 0; r < 3; ++r) if (n + r < p.N) o[r] = v[r];
    } else {
        unsigned short* const o = reinterpret_cast<unsigned short*>(p.out) + at;
        const uint2 w = p.type == 0 ? (uint2){elem_pack2<0>(v[0], v[1]), elem_pack2<0>(v[2], v[3])} : (uint2){elem_pack2<1>(v[0], v[1]), elem_pack2<1>(v[2], v[3])};
        if (n + 4 <= p.N) *reinterpret_cast<mx_u64_a2*>(o) = w;
        else for (int r = 0; r < 3; ++r) if (n + r < p.N) o[r] = (unsigned short)((r < 2 ? w.x : w.y) >> (16 * (r & 1)));
    }
}

// Stores and residual loads of whole lines.  A lane of the accumulators has 16-byte pieces of one token, and neighbouring lanes
// are neighbouring TOKENS: stored as they lie, a kilobyte of output is 64 addresses in 16 half lines.  So pairs of pieces (of
// 16-bit types columns c and c + 32, of fp32 c and c + 4) go round the lanes until lane l holds piece l % 8 of a 128-byte line of
// token l / 8, in the first of the two for tokens 0 ... 7 of the fragment and in the second for 8 ... 15; residuals take the same
// way back.  (Before and after, with the bands of 4 and 8 tiles of that time: 8192 x 10240 x 1280, 256 x 256 tiles, 4 bits 90 and
// 86 us, with residual 121 and 117; 4096 x 10240 x 1280 fp32 86 and 79.  Stores past the caches gained nothing, and whatever
// reads the output next had to fetch it from memory: 8192 x 10240 x 5120 with the quantisation of its output 241 us, and 232
// like this.)
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) mx_u32x4_a2;
__device__ __forceinline__ void mx_swap_rows(u32x4& a, u32x4& b, bool upper) {       // rows 0 - 7's b for rows 8 - 15's a; its own inverse
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned got = __builtin_amdgcn_update_dpp(0, upper ? a[j] : b[j], 0x128, 0xf, 0xf, true);     // row_ror:8
        a[j] = upper ? got : a[j];
        b[j] = upper ? b[j] : got;
    }
}
__device__ __forceinline__ void mx_permute(u32x4& a, int from) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __builtin_amdgcn_ds_bpermute(from, a[j]);
}

// A wave's MF x 16 tokens (from m on) x 64 columns (from c on): bias, residual, one rounding.  Straight code for each type, the
// residuals of several fragments asked for before the first of them is stored - the compiler cannot know that a store to `out`
// leaves them alone.
template <int TYPE, bool RES, int MF> __device__ __forceinline__ void mx_store_tile(const MxGemmDev& p, int64_t m, int64_t c, int lane, const f32x4 (&acc)[MF][4]) {
    typedef typename MxElem<TYPE>::type E;
    constexpr int PAIRS = TYPE == 2 ? 2 : 1, PIECE = 16 / (int)sizeof(E), TOGETHER = TYPE == 2 || MF < 4 ? 2 : 4;
    const int row = lane & 15, q = lane >> 4, t8 = lane >> 3, c8 = lane & 7;
    const bool upper = row & 8;
    const int there = 4 * (TYPE == 2 ? t8 + 8 * (c8 & 1) + 16 * (c8 >> 1) : t8 + 8 * (c8 >> 2) + 16 * (c8 & 3));
    const int back = 4 * (8 * (row & 7) + (TYPE == 2 ? 2 * q + (row >> 3) : q + 4 * (row >> 3)));
    float b[16];
    if (p.bias) {
        mx_load8<2>(p.bias + c + 8 * q, 8, b);
        mx_load8<2>(p.bias + c + 8 * q + 32, 8, b + 8);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) b[j] = 0.0f;
    }
    const E* const res = reinterpret_cast<const E*>(p.res) + c + c8 * PIECE;
    E* const out = reinterpret_cast<E*>(p.out) + c + c8 * PIECE;
#pragma unroll
    for (int i0 = 0; i0 < MF; i0 += TOGETHER) {
        u32x4 r[TOGETHER][PAIRS][2];
        if constexpr (RES) {
#pragma unroll
            for (int i = 0; i < TOGETHER; ++i)
#pragma unroll
                for (int h = 0; h < PAIRS; ++h)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        r[i][h][k] = *reinterpret_cast<const mx_u32x4_a2*>(res + min(m + 16 * (i0 + i) + 8 * k + t8, p.M - 1) * p.ld_res + 32 * h);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
            float a[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) a[j] = acc[i0 + i][j / 4][j % 4] + b[j];
            if constexpr (RES) {
#pragma unroll
                for (int h = 0; h < PAIRS; ++h) {
                    mx_permute(r[i][h][0], back);
                    mx_permute(r[i][h][1], back);
                    mx_swap_rows(r[i][h][0], r[i][h][1], upper);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float d[8];
                        if constexpr (TYPE == 2) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) d[j] = __uint_as_float(r[i][h][k][j]);
                        } else {
                            elem_unpack8<TYPE>(__builtin_bit_cast(uint4, r[i][h][k]), d);
                        }
#pragma unroll
                        for (int j = 0; j < PIECE; ++j) a[8 * h + PIECE * k + j] += d[j];
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < PAIRS; ++h) {
                u32x4 v[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (TYPE == 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[k][j] = __float_as_uint(a[8 * h + 4 * k + j]);
                    } else {
                        v[k] = __builtin_bit_cast(u32x4, elem_pack8<TYPE>(a + 8 * k));
                    }
                }
                mx_swap_rows(v[0], v[1], upper);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    mx_permute(v[k], there);
                    const int64_t t = m + 16 * (i0 + i) + 8 * k + t8;
                    if (t < p.M) *reinterpret_cast<mx_u32x4_a2*>(out + t * p.ld_out + 32 * h) = v[k];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

template <int T> struct MxRaw8 {             // 8 values as they lie in memory
    uint4 v;
    __device__ __forceinline__ void load(const unsigned short* p) { v = *reinterpret_cast<const mx_u128_a2*>(p); }
    __device__ __forceinline__ void clear() { v = (uint4){0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void values(float* f) const { elem_unpack8<T>(v, f); }
};
template <> struct MxRaw8<2> {
    f32x4 v[2];
    __device__ __forceinline__ void load(const float* p) { v[0] = reinterpret_cast<const mx_f128_a4*>(p)[0]; v[1] = reinterpret_cast<const mx_f128_a4*>(p)[1]; }
    __device__ __forceinline__ void clear() { v[0] = v[1] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ void values(float* f) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = v[j / 4][j % 4];
    }
};

// ---- direct form --------------------------------------------------------------------------------------------------------
// Few tokens: the weights' bytes are the work, and a workgroup has to have many of them in flight.  It takes NF of a group's
// four fragments for MT x 16 tokens; its KW waves take every KW-th k-step from memory straight into
// registers, U k-steps ahead of the ones they multiply, and join their sums through LDS in a fixed order.
// SRC >= 0: x is a plain matrix of that type (mx_src_type), of which every workgroup quantises its rows for itself (mx_fused),
// into LDS while its first weights are on their way: one launch instead of two.
template <int FMT, int MT, int NF, int KW, int U, int SRC>
__global__ __launch_bounds__(64 * KW) void sdmi_mx_direct_kernel(MxGemmDev p) {
    extern __shared__ unsigned char smem[];
    constexpr int RB = FMT == SDMI_MX_FP8 ? 128 : 64;      // bytes of a row's k-step
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, q = lane >> 4;
    constexpr int PARTS = 4 / NF;
    const int64_t grp = blockIdx.x / PARTS, m0 = (int64_t)blockIdx.y * (16 * MT);
    const int f0 = (int)(blockIdx.x % PARTS) * NF;
    const int nk = (int)p.ksteps, mine = (nk - wave + KW - 1) / KW;                 // k-steps of this wave (<= 0: none)
    const unsigned char* const wc = p.wc + (grp * p.ksteps + wave) * 4096 + f0 * 1024 + lane * 16;
    const unsigned char* const ws = p.ws + (grp * p.ksteps + wave) * 256 + lane * 4;
    const unsigned char* xc[MT];
    const unsigned char* xs[MT];
    f32x4 acc[MT][NF];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) {
        const int64_t r = min(m0 + mi * 16 + row, p.M - 1);
        if constexpr (SRC < 0) {
            xc[mi] = p.xc + (wave * (RB / 64) * p.M + r) * 64 + q * 16;
            xs[mi] = p.xs + (wave * p.M + r) * 4 + q;
        }
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[mi][f] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    uint4 w[2][U][NF], a[2][U][SRC < 0 ? MT : 1], b[2][U][SRC < 0 && FMT == SDMI_MX_FP8 ? MT : 1];
    int wsc[2][U], xsc[2][U][SRC < 0 ? MT : 1];
    auto load = [&](int buf, int i0) {                     // k-steps i0 .. i0 + U of this wave (past the end: the last one again)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = (int64_t)min(i0 + u, mine - 1) * KW;
#pragma unroll
            for (int f = 0; f < NF; ++f) w[buf][u][f] = *reinterpret_cast<const uint4*>(wc + at * 4096 + f * 1024);
            wsc[buf][u] = *reinterpret_cast<const int*>(ws + at * 256);
            if constexpr (SRC < 0) {
#pragma unroll
                for (int mi = 0; mi < MT; ++mi) {
                    a[buf][u][mi] = *reinterpret_cast<const uint4*>(xc[mi] + at * p.M * RB);
                    if constexpr (FMT == SDMI_MX_FP8) b[buf][u][mi] = *reinterpret_cast<const uint4*>(xc[mi] + at * p.M * RB + p.M * 64);
                    xsc[buf][u][mi] = xs[mi][at * p.M * 4];
                }
            }
        }
    };
    if (mine > 0) load(0, 0);
    if (mine > U) load(1, U);
    // the wave stores fragments wave, wave + KW ... of the output; their bias and residual travel behind the first weights
    constexpr int OWN = (MT * NF + KW - 1) / KW;
    auto place = [&](int i, int64_t& m, int64_t& n) {
        const int t = wave + i * KW, f = f0 + t % NF;
        m = m0 + t / NF * 16 + row;
        n = grp * 64 + 32 * (f >> 1) + 8 * q + 4 * (f & 1);
        return t < MT * NF && m < p.M && n < p.N;
    };
    uint4 bias[OWN], res[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        int64_t m, n;
        const bool stores = place(i, m, n);
        bias[i] = res[i] = (uint4){0u, 0u, 0u, 0u};
        if (stores && p.bias) bias[i] = mx_quad_load(p.bias, n, 2, p.N - n);
        if (stores && p.res) res[i] = mx_quad_load(p.res, m * p.ld_res + n, p.type, p.N - n);
    }
    unsigned char* const own = smem;                       // SRC >= 0: [nk][rows][RB] codes, then [nk][rows][4] scales
    const int rows = (int)min(p.M - m0, (int64_t)(16 * MT));
    unsigned char* const own_s = smem + nk * rows * RB;
    if constexpr (SRC >= 0) {
        // the wave quantises the k-steps that it alone will read: four (k-step, row) pairs at a time, 16 lanes each, and the
        // 16 MT rows of a k-step on their way together (rows and pairs past the end: the last one again)
        typedef typename MxElem<SRC>::type E;
        constexpr int AT = 4 * MT;
        const E* const x = reinterpret_cast<const E*>(p.x) + m0 * p.ldx;
        const int sh = rows > 1 ? 32 - __builtin_clz(rows - 1) : 0, pairs = mine << sh;          // (rows rounded up to a power of two)
        for (int j0 = 0; j0 < pairs; j0 += 4 * AT) {
            MxRaw8<SRC> raw[AT];
            int at[AT];
#pragma unroll
            for (int u = 0; u < AT; ++u) {
                const int j = min(j0 + 4 * u + q, pairs - 1), step = wave + (j >> sh) * KW, r = min(j & ((1 << sh) - 1), rows - 1);
                const int64_t k0 = (int64_t)step * MX_KSTEP + row * 8;
                at[u] = step * rows + r;
                raw[u].load(x + r * p.ldx + min(k0, p.K - 8));                   // (K is whole eights: mx_fused)
                if (k0 >= p.K) raw[u].clear();
            }
#pragma unroll
            for (int u = 0; u < AT; ++u) {
                float f[8];
                raw[u].values(f);
                uint2 c;
                const unsigned dw = mx_quantise8<FMT>(f, lane, c);
                if constexpr (FMT == SDMI_MX_FP8) *reinterpret_cast<uint2*>(own + at[u] * RB + row * 8) = c;
                else *reinterpret_cast<unsigned*>(own + at[u] * RB + row * 4) = c.x;
                if (row == 0) *reinterpret_cast<unsigned*>(own_s + at[u] * 4) = dw;
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // other lanes of this wave read them
    }
    auto multiply = [&](int buf, int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u >= mine) break;                     // (uniform)
#pragma unroll
            for (int mi = 0; mi < MT; ++mi) {
                i32x8 x;
                int sc;
                if constexpr (SRC < 0) {
                    if constexpr (FMT == SDMI_MX_FP8) x = mx_op8(a[buf][u][mi], b[buf][u][mi]);
                    else x = mx_op4(a[buf][u][mi]);
                    sc = xsc[buf][u][mi];
                } else {
                    const int at = (wave + (i0 + u) * KW) * rows + min(mi * 16 + row, rows - 1);
                    const uint4 lo = *reinterpret_cast<const uint4*>(own + at * RB + q * 16);
                    if constexpr (FMT == SDMI_MX_FP8) x = mx_op8(lo, *reinterpret_cast<const uint4*>(own + at * RB + q * 16 + 64));
                    else x = mx_op4(lo);
                    sc = own_s[at * 4 + q];
                }
                const int s4 = wsc[buf][u] >> (8 * f0);
#pragma unroll
                for (int f = 0; f < NF; ++f) acc[mi][f] = mx_mfma_f<FMT>(f, mx_op4(w[buf][u][f]), x, acc[mi][f], s4, sc);
            }
        }
    };
    for (int i = 0; i < mine; i += 2 * U) {
        multiply(0, i);
        if (i + 2 * U < mine) load(0, i + 2 * U);
        if (i + U < mine) multiply(1, i + U);
        if (i + 3 * U < mine) load(1, i + 3 * U);
    }
    if constexpr (SRC >= 0) __syncthreads();               // the codes' place becomes that of the sums
    f32x4* const part = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
#pragma unroll
        for (int f = 0; f < NF; ++f) part[((wave * MT + mi) * NF + f) * 64 + lane] = acc[mi][f];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
        int64_t m, n;
        if (!place(i, m, n)) continue;
        const int t = wave + i * KW;
        f32x4 v = part[t * 64 + lane];
#pragma unroll
        for (int k = 1; k < KW; ++k) v += part[(k * MT * NF + t) * 64 + lane];
        if (p.bias) v += mx_quad_values(bias[i], 2);
        if (p.res) v += mx_quad_values(res[i], p.type);
        mx_quad_store(p, m, n, v);
    }
}

// ---- tiled form ---------------------------------------------------------------------------------------------------------
// A workgroup computes BM tokens x 64 WGN columns; wave (wm, wn) MF x 16 tokens x one group of 64 columns.  A k-step's codes
// and scales come through a ring of ST LDS stages, filled by LDS-DMA: weights and their scales as they lie in memory, rows of
// activations with their 16-byte chunks exchanged (chunk c of row r lies at c ^ swizzle(r)), so that the 16 rows of a fragment
// read meet no bank twice - an LDS-DMA writes in lane order, so the exchange is made on the side of the global address.
// One barrier a k-step, in its middle.
// `mask`: the lanes that load, all or none.  A fill past the last k-step is issued with none: it moves nothing and still counts
// as issued and landed, so that every k-step waits for the same number of instructions and the loop has no branch.
#define MX_GLDS(NAME, OP)                                                                                            \
    __device__ __forceinline__ void NAME(unsigned d0, const void* sb, unsigned v0, unsigned mask) {                   \
        unsigned keep;                                                                                               \
        uint64_t all;                                                                                                \
        asm volatile(SDMI_M0_SAVE "s_mov_b32 m0, %[d0]\n\ts_mov_b64 %[all], exec\n\ts_mov_b32 exec_lo, %[mask]\n\ts_mov_b32 exec_hi, %[mask]\n\ts_nop 0\n\t"  \
                     OP " %[v0], %[sb]\n\ts_mov_b64 exec, %[all]\n\t" SDMI_M0_REST                                   \
                     : [keep] "=&s"(keep), [all] "=&s"(all)                                                          \
                     : [d0] "s"(d0), [sb] "s"(sb), [v0] "v"(v0), [mask] "s"(__builtin_amdgcn_readfirstlane(mask))                                    \
                     : "memory");                                                                                    \
    }
MX_GLDS(mx_glds16, "global_load_lds_dwordx4")
MX_GLDS(mx_glds4, "global_load_lds_dword")

// all but the youngest N fill instructions have landed, and so have the LDS reads
template <int N> __device__ __forceinline__ void mx_wait() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory"); }

template <int FMT, int BM, int WGM, int WGN, int ST> struct MxTile {
    static constexpr int RB = FMT == SDMI_MX_FP8 ? 128 : 64;                     // bytes of a row's k-step
    static constexpr int NW = WGM * WGN, THREADS = 64 * NW, BN = 64 * WGN, MF = BM / WGM / 16;
    static constexpr int HALF = MF / 2, HR = HALF * 16;                          // fragments and rows of a wave's half
    static constexpr int XJ = (BM / 2 + 63) / 64;                                // scale instructions of a half
    static constexpr int A_BYTES = BM * RB, W_BYTES = WGN * 4096, AS_BYTES = 2 * XJ * 256, WS_BYTES = WGN * 256;
    static constexpr int STAGE = A_BYTES + W_BYTES + AS_BYTES + WS_BYTES;
    static constexpr int AI = A_BYTES / 1024 / NW, WI = W_BYTES / 1024 / NW;     // LDS-DMA instructions of a wave and stage
    static constexpr int SJ = 2 * XJ + WGN, SI = (SJ + NW - 1) / NW;             // scale instructions: the halves', one a group
    static constexpr int PER = AI + WI + SI, LDS = STAGE * ST;
    static_assert(A_BYTES % (1024 * NW) == 0 && W_BYTES % (1024 * NW) == 0 && MF % 2 == 0 && MF * 16 * WGM == BM, "tile");
    static_assert(AI % 2 == 0 || AI == 1, "halves");
    static_assert((ST - 1) * PER < 64 && LDS <= 160 * 1024, "ring");
};

template <int FMT, int BM, int WGM, int WGN, int ST>
__global__ __launch_bounds__(64 * WGM * WGN, 2) void sdmi_mx_tiled_kernel(MxGemmDev p) {
    typedef MxTile<FMT, BM, WGM, WGN, ST> T;
    extern __shared__ unsigned char smem[];
    const unsigned lds_base = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)smem;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN, row = lane & 15, q = lane >> 4;

    // Workgroups go round the 8 XCDs; each XCD takes a run of consecutive tiles, and a run walks BAND token tiles before the next
    // column tile, so that the tiles an XCD works on together - 32 of 256 x 256, 64 of the smaller ones - are a compact patch
    // and share their operands in its L2.  Heights that are no power of two: with 4 or 8 the runs of all XCDs start in the same
    // column tile of their bands and write lines a power of two apart at a time (8192 x 10240 x 1280, 4 bits: 256 x 256 tiles
    // 86 us with 4, 76 with 5, 128 x 128 ones 96 with 8, 79 with 7; 4096 x 5120 x 5120 the same with either).
    const unsigned tm = (unsigned)((p.M + BM - 1) / BM), tn = (unsigned)((p.N + T::BN - 1) / T::BN), total = tm * tn;
    const unsigned xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
    const unsigned id = (xcd < more ? xcd * (each + 1) : more + xcd * each) + (blockIdx.x >> 3);
    constexpr unsigned BAND = BM == 256 ? 5 : 7;
    const unsigned band = id / (BAND * tn), height = min(BAND, tm - band * BAND), in_band = id - band * BAND * tn;
    const int64_t m0 = (int64_t)(band * BAND + in_band % height) * BM;
    const int64_t g0 = (int64_t)(in_band / height) * WGN, groups = (p.N + 63) >> 6;

    const int nk = (int)p.ksteps;

    // Fills.  A wave's tokens are two halves of HR rows: with the weights go the first halves ("X" of a stage), the second
    // halves ("Y") follow half a k-step later, as they are read, so that each place in the ring is free again half a k-step
    // earlier than it would be as a whole and the fills run ST - 1 / 2 k-steps ahead.
    // Row j of X is row j % HR of the first half of wave row j / HR.  Per-lane offsets are constant over the k-steps.
    auto tile_row = [](int j, bool y) { return j / T::HR * (2 * T::HR) + j % T::HR + (y ? T::HR : 0); };
    const int64_t a_step = p.M * T::RB;
    unsigned a_off[T::AI], w_off[T::WI], s_off[T::SI], a_dst[T::AI], s_dst[T::SI];
    int64_t a_add[T::AI];
    bool a_y[T::AI], s_y[T::SI];
    const unsigned char* s_src[T::SI];
    int64_t s_step[T::SI];
#pragma unroll
    for (int i = 0; i < T::AI; ++i) {
        a_y[i] = T::AI == 1 ? wave >= T::NW / 2 : i >= T::AI / 2;                // an instruction takes 16 rows of a plane
        const int c = T::AI == 1 ? wave % (T::NW / 2) : (i % (T::AI / 2)) * T::NW + wave, plane = c / (BM / 32);
        const int first = tile_row(c % (BM / 32) * 16, a_y[i]), r = first + (lane >> 2);
        const int64_t rr = min((int64_t)r, p.M - 1 - m0);                        // rows past the end repeat the last one
        a_off[i] = (unsigned)rr * 64 + ((lane & 3) ^ ((r >> 1) & 3)) * 16;
        a_add[i] = plane * p.M * 64 - (a_y[i] ? a_step : 0);
        a_dst[i] = (plane * BM + first) * 64;
    }
#pragma unroll
    for (int i = 0; i < T::WI; ++i) {
        const int c = i * T::NW + wave;
        const int64_t g = min((int64_t)(c >> 2), groups - 1 - g0);
        w_off[i] = (unsigned)(g * p.ksteps * 4096) + (c & 3) * 1024 + lane * 16;
    }
#pragma unroll
    for (int i = 0; i < T::SI; ++i) {
        const int job = (i * T::NW + wave) % T::SJ;                              // (a job done twice writes the same bytes twice)
        s_y[i] = job >= T::XJ && job < 2 * T::XJ;
        s_dst[i] = T::A_BYTES + T::W_BYTES + job * 256;
        if (job < 2 * T::XJ) {
            const int jr = (job % T::XJ * 64 + lane) % (BM / 2);
            const int64_t r = min(m0 + tile_row(jr, s_y[i]), p.M - 1);
            s_off[i] = (unsigned)((r - m0) * 4);
            s_src[i] = p.xs + m0 * 4;
            s_step[i] = p.M * 4;
        } else {
            const int64_t g = min(g0 + (job - 2 * T::XJ), groups - 1);
            s_off[i] = lane * 4;
            s_src[i] = p.ws + g * p.ksteps * 256;
            s_step[i] = 256;
        }
        if (s_y[i]) s_src[i] -= s_step[i];
    }
    const unsigned char* a_src = p.xc + m0 * 64;
    const unsigned char* w_src = p.wc + g0 * p.ksteps * 4096;
    // Instruction j of the PER of a fill: X of the k-step that the sources point at into stage x, Y of the one before into y.
    auto fill_piece = [&](int j, unsigned x, unsigned y, unsigned xmask, unsigned ymask) {
        if (j < T::AI) {
            const bool late = a_y[j];
            mx_glds16(lds_base + (late ? y : x) * T::STAGE + a_dst[j], a_src + a_add[j], a_off[j], late ? ymask : xmask);
        } else if (j < T::AI + T::WI) {
            const int i = j - T::AI;
            mx_glds16(lds_base + x * T::STAGE + T::A_BYTES + (i * T::NW + wave) * 1024, w_src, w_off[i], xmask);
        } else {
            const int i = j - T::AI - T::WI;
            mx_glds4(lds_base + (s_y[i] ? y : x) * T::STAGE + s_dst[i], s_src[i], s_off[i], s_y[i] ? ymask : xmask);
        }
    };
    auto fill_done = [&]() {
#pragma unroll
        for (int i = 0; i < T::SI; ++i) s_src[i] += s_step[i];
        a_src += a_step;
        w_src += 4096;
    };

    f32x4 acc[T::MF][4];
#pragma unroll
    for (int mi = 0; mi < T::MF; ++mi)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[mi][f] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // the ring before the first k-step: X 0, then Y s and X s + 1 in pairs
#pragma unroll
    for (int i = 0; i < ST; ++i) {
#pragma unroll
        for (int j = 0; j < T::PER; ++j) fill_piece(j, i, i > 0 ? i - 1 : 0, i < nk ? ~0u : 0u, i > 0 && i - 1 < nk ? ~0u : 0u);
        fill_done();
    }
    const int arow = wm * T::MF * 16 + row;
    const int a_at = arow * 64 + (q ^ ((row >> 1) & 3)) * 16;
    const int w_at = T::A_BYTES + wn * 4096 + lane * 16;
    const int as_at = T::A_BYTES + T::W_BYTES + (wm * T::HR + row) * 4 + q, ws_at = T::A_BYTES + T::W_BYTES + T::AS_BYTES + wn * 256 + lane * 4;
    // Two k-steps overlap.  The MF x 4 matrix instructions of a k-step go in MF slots of four, with the other instructions
    // spread between the slots: slot mi reads the activations of slot mi + AHEAD; from slot TURN on, behind the barrier that
    // publishes Y of this k-step and X of the next, the slots also issue the next fill and read the weights and first
    // activations of k-step s + 1.  So the matrix pipe waits neither for a burst of loads nor for LDS behind the barrier.
    constexpr int AHEAD = 1, TURN = T::HALF - AHEAD, SLOTS = T::MF - TURN;
    static_assert(TURN >= 0, "the slot of the wait and the barrier");
    struct Act { uint4 a, b; int s; };
    struct Step { uint4 w[4]; int ws; Act x[AHEAD]; };
    auto read_act = [&](const unsigned char* st, int mi) {
        Act x;
        x.a = *reinterpret_cast<const uint4*>(st + a_at + mi * 1024);
        if constexpr (FMT == SDMI_MX_FP8) x.b = *reinterpret_cast<const uint4*>(st + a_at + BM * 64 + mi * 1024);
        x.s = st[as_at + mi % T::HALF * 64 + mi / T::HALF * T::XJ * 256];
        return x;
    };
    unsigned cur = 0, prev = ST - 1;
    auto step = [&](auto more, const Step& c, Step& n, int s) {                  // more: k-step s + 1 exists
        constexpr bool MORE = decltype(more)::value;
        const unsigned char* const st = smem + cur * T::STAGE;
        const unsigned next = cur + 1 == ST ? 0 : cur + 1;
        const unsigned char* const nst = smem + next * T::STAGE;
        const unsigned xmask = s + ST < nk ? ~0u : 0u, ymask = s + ST - 1 < nk ? ~0u : 0u;
        Act x[T::MF];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) x[i] = c.x[i];
#pragma unroll
        for (int mi = 0; mi < T::MF; ++mi) {
            if (mi == TURN) {
                mx_wait<(ST - 2) * T::PER>();
                asm volatile("s_barrier" ::: "memory");
            }
            if (mi + AHEAD < T::MF) x[mi + AHEAD] = read_act(st, mi + AHEAD);
            if (mi >= TURN && MORE) {
                const int k = mi - TURN;
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    if (f >= k * 4 / SLOTS && f < (k + 1) * 4 / SLOTS) n.w[f] = *reinterpret_cast<const uint4*>(nst + w_at + f * 1024);
                if (mi == T::MF - 1) n.ws = *reinterpret_cast<const int*>(nst + ws_at);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    if (mi + AHEAD - i == T::MF) n.x[i] = read_act(nst, i);
#pragma unroll
                for (int j = 0; j < T::PER; ++j)
                    if (j >= k * T::PER / SLOTS && j < (k + 1) * T::PER / SLOTS) fill_piece(j, cur, prev, xmask, ymask);
            }
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                if constexpr (FMT == SDMI_MX_FP8) acc[mi][f] = mx_mfma_f<FMT>(f, mx_op4(c.w[f]), mx_op8(x[mi].a, x[mi].b), acc[mi][f], c.ws, x[mi].s);
                else acc[mi][f] = mx_mfma_f<FMT>(f, mx_op4(c.w[f]), mx_op4(x[mi].a), acc[mi][f], c.ws, x[mi].s);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (MORE) {
            fill_done();
            prev = cur;
            cur = next;
        }
    };
    Step even, odd;
    mx_wait<(ST - 1) * T::PER>();
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int f = 0; f < 4; ++f) even.w[f] = *reinterpret_cast<const uint4*>(smem + w_at + f * 1024);
    even.ws = *reinterpret_cast<const int*>(smem + ws_at);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) even.x[i] = read_act(smem, i);
    // Two k-steps a trip, so that the fragments of one and of the next change places without moves; an odd number is evened out
    // in front.  One loop with one exit: with several the compiler no longer accumulates in place and spills.
    int s = 0;
    if ((nk - 1) & 1) {
        step(std::true_type(), even, odd, 0);
        even = odd;
        s = 1;
    }
    for (; s + 1 < nk; s += 2) {
        step(std::true_type(), even, odd, s);
        step(std::true_type(), odd, even, s + 1);
    }
    step(std::false_type(), even, odd, s);

    const int64_t m = m0 + arow, c = (g0 + wn) * 64;
    if (c + 64 <= p.N) {
        auto store = [&](auto res) {
            constexpr bool RES = decltype(res)::value;
            if (p.type == 0) mx_store_tile<0, RES>(p, m0 + wm * T::MF * 16, c, lane, acc);
            else if (p.type == 1) mx_store_tile<1, RES>(p, m0 + wm * T::MF * 16, c, lane, acc);
            else mx_store_tile<2, RES>(p, m0 + wm * T::MF * 16, c, lane, acc);
        };
        if (p.res) store(std::true_type());
        else store(std::false_type());
        return;
    }
#pragma unroll
    for (int mi = 0; mi < T::MF; ++mi) {                                         // the last columns, in quads
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t n = c + 32 * (f >> 1) + 8 * q + 4 * (f & 1);
            if (m + mi * 16 < p.M && n < p.N) {
                f32x4 v = acc[mi][f];
                if (p.bias) v += mx_quad_values(mx_quad_load(p.bias, n, 2, p.N - n), 2);
                if (p.res) v += mx_quad_values(mx_quad_load(p.res, (m + mi * 16) * p.ld_res + n, p.type, p.N - n), p.type);
                mx_quad_store(p, m + mi * 16, n, v);
            }
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (the packing kernel's threads, one for a block of 32, in one launch)
static bool mx_weight_ok(int64_t N, int64_t K) {
    return N > 0 && N <= MX_MAX_DIM && K > 0 && K <= MX_MAX_DIM && ((N + 63) / 64 * 64 * mx_ksteps(K) * 4 + 255) / 256 <= mx_grid_blocks(256);
}
extern "C" int64_t sdmi_mx_weight_codes_bytes(int64_t N, int64_t K) { return mx_weight_ok(N, K) ? (N + 63) / 64 * mx_ksteps(K) * 4096 : -1; }
extern "C" int64_t sdmi_mx_weight_scales_bytes(int64_t N, int64_t K) { return mx_weight_ok(N, K) ? (N + 63) / 64 * mx_ksteps(K) * 256 : -1; }

extern "C" int sdmi_mx_pack_linear(const void* w, int64_t ldw, int64_t N, int64_t K, int32_t dtype, void* codes, void* scales, void* stream) {
    const int t = mx_src_type(dtype);
    if (!w || !codes || !scales || t < 0 || !mx_weight_ok(N, K) || ldw < K) return SDMI_ERR_BAD_ARG;
    if (!aligned16(codes) || !aligned16(scales)) return SDMI_ERR_ALIGNMENT;
    const int64_t n = (N + 63) / 64 * 64 * mx_ksteps(K) * 4, blocks = (n + 255) / 256;
    hipStream_t st = (hipStream_t)stream;
    unsigned char *c = (unsigned char*)codes, *s = (unsigned char*)scales;
    if (t == 0) sdmi_mx_pack_kernel<0><<<(unsigned)blocks, 256, 0, st>>>((const unsigned short*)w, ldw, N, K, c, s);
    else if (t == 1) sdmi_mx_pack_kernel<1><<<(unsigned)blocks, 256, 0, st>>>((const unsigned short*)w, ldw, N, K, c, s);
    else sdmi_mx_pack_kernel<2><<<(unsigned)blocks, 256, 0, st>>>((const float*)w, ldw, N, K, c, s);
    SDMI_CHECK_LAUNCH();
    return SDMI_OK;
}

static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

static bool mx_args_ok(const sdmi_mx_gemm_args* a) {
    if (!a || !mx_sizes_ok(a->M, a->K) || !mx_weight_ok(a->N, a->K)) return false;
    if ((a->fmt != SDMI_MX_FP8 && a->fmt != SDMI_MX_FP4) || a->algo < 0 || a->algo > SDMI_MX_ALGOS) return false;
    return !a->x || (mx_src_type(a->x_dtype) >= 0 && a->ldx >= a->K);
}

// Which kernel runs a product: the cheapest by a model of rounds.  A kernel's workgroups take `rows` x `cols` of the output; a
// launch costs `fixed` us, a unit of K `first` for the first workgroup on each of the 256 CUs, and every further round of them
// `round` and `more` a unit.  (Direct kernels: the unit is eight k-steps, one for each wave; tiled ones: one k-step.)  Least
// squares over a sweep of 1 ... 8192 rows and twenty (N, K) from 320 x 320 to 20480 x 2560 and 5120 x 10240, of each kernel
// at the sizes where it is near the fastest; over the sweep the pick takes 1.005 (8-bit) and 1.003 (4-bit) times the fastest
// one's time on average, 1.11 at worst (32 x 640 x 640, half a microsecond; profiles/mx_kernel_choice.txt has all of it).
// Examples, us, 8-bit activations (direct kernels by their outputs a workgroup, D, tiled ones T):
//     32 x 10240 x 5120: D 32 x 64  9.4, D 48 x 64 10.5, D 16 x 64 12.4, D 16 x 32 12.7
//     48 x  5120 x 5120: D 16 x 64  7.7, D 32 x 64  8.5, D 16 x 32  9.3, D 48 x 64 10.4
//    128 x  5120 x 5120: D 48 x 64 10.8, D 32 x 64 14.1, T 64 x 128 15.4, T 128 x 128 21.1
//    256 x  1280 x 1280: D 32 x 64  4.9, D 48 x 64  5.5, T 64 x 128  6.6, T 128 x 128  8.5
//    512 x  5120 x 1280: T 128 x 128  9.5, T 64 x 128  9.6, D 48 x 64 16.0, T 256 x 256 17.0
//   1024 x  5120 x 5120: T 64 x 128 30.2, T 128 x 256 30.8, T 128 x 128 32.8, T 256 x 256 47.7
//   4096 x  5120 x 5120: T 128 x 128 82.3, T 64 x 128 94.3, T 256 x 256 99.8 (320 tiles: two rounds)
//   8192 x  5120 x 5120: T 256 x 256 158, T 128 x 256 158, T 128 x 128 164
// Activations are read again by every column group and weights by every row tile, from L2, which is what the direct kernels'
// shapes trade (96 x 5120 x 5120: 48 x 32 and 64 x 32 15.2 and 15.3 us, 32 x 64 8.9).
// Parts of K in several workgroups of a tiled kernel and a second launch that joins them were measured too (two and four parts)
// and won by 6 % at most, at one size: the workgroups of a direct kernel split K among their waves already.
enum MxKind { MX_D16x32, MX_D16x64, MX_D32x64, MX_D48x64, MX_T64x128, MX_T128x128, MX_T128x256, MX_T256x256, MX_KINDS };
struct MxCost { int rows, cols, unit; struct { double fixed, first, round, more; } us[2]; };      // [0]: 8-bit activations, [1]: 4-bit
static const MxCost MX_COST[MX_KINDS] = {
    {16, 32, 8, {{3.533, 0.425, 0.143, 0.475}, {3.547, 0.335, 0.280, 0.333}}},
    {16, 64, 8, {{3.471, 0.615, 0.875, 0.599}, {3.600, 0.478, 0.631, 0.536}}},
    {32, 64, 8, {{3.419, 0.865, 1.180, 0.968}, {3.572, 0.613, 0.824, 0.766}}},
    {48, 64, 8, {{3.466, 1.178, 1.621, 1.235}, {3.741, 0.776, 1.520, 0.929}}},
    {64, 128, 1, {{4.050, 0.286, 0.984, 0.193}, {4.069, 0.268, 1.036, 0.127}}},
    {128, 128, 1, {{4.844, 0.423, 1.385, 0.351}, {4.808, 0.323, 1.480, 0.222}}},
    {128, 256, 1, {{6.283, 0.625, 3.900, 0.717}, {6.287, 0.484, 3.799, 0.524}}},
    {256, 256, 1, {{8.431, 1.113, 6.373, 1.182}, {8.944, 0.678, 6.108, 0.793}}},
};
static_assert(MX_KINDS == SDMI_MX_ALGOS, "sdmi_mx_gemm_args.algo");
static int64_t mx_rounds(const sdmi_mx_gemm_args* a, int kind) {
    const MxCost& c = MX_COST[kind];
    return ((a->M + c.rows - 1) / c.rows * ((a->N + c.cols - 1) / c.cols) + 255) / 256;
}
static double mx_cost(const sdmi_mx_gemm_args* a, int kind) {
    const MxCost& c = MX_COST[kind];
    const auto& us = c.us[a->fmt == SDMI_MX_FP8 ? 0 : 1];
    const double units = (double)((mx_ksteps(a->K) + c.unit - 1) / c.unit);
    return us.fixed + us.first * units + (double)(mx_rounds(a, kind) - 1) * (us.round + us.more * units);
}
// Whether a kernel's workgroups fit a launch: rows go along y in the direct kernels (512 threads), all tiles along x in the tiled
// ones (two wave rows for every 64 columns).
static bool mx_fits(const sdmi_mx_gemm_args* a, int kind) {
    const MxCost& c = MX_COST[kind];
    const int64_t ny = (a->M + c.rows - 1) / c.rows, nx = (a->N + c.cols - 1) / c.cols;
    return c.unit > 1 ? ny <= 65535 && nx <= mx_grid_blocks(512) : ny * nx <= mx_grid_blocks(2 * c.cols);
}
static MxKind mx_kind(const sdmi_mx_gemm_args* a) {                              // MX_KINDS: none
    if (a->algo) return mx_fits(a, a->algo - 1) ? (MxKind)(a->algo - 1) : MX_KINDS;
    int best = MX_KINDS;
    double least = 0.0;
    for (int i = MX_KINDS - 1; i >= 0; --i) {
        const double cost = mx_cost(a, i);
        if ((best == MX_KINDS || cost < least) && mx_fits(a, i)) { best = i; least = cost; }
    }
    return (MxKind)best;
}

// The direct kernel quantises plain activations itself where that is little work beside the product, since a launch less is 4 us
// less of the caller's time (8 or 12 for an eager call) and about one on the GPU.  Each workgroup quantises its own rows, 16 (k-step,
// row) pairs of a wave a trip, so the rule counts trips and rounds of workgroups on the 256 CUs.  GPU time alone, us, fused and
// apart: one trip, 16 x 1280 x 1024 4.3 and 5.3, 1 x 10240 x 5120 7.6 and 9.1; three, 16 x 2560 x 2560 6.4 and 5.9; a second round
// of workgroups, 16 x 20480 x 1024 7.6 and 7.9, but with more trips 8 x 20480 x 4096 15.1 and 12.9; 32 rows a workgroup where that
// saves the second round, 231 x 1280 x 1024 6.6 and 6.2, 32 x 10240 x 1024 6.7 and 6.6.
enum MxFused { MX_APART, MX_FUSED16x32, MX_FUSED16x64, MX_FUSED32x64 };
static MxFused mx_fused(const sdmi_mx_gemm_args* a) {
    if (!a->x || a->algo || a->M > 8192 || a->K % 8) return MX_APART;            // (eight values are a lane's load)
    int64_t rows = 1;                                                            // of a workgroup, as the kernel counts them
    while (rows < 16 && rows < a->M) rows *= 2;
    const int64_t trips = (rows * ((mx_ksteps(a->K) + 7) / 8) + 15) / 16, r16 = (a->M + 15) / 16, c64 = (a->N + 63) / 64;
    if (trips > 3) return MX_APART;
    if (r16 * ((a->N + 31) / 32) <= 256) return MX_FUSED16x32;
    if (r16 * c64 <= 256) return MX_FUSED16x64;
    if (trips > 1) return MX_APART;
    if ((r16 + 1) / 2 * c64 <= 256) return MX_FUSED32x64;
    return r16 * c64 <= 512 ? MX_FUSED16x64 : MX_APART;
}

// How a product runs and the workspace it needs; false: not at all, said before anything of it is launched.
struct MxPlan { MxFused fused; MxKind kind; int64_t workspace; };
static bool mx_plan(const sdmi_mx_gemm_args* a, MxPlan* p) {
    if (!mx_args_ok(a)) return false;
    p->fused = mx_fused(a);
    p->kind = p->fused ? MX_KINDS : mx_kind(a);
    p->workspace = !a->x || a->M == 0 || p->fused ? 0 : up256(a->M * mx_row_bytes(a->K, a->fmt)) + up256(a->M * mx_ksteps(a->K) * 4);
    return p->fused || p->kind != MX_KINDS;
}

extern "C" int64_t sdmi_mx_gemm_workspace_bytes(const sdmi_mx_gemm_args* a) {
    MxPlan p;
    return mx_plan(a, &p) ? p.workspace : -1;
}

template <int FMT, int BM, int WGM, int WGN, int ST> static int tiled_launch(const MxGemmDev& d, hipStream_t st) {
    typedef MxTile<FMT, BM, WGM, WGN, ST> T;
    static_assert(T::THREADS == 2 * T::BN, "mx_fits");
    static SdmiPerDeviceOnce once;
    const auto kernel = sdmi_mx_tiled_kernel<FMT, BM, WGM, WGN, ST>;
    if (T::LDS > 65536) {
        const int r = once.run([&] { return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS) == hipSuccess; });
        if (r != SDMI_OK) return r;
    }
    const int64_t tiles = (d.M + BM - 1) / BM * ((d.N + T::BN - 1) / T::BN);
    kernel<<<(unsigned)tiles, T::THREADS, T::LDS, st>>>(d);
    SDMI_CHECK_LAUNCH();
    return SDMI_OK;
}

template <int FMT, int MT, int NF, int KW, int U, int SRC> static int direct_launch(const MxGemmDev& d, hipStream_t st) {
    const int sums = KW * MT * NF * 1024, codes = SRC < 0 ? 0 : (int)(d.ksteps * (d.M < 16 * MT ? d.M : 16 * MT) * (mx_row_bytes(128, FMT) + 4));
    const int64_t nx = (d.N + 63) / 64 * (4 / NF), ny = (d.M + 16 * MT - 1) / (16 * MT);
    if (KW * MT * NF * 1024 > 65536) {
        static SdmiPerDeviceOnce once;
        const int r = once.run([&] { return hipFuncSetAttribute(reinterpret_cast<const void*>(sdmi_mx_direct_kernel<FMT, MT, NF, KW, U, SRC>), hipFuncAttributeMaxDynamicSharedMemorySize, KW * MT * NF * 1024) == hipSuccess; });
        if (r != SDMI_OK) return r;
    }
    sdmi_mx_direct_kernel<FMT, MT, NF, KW, U, SRC><<<dim3((unsigned)nx, (unsigned)ny), 64 * KW, sums > codes ? sums : codes, st>>>(d);
    SDMI_CHECK_LAUNCH();
    return SDMI_OK;
}

template <int FMT, int MT, int NF> static int direct_fused(const MxGemmDev& d, int src, hipStream_t st) {
    return src == 0 ? direct_launch<FMT, MT, NF, 8, 2, 0>(d, st) : src == 1 ? direct_launch<FMT, MT, NF, 8, 2, 1>(d, st) : direct_launch<FMT, MT, NF, 8, 2, 2>(d, st);
}

template <int FMT> static int mx_launch(const MxGemmDev& d, MxKind kind, MxFused fused, int src, hipStream_t st) {
    switch (fused) {
        case MX_FUSED16x32: return direct_fused<FMT, 1, 2>(d, src, st);
        case MX_FUSED16x64: return direct_fused<FMT, 1, 4>(d, src, st);
        case MX_FUSED32x64: return direct_fused<FMT, 2, 4>(d, src, st);
        default: break;
    }
    switch (kind) {
        case MX_D16x32: return direct_launch<FMT, 1, 2, 8, 2, -1>(d, st);
        case MX_D16x64: return direct_launch<FMT, 1, 4, 8, 2, -1>(d, st);
        case MX_D32x64: return direct_launch<FMT, 2, 4, 8, 1, -1>(d, st);
        case MX_D48x64: return direct_launch<FMT, 3, 4, 8, 1, -1>(d, st);
        // Rings no deeper than leaves room for three workgroups on a CU, whose starts and stores then run under each other's
        // products (with an earlier epilogue, 4096 x 10240 x 1280, 64 x 128: 8 bits 76.8 -> 69.5 us, 4 bits 62.0 -> 53.5; 128 x 128,
        // 4 bits 48.9 -> 44.8).  With 8-bit operands that is two stages of 128 x 128, which wait for their loads when they are few
        // on a CU.  Two and three stages, us: 160 tiles (512 x 5120 x 5120) 29.7 and 23.9, 480 (1536 x 5120 x 5120) 38.1 and 36.5,
        // 520 (1664 x 5120 x 2560) 28.2 and 31.0, 1000 (3200 x 5120 x 5120) 70.7 and 68.1, 1280 (4096 x 5120 x 5120) 83.5 and 85.8, 2560
        // (4096 x 10240 x 1280) 49.5 and 54.9.
        case MX_T64x128: return tiled_launch<FMT, 64, 2, 2, 3>(d, st);
        case MX_T128x128:
            if constexpr (FMT == SDMI_MX_FP8)
                if ((d.M + 127) / 128 * ((d.N + 127) / 128) > 512) return tiled_launch<FMT, 128, 2, 2, 2>(d, st);
            return tiled_launch<FMT, 128, 2, 2, 3>(d, st);
        case MX_T128x256: return tiled_launch<FMT, 128, 2, 4, 4>(d, st);
        default: return tiled_launch<FMT, 256, 2, 4, FMT == SDMI_MX_FP8 ? 3 : 4>(d, st);      // (three 8-bit stages fill the LDS)
    }
}

extern "C" int sdmi_mx_gemm(const sdmi_mx_gemm_args* a, void* stream) {
    MxPlan plan;
    if (!mx_plan(a, &plan) || !a->w_codes || !a->w_scales || !a->out || (!a->x && (!a->x_codes || !a->x_scales))) return SDMI_ERR_BAD_ARG;
    const int type = mx_src_type(a->out_dtype);
    if (type < 0 || a->ld_out < a->N || (a->res && a->ld_res < a->N)) return SDMI_ERR_BAD_ARG;
    if (!aligned16(a->w_codes) || !aligned16(a->w_scales) || (!a->x && (!aligned16(a->x_codes) || !aligned16(a->x_scales)))) return SDMI_ERR_ALIGNMENT;
    if (a->M == 0) return SDMI_OK;
    if (plan.workspace > 0 && (!a->workspace || a->workspace_bytes < plan.workspace || !aligned16(a->workspace))) return SDMI_ERR_WORKSPACE;
    MxGemmDev d = {};
    d.xc = (const unsigned char*)a->x_codes; d.xs = (const unsigned char*)a->x_scales;
    const int src = plan.fused ? mx_src_type(a->x_dtype) : -1;
    if (plan.fused) {
        d.x = a->x; d.ldx = a->ldx;
    } else if (a->x) {
        unsigned char* const ws = (unsigned char*)a->workspace;
        unsigned char* const xs = ws + up256(a->M * mx_row_bytes(a->K, a->fmt));
        const int st = sdmi_mx_quantize(a->x, a->ldx, a->M, a->K, a->x_dtype, ws, xs, a->fmt, stream);
        if (st != SDMI_OK) return st;
        d.xc = ws; d.xs = xs;
    }
    d.wc = (const unsigned char*)a->w_codes; d.ws = (const unsigned char*)a->w_scales;
    d.bias = a->bias; d.res = a->res; d.out = a->out;
    d.M = a->M; d.N = a->N; d.K = a->K; d.ksteps = mx_ksteps(a->K); d.ld_res = a->ld_res; d.ld_out = a->ld_out;
    d.type = type;
    return a->fmt == SDMI_MX_FP8 ? mx_launch<SDMI_MX_FP8>(d, plan.kind, plan.fused, src, (hipStream_t)stream) : mx_launch<SDMI_MX_FP4>(d, plan.kind, plan.fused, src, (hipStream_t)stream);
}
