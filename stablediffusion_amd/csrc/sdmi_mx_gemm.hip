// sdmi_mx_gemm: out[m, n] = sum_k x[m, k] w[n, k] + bias[n] + res[m, n] with 4-bit block-scaled weights and 8- or 4-bit
// block-scaled activations, on v_mfma_scale_f32_16x16x128_f8f6f4 (fp32 accumulation, one rounding at the end).
//
// The instruction's first operand is the weights, so that an accumulator register quad is 4 consecutive rows of the WEIGHT
// fragment at one token.  Lane l of an operand holds row l % 16; a 4-bit lane the 32 values of k-block l / 16 (16 bytes),
// an 8-bit lane the values [16 (l / 16), + 16) and 64 further on; the lane's scale is that of block l / 16 either way.
//
// Packed weights: per group of 64 output columns and k-step of 128, four fragments of 64 lanes x 16 bytes, then (in a second
// buffer) 64 lanes x 4 scale bytes, one for each fragment (the instruction selects the byte).  Fragment f, row 4 g + r holds
// column 16 g + 4 f + r of its group: the four accumulator quads of a lane are then 16 CONSECUTIVE columns, stored as two
// 16-byte vectors, and the four lanes of a token write a whole 128-byte line.
#include "sdmi_mx.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;

// ---- packing -----------------------------------------------------------------------------------------------------------
template <int T>
__global__ __launch_bounds__(256) void sdmi_mx_pack_kernel(const typename MxElem<T>::type* w, int64_t ldw, int64_t N, int64_t K,
                                                           unsigned char* codes, unsigned char* scales, int vec) {
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
        mx_load8<T>(w + (n < N ? n : 0) * ldw + k0, have, vec, f[j]);
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
    const int nl = (int)(n & 63), frag = (nl & 15) >> 2, lane = (int)(kb & 3) * 16 + (nl >> 4) * 4 + (nl & 3);
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
    int64_t M, N, ksteps, ld_res, ld_out;
    int type, vec_out;         // of out and res: 0 bf16, 1 f16, 2 fp32
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

// out[m, n .. n + 4) for one lane: bias, residual, one rounding
__device__ __forceinline__ void mx_store_quad(const MxGemmDev& p, int64_t m, int64_t n, f32x4 v) {
    if (m >= p.M) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (n + r >= p.N) break;
        float a = v[r];
        if (p.bias) a += p.bias[n + r];
        if (p.type == 2) {
            if (p.res) a += reinterpret_cast<const float*>(p.res)[m * p.ld_res + n + r];
            reinterpret_cast<float*>(p.out)[m * p.ld_out + n + r] = a;
        } else {
            if (p.res) {
                const unsigned short b = reinterpret_cast<const unsigned short*>(p.res)[m * p.ld_res + n + r];
                a += p.type == 0 ? elem_to_f32<0>(b) : elem_to_f32<1>(b);
            }
            reinterpret_cast<unsigned short*>(p.out)[m * p.ld_out + n + r] = p.type == 0 ? elem_from_f32<0>(a) : elem_from_f32<1>(a);
        }
    }
}

// Few rows: a workgroup takes one weight fragment (16 columns) and MT x 16 tokens; its four waves take every fourth k-step
// straight from memory into registers and join their sums through LDS in a fixed order.
template <int FMT, int MT>
__global__ __launch_bounds__(256) void sdmi_mx_direct_kernel(MxGemmDev p) {
    __shared__ f32x4 part[4][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q = lane >> 4;
    const int64_t grp = blockIdx.x >> 2, m0 = (int64_t)blockIdx.y * (16 * MT);
    const int frag = blockIdx.x & 3;
    constexpr int RB = FMT == SDMI_MX_FP8 ? 128 : 64;      // bytes of a row's k-step
    const unsigned char* const wc = p.wc + grp * p.ksteps * 4096 + frag * 1024 + lane * 16;
    const unsigned char* const ws = p.ws + grp * p.ksteps * 256 + lane * 4 + frag;
    const unsigned char* xc[MT];
    int64_t xr[MT];
    f32x4 acc[MT];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) {
        xr[mi] = min(m0 + mi * 16 + row, p.M - 1);
        xc[mi] = p.xc + xr[mi] * p.ksteps * RB + q * 16;
        acc[mi] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    for (int64_t s = wave; s < p.ksteps; s += 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(wc + s * 4096);
        const int wsc = ws[s * 256];
#pragma unroll
        for (int mi = 0; mi < MT; ++mi) {
            const int xsc = p.xs[(s * p.M + xr[mi]) * 4 + q];
            const uint4 a = *reinterpret_cast<const uint4*>(xc[mi] + s * RB);
            if constexpr (FMT == SDMI_MX_FP8) {
                const uint4 b = *reinterpret_cast<const uint4*>(xc[mi] + s * RB + 64);
                acc[mi] = mx_mfma<FMT, 0>(mx_op4(w), mx_op8(a, b), acc[mi], wsc, xsc);
            } else {
                acc[mi] = mx_mfma<FMT, 0>(mx_op4(w), mx_op4(a), acc[mi], wsc, xsc);
            }
        }
    }
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) part[wave][mi][lane] = acc[mi];
    __syncthreads();
    for (int mi = wave; mi < MT; mi += 4) {
        const f32x4 v = (part[0][mi][lane] + part[1][mi][lane]) + (part[2][mi][lane] + part[3][mi][lane]);
        mx_store_quad(p, m0 + mi * 16 + row, grp * 64 + 16 * q + 4 * frag, v);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
constexpr int64_t MX_MAX_DIM = (int64_t)1 << 24;

extern "C" int64_t sdmi_mx_weight_codes_bytes(int64_t N, int64_t K) { return N <= 0 || K <= 0 ? -1 : (N + 63) / 64 * mx_ksteps(K) * 4096; }
extern "C" int64_t sdmi_mx_weight_scales_bytes(int64_t N, int64_t K) { return N <= 0 || K <= 0 ? -1 : (N + 63) / 64 * mx_ksteps(K) * 256; }

extern "C" int sdmi_mx_pack_linear(const void* w, int64_t ldw, int64_t N, int64_t K, int32_t dtype, void* codes, void* scales, void* stream) {
    const int t = mx_src_type(dtype);
    if (!w || !codes || !scales || t < 0 || N <= 0 || K <= 0 || N > MX_MAX_DIM || K > MX_MAX_DIM || ldw < K) return SDMI_ERR_BAD_ARG;
    if (!aligned16(codes) || !aligned16(scales)) return SDMI_ERR_ALIGNMENT;
    const int64_t n = (N + 63) / 64 * 64 * mx_ksteps(K) * 4, blocks = (n + 255) / 256;
    if (blocks >= ((int64_t)1 << 31)) return SDMI_ERR_BAD_ARG;
    const int vec = aligned16(w) && ldw % (t == 2 ? 4 : 8) == 0;
    hipStream_t st = (hipStream_t)stream;
    unsigned char *c = (unsigned char*)codes, *s = (unsigned char*)scales;
    if (t == 0) sdmi_mx_pack_kernel<0><<<(unsigned)blocks, 256, 0, st>>>((const unsigned short*)w, ldw, N, K, c, s, vec);
    else if (t == 1) sdmi_mx_pack_kernel<1><<<(unsigned)blocks, 256, 0, st>>>((const unsigned short*)w, ldw, N, K, c, s, vec);
    else sdmi_mx_pack_kernel<2><<<(unsigned)blocks, 256, 0, st>>>((const float*)w, ldw, N, K, c, s, vec);
    SDMI_CHECK_LAUNCH();
    return SDMI_OK;
}

static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

static bool mx_args_ok(const sdmi_mx_gemm_args* a) {
    if (!a || a->M < 0 || a->N <= 0 || a->K <= 0 || a->M >= ((int64_t)1 << 31) || a->N > MX_MAX_DIM || a->K > MX_MAX_DIM) return false;
    if (a->fmt != SDMI_MX_FP8 && a->fmt != SDMI_MX_FP4) return false;
    return !a->x || (mx_src_type(a->x_dtype) >= 0 && a->ldx >= a->K);
}

extern "C" int64_t sdmi_mx_gemm_workspace_bytes(const sdmi_mx_gemm_args* a) {
    if (!mx_args_ok(a)) return -1;
    if (!a->x || a->M == 0) return 0;
    return up256(a->M * mx_row_bytes(a->K, a->fmt)) + up256(a->M * mx_ksteps(a->K) * 4);
}

template <int FMT> static int mx_launch(const MxGemmDev& d, hipStream_t st) {
    const unsigned nx = (unsigned)((d.N + 63) / 64 * 4);
    const int mt = d.M <= 16 ? 1 : d.M <= 32 ? 2 : 4;
    const int64_t ny = (d.M + 16 * mt - 1) / (16 * mt);
    if (ny > 65535) return SDMI_ERR_BAD_ARG;
    const dim3 g(nx, (unsigned)ny);
    if (mt == 1) sdmi_mx_direct_kernel<FMT, 1><<<g, 256, 0, st>>>(d);
    else if (mt == 2) sdmi_mx_direct_kernel<FMT, 2><<<g, 256, 0, st>>>(d);
    else sdmi_mx_direct_kernel<FMT, 4><<<g, 256, 0, st>>>(d);
    SDMI_CHECK_LAUNCH();
    return SDMI_OK;
}

extern "C" int sdmi_mx_gemm(const sdmi_mx_gemm_args* a, void* stream) {
    if (!mx_args_ok(a) || !a->w_codes || !a->w_scales || !a->out || (!a->x && (!a->x_codes || !a->x_scales))) return SDMI_ERR_BAD_ARG;
    const int type = mx_src_type(a->out_dtype);
    if (type < 0 || a->ld_out < a->N || (a->res && a->ld_res < a->N)) return SDMI_ERR_BAD_ARG;
    if (!aligned16(a->w_codes) || !aligned16(a->w_scales) || (!a->x && (!aligned16(a->x_codes) || !aligned16(a->x_scales)))) return SDMI_ERR_ALIGNMENT;
    if (a->M == 0) return SDMI_OK;
    MxGemmDev d = {};
    d.xc = (const unsigned char*)a->x_codes; d.xs = (const unsigned char*)a->x_scales;
    if (a->x) {
        const int64_t need = sdmi_mx_gemm_workspace_bytes(a);
        if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)) return SDMI_ERR_WORKSPACE;
        unsigned char* const ws = (unsigned char*)a->workspace;
        unsigned char* const xs = ws + up256(a->M * mx_row_bytes(a->K, a->fmt));
        const int st = sdmi_mx_quantize(a->x, a->ldx, a->M, a->K, a->x_dtype, ws, xs, a->fmt, stream);
        if (st != SDMI_OK) return st;
        d.xc = ws; d.xs = xs;
    }
    d.wc = (const unsigned char*)a->w_codes; d.ws = (const unsigned char*)a->w_scales;
    d.bias = a->bias; d.res = a->res; d.out = a->out;
    d.M = a->M; d.N = a->N; d.ksteps = mx_ksteps(a->K); d.ld_res = a->ld_res; d.ld_out = a->ld_out;
    d.type = type;
    return a->fmt == SDMI_MX_FP8 ? mx_launch<SDMI_MX_FP8>(d, (hipStream_t)stream) : mx_launch<SDMI_MX_FP4>(d, (hipStream_t)stream);
}
