// sdmi_mx: the element-wise and row-wise operators around the block-scaled product (sdmi_mx_gemm.hip): quantisation of a
// matrix and its reading back, the gated activation, the RMS norm with the residual's addition - each with a 16-bit, fp32 or
// block-scaled result - and the packing of weights.  All of them are bound by bytes: every input is read once in 16-byte
// vectors, statistics stay in registers, the result is written once in the form its reader takes.
#include "sdmi_mx.h"

// ---- one k-step per 16 lanes -------------------------------------------------------------------------------------------
// A block of 256 threads owns a tile of 16 rows x STEPS k-steps: 16 lanes hold one k-step of one row, 8 values a lane.  So a
// row is read in 256-byte runs, the 16 rows of a code plane are written as one KB, and the 16 scale dwords of a k-step lie next
// to each other.  STEPS = 4 keeps four (gated: eight) loads a lane in flight; a launch too small to fill the chip with such
// tiles takes STEPS = 1, four times the waves with a quarter of the instructions each (gated 1 x 1280: 5.2 -> 3.2 us, 154 x 4096: 5.6 -> 3.5).
constexpr int EL_ROWS = 16;

struct MxElemArgs {
    const void* x;
    int64_t ldx, rows, K;      // gated: K = the width of one half, the gate starts at column K
    int64_t row0;              // the launch's first row
    void* out;                 // FMT none: [rows][ld_out] of the source's type or the given one
    int64_t ld_out;
    unsigned char* codes;
    unsigned char* scales;
    unsigned ktiles;
};

// OP 0: x   1: a gelu(b)   2: a silu(b)        FMT -1: plain result of type TO
template <int T, int OP, int FMT, int TO, int EL_STEPS>
__global__ __launch_bounds__(256) void sdmi_mx_elem_kernel(MxElemArgs p) {
    typedef typename MxElem<T>::type E;
    const unsigned tile_r = blockIdx.x / p.ktiles, tile_k = blockIdx.x - tile_r * p.ktiles;
    const int lane = threadIdx.x & 63, sub = threadIdx.x & 15;
    const int64_t row = p.row0 + (int64_t)tile_r * EL_ROWS + (threadIdx.x >> 4);
    const int64_t nsteps = mx_ksteps(p.K);
    const int64_t src_row = row < p.rows ? row : p.rows - 1;     // (the 16 lanes of a row past the end work on the last one and store nothing)
    const E* const xr = reinterpret_cast<const E*>(p.x) + src_row * p.ldx;
    float f[EL_STEPS][8], g[OP ? EL_STEPS : 1][8];
#pragma unroll
    for (int s = 0; s < EL_STEPS; ++s) {
        const int64_t k0 = ((int64_t)tile_k * EL_STEPS + s) * MX_KSTEP + sub * 8;
        const int n = (int)max((int64_t)0, min((int64_t)8, p.K - k0));
        mx_load8<T>(xr + k0, n, f[s]);
        if constexpr (OP != 0) mx_load8<T>(xr + p.K + k0, n, g[s]);
    }
#pragma unroll
    for (int s = 0; s < EL_STEPS; ++s) {
        const int64_t step = (int64_t)tile_k * EL_STEPS + s;
        if (step >= nsteps) break;                               // (uniform)
        const int64_t k0 = step * MX_KSTEP + sub * 8;
        const int n = (int)max((int64_t)0, min((int64_t)8, p.K - k0));
        if constexpr (OP != 0) mx_gate8<OP, FMT < 0 && TO == 2>(f[s], g[s]);
        if constexpr (FMT < 0) {
            if (row < p.rows && n > 0)
                mx_store8<TO>(reinterpret_cast<typename MxElem<TO>::type*>(p.out) + row * p.ld_out + k0, n, f[s]);
        } else {
            uint2 c;
            const unsigned dw = mx_quantise8<FMT>(f[s], lane, c);
            if (row < p.rows) {
                if constexpr (FMT == SDMI_MX_FP8)
                    *reinterpret_cast<uint2*>(p.codes + ((step * 2 + (sub >> 3)) * p.rows + row) * 64 + (sub & 7) * 8) = c;
                else
                    *reinterpret_cast<unsigned*>(p.codes + (step * p.rows + row) * 64 + sub * 4) = c.x;
                if (sub == 0) *reinterpret_cast<unsigned*>(p.scales + (step * p.rows + row) * 4) = dw;
            }
        }
    }
}

// The values that codes and scales stand for.  Every code has at most four significant bits: a bf16 holds the value exactly
// (down to its subnormals), an f16 rounds it to its own range.
template <int FMT, int TO, int EL_STEPS>
__global__ __launch_bounds__(256) void sdmi_mx_dequantise_kernel(MxElemArgs p) {
    const unsigned tile_r = blockIdx.x / p.ktiles, tile_k = blockIdx.x - tile_r * p.ktiles;
    const int sub = threadIdx.x & 15;
    const int64_t row = p.row0 + (int64_t)tile_r * EL_ROWS + (threadIdx.x >> 4), nsteps = mx_ksteps(p.K);
    if (row >= p.rows) return;
    uint2 c[EL_STEPS];
    unsigned char sc[EL_STEPS];
#pragma unroll
    for (int s = 0; s < EL_STEPS; ++s) {
        const int64_t step = (int64_t)tile_k * EL_STEPS + s;
        if (step >= nsteps) break;
        if constexpr (FMT == SDMI_MX_FP8) c[s] = *reinterpret_cast<const uint2*>(p.codes + ((step * 2 + (sub >> 3)) * p.rows + row) * 64 + (sub & 7) * 8);
        else c[s].x = *reinterpret_cast<const unsigned*>(p.codes + (step * p.rows + row) * 64 + sub * 4);
        sc[s] = p.scales[(step * p.rows + row) * 4 + (sub >> 2)];
    }
#pragma unroll
    for (int s = 0; s < EL_STEPS; ++s) {
        const int64_t step = (int64_t)tile_k * EL_STEPS + s;
        if (step >= nsteps) break;
        const int64_t k0 = step * MX_KSTEP + sub * 8;
        const int n = (int)max((int64_t)0, min((int64_t)8, p.K - k0));
        if (n == 0) continue;
        float f[8];
        if constexpr (FMT == SDMI_MX_FP8) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[s].x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[s].x, true);
            const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[s].y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[s].y, true);
            f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1]; f[4] = d[0]; f[5] = d[1]; f[6] = e[0]; f[7] = e[1];
        } else {
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s].x, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s].x, 1.0f, 1);
            const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s].x, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s].x, 1.0f, 3);
            f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1]; f[4] = d[0]; f[5] = d[1]; f[6] = e[0]; f[7] = e[1];
        }
        // 2^(byte - 127): byte 0 is the subnormal 2^-127, byte 255 a NaN
        const unsigned byte = sc[s];
        const float scale = __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= scale;
        mx_store8<TO>(reinterpret_cast<typename MxElem<TO>::type*>(p.out) + row * p.ld_out + k0, n, f);
    }
}

// ---- RMS norm ----------------------------------------------------------------------------------------------------------
// s = x + res (stored in x's type), y = s / sqrt(mean s^2 + eps) * gamma, of the fp32 sum.  TPR threads hold a row in
// registers, U chunks of 8 values each, so that a row is read once.
struct MxNormArgs {
    const void* x;
    const void* res;           // NULL: s = x
    const float* gamma;
    void* sum_out;
    void* out;
    unsigned char* codes;
    unsigned char* scales;
    int64_t ldx, ld_res, rows, C, row0;      // row0: the launch's first row
    double inv_c;
    float eps;
};

template <int T, int FMT, int TO, int TPR, int U>
__global__ __launch_bounds__(256) void sdmi_rmsnorm_kernel(MxNormArgs p) {
    typedef typename MxElem<T>::type E;
    constexpr int RPB = 256 / TPR;
    __shared__ double part[RPB][TPR / 64];
    const int t = threadIdx.x % TPR, r = threadIdx.x / TPR, lane = threadIdx.x & 63;
    // Workgroups go round the 8 XCDs; of every 64 each XCD takes 8 neighbours, whose codes and scales share cache lines of its
    // L2 (16384 x 5120 with residual and 8-bit output: 129 -> 120 us; runs of 2 and 32 the same or slower, one run an XCD 152:
    // eight far places of memory at a time).
    constexpr unsigned RUN = 8;
    unsigned block = blockIdx.x;
    if (block < gridDim.x / (8 * RUN) * (8 * RUN)) block = block / (8 * RUN) * (8 * RUN) + (block & 7) * RUN + block % (8 * RUN) / 8;
    const int64_t row = p.row0 + (int64_t)block * RPB + r, srow = row < p.rows ? row : p.rows - 1;
    const E* const xr = reinterpret_cast<const E*>(p.x) + srow * p.ldx;
    float f[U][8], q[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t c0 = ((int64_t)u * TPR + t) * 8;
        const int n = (int)max((int64_t)0, min((int64_t)8, p.C - c0));
        mx_load8<T>(xr + c0, n, f[u]);
    }
    if (p.res) {
        const E* const rr = reinterpret_cast<const E*>(p.res) + srow * p.ld_res;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t c0 = ((int64_t)u * TPR + t) * 8;
            const int n = (int)max((int64_t)0, min((int64_t)8, p.C - c0));
            mx_load8<T>(rr + c0, n, q[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) f[u][j] += q[u][j];
    }
    // In fp64, which costs nothing beside the bytes: every value of a row is scaled by the same number, so an error in it moves
    // all of them towards the same side of the codes' rounding borders; and no square overflows or vanishes.
    double ss = 0.0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fma((double)f[u][j], (double)f[u][j], ss);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
    if constexpr (TPR > 64) {
        if (lane == 0) part[r][t >> 6] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) ss += part[r][w];
    }
    // 1 / sqrt(v), one Newton step from the approximation, as the sum of two fp32 numbers.  Of rows of subnormals it lies past
    // fp32's largest number, of rows near that one among the subnormals: there `up` brings it back, and the values with it.
    const double v = ss * p.inv_c + (double)p.eps;
    double r1 = __builtin_amdgcn_rsq(v);
    if (v > 0.0 && v < 1e300) r1 *= fma(-0.5 * v * r1, r1, 1.5);
    const float up = r1 > 0x1p96 ? 0x1p64f : r1 < 0x1p-96 ? 0x1p-64f : 1.0f;
    r1 *= r1 > 0x1p96 ? 0x1p-64 : r1 < 0x1p-96 ? 0x1p64 : 1.0;
    const float r0 = (float)r1, lo = r0 < 3e38f ? (float)(r1 - (double)r0) : 0.0f;
    const int64_t nsteps = mx_ksteps(p.C);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t c0 = ((int64_t)u * TPR + t) * 8;
        const int n = (int)max((int64_t)0, min((int64_t)8, p.C - c0));
        if (p.sum_out && row < p.rows && n > 0)
            mx_store8<T>(reinterpret_cast<E*>(p.sum_out) + row * p.C + c0, n, f[u]);
        float gm[8];
        mx_load8<2>(p.gamma + c0, n, gm);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float s = f[u][j] * up;
            gm[j] *= fmaf(s, r0, s * lo);
        }
        if constexpr (FMT < 0) {
            if (row < p.rows && n > 0)
                mx_store8<TO>(reinterpret_cast<typename MxElem<TO>::type*>(p.out) + row * p.C + c0, n, gm);
        } else {
            const int64_t step = c0 / MX_KSTEP;
            if (step >= nsteps) continue;                        // (whole groups of 16 lanes)
            uint2 c;
            const unsigned dw = mx_quantise8<FMT>(gm, lane, c);
            if (row < p.rows) {
                if constexpr (FMT == SDMI_MX_FP8)
                    *reinterpret_cast<uint2*>(p.codes + (c0 / 64 * p.rows + row) * 64 + (c0 & 63)) = c;
                else
                    *reinterpret_cast<unsigned*>(p.codes + (step * p.rows + row) * 64 + ((c0 & 127) >> 1)) = c.x;
                if ((lane & 15) == 0) *reinterpret_cast<unsigned*>(p.scales + (step * p.rows + row) * 4) = dw;
            }
        }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool fmt_ok(int32_t fmt) { return fmt == SDMI_MX_FP8 || fmt == SDMI_MX_FP4; }

extern "C" int64_t sdmi_mx_codes_bytes(int64_t rows, int64_t K, int32_t fmt) {
    return !mx_sizes_ok(rows, K) || !fmt_ok(fmt) ? -1 : rows * mx_row_bytes(K, fmt);
}
extern "C" int64_t sdmi_mx_scales_bytes(int64_t rows, int64_t K) { return !mx_sizes_ok(rows, K) ? -1 : rows * mx_ksteps(K) * 4; }

// The k-steps of a tile, and a launch for every `rows` rows: all of them but where the tiles are more than a grid holds.
struct ElemGrid { int64_t rows; int steps; };
static ElemGrid elem_grid(int64_t rows, int64_t K, MxElemArgs* a) {
    const int64_t rt = (rows + EL_ROWS - 1) / EL_ROWS, ks = mx_ksteps(K);
    const int steps = rt * ((ks + 3) / 4) >= 1024 ? 4 : 1;
    a->ktiles = (unsigned)((ks + steps - 1) / steps);
    return {mx_grid_blocks(256) / a->ktiles * EL_ROWS, steps};
}
template <class F> static int elem_rows(MxElemArgs a, const ElemGrid& g, F&& launch) {
    for (; a.row0 < a.rows; a.row0 += g.rows) {
        const int64_t rows = a.rows - a.row0 < g.rows ? a.rows - a.row0 : g.rows;
        launch(a, (unsigned)((rows + EL_ROWS - 1) / EL_ROWS * a.ktiles));
        SDMI_CHECK_LAUNCH();
    }
    return SDMI_OK;
}

template <int T, int OP, int FMT, int TO> static int elem_steps(const MxElemArgs& a, const ElemGrid& g, hipStream_t st) {
    return elem_rows(a, g, [&](const MxElemArgs& b, unsigned blocks) {
        if (g.steps == 4) sdmi_mx_elem_kernel<T, OP, FMT, TO, 4><<<blocks, 256, 0, st>>>(b);
        else sdmi_mx_elem_kernel<T, OP, FMT, TO, 1><<<blocks, 256, 0, st>>>(b);
    });
}
template <int T, int OP>
static int elem_launch(const MxElemArgs& a, int fmt, int to, const ElemGrid& g, hipStream_t st) {
    if (fmt == SDMI_MX_FP8) return elem_steps<T, OP, SDMI_MX_FP8, 0>(a, g, st);
    if (fmt == SDMI_MX_FP4) return elem_steps<T, OP, SDMI_MX_FP4, 0>(a, g, st);
    if constexpr (OP == 0) return SDMI_ERR_BAD_ARG;
    else return to == 0 ? elem_steps<T, OP, -1, 0>(a, g, st) : to == 1 ? elem_steps<T, OP, -1, 1>(a, g, st) : elem_steps<T, OP, -1, 2>(a, g, st);
}

extern "C" int sdmi_mx_quantize(const void* x, int64_t ldx, int64_t rows, int64_t K, int32_t dtype, void* codes, void* scales,
                                int32_t fmt, void* stream) {
    const int t = mx_src_type(dtype);
    if (!x || !codes || !scales || t < 0 || !fmt_ok(fmt) || !mx_sizes_ok(rows, K) || ldx < K) return SDMI_ERR_BAD_ARG;
    if (!aligned16(codes) || !aligned16(scales)) return SDMI_ERR_ALIGNMENT;
    if (rows == 0) return SDMI_OK;
    MxElemArgs a = {};
    a.x = x; a.ldx = ldx; a.rows = rows; a.K = K; a.codes = (unsigned char*)codes; a.scales = (unsigned char*)scales;
    const ElemGrid g = elem_grid(rows, K, &a);
    hipStream_t st = (hipStream_t)stream;
    return t == 0 ? elem_launch<0, 0>(a, fmt, 0, g, st) : t == 1 ? elem_launch<1, 0>(a, fmt, 0, g, st) : elem_launch<2, 0>(a, fmt, 0, g, st);
}

extern "C" int sdmi_gated(const void* x, int64_t ldx, int64_t rows, int64_t inner, int32_t dtype, int32_t act, void* out,
                          int32_t out_dtype, void* scales, int32_t fmt, void* stream) {
    const int t = mx_src_type(dtype), to = fmt == SDMI_MX_NONE ? mx_src_type(out_dtype) : 0;
    if (!x || !out || t < 0 || to < 0 || (act != 0 && act != 1) || (fmt != SDMI_MX_NONE && (!fmt_ok(fmt) || !scales)) ||
        !mx_sizes_ok(rows, inner) || ldx < 2 * inner) return SDMI_ERR_BAD_ARG;
    if (fmt != SDMI_MX_NONE && (!aligned16(out) || !aligned16(scales))) return SDMI_ERR_ALIGNMENT;
    if (rows == 0) return SDMI_OK;
    MxElemArgs a = {};
    a.x = x; a.ldx = ldx; a.rows = rows; a.K = inner; a.codes = (unsigned char*)out; a.scales = (unsigned char*)scales;
    a.out = out; a.ld_out = inner;
    const ElemGrid g = elem_grid(rows, inner, &a);
    hipStream_t st = (hipStream_t)stream;
    if (act == 0)
        return t == 0 ? elem_launch<0, 1>(a, fmt, to, g, st) : t == 1 ? elem_launch<1, 1>(a, fmt, to, g, st) : elem_launch<2, 1>(a, fmt, to, g, st);
    return t == 0 ? elem_launch<0, 2>(a, fmt, to, g, st) : t == 1 ? elem_launch<1, 2>(a, fmt, to, g, st) : elem_launch<2, 2>(a, fmt, to, g, st);
}

extern "C" int sdmi_mx_dequantize(const void* codes, const void* scales, int64_t rows, int64_t K, int32_t fmt, void* out,
                                  int64_t ld_out, int32_t out_dtype, void* stream) {
    const int to = mx_src_type(out_dtype);
    if (!codes || !scales || !out || to < 0 || !fmt_ok(fmt) || !mx_sizes_ok(rows, K) || ld_out < K) return SDMI_ERR_BAD_ARG;
    if (!aligned16(codes) || !aligned16(scales)) return SDMI_ERR_ALIGNMENT;
    if (rows == 0) return SDMI_OK;
    MxElemArgs a = {};
    a.rows = rows; a.K = K; a.codes = (unsigned char*)codes; a.scales = (unsigned char*)scales; a.out = out; a.ld_out = ld_out;
    const ElemGrid g = elem_grid(rows, K, &a);
    hipStream_t st = (hipStream_t)stream;
#define SDMI_DQ(F, O) elem_rows(a, g, [&](const MxElemArgs& b, unsigned blocks) { \
        if (g.steps == 4) sdmi_mx_dequantise_kernel<F, O, 4><<<blocks, 256, 0, st>>>(b); else sdmi_mx_dequantise_kernel<F, O, 1><<<blocks, 256, 0, st>>>(b); })
    if (fmt == SDMI_MX_FP8) return to == 0 ? SDMI_DQ(SDMI_MX_FP8, 0) : to == 1 ? SDMI_DQ(SDMI_MX_FP8, 1) : SDMI_DQ(SDMI_MX_FP8, 2);
    return to == 0 ? SDMI_DQ(SDMI_MX_FP4, 0) : to == 1 ? SDMI_DQ(SDMI_MX_FP4, 1) : SDMI_DQ(SDMI_MX_FP4, 2);
#undef SDMI_DQ
}

template <int T, int FMT, int TO, int TPR, int U> static int norm_rows(MxNormArgs a, hipStream_t st) {
    constexpr int RPB = 256 / TPR;
    for (; a.row0 < a.rows; a.row0 += mx_grid_blocks(256) * RPB) {             // (one launch but for more rows than a grid holds)
        const int64_t blocks = (a.rows - a.row0 + RPB - 1) / RPB;
        sdmi_rmsnorm_kernel<T, FMT, TO, TPR, U><<<(unsigned)(blocks < mx_grid_blocks(256) ? blocks : mx_grid_blocks(256)), 256, 0, st>>>(a);
        SDMI_CHECK_LAUNCH();
    }
    return SDMI_OK;
}

template <int T, int FMT, int TO>
static int norm_launch(const MxNormArgs& a, hipStream_t st) {
    // As few threads a row as hold it in one chunk of 8 values each, and from 2048 values on 256 threads with as many chunks as
    // the row needs and no more: an empty chunk costs registers and instructions (16384 x 5120: 256 x 3 120 us, 256 x 4 143,
    // 128 x 5 148, 512 x 2 127, 64 x 10 208; 32768 x 1024: 128 x 1 47 us, 64 x 2 50, 256 x 1 58).
    if (a.C <= 512) return norm_rows<T, FMT, TO, 64, 1>(a, st);
    if (a.C <= 1024) return norm_rows<T, FMT, TO, 128, 1>(a, st);
    switch ((a.C + 2047) / 2048) {
        case 1: return norm_rows<T, FMT, TO, 256, 1>(a, st);
        case 2: return norm_rows<T, FMT, TO, 256, 2>(a, st);
        case 3: return norm_rows<T, FMT, TO, 256, 3>(a, st);
        case 4: return norm_rows<T, FMT, TO, 256, 4>(a, st);
        case 5: return norm_rows<T, FMT, TO, 256, 5>(a, st);
        case 6: return norm_rows<T, FMT, TO, 256, 6>(a, st);
        case 7: return norm_rows<T, FMT, TO, 256, 7>(a, st);
        default: return norm_rows<T, FMT, TO, 256, 8>(a, st);
    }
}

template <int T> static int norm_type(const MxNormArgs& a, int fmt, int to, hipStream_t st) {
    if (fmt == SDMI_MX_FP8) return norm_launch<T, SDMI_MX_FP8, 0>(a, st);
    if (fmt == SDMI_MX_FP4) return norm_launch<T, SDMI_MX_FP4, 0>(a, st);
    return to == 0 ? norm_launch<T, -1, 0>(a, st) : to == 1 ? norm_launch<T, -1, 1>(a, st) : norm_launch<T, -1, 2>(a, st);
}

extern "C" int sdmi_rmsnorm(const void* x, int64_t ldx, const void* res, int64_t ld_res, const float* gamma, float eps,
                            int64_t rows, int64_t C, int32_t dtype, void* sum_out, void* out, int32_t out_dtype, void* scales,
                            int32_t fmt, void* stream) {
    const int t = mx_src_type(dtype), to = fmt == SDMI_MX_NONE ? mx_src_type(out_dtype) : 0;
    if (!x || !gamma || !out || t < 0 || to < 0 || (fmt != SDMI_MX_NONE && (!fmt_ok(fmt) || !scales)) || !mx_sizes_ok(rows, C) ||
        C > SDMI_RMSNORM_MAX_C || ldx < C || (res && (ld_res < C || !sum_out)) || !(eps >= 0.0f)) return SDMI_ERR_BAD_ARG;
    if (!aligned16(gamma) || (fmt != SDMI_MX_NONE && (!aligned16(out) || !aligned16(scales)))) return SDMI_ERR_ALIGNMENT;
    if (rows == 0) return SDMI_OK;
    MxNormArgs a = {};
    a.x = x; a.res = res; a.gamma = gamma; a.sum_out = res ? sum_out : nullptr; a.out = out;
    a.codes = (unsigned char*)out; a.scales = (unsigned char*)scales;
    a.ldx = ldx; a.ld_res = ld_res; a.rows = rows; a.C = C; a.inv_c = 1.0 / (double)C; a.eps = eps;
    hipStream_t st = (hipStream_t)stream;
    return t == 0 ? norm_type<0>(a, fmt, to, st) : t == 1 ? norm_type<1>(a, fmt, to, st) : norm_type<2>(a, fmt, to, st);
}
