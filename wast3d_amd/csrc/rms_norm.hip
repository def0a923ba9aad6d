// Root-mean-square norm of feature rows, with the residual's addition in front and, optionally, e4m3 rows with one E8M0 scale each behind (the format of
// w3d_quantize_rows_fp8, so that normalised rows — equal norms: the L2 match is a cosine match — go straight into w3d_knn_fp8).
//
//   s = x + residual;  r = 1 / sqrt(mean(s^2) + eps);  y = s r w
//   given dy (and ds, what reaches s from elsewhere):  g = dy w;  x^ = s r;  dx = r (g - x^ mean(g x^)) + ds;  dw = sum over rows of dy x^
// The backward pass forms s again from x and the residual, unrounded: from the rounded s its error would show in dw (1.5 x the error of one rounding).
//
// Bound by HBM: every element is read once and written once.  A row stays in registers between its sum and its output, in f32.  Sums are f32 for 16-bit rows, 64-bit where a bf16 row's
// squares leave f32's range.
// For 8-bit rows the forward pass is 64-bit between the loads and one rounding to f32: what 32 bits lose (2^-23 or so) moves values over e4m3's borders by whole steps: 100 - 127 of 256 million at
// 1 000 000 x 256, none this way (at the same speed).  f32 rows are formed alike, so that quantising them afterwards gives the same bytes.
// G lanes share a row (a wave holds 64 / G rows), 8 elements per lane and vector, NV vectors per lane: G x NV is the smallest that covers the row, wide
// rows take the whole block of 256 lanes.  Rows beyond 8 192 elements are read again instead of kept (second and third reading come from L2).
//
// Measured, bf16: 1 000 000 x 256 with a residual into 8 bits 326 us (5.5 TB/s); 65 536 x 256 with a residual 22.8 us, backward 27.2 + 4.4 us (fold of dw); kept rows 4.7 - 6.4 TB/s forward,
// 3.4 - 5.4 backward (131 072 x 256 .. 16 384 x 8 192), rows read again 3.4 - 3.7 and 2.4 (16 384 wide).
#include <type_traits>
#include "rows16.h"

namespace {

constexpr int NORM_BLOCK = 256, MAX_WIDTH = 1 << 30;      // (columns are 32-bit)

struct NormArgs {
    const char *x, *res, *w;
    char *y, *s;
    float *rstd;
    uint8_t *q;
    int32_t *scale;
    int64_t R;
    int d, w_f32;
    float eps;
    double inv_d;
};

template <int DT>
__device__ __forceinline__ void load_weight(const char *w, int w_f32, int c, int d, float (&v)[8]) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 1.f;
    } else if (w_f32) load8<W3D_DTYPE_F32>(w + (int64_t)c * 4, d - c, v);
    else load8<DT>(w + (int64_t)c * Elem<DT>::B, d - c, v);
}

// 8 elements of s = x + residual, in f32
template <int DT, typename A>
__device__ __forceinline__ void sum_row(const A &a, int64_t at, int c, float (&s)[8]) {
    load8<DT>(a.x + (at + c) * Elem<DT>::B, a.d - c, s);
    if (a.res) {
        float t[8];
        load8<DT>(a.res + (at + c) * Elem<DT>::B, a.d - c, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += t[i];
    }
}

// sum / maximum over the G lanes of a row; G = 256: over the block (red: 4 floats of LDS per slot; every lane of the block calls)
template <int G, bool MAX, typename T>
__device__ __forceinline__ T group_reduce(T v, T *red) {
    auto op = [](T a, T b) { return MAX ? (T)fmaxf(a, b) : a + b; };
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
    if (G == 256) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = op(op(red[0], red[1]), op(red[2], red[3]));
    }
    return v;
}

// The forward pass's type: 64 bits for 8-bit rows, and for f32 ones (the same rows, quantised afterwards, are the same bytes)
template <int DT, bool Q> struct Wide { typedef typename std::conditional<Q || DT == W3D_DTYPE_F32, double, float>::type T; };
// Has a 32-bit sum of squares left f32's range, or come near its end?  (bf16 rows past 1.8e19 or below 1e-15 or so, rows of zeros: they are summed again in 64 bits.  In 64 bits throughout, 65 536 x 256 from the
// caches take 14.8 us instead of 13.8.)
template <int DT> __device__ __forceinline__ bool out_of_range(float sum) { return DT == W3D_DTYPE_BF16 && !(sum >= 0x1p-100f && sum <= 0x1.fffffep127f); }
template <int DT> __device__ __forceinline__ bool out_of_range(double) { return false; }
__device__ __forceinline__ float inverse_rms(float sum, const NormArgs &a) { return 1.0f / sqrtf(sum * (float)a.inv_d + a.eps); }
// 1 / sqrt(mean + eps) of a row's 64-bit sum of squares: the instruction's estimate and two Newton steps.  Where they give no number (a mean of 0, infinity, NaN) the estimate stands: infinity, 0, NaN.
__device__ __forceinline__ double inverse_rms(double sum, const NormArgs &a) {
    const double v = sum * a.inv_d + (double)a.eps, r0 = __builtin_amdgcn_rsq(v);
    double r = r0;
#pragma unroll
    for (int i = 0; i < 2; ++i) r = r * fma(-0.5 * v * r, r, 1.5);
    return r > 0.0 ? r : r0;
}

// the E8M0 exponent of a row: the smallest power of two that takes amax into e4m3's range (448 = 0.875 2^9), 127 for a row of zeros (or one without a finite maximum below 2^127)
__device__ __forceinline__ int e8m0_of(float amax) {
    int ex = 0;
    const float m = frexpf(amax, &ex);
    int e = (m <= 0.875f ? ex - 9 : ex - 8) + 127;
    if (!(amax > 0.f)) e = 127;
    return min(max(e, 1), 254);
}
__device__ __forceinline__ void store_fp8(uint8_t *p, int n, const float (&v)[8], float inv) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = v[i] * inv, t[i] = t[i] != t[i] ? t[i] : fminf(fmaxf(t[i], -448.f), 448.f);   // (a NaN stays one)
    int w[2] = {0, 0};
    w[0] = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], w[0], false);
    w[0] = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w[0], true);
    w[1] = __builtin_amdgcn_cvt_pk_fp8_f32(t[4], t[5], w[1], false);
    w[1] = __builtin_amdgcn_cvt_pk_fp8_f32(t[6], t[7], w[1], true);
    if (n >= 8) { __builtin_memcpy(p, w, 8); return; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
}

template <int DT, int G, int NV, bool Q>
__global__ __launch_bounds__(NORM_BLOCK) void rms_norm_kernel(NormArgs a) {
    typedef typename Wide<DT, Q>::T T;
    constexpr int EB = Elem<DT>::B, RPB = NORM_BLOCK / G;
    __shared__ float red[4];
    __shared__ T red_sum[4];
    __shared__ double red_again[4];
    const int gl = threadIdx.x & (G - 1), c0 = gl * 8;
    float w[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) load_weight<DT>(a.w, a.w_f32, c0 + v * G * 8, a.d, w[v]);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.R; r0 += (int64_t)gridDim.x * RPB) {        // (uniform over the block: group_reduce<256> has barriers)
        const int64_t r = r0 + threadIdx.x / G;
        const bool live = r < a.R;
        const int64_t at = (live ? r : a.R - 1) * a.d;
        float s[NV][8];
        T sum = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * G * 8;
            sum_row<DT>(a, at, c, s[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fma((T)s[v][i], (T)s[v][i], sum);
        sum = group_reduce<G, false>(sum, red_sum);
        T rs = inverse_rms(sum, a);
        if (out_of_range<DT>(sum)) {                                        // (alike for all lanes of a row)
            double again = 0;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) again = fma((double)s[v][i], (double)s[v][i], again);
            rs = (T)inverse_rms(group_reduce<G, false>(again, red_again), a);
        }
        if (a.rstd && live && gl == 0) a.rstd[r] = (float)rs;
        if (a.s && live) {
#pragma unroll
            for (int v = 0; v < NV; ++v) { const int c = c0 + v * G * 8; store8<DT>(a.s + (at + c) * EB, a.d - c, s[v]); }
        }
        float amax = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) { s[v][i] = (float)((T)s[v][i] * rs * (T)w[v][i]); amax = fmaxf(amax, fabsf(s[v][i])); }
        if (!Q && live) {
#pragma unroll
            for (int v = 0; v < NV; ++v) { const int c = c0 + v * G * 8; store8<DT>(a.y + (at + c) * EB, a.d - c, s[v]); }
        }
        if (Q) {
            const int e = e8m0_of(group_reduce<G, true>(amax, red));
            const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
            if (live) {
                if (gl == 0) a.scale[r] = e;
#pragma unroll
                for (int v = 0; v < NV; ++v) { const int c = c0 + v * G * 8; store_fp8(a.q + at + c, a.d - c, s[v], inv); }
            }
        }
    }
}

// rows of more than 256 x 8 x 4 elements: one block per row, the row read again for every pass over it
template <int DT, bool Q>
__global__ __launch_bounds__(NORM_BLOCK) void rms_norm_wide_kernel(NormArgs a) {
    typedef typename Wide<DT, Q>::T T;
    constexpr int EB = Elem<DT>::B;
    __shared__ float red[4];
    __shared__ T red_sum[4];
    __shared__ double red_again[4];
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const int64_t at = r * a.d;
        float s[8], w[8];
        T sum = 0;
        for (int c = threadIdx.x * 8; c < a.d; c += NORM_BLOCK * 8) {
            sum_row<DT>(a, at, c, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fma((T)s[i], (T)s[i], sum);
        }
        sum = group_reduce<256, false>(sum, red_sum);
        T rs = inverse_rms(sum, a);
        if (out_of_range<DT>(sum)) {
            double again = 0;
            for (int c = threadIdx.x * 8; c < a.d; c += NORM_BLOCK * 8) {
                sum_row<DT>(a, at, c, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) again = fma((double)s[i], (double)s[i], again);
            }
            rs = (T)inverse_rms(group_reduce<256, false>(again, red_again), a);
        }
        if (a.rstd && threadIdx.x == 0) a.rstd[r] = (float)rs;
        float amax = 0.f;
        for (int c = threadIdx.x * 8; c < a.d; c += NORM_BLOCK * 8) {
            sum_row<DT>(a, at, c, s);
            load_weight<DT>(a.w, a.w_f32, c, a.d, w);
            if (a.s) store8<DT>(a.s + (at + c) * EB, a.d - c, s);
#pragma unroll
            for (int i = 0; i < 8; ++i) { s[i] = (float)((T)s[i] * rs * (T)w[i]); amax = c + i < a.d ? fmaxf(amax, fabsf(s[i])) : amax; }
            if (!Q) store8<DT>(a.y + (at + c) * EB, a.d - c, s);
        }
        if (!Q) continue;
        const int e = e8m0_of(group_reduce<256, true>(amax, red));
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
        if (threadIdx.x == 0) a.scale[r] = e;
        for (int c = threadIdx.x * 8; c < a.d; c += NORM_BLOCK * 8) {
            sum_row<DT>(a, at, c, s);
            load_weight<DT>(a.w, a.w_f32, c, a.d, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = (float)((T)s[i] * rs * (T)w[i]);
            store_fp8(a.q + at + c, a.d - c, s, inv);
        }
    }
}

// ---- backward: the rows of a block are walked by the same lanes, so every lane keeps the weight gradient of its own columns in registers; the block's rows are folded in LDS, the
// blocks' partial sums by a second launch in a fixed order (no atomics: the same bits every time)
struct NormBwdArgs {
    const char *x, *res, *w, *dy, *ds;
    const float *rstd;
    char *dx;
    float *part;                 // [gridDim.x][d] or NULL
    int64_t R;
    int d, w_f32;
    float inv_d;
};

template <int DT, int G, int NV>
__global__ __launch_bounds__(NORM_BLOCK) void rms_norm_bwd_kernel(NormBwdArgs a) {
    constexpr int EB = Elem<DT>::B, RPB = NORM_BLOCK / G;
    __shared__ float red[4];
    __shared__ float fold[RPB > 1 ? NORM_BLOCK * NV * 8 : 1];
    const int gl = threadIdx.x & (G - 1), c0 = gl * 8;
    float w[NV][8], dw[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        load_weight<DT>(a.w, a.w_f32, c0 + v * G * 8, a.d, w[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[v][i] = 0.f;
    }
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.R; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + threadIdx.x / G;
        const bool live = r < a.R;
        const int64_t rr = live ? r : a.R - 1, at = rr * a.d;
        const float rs = a.rstd[rr];
        float x[NV][8], g[NV][8], dot = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * G * 8;
            sum_row<DT>(a, at, c, x[v]);
            load8<DT>(a.dy + (at + c) * EB, a.d - c, g[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[v][i] *= rs;
                if (live) dw[v][i] = fmaf(g[v][i], x[v][i], dw[v][i]);
                g[v][i] *= w[v][i];
                dot = fmaf(g[v][i], x[v][i], dot);
            }
        dot = group_reduce<G, false>(dot, red) * a.inv_d;
        if (!live || !a.dx) continue;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = c0 + v * G * 8;
            float t[8];
            if (a.ds) load8<DT>(a.ds + (at + c) * EB, a.d - c, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[v][i] = rs * (g[v][i] - x[v][i] * dot) + (a.ds ? t[i] : 0.f);
            store8<DT>(a.dx + (at + c) * EB, a.d - c, x[v]);
        }
    }
    if (!a.part) return;
    if (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) fold[(v * 8 + i) * NORM_BLOCK + threadIdx.x] = dw[v][i];
        __syncthreads();
        if (threadIdx.x >= G) return;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 1; j < RPB; ++j) dw[v][i] += fold[(v * 8 + i) * NORM_BLOCK + j * G + gl];
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = c0 + v * G * 8;
        store8<W3D_DTYPE_F32>(a.part + (int64_t)blockIdx.x * a.d + c, a.d - c, dw[v]);
    }
}

template <int DT>
__global__ __launch_bounds__(NORM_BLOCK) void rms_norm_bwd_wide_kernel(NormBwdArgs a) {
    constexpr int EB = Elem<DT>::B;
    __shared__ float red[4];
    for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
        const int64_t at = r * a.d;
        const float rs = a.rstd[r];
        float dot = 0.f, x[8], g[8], w[8];
        for (int c = threadIdx.x * 8; c < a.d; c += NORM_BLOCK * 8) {
            sum_row<DT>(a, at, c, x);
            load8<DT>(a.dy + (at + c) * EB, a.d - c, g);
            load_weight<DT>(a.w, a.w_f32, c, a.d, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) dot = fmaf(g[i] * w[i], x[i] * rs, dot);
        }
        dot = group_reduce<256, false>(dot, red) * a.inv_d;
        for (int c = threadIdx.x * 8; c < a.d; c += NORM_BLOCK * 8) {
            float t[8];
            sum_row<DT>(a, at, c, x);
            load8<DT>(a.dy + (at + c) * EB, a.d - c, g);
            load_weight<DT>(a.w, a.w_f32, c, a.d, w);
            if (a.ds) load8<DT>(a.ds + (at + c) * EB, a.d - c, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = rs * (g[i] * w[i] - x[i] * rs * dot) + (a.ds ? t[i] : 0.f);
            store8<DT>(a.dx + (at + c) * EB, a.d - c, x);
        }
    }
}
// the weight gradient of such rows: a lane owns 8 columns and walks the rows gridDim.y apart
template <int DT>
__global__ __launch_bounds__(NORM_BLOCK) void rms_norm_dw_wide_kernel(NormBwdArgs a) {
    constexpr int EB = Elem<DT>::B;
    const int c = (blockIdx.x * NORM_BLOCK + threadIdx.x) * 8;
    if (c >= a.d) return;
    float dw[8] = {};
    for (int64_t r = blockIdx.y; r < a.R; r += gridDim.y) {
        float x[8], g[8];
        sum_row<DT>(a, r * a.d, c, x);
        load8<DT>(a.dy + (r * a.d + c) * EB, a.d - c, g);
        const float rs = a.rstd[r];
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[i] = fmaf(g[i], x[i] * rs, dw[i]);
    }
    store8<W3D_DTYPE_F32>(a.part + (int64_t)blockIdx.y * a.d + c, a.d - c, dw);
}

// blocks of the backward pass = partial sums of the weight gradient
static int bwd_blocks(int64_t R, int rows_per_block) {
    const int64_t n = (R + rows_per_block - 1) / rows_per_block;
    return (int)(n < 1 ? 1 : n > 1024 ? 1024 : n);
}
struct Shape { int g, nv; };
// Lanes per row and vectors per lane: the smallest power-of-two group whose one vector covers the row; past 512 elements a wave holds two vectors a lane, past 1 024 the block takes the row.
// us forward | backward with dw, bf16, this choice against the next one: 131 072 x 64, 8 lanes 10.2 | 19.2, 16 lanes 13.9 | 23.9; x 256, 32 lanes 23.5 | 39.6, 64 lanes 32.9 | 61.1; x 1 024,
// two vectors 98.6 | 152, the block 117 | 256; 65 536 x 2 048, the block 97.6 | 163, four vectors of a wave 111 | 232; 32 768 x 4 096, the block 99 | 162, eight vectors of a wave 204 | 405.
static Shape shape_of(int d) {
    const int v = (d + 7) / 8;
    for (int g = 8; g <= 64; g *= 2)
        if (v <= g) return {g, 1};
    if (v <= 128) return {64, 2};
    if (v <= 256) return {256, 1};
    if (v <= 512) return {256, 2};
    if (v <= 1024) return {256, 4};
    return {0, 0};
}

template <int DT, bool Q>
static int launch_fwd(const NormArgs &a, hipStream_t st) {
    const Shape sh = shape_of(a.d);
    if (!sh.g) {
        hipLaunchKernelGGL((rms_norm_wide_kernel<DT, Q>), dim3((unsigned)(a.R < 4096 ? a.R : 4096)), dim3(NORM_BLOCK), 0, st, a);
        return W3D_OK;
    }
    // Two turns a block, or 8 192 blocks if that is more turns for rows that take a whole block (which load the weight for one row at a time).  Blocks at 1 000 000 x 256 with a residual, into
    // 8 bits | bf16: 4 096 370 us | 375, 8 192 364 | 377, 65 536 (two turns) 326 | 344, 125 000 346 | 329; at 131 072 x 256 8 192 (two turns) 23.5, 16 384 24.8; at 130 055 x 1 032 8 192 129,
    // 65 536 149; at 16 384 x 8 192 8 192 113, 16 384 128.
    const int64_t turns = (a.R + NORM_BLOCK / sh.g - 1) / (NORM_BLOCK / sh.g), two = (turns + 1) / 2, most = 1 << 22;
    const dim3 grid((unsigned)(turns < 8192 ? turns : sh.g == 256 || two < 8192 ? 8192 : two < most ? two : most)), block(NORM_BLOCK);
#define W3D_NORM(G, NV) hipLaunchKernelGGL((rms_norm_kernel<DT, G, NV, Q>), grid, block, 0, st, a)
    if (sh.g == 8) W3D_NORM(8, 1);
    else if (sh.g == 16) W3D_NORM(16, 1);
    else if (sh.g == 32) W3D_NORM(32, 1);
    else if (sh.g == 64 && sh.nv == 1) W3D_NORM(64, 1);
    else if (sh.g == 64 && sh.nv == 2) W3D_NORM(64, 2);
    else if (sh.nv == 1) W3D_NORM(256, 1);
    else if (sh.nv == 2) W3D_NORM(256, 2);
    else W3D_NORM(256, 4);
#undef W3D_NORM
    return W3D_OK;
}
template <int DT>
static int launch_bwd(const NormBwdArgs &a, int blocks, hipStream_t st) {
    const Shape sh = shape_of(a.d);
    const dim3 block(NORM_BLOCK);
    if (!sh.g) {
        if (a.dx) hipLaunchKernelGGL(rms_norm_bwd_wide_kernel<DT>, dim3((unsigned)(a.R < 4096 ? a.R : 4096)), block, 0, st, a);
        if (a.part) hipLaunchKernelGGL(rms_norm_dw_wide_kernel<DT>, dim3((a.d + 2047) / 2048, blocks), block, 0, st, a);
        return W3D_OK;
    }
#define W3D_NORM(G, NV) hipLaunchKernelGGL((rms_norm_bwd_kernel<DT, G, NV>), dim3(blocks), block, 0, st, a)
    if (sh.g == 8) W3D_NORM(8, 1);
    else if (sh.g == 16) W3D_NORM(16, 1);
    else if (sh.g == 32) W3D_NORM(32, 1);
    else if (sh.g == 64 && sh.nv == 1) W3D_NORM(64, 1);
    else if (sh.g == 64 && sh.nv == 2) W3D_NORM(64, 2);
    else if (sh.nv == 1) W3D_NORM(256, 1);
    else if (sh.nv == 2) W3D_NORM(256, 2);
    else W3D_NORM(256, 4);
#undef W3D_NORM
    return W3D_OK;
}
static int blocks_for(int64_t R, int d) {
    const Shape sh = shape_of(d);
    if (!sh.g) {                                                          // strips of rows: 2 048 blocks together with those across the columns
        const int across = (d + NORM_BLOCK * 8 - 1) / (NORM_BLOCK * 8), strips = (2048 + across - 1) / across;
        return (int)(R < strips ? R : strips);
    }
    return bwd_blocks(R, NORM_BLOCK / sh.g);
}
static bool dtype_ok(int t) { return t == W3D_DTYPE_F32 || t == W3D_DTYPE_BF16 || t == W3D_DTYPE_F16; }

}  // namespace

static int rms_norm_any(const void *x, const void *residual, const void *weight, int weight_dtype, int64_t R, int d, int dtype, float eps, void *y, void *s, float *rstd,
                        void *q, int32_t *scale, w3d_stream_t stream) {
    if (R < 0 || d < 1 || !dtype_ok(dtype) || !(eps >= 0.f)) return W3D_ERR_ARG;
    if (weight && weight_dtype != dtype && weight_dtype != W3D_DTYPE_F32) return W3D_ERR_ARG;
    if (d > MAX_WIDTH) return W3D_ERR_UNSUPPORTED;
    if (R == 0) return W3D_OK;
    if (!x || (s && !residual)) return W3D_ERR_ARG;
    NormArgs a = {(const char *)x, (const char *)residual, (const char *)weight, (char *)y, (char *)s, rstd, (uint8_t *)q, scale, R, d,
                  weight_dtype == W3D_DTYPE_F32 && dtype != W3D_DTYPE_F32, eps, 1.0 / (double)d};
    hipStream_t st = w3d_s(stream);
    if (dtype == W3D_DTYPE_F32) q ? launch_fwd<W3D_DTYPE_F32, true>(a, st) : launch_fwd<W3D_DTYPE_F32, false>(a, st);
    else if (dtype == W3D_DTYPE_BF16) q ? launch_fwd<W3D_DTYPE_BF16, true>(a, st) : launch_fwd<W3D_DTYPE_BF16, false>(a, st);
    else q ? launch_fwd<W3D_DTYPE_F16, true>(a, st) : launch_fwd<W3D_DTYPE_F16, false>(a, st);
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}

extern "C" int w3d_rms_norm_fwd(const void *x, const void *residual, const void *weight, int weight_dtype, int64_t R, int d, int dtype, float eps, void *y, void *s, float *rstd,
                                w3d_stream_t stream) {
    if (R > 0 && !y) return W3D_ERR_ARG;
    return rms_norm_any(x, residual, weight, weight_dtype, R, d, dtype, eps, y, s, rstd, nullptr, nullptr, stream);
}
extern "C" int w3d_rms_norm_fp8(const void *x, const void *residual, const void *weight, int weight_dtype, int64_t R, int d, int dtype, float eps, void *q, int32_t *scale_e8m0,
                                void *s, w3d_stream_t stream) {
    if (R > 0 && (!q || !scale_e8m0)) return W3D_ERR_ARG;
    return rms_norm_any(x, residual, weight, weight_dtype, R, d, dtype, eps, nullptr, s, nullptr, q, scale_e8m0, stream);
}
extern "C" size_t w3d_rms_norm_bwd_workspace_bytes(int64_t R, int d) {
    if (R < 1 || d < 1) return 0;
    return (size_t)blocks_for(R, d) * (size_t)d * 4;
}
int w3d_fold_columns(const float *part, int parts, int64_t ld, int64_t n, void *out, int out_dtype, hipStream_t st);      // columns.hip

extern "C" int w3d_rms_norm_bwd(const void *x, const void *residual, const void *weight, int weight_dtype, const float *rstd, const void *dy, const void *ds, int64_t R, int d, int dtype, void *dx,
                                void *dweight, void *workspace, size_t workspace_bytes, w3d_stream_t stream) {
    if (R < 0 || d < 1 || !dtype_ok(dtype) || (!dx && !dweight)) return W3D_ERR_ARG;
    if ((weight || dweight) && weight_dtype != dtype && weight_dtype != W3D_DTYPE_F32) return W3D_ERR_ARG;
    if (R > 0 && (!x || !rstd || !dy)) return W3D_ERR_ARG;
    if (d > MAX_WIDTH) return W3D_ERR_UNSUPPORTED;
    hipStream_t st = w3d_s(stream);
    const int blocks = R > 0 ? blocks_for(R, d) : 0;
    if (R > 0) {
        if (dweight && (!workspace || workspace_bytes < w3d_rms_norm_bwd_workspace_bytes(R, d))) return W3D_ERR_WORKSPACE;
        NormBwdArgs a = {(const char *)x, (const char *)residual, (const char *)weight, (const char *)dy, (const char *)ds, rstd, (char *)dx, dweight ? (float *)workspace : nullptr, R, d,
                         weight_dtype == W3D_DTYPE_F32 && dtype != W3D_DTYPE_F32, 1.0f / (float)d};
        if (dtype == W3D_DTYPE_F32) launch_bwd<W3D_DTYPE_F32>(a, blocks, st);
        else if (dtype == W3D_DTYPE_BF16) launch_bwd<W3D_DTYPE_BF16>(a, blocks, st);
        else launch_bwd<W3D_DTYPE_F16>(a, blocks, st);
        W3D_CHECK_LAUNCH();
    }
    if (dweight) return w3d_fold_columns((const float *)workspace, blocks, d, d, dweight, weight_dtype, st);     // (no rows: zeros)
    return W3D_OK;
}
