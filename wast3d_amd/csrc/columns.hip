// Column sums of row-major matrices in two launches of fixed order (no atomics: the same bits every time): partial sums per strip of rows, then the fold over the strips.
#include "rows16.h"

namespace {

// out[c] = sum over p of part[p][c]: 64 columns per block, its sixteen waves take every sixteenth strip, eight loads in flight each (the strips are few and the launch short: latency; 128 strips of
// 4 096 columns 4.9 us)
template <int DT>
__global__ __launch_bounds__(1024) void fold_columns_kernel(const float *__restrict__ part, int parts, int64_t ld, int64_t n, void *__restrict__ out) {
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < n; c0 += (int64_t)gridDim.x * 64) {
        const int64_t c = c0 + lane;
        float s[8] = {};
        if (c < n) {
            int p = w;
            for (; p + 112 < parts; p += 128)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] += part[(int64_t)(p + 16 * i) * ld + c];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (p + 16 * i < parts) s[i] += part[(int64_t)(p + 16 * i) * ld + c];
        }
        sm[w][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        __syncthreads();
        if (w == 0 && c < n) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) t += sm[i][lane];
            store1<DT>((char *)out + c * Elem<DT>::B, t);
        }
        __syncthreads();                                     // (the next columns' sums)
    }
}

// part[strip][c] = sum of x[r][c] over the strip's rows: a lane owns one column, the four waves of a block every fourth row of the strip
template <int DT>
__global__ __launch_bounds__(256) void column_sums_kernel(const char *__restrict__ x, int64_t R, int64_t n, int64_t rows_per_strip, float *__restrict__ part, int64_t ld) {
    __shared__ float sm[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    const int64_t r0 = (int64_t)blockIdx.y * rows_per_strip, r1 = min(R, r0 + rows_per_strip);
    float s0 = 0.f, s1 = 0.f;
    if (c < n) {
        int64_t r = r0 + w;
        for (; r + 4 < r1; r += 8) {
            s0 += load1<DT>(x + (r * n + c) * Elem<DT>::B);
            s1 += load1<DT>(x + ((r + 4) * n + c) * Elem<DT>::B);
        }
        if (r < r1) s0 += load1<DT>(x + (r * n + c) * Elem<DT>::B);
    }
    sm[w][lane] = s0 + s1;
    __syncthreads();
    if (w == 0 && c < n) part[(int64_t)blockIdx.y * ld + c] = (sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]);
}

}  // namespace

// fold of `parts` rows of partial sums (0 parts: zeros) into out[n] of the given dtype
int w3d_fold_columns(const float *part, int parts, int64_t ld, int64_t n, void *out, int out_dtype, hipStream_t st) {
    if (n < 1) return W3D_OK;
    const int64_t cols = (n + 63) / 64;
    const dim3 grid((unsigned)(cols < 65536 ? cols : 65536)), block(1024);      // (a launch has less than 2^32 threads; the weight gradient of no rows can be longer)
    if (out_dtype == W3D_DTYPE_F32) hipLaunchKernelGGL(fold_columns_kernel<W3D_DTYPE_F32>, grid, block, 0, st, part, parts, ld, n, out);
    else if (out_dtype == W3D_DTYPE_BF16) hipLaunchKernelGGL(fold_columns_kernel<W3D_DTYPE_BF16>, grid, block, 0, st, part, parts, ld, n, out);
    else hipLaunchKernelGGL(fold_columns_kernel<W3D_DTYPE_F16>, grid, block, 0, st, part, parts, ld, n, out);
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}

// strips of a column sum over R rows of n columns: enough blocks to fill the chip, at least 32 rows each
int w3d_column_strips(int64_t R, int64_t n) {
    const int64_t bx = (n + 63) / 64, want = (2048 + bx - 1) / bx, most = (R + 31) / 32;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 1024 ? 1024 : s);
}
int w3d_column_sums(const void *x, int64_t R, int64_t n, int dtype, float *part, int64_t ld, hipStream_t st) {
    const int strips = w3d_column_strips(R, n);
    const int64_t rps = (R + strips - 1) / strips;
    const dim3 grid((unsigned)((n + 63) / 64), (unsigned)strips), block(256);
    if (dtype == W3D_DTYPE_F32) hipLaunchKernelGGL(column_sums_kernel<W3D_DTYPE_F32>, grid, block, 0, st, (const char *)x, R, n, rps, part, ld);
    else if (dtype == W3D_DTYPE_BF16) hipLaunchKernelGGL(column_sums_kernel<W3D_DTYPE_BF16>, grid, block, 0, st, (const char *)x, R, n, rps, part, ld);
    else hipLaunchKernelGGL(column_sums_kernel<W3D_DTYPE_F16>, grid, block, 0, st, (const char *)x, R, n, rps, part, ld);
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}
