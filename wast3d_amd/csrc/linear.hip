// Linear and gated linear layers on feature rows: z = x W^T + b;  y = act(z) + residual  /  y = act(x Wg^T + bg) * (x Wu^T + bu), and their gradients.
//
// Three kernels do the products (gemm_tile.h has the tile):
//   * few rows: the weights are read once, straight into MFMA fragments, by as many waves as there are; the rows are the other operand
//   * tiles of 256 x 256 (gemm_pipe.h), 128 x 128 or 64 x 64 (gemm_tile.h) through LDS
//   * when the tiles are few for 256 CUs the contraction is cut into slices; partial tiles are added in slice order, and the epilogue applied, by a second launch
//
// Backward from nothing but the inputs (16-bit rows, z not given): z is formed again and turned into dz in the epilogue, where the column sums for the bias
// gradient are taken too.  Backward from the z that the forward pass kept (always for f32, at a tenth of the 16-bit rate): one pass over z and dy (dz_kernel).  z is kept in 32 bits (16 would put
// their rounding into every gradient): 8 bytes an output written and read against 2 K operations, even at K of 900 or so.  dz is rounded once to the operands' type (it is an operand of two
// products); sums are f32.
//
// One translation unit per operand type (W3D_LIN_DT: the tiles), one for the entry points.
#include "gemm_pipe.h"

int w3d_fold_columns(const float *part, int parts, int64_t ld, int64_t n, void *out, int out_dtype, hipStream_t st);      // columns.hip
int w3d_column_strips(int64_t R, int64_t n);
int w3d_column_sums(const void *x, int64_t R, int64_t n, int dtype, float *part, int64_t ld, hipStream_t st);

namespace {
enum { PROD_LINEAR = 0, PROD_GATED = 1, PROD_LINEAR_BWD = 2, PROD_GATED_BWD = 3, PROD_DX = 4, PROD_DW = 5 };
constexpr int SKINNY_ROWS = 64;
}  // namespace

// launches of one operand type's kernels
int w3d_lin_tiles_f32(const GemmArgs &a, int prod, int tile, int z, hipStream_t st);
int w3d_lin_tiles_bf16(const GemmArgs &a, int prod, int tile, int z, hipStream_t st);
int w3d_lin_tiles_f16(const GemmArgs &a, int prod, int tile, int z, hipStream_t st);
int w3d_lin_tiles_fp8(const GemmArgs &a, int prod, int tile, int z, hipStream_t st);
int w3d_lin_skinny_f32(const GemmArgs &a, int prod, hipStream_t st);
int w3d_lin_skinny_bf16(const GemmArgs &a, int prod, hipStream_t st);
int w3d_lin_skinny_f16(const GemmArgs &a, int prod, hipStream_t st);
int w3d_lin_skinny_fp8(const GemmArgs &a, int prod, hipStream_t st);

#ifdef W3D_LIN_DT
namespace {

int launch_kernel(void (*kernel)(GemmArgs), int threads, int lds, const GemmArgs &a, int z, hipStream_t st) {
    if (lds > 65536) W3D_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    const int64_t blocks = (int64_t)a.tiles_m * a.tiles_n * a.slices;
    if (blocks < 1 || blocks * threads > 0xffffffffll) return W3D_ERR_UNSUPPORTED;             // (a launch has less than 2^32 threads)
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, 1, z), dim3(threads), lds, st, a);
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}
template <int LX, int LW, int EPI, int BM, int BN, int WM, int WN>
int launch_tile(const GemmArgs &a, int z, hipStream_t st) {
    typedef Gemm<W3D_LIN_DT, LX, LW, EPI, BM, BN, WM, WN> G;
    return launch_kernel(gemm_kernel<W3D_LIN_DT, LX, LW, EPI, BM, BN, WM, WN>, G::NT, G::LDS_BYTES, a, z, st);
}
template <int LX, int LW, int EPI>
int launch_shape(const GemmArgs &a, int tile, int z, hipStream_t st) {
    if constexpr (W3D_LIN_DT != W3D_DTYPE_F32) {
        if (tile == 256) {
            typedef Pipe<W3D_LIN_DT, LX, LW, EPI> P;
            return launch_kernel(gemm_pipe_kernel<W3D_LIN_DT, LX, LW, EPI>, P::NT, P::LDS_BYTES, a, z, st);
        }
    }
    if (tile == 128) return launch_tile<LX, LW, EPI, 128, 128, 2, 2>(a, z, st);
    return launch_tile<LX, LW, EPI, 64, 64, 4, 1>(a, z, st);
}
int launch_prod(const GemmArgs &a, int prod, int tile, int z, hipStream_t st) {
    switch (prod) {
        case PROD_LINEAR: return launch_shape<K_ROWS, K_ROWS, EPI_LINEAR>(a, tile, z, st);
        case PROD_GATED: return launch_shape<K_ROWS, K_ROWS, EPI_GATED>(a, tile, z, st);
        default: break;
    }
    if constexpr (W3D_LIN_DT != W3D_DTYPE_FP8_E4M3) {
        switch (prod) {
            case PROD_DX: return launch_shape<K_ROWS, M_ROWS, EPI_STORE>(a, tile, z, st);
            case PROD_DW: return launch_shape<M_ROWS, M_ROWS, EPI_STORE>(a, tile, z, st);
            default: break;
        }
    }
    if constexpr (W3D_LIN_DT == W3D_DTYPE_BF16 || W3D_LIN_DT == W3D_DTYPE_F16) {
        switch (prod) {
            case PROD_LINEAR_BWD: return launch_shape<K_ROWS, K_ROWS, EPI_LINEAR_BWD>(a, tile, z, st);
            case PROD_GATED_BWD: return launch_shape<K_ROWS, K_ROWS, EPI_GATED_BWD>(a, tile, z, st);
            default: break;
        }
    }
    return W3D_ERR_UNSUPPORTED;
}

// ---- few rows.  Bound by the weights: every one is read once.  A block owns 16 columns (of each half of a gated layer); its waves share the contraction in turns of STEP_RUN steps of 64
// bytes, a lane loading 16 bytes of one weight row per step, so that a row's 256 consecutive bytes are in flight together (runs of 8 steps: 9.5 instead of 10.3 us for one row below, but 13.0 instead of 12.1 for 16); rows of any
// alignment are read in place.  The waves' partial sums meet in LDS.  Measured, weights from HBM: bf16 4096 -> 4096, 1 row 10.3 us (3.2 TB/s with the launch), 16 rows 12.1; fp8 8.1 and 8.5; gated 1024 -> 2816
// 5.9 us.
template <int EPI, int RF>
__global__ __launch_bounds__(512) void skinny_kernel(GemmArgs a) {
    constexpr int DT = W3D_LIN_DT, EB = Elem<DT>::B, WAVES = 8, KPSTEP = 64 / EB, STEP_RUN = 4;
    constexpr bool GATED = EPI == EPI_GATED;
    constexpr int PARTS = GATED ? 2 : 1;
    __shared__ f32x4 sums[WAVES][PARTS * RF][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int64_t n = n0 + (lane & 15) < a.N ? n0 + (lane & 15) : a.N - 1;                    // (rows past the end: the last one again, never stored)
    const uint8_t *wr[PARTS];
    wr[0] = a.w + n * a.ldw;
    if (GATED) wr[PARTS - 1] = a.w2 + n * a.ldw;
    const uint8_t *xr[RF];
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int64_t m = 16 * i + (lane & 15);
        xr[i] = a.x + (m < a.M ? m : a.M - 1) * a.ldx;
    }
    f32x4 acc[PARTS][RF];
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[p][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const uint8_t *row, int64_t k) -> i32x4 {                                 // 16 bytes from contraction index k, zeros behind the end
        i32x4 v = {0, 0, 0, 0};
        const int64_t left = a.K - k;
        if (left >= 16 / EB) { __builtin_memcpy(&v, row + k * EB, 16); return v; }
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16 / EB; ++e)
            if (e < left) {
                uint32_t b = 0;
                __builtin_memcpy(&b, row + (k + e) * EB, EB);
                w[e * EB / 4] |= b << (8 * ((e * EB) & 3));
            }
        __builtin_memcpy(&v, w, 16);
        return v;
    };
    const int64_t steps = (a.K + KPSTEP - 1) / KPSTEP;
    for (int64_t s0 = (int64_t)wave * STEP_RUN; s0 < steps; s0 += WAVES * STEP_RUN) {
        i32x4 wf[PARTS][STEP_RUN], xf[RF][STEP_RUN];
#pragma unroll
        for (int s = 0; s < STEP_RUN; ++s) {
            const int64_t k = (s0 + s) * KPSTEP + q * (16 / EB);                              // (steps past the end load zeros)
#pragma unroll
            for (int p = 0; p < PARTS; ++p) wf[p][s] = load(wr[p], k);
#pragma unroll
            for (int i = 0; i < RF; ++i) xf[i][s] = load(xr[i], k);
        }
#pragma unroll
        for (int s = 0; s < STEP_RUN; s += 2)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int i = 0; i < RF; ++i) {
                    const i32x4 w2[2] = {wf[p][s], wf[p][s + 1]}, x2[2] = {xf[i][s], xf[i][s + 1]};
                    acc[p][i] = mfma_step<DT>(w2, x2, 0, acc[p][i]);
                    acc[p][i] = mfma_step<DT>(w2, x2, 1, acc[p][i]);
                }
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int i = 0; i < RF; ++i) sums[wave][p * RF + i][lane] = acc[p][i];
    __syncthreads();
    // fragment i is summed and finished by wave i: lane = row 16 i + (lane & 15), columns n0 + 4 q .. + 3
    if (wave >= RF) return;
    const int64_t m = 16 * wave + (lane & 15);
    float v[4], u[4] = {};
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) t += sums[w][p * RF + wave][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) (p ? u : v)[e] = t[e];
    }
    if (m >= a.M) return;
    auto out = [&](auto ot) {
        constexpr int OT = decltype(ot)::value, OB = Elem<OT>::B;
        const int64_t c = n0 + 4 * q;
        with_act(a.act, [&](auto act_c) {
            constexpr int ACT = decltype(act_c)::value;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (c + e >= a.N) break;
                if (DT == W3D_DTYPE_FP8_E4M3) {
                    v[e] = __builtin_ldexpf(v[e], a.xs[m] + a.ws[c + e] - 254);
                    if (GATED) u[e] = __builtin_ldexpf(u[e], a.xs[m] + a.ws2[c + e] - 254);
                }
                const float z = v[e] + bias_at<OT>(a.bias, a.bias_f32, c + e, a.N), z2 = GATED ? u[e] + bias_at<OT>(a.bias2, a.bias_f32, c + e, a.N) : 0.f;
                if (DT != W3D_DTYPE_FP8_E4M3 && a.z) { a.z[m * a.part_ld + c + e] = z; if (GATED) a.z[m * a.part_ld + a.part_ld / 2 + c + e] = z2; }
                float y = act_fwd<ACT, OT>(z);
                if (GATED) y *= z2;
                else if (a.res) y += load1<OT>(a.res + (m * a.N + c + e) * OB);
                store1<OT>(a.out + m * a.ld_out + (c + e) * OB, y);
            }
        });
    };
    if constexpr (DT != W3D_DTYPE_FP8_E4M3) out(std::integral_constant<int, DT>());
    else if (a.out_dt == W3D_DTYPE_BF16) out(std::integral_constant<int, W3D_DTYPE_BF16>());
    else out(std::integral_constant<int, W3D_DTYPE_F16>());
}
template <int EPI>
int launch_skinny(const GemmArgs &a, hipStream_t st) {
    const int64_t blocks = (a.N + 15) / 16;
    if (blocks > 0x7fffffff) return W3D_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)blocks), block(512);
    if (a.M <= 16) hipLaunchKernelGGL((skinny_kernel<EPI, 1>), grid, block, 0, st, a);
    else if (a.M <= 32) hipLaunchKernelGGL((skinny_kernel<EPI, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((skinny_kernel<EPI, 4>), grid, block, 0, st, a);
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}
}  // namespace

#if W3D_LIN_DT == 0
#define W3D_LIN_NAME(f) f##_f32
#elif W3D_LIN_DT == 1
#define W3D_LIN_NAME(f) f##_bf16
#elif W3D_LIN_DT == 2
#define W3D_LIN_NAME(f) f##_f16
#else
#define W3D_LIN_NAME(f) f##_fp8
#endif
int W3D_LIN_NAME(w3d_lin_tiles)(const GemmArgs &a, int prod, int tile, int z, hipStream_t st) { return launch_prod(a, prod, tile, z, st); }
int W3D_LIN_NAME(w3d_lin_skinny)(const GemmArgs &a, int prod, hipStream_t st) {
    return prod == PROD_GATED ? launch_skinny<EPI_GATED>(a, st) : launch_skinny<EPI_LINEAR>(a, st);
}

#else  // ---------------------------------------------------------------- entry points

namespace {

// Partial sums of a sliced product: part[slice][m][ld] -> the epilogue of the product.  A block
// takes 64 columns of a strip of rows (a multiple of JOIN_ROWS), JOIN_ROWS at a time (a quarter per wave), so that the column sums of dz are complete per strip; up to 8
// slices of every row are loaded before the first sum (one after another, 16 slices of 16 rows waited 12 us).  Measured: 4 slices of 1024 x 4096 in f32, 75 MB, 18 us.
constexpr int JOIN_ROWS = 16;
template <int OT, int EPI>
__global__ __launch_bounds__(256) void join_slices_kernel(GemmArgs a) {
    constexpr int OB = Elem<OT>::B;
    constexpr bool GATED = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
    __shared__ float sums[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = (int64_t)blockIdx.x * 64 + lane, r_end = min(a.M, ((int64_t)blockIdx.y + 1) * a.strip);
    const int64_t pad = EPI == EPI_LINEAR_BWD ? a.ld_out / OB : EPI == EPI_GATED_BWD ? a.half_out / OB : a.N;
    const bool in = n < a.N, store = n < pad;
    const float b0 = bias_at<OT>(a.bias, a.bias_f32, n, a.N), b1 = GATED ? bias_at<OT>(a.bias2, a.bias_f32, n, a.N) : 0.f;
    const int s0 = a.ws && in ? a.ws[n] - 254 : 0, s1 = GATED && a.ws2 && in ? a.ws2[n] - 254 : 0;
    const int64_t z = blockIdx.z, slice = a.M * a.part_ld;
    float c0 = 0.f, c1 = 0.f;
    for (int64_t r0 = (int64_t)blockIdx.y * a.strip; r0 < r_end; r0 += JOIN_ROWS) {
    float v[JOIN_ROWS / 4] = {}, u[JOIN_ROWS / 4] = {};
    const float *p[JOIN_ROWS / 4];                                                             // (rows and columns past the end load the last ones; never stored)
#pragma unroll
    for (int i = 0; i < JOIN_ROWS / 4; ++i) p[i] = a.part + (z * a.slices * a.M + min(r0 + 4 * i + wave, r_end - 1)) * a.part_ld + min(n, a.N - 1);
    auto add = [&](auto run) {                                                                 // RUN slices of every row: all loads first, then the sums in slice order
        constexpr int RUN = decltype(run)::value;
        float l[JOIN_ROWS / 4][RUN], h[JOIN_ROWS / 4][RUN];
#pragma unroll
        for (int i = 0; i < JOIN_ROWS / 4; ++i) {
#pragma unroll
            for (int k = 0; k < RUN; ++k) {
                l[i][k] = p[i][k * slice];
                if (GATED) h[i][k] = p[i][k * slice + a.part_ld / 2];
            }
            p[i] += RUN * slice;
        }
#pragma unroll
        for (int i = 0; i < JOIN_ROWS / 4; ++i)
#pragma unroll
            for (int k = 0; k < RUN; ++k) {
                v[i] += l[i][k];
                if (GATED) u[i] += h[i][k];
            }
    };
    int left = a.slices;
    for (; left >= 8; left -= 8) add(std::integral_constant<int, 8>());
    if (left & 4) add(std::integral_constant<int, 4>());
    if (left & 2) add(std::integral_constant<int, 2>());
    if (left & 1) add(std::integral_constant<int, 1>());
    with_act(a.act, [&](auto act_c) {
        constexpr int ACT = decltype(act_c)::value;
#pragma unroll
        for (int i = 0; i < JOIN_ROWS / 4; ++i) {
            const int64_t m = r0 + 4 * i + wave;
            if (!store || m >= r_end) continue;
            float x = v[i], y = u[i];
            if (a.xs) { x = __builtin_ldexpf(x, a.xs[m] + s0); if (GATED) y = __builtin_ldexpf(y, a.xs[m] + s1); }
            x += b0; y += b1;
            if ((EPI == EPI_LINEAR || EPI == EPI_GATED) && a.z && in) { a.z[m * a.part_ld + n] = x; if (GATED) a.z[m * a.part_ld + a.part_ld / 2 + n] = y; }
            uint8_t *o = (EPI == EPI_STORE && z ? a.out2 : a.out) + m * a.ld_out + n * OB;
            if (EPI == EPI_STORE) store1<OT>(o, x);
            else if (EPI == EPI_LINEAR) {
                x = act_fwd<ACT, OT>(x);
                if (a.res) x += load1<OT>(a.res + (m * a.N + n) * OB);
                store1<OT>(o, x);
            } else if (EPI == EPI_GATED) store1<OT>(o, act_fwd<ACT, OT>(x) * y);
            else {
                float act, der;
                act_both<ACT, OT>(x, act, der);
                const float dy = in ? load1<OT>(a.dy + (m * a.N + n) * OB) : 0.f;
                if (EPI == EPI_LINEAR_BWD) x = in ? through<ACT>(dy, x, der) : 0.f;
                else { x = in ? through<ACT>(dy, x, der, y) : 0.f; y = in ? dy * act : 0.f; store1<OT>(o + a.half_out, y); c1 += y; }
                store1<OT>(o, x);
                c0 += x;
            }
        }
    });
    }
    if ((EPI == EPI_LINEAR_BWD || EPI == EPI_GATED_BWD) && a.colsum) {
        sums[0][wave][lane] = c0;
        if (GATED) sums[1][wave][lane] = c1;
        __syncthreads();
        if (wave < (GATED ? 2 : 1) && in)
            a.colsum[(int64_t)blockIdx.y * a.colsum_ld + wave * (a.colsum_ld / 2) + n] = (sums[wave][0][lane] + sums[wave][1][lane]) + (sums[wave][2][lane] + sums[wave][3][lane]);
    }
}
// rows of a strip: JOIN_ROWS, more where the strips would be over 1 024
int64_t strip_rows(int64_t M) { return (M / 1024 + JOIN_ROWS) / JOIN_ROWS * JOIN_ROWS; }
template <int OT>
int join_as(GemmArgs a, int prod, int z, hipStream_t st) {
    const int64_t cols = prod == PROD_LINEAR_BWD ? a.ld_out / Elem<OT>::B : prod == PROD_GATED_BWD ? a.half_out / Elem<OT>::B : a.N;
    a.strip = strip_rows(a.M);
    const int64_t strips = (a.M + a.strip - 1) / a.strip;
    const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)strips, z), block(256);
    switch (prod) {
        case PROD_LINEAR: hipLaunchKernelGGL((join_slices_kernel<OT, EPI_LINEAR>), grid, block, 0, st, a); break;
        case PROD_GATED: hipLaunchKernelGGL((join_slices_kernel<OT, EPI_GATED>), grid, block, 0, st, a); break;
        case PROD_LINEAR_BWD: if constexpr (OT != W3D_DTYPE_F32) hipLaunchKernelGGL((join_slices_kernel<OT, EPI_LINEAR_BWD>), grid, block, 0, st, a); break;      // (f32 calls keep z)
        case PROD_GATED_BWD: if constexpr (OT != W3D_DTYPE_F32) hipLaunchKernelGGL((join_slices_kernel<OT, EPI_GATED_BWD>), grid, block, 0, st, a); break;
        default: hipLaunchKernelGGL((join_slices_kernel<OT, EPI_STORE>), grid, block, 0, st, a); break;
    }
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}

// dz (both halves of it), and its column sums per strip of rows, from the z that the forward pass kept: a.part = z.  Bound by HBM: a lane takes 8 columns, the four waves of a block every fourth
// row of the strip.  Padding columns become zeros (z and dy are read as zeros there).  A step of 16 384 rows 1024 -> 4096 590 us with it, 613 with the product once more.
template <int OT, bool GATED>
__global__ __launch_bounds__(256) void dz_kernel(GemmArgs a) {
    constexpr int OB = Elem<OT>::B;
    __shared__ float sums[4][64 * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = ((int64_t)blockIdx.x * 64 + lane) * 8, pad = (GATED ? a.half_out : a.ld_out) / OB;
    const int64_t r_begin = (int64_t)blockIdx.y * a.strip, r_end = min(a.M, r_begin + a.strip);
    const int in = (int)max(a.N - n, (int64_t)0), room = (int)(pad - n);
    float c0[8] = {}, c1[8] = {};
    if (room > 0)
        with_act(a.act, [&](auto act_c) {
            constexpr int ACT = decltype(act_c)::value;
#pragma unroll 2
            for (int64_t r = r_begin + wave; r < r_end; r += 4) {
                float v[8], u[8], t[8];
                load8<W3D_DTYPE_F32>(a.part + r * a.part_ld + n, in, v);
                if (GATED) load8<W3D_DTYPE_F32>(a.part + r * a.part_ld + a.part_ld / 2 + n, in, u);
                load8<OT>(a.dy + (r * a.N + n) * OB, in, t);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float f, d;
                    act_both<ACT, OT>(v[e], f, d);
                    if (GATED) { v[e] = through<ACT>(t[e], v[e], d, u[e]); u[e] = t[e] * f; c1[e] += u[e]; }
                    else v[e] = through<ACT>(t[e], v[e], d);
                    c0[e] += v[e];
                }
                uint8_t *o = a.out + r * a.ld_out + n * OB;
                store8<OT>(o, room, v);
                if (GATED) store8<OT>(o + a.half_out, room, u);
            }
        });
    if (!a.colsum) return;
#pragma unroll
    for (int h = 0; h < (GATED ? 2 : 1); ++h) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[wave][e * 64 + lane] = h ? c1[e] : c0[e];
        __syncthreads();
#pragma unroll
        for (int e = 2 * wave; e < 2 * wave + 2; ++e)
            if (n + e < a.N)
                a.colsum[(int64_t)blockIdx.y * a.colsum_ld + h * (a.colsum_ld / 2) + n + e] =
                    (sums[0][e * 64 + lane] + sums[1][e * 64 + lane]) + (sums[2][e * 64 + lane] + sums[3][e * 64 + lane]);
    }
}
template <int OT>
int dz_as(GemmArgs a, bool gated, hipStream_t st) {
    const int64_t pad = (gated ? a.half_out : a.ld_out) / Elem<OT>::B;
    a.strip = strip_rows(a.M);
    const dim3 grid((unsigned)((pad + 511) / 512), (unsigned)((a.M + a.strip - 1) / a.strip)), block(256);
    if (gated) hipLaunchKernelGGL((dz_kernel<OT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((dz_kernel<OT, false>), grid, block, 0, st, a);
    W3D_CHECK_LAUNCH();
    return W3D_OK;
}

int eb_of(int dtype) { return dtype == W3D_DTYPE_F32 ? 4 : dtype == W3D_DTYPE_FP8_E4M3 ? 1 : 2; }
bool float_dtype(int t) { return t == W3D_DTYPE_F32 || t == W3D_DTYPE_BF16 || t == W3D_DTYPE_F16; }
int64_t ceil_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
bool aligned16(const void *p, int64_t ld) { return !(((uintptr_t)p) & 15) && ld % 16 == 0; }

// How a product is cut: tile size and slices of the contraction, by the time they would take.  Microseconds, fitted to every tile with 1, 2 and 4 slices on 12 sizes of rows 100 .. 65 536 and
// widths 100 .. 4 096: `lone`, a 128-byte slab of a block that has its CU for itself; `busy`, the same of a block among others, per block on the CU; `round`, start and epilogue of a block.
// Slices write and read their f32 tiles (2.5 TB/s, and the second launch).  The choices take 4 % longer than the best of all 13 over 18 such sizes, forward, dx and dW.
struct TileCost { double lone[3], busy[3], round[3]; };      // of 64, 128, 256
constexpr TileCost COST_16 = {{0.35, 0.6, 1.2}, {0.22, 0.6, 1.3}, {4, 5, 10}}, COST_DW = {{0.57, 0.77, 1.35}, {0.24, 0.5, 1.35}, {4, 5, 10}}, COST_FP8 = {{0.35, 0.6, 0.9}, {0.22, 0.6, 0.9}, {4, 5, 10}},
                   COST_F32 = {{0.72, 2.25, 0}, {0.62, 2.25, 0}, {4, 5, 0}}, COST_FEW = {{0.8, 0, 0}, {0.4, 0, 0}, {4, 0, 0}};
enum Products { PLAIN, DW, FEW };      // DW: both operands M_ROWS; FEW: at most SKINNY_ROWS rows (one row of 64-wide tiles; the weights come from HBM, a slab waits for them)
struct Cut { int tile, slices; int64_t tiles_m, tiles_n; double us; };
// vec: rows of everything the epilogue touches are aligned, too (the 256 x 256 tile needs it)
Cut cut_of(int64_t M, int64_t N, int64_t K, int dtype, bool gated, bool vec, int batch, Products kind = PLAIN) {
    const int parts = gated ? 2 : 1;
    const int64_t slabs = (K * eb_of(dtype) + SLAB - 1) / SLAB;
    Cut best = {};
    double best_t = 0;
    for (int tile = 64; tile <= 256; tile *= 2) {
        if ((tile == 256 && (!vec || dtype == W3D_DTYPE_F32)) || (tile > 64 && kind == FEW)) break;
        const int bn = tile / parts;
        const int64_t tm = (M + tile - 1) / tile, tn = (N + bn - 1) / bn, tiles = tm * tn * batch;
        const int k = tile == 64 ? 0 : tile == 128 ? 1 : 2;
        const TileCost &c = dtype == W3D_DTYPE_F32 ? COST_F32 : kind == FEW ? COST_FEW : dtype == W3D_DTYPE_FP8_E4M3 ? COST_FP8 : kind == DW ? COST_DW : COST_16;
        const int per_cu = tile == 256 ? 1 : tile == 128 ? 2 : 4;
        for (int s = 1; s <= 32 && (s == 1 || slabs / s >= 4); ++s) {
            const double cu = (double)((tiles * s + 255) / 256), rounds = (double)((tiles * s + 256 * per_cu - 1) / (256 * per_cu)), n = (double)((slabs + s - 1) / s);
            const double a = n * c.busy[k] * cu, b = n * c.lone[k] * rounds;
            double t = (a > b ? a : b) + c.round[k] * rounds;
            if (s > 1) t += 3.0 + 8.0 * (double)s * (double)batch * (double)M * (double)N * parts / 2.5e6;
            if (best_t == 0 || t < best_t) { best_t = t; best = {tile, s, tm, tn, t}; }
        }
    }
    return best;
}
// Few rows: do they take skinny_kernel or 64-wide tiles over a sliced contraction?  A skinny block reads its 16 weight rows and ALL of the rows, 27 bytes a nanosecond (measured at 64 .. 16 384
// columns); long rows onto few columns leave it short of blocks, and many long rows are read once per 16 columns.  us, skinny | tiles, weights from HBM: bf16 4096 -> 4096 1 row 10.3 | 14.2,
// 16 rows 12.1 | 15.1, 32 rows 17.1 | 15.5, 64 rows 24.7 | 20.7; 1024 -> 4096 64 rows 8.2 | 12.1; 8192 -> 64 1 row 11.3 | 8.0, 64 rows 37.8 | 9.2; 2048 -> 16384 16 rows 23.4 | 32.0, 64 rows
// 46.3 | 31.8; f32 512 -> 512 64 rows 8.4 | 8.5; f32 4096 -> 4096 16 rows 21.4 | 29.3, 64 rows 55.3 | 36.3.  Unaligned operands are read in place, which beats copying the weights.
bool few_rows(int64_t R, int64_t K, int64_t N, int dtype, bool gated, bool unaligned, const Cut &tiles) {
    if (R > SKINNY_ROWS || unaligned) return R <= SKINNY_ROWS;
    const double blocks = (double)((N + 15) / 16), cu = blocks > 256 ? blocks / 256 : 1;
    return 2.5 + cu * 16.0 * ((gated ? 2 : 1) + (double)R / 16) * (double)K * eb_of(dtype) / 27e3 <= tiles.us;
}
Cut forward_cut(int64_t R, int64_t K, int64_t N, int dtype, bool gated, bool vec) { return cut_of(R, N, K, dtype, gated, vec, 1, R <= SKINNY_ROWS ? FEW : PLAIN); }
size_t part_bytes(const Cut &c, int64_t M, int64_t N, bool gated, int batch) {
    return c.slices > 1 ? (size_t)batch * c.slices * M * ceil_to(N, 16) * (gated ? 2 : 1) * 4 : 0;
}

// floats of a row of partial sums, or of kept values before the activation
int64_t z_stride(int64_t N, bool gated) { return ceil_to(N, 16) * (gated ? 2 : 1); }
// the second launch of a sliced product
int join(const GemmArgs &a, int prod, int z, hipStream_t st) {
    switch (a.out_dt) {
        case W3D_DTYPE_F32: return join_as<W3D_DTYPE_F32>(a, prod, z, st);
        case W3D_DTYPE_BF16: return join_as<W3D_DTYPE_BF16>(a, prod, z, st);
        default: return join_as<W3D_DTYPE_F16>(a, prod, z, st);
    }
}
int run_product(GemmArgs &a, int prod, int dtype, const Cut &c, int z, hipStream_t st) {
    a.slices = c.slices;
    if (c.tiles_m > 0x7fffffff || c.tiles_n > 0x7fffffff) return W3D_ERR_UNSUPPORTED;
    a.tiles_m = (int)c.tiles_m; a.tiles_n = (int)c.tiles_n;
    a.part_ld = z_stride(a.N, prod == PROD_GATED || prod == PROD_GATED_BWD);
    int rc;
    switch (dtype) {
        case W3D_DTYPE_F32: rc = w3d_lin_tiles_f32(a, prod, c.tile, z, st); break;
        case W3D_DTYPE_BF16: rc = w3d_lin_tiles_bf16(a, prod, c.tile, z, st); break;
        case W3D_DTYPE_F16: rc = w3d_lin_tiles_f16(a, prod, c.tile, z, st); break;
        default: rc = w3d_lin_tiles_fp8(a, prod, c.tile, z, st); break;
    }
    return rc != W3D_OK || c.slices == 1 ? rc : join(a, prod, z, st);
}

// 32-bit offsets inside a tile: rows of less than 8 MB
bool row_ok(int64_t ld) { return ld < (8 << 20); }

// ---- operands whose rows are not aligned (an odd width, a view that starts anywhere) are copied once per call into rows padded with zeros to 16 bytes; the few-row form reads them in place.
// One wave per row, 16 bytes a lane; one launch for all of a call's operands.  (Staging such rows through registers instead: 4999 x 999 -> 515 f16 in training 162 us.)
struct Copy { const uint8_t *src; uint8_t *dst; int64_t rows, cols, ld; };      // cols: elements, ld: bytes
struct Copies { Copy c[4]; int n; };
template <int EB>
__global__ __launch_bounds__(256) void align_rows_kernel(Copies a) {
    const int lane = threadIdx.x & 63;
    int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t waves = (int64_t)gridDim.x * 4;
    for (int j = 0; j < a.n; ++j) {
        const Copy &c = a.c[j];
        for (; w < c.rows; w += waves) {
            const uint8_t *src = c.src + w * c.cols * EB;
            uint8_t *dst = c.dst + w * c.ld;
            for (int64_t k = lane * 16; k < c.ld; k += 1024) {
                const int64_t left = c.cols * EB - k;
                uint32_t v[4] = {0, 0, 0, 0};
                if (left >= 16) __builtin_memcpy(v, src + k, 16);
                else
#pragma unroll
                    for (int e = 0; e < 16; e += EB)
                        if (e < left) {
                            uint32_t b = 0;
                            __builtin_memcpy(&b, src + k + e, EB);
                            v[e / 4] |= b << (8 * (e & 3));
                        }
                *reinterpret_cast<uint4 *>(dst + k) = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
        w -= c.rows;                                                     // the rows of the copies are one sequence
    }
}
int64_t copy_bytes(int64_t rows, int64_t cols, int eb) { return ceil_to(rows * ceil_to(cols * eb, 16), 256); }
bool unaligned(const void *p, int64_t ld) { return p && !aligned16(p, ld); }
struct Aligner {
    uint8_t *at;
    Copies todo;
    int eb;
    // where the operand's copy will be
    const uint8_t *copy(const void *p, int64_t rows, int64_t cols, int64_t &ld) {
        ld = ceil_to(cols * eb, 16);
        uint8_t *dst = at;
        at += copy_bytes(rows, cols, eb);
        todo.c[todo.n++] = {(const uint8_t *)p, dst, rows, cols, ld};
        return dst;
    }
    int run(hipStream_t st) const {
        if (!todo.n) return W3D_OK;
        int64_t rows = 0;
        for (int i = 0; i < todo.n; ++i) rows += todo.c[i].rows;
        const dim3 grid(w3d_grid(rows, 4, 4096)), block(256);
        if (eb == 4) hipLaunchKernelGGL(align_rows_kernel<4>, grid, block, 0, st, todo);
        else if (eb == 2) hipLaunchKernelGGL(align_rows_kernel<2>, grid, block, 0, st, todo);
        else hipLaunchKernelGGL(align_rows_kernel<1>, grid, block, 0, st, todo);
        W3D_CHECK_LAUNCH();
        return W3D_OK;
    }
};

int forward(const void *x, const int32_t *xs, const void *w, const int32_t *ws, const void *w2, const int32_t *ws2, const void *bias, const void *bias2, int bias_dtype,
            const void *residual, int64_t R, int64_t K, int64_t N, int dtype, int out_dtype, int act, bool gated, void *y, float *z, void *workspace, size_t workspace_bytes, hipStream_t st) {
    if (R < 0 || K < 1 || N < 1 || act < 0 || act > ACT_SIGMOID || !float_dtype(out_dtype)) return W3D_ERR_ARG;
    if ((bias || bias2) && bias_dtype != out_dtype && bias_dtype != W3D_DTYPE_F32) return W3D_ERR_ARG;
    if (R == 0) return W3D_OK;
    if (!x || !w || !y || (gated && !w2) || ((uintptr_t)z & 15)) return W3D_ERR_ARG;
    const int eb = eb_of(dtype);
    if (!row_ok(K * eb) || !row_ok(N * eb_of(out_dtype))) return W3D_ERR_UNSUPPORTED;
    GemmArgs a = {};
    a.x = (const uint8_t *)x; a.w = (const uint8_t *)w; a.w2 = (const uint8_t *)w2;
    a.ldx = a.ldw = K * eb; a.M = R; a.N = N; a.K = K;
    a.bias = (const uint8_t *)bias; a.bias2 = (const uint8_t *)bias2; a.bias_f32 = bias_dtype == W3D_DTYPE_F32 && out_dtype != W3D_DTYPE_F32;
    a.res = (const uint8_t *)residual; a.xs = xs; a.ws = ws; a.ws2 = ws2;
    a.out = (uint8_t *)y; a.ld_out = N * eb_of(out_dtype); a.act = act; a.out_dt = out_dtype; a.z = z; a.part_ld = z_stride(N, gated);
    const bool vec = aligned16(y, a.ld_out) && aligned16(residual, 0);
    const int prod = gated ? PROD_GATED : PROD_LINEAR;
    // (all operands of one side have one row length: an unaligned second weight matrix takes the first along)
    const bool ux = unaligned(x, K * eb), uw = unaligned(w, K * eb) || unaligned(w2, K * eb);
    const Cut c = forward_cut(R, K, N, dtype, gated, vec);
    if (few_rows(R, K, N, dtype, gated, ux || uw, c)) {
        switch (dtype) {
            case W3D_DTYPE_F32: return w3d_lin_skinny_f32(a, prod, st);
            case W3D_DTYPE_BF16: return w3d_lin_skinny_bf16(a, prod, st);
            case W3D_DTYPE_F16: return w3d_lin_skinny_f16(a, prod, st);
            default: return w3d_lin_skinny_fp8(a, prod, st);
        }
    }
    Aligner al = {(uint8_t *)workspace, {}, eb};
    const int64_t copies = (ux ? copy_bytes(R, K, eb) : 0) + (uw ? (gated ? 2 : 1) * copy_bytes(N, K, eb) : 0);
    const size_t need = (size_t)copies + part_bytes(c, R, N, gated, 1);
    if (need && (!workspace || (((uintptr_t)workspace) & 15) || workspace_bytes < need)) return W3D_ERR_WORKSPACE;
    if (copies) {
        if (ux) a.x = al.copy(x, R, K, a.ldx);
        if (uw) { a.w = al.copy(w, N, K, a.ldw); if (gated) a.w2 = al.copy(w2, N, K, a.ldw); }
        const int rc = al.run(st);
        if (rc != W3D_OK) return rc;
    }
    a.part = (float *)((uint8_t *)workspace + copies);
    return run_product(a, prod, dtype, c, 1, st);
}

// what a call may need: by its sizes, and for tensors that may start at any element (views) the copies on top
size_t forward_bytes(int64_t R, int64_t K, int64_t N, int dtype, bool gated, bool views) {
    if (K < 1 || N < 1) return 0;
    const int eb = eb_of(dtype);
    size_t most = 0;
    for (int vec = 0; vec < 2; ++vec) {
        const Cut c = forward_cut(R, K, N, dtype, gated, vec);
        if (few_rows(R, K, N, dtype, gated, K * eb % 16 != 0, c)) continue;
        const size_t b = part_bytes(c, R, N, gated, 1);
        most = b > most ? b : most;
    }
    if (R <= SKINNY_ROWS) return most;                                                        // (no copies)
    return most + (views || K * eb % 16 ? (size_t)(copy_bytes(R, K, eb) + (gated ? 2 : 1) * copy_bytes(N, K, eb)) : 0);
}

// ---- backward.  Workspace: aligned copies | dz | column sums | partial tiles (of one product at a time)
struct Bwd {
    int64_t pad, ld_dz;          // columns of one half of dz, bytes of a row of dz
    int64_t copies, dz_bytes, strips, colsum_ld, colsum_bytes, part;
};
int64_t max64(int64_t a, int64_t b) { return a > b ? a : b; }
// strips of partial column sums that the product forming dz writes: one per tile row and row of waves, or the joining launch's
int64_t join_strips(int64_t R) { return (R + strip_rows(R) - 1) / strip_rows(R); }
int64_t strips_of(const Cut &c, int64_t R) { return c.slices > 1 ? join_strips(R) : c.tiles_m * (c.tile == 64 ? 4 : 2); }
// kept: z is there; cx, cw, cdy: the rows of x, of the weights, of dy (as an operand) are copied
Bwd bwd_plan(int64_t R, int64_t K, int64_t N, int dtype, bool gated, bool no_act, bool kept, bool cx, bool cw, bool cdy) {
    Bwd b;
    const int eb = eb_of(dtype), parts = gated ? 2 : 1;
    b.copies = (cx ? copy_bytes(R, K, eb) : 0) + (cw ? parts * copy_bytes(N, K, eb) : 0) + (cdy ? copy_bytes(R, N, eb) : 0);
    b.pad = ceil_to(N, gated ? 64 : 16 / eb);
    b.ld_dz = b.pad * parts * eb;
    b.dz_bytes = no_act ? 0 : ceil_to(R * b.ld_dz, 256);
    b.colsum_ld = ceil_to(N, 16) * parts;
    b.part = 0;
    b.strips = no_act ? w3d_column_strips(R, N) : kept ? join_strips(R) : 0;
    for (int vec = 0; vec < 2; ++vec) {
        const Cut z = cut_of(R, gated ? b.pad : N, K, dtype, gated, vec, 1), dx = cut_of(R, K, gated ? 2 * b.pad : N, dtype, false, vec, 1), dw = cut_of(N, K, R, dtype, false, vec, parts, DW);
        if (!no_act && !kept) {
            b.strips = max64(b.strips, strips_of(z, R));
            b.part = max64(b.part, (int64_t)part_bytes(z, R, N, gated, 1));
        }
        b.part = max64(b.part, max64((int64_t)part_bytes(dx, R, K, false, 1), (int64_t)part_bytes(dw, N, K, false, parts)));
    }
    b.colsum_bytes = ceil_to(b.strips * b.colsum_ld * 4, 256);
    return b;
}

int backward(const void *x, const void *w, const void *w2, const void *bias, const void *bias2, int bias_dtype, const void *dy, const float *z, int64_t R, int64_t K, int64_t N, int dtype,
             int act, bool gated, void *dx, void *dw, void *dw2, void *db, void *db2, void *workspace, size_t workspace_bytes, hipStream_t st) {
    if (R < 0 || K < 1 || N < 1 || act < 0 || act > ACT_SIGMOID || !float_dtype(dtype)) return W3D_ERR_ARG;
    if ((bias || bias2 || db || db2) && bias_dtype != dtype && bias_dtype != W3D_DTYPE_F32) return W3D_ERR_ARG;
    if (!dx && !dw && !dw2 && !db && !db2) return W3D_ERR_ARG;
    const int eb = eb_of(dtype), parts = gated ? 2 : 1;
    if (!row_ok(K * eb) || !row_ok((N + 64) * eb * parts)) return W3D_ERR_UNSUPPORTED;
    if (R > 0 && (!x || !w || !dy || (gated && !w2) || ((uintptr_t)z & 15))) return W3D_ERR_ARG;
    const bool no_act = !gated && act == ACT_NONE;
    if (R > 0 && dtype == W3D_DTYPE_F32 && !no_act && !z) return W3D_ERR_ARG;
    const bool again = !no_act && !z;                                                         // z is formed again
    const bool cx = R > 0 && (again || dw || dw2) && unaligned(x, K * eb), cw = R > 0 && (again || dx) && (unaligned(w, K * eb) || unaligned(w2, K * eb)),
               cdy = R > 0 && no_act && (dx || dw) && unaligned(dy, N * eb);
    const Bwd b = bwd_plan(R, K, N, dtype, gated, no_act, z != nullptr, cx, cw, cdy);
    uint8_t *ws = (uint8_t *)workspace;
    if (R > 0) {
        const size_t need = (size_t)(b.copies + b.dz_bytes + b.colsum_bytes + b.part);
        if (need && (!ws || (((uintptr_t)ws) & 15) || workspace_bytes < need)) return W3D_ERR_WORKSPACE;
    }
    uint8_t *dz_buf = ws + b.copies;
    float *colsum = (float *)(dz_buf + b.dz_bytes), *part = (float *)(dz_buf + b.dz_bytes + b.colsum_bytes);
    const uint8_t *X = (const uint8_t *)x, *W = (const uint8_t *)w, *W2 = (const uint8_t *)w2, *dz = (const uint8_t *)dy;
    int64_t ldx = K * eb, ldw = K * eb, ld_dz = N * eb, strips = 0;
    Aligner al = {ws, {}, eb};
    if (cx) X = al.copy(x, R, K, ldx);
    if (cw) { W = al.copy(w, N, K, ldw); if (gated) W2 = al.copy(w2, N, K, ldw); }
    if (cdy) dz = al.copy(dy, R, N, ld_dz);
    int rc = al.run(st);
    if (rc != W3D_OK) return rc;
    if (R > 0 && !no_act) {
        GemmArgs a = {};
        a.x = X; a.w = W; a.w2 = W2; a.ldx = ldx; a.ldw = ldw; a.M = R; a.N = N; a.K = K;
        a.bias = (const uint8_t *)bias; a.bias2 = (const uint8_t *)bias2; a.bias_f32 = bias_dtype == W3D_DTYPE_F32 && dtype != W3D_DTYPE_F32;
        a.dy = (const uint8_t *)dy; a.out = dz_buf; a.ld_out = b.ld_dz; a.half_out = b.pad * eb; a.act = act; a.out_dt = dtype;
        a.colsum = db || db2 ? colsum : nullptr; a.colsum_ld = b.colsum_ld; a.part = part;
        const int prod = gated ? PROD_GATED_BWD : PROD_LINEAR_BWD;
        if (z) {
            a.part = const_cast<float *>(z); a.part_ld = z_stride(N, gated);
            rc = dtype == W3D_DTYPE_F32 ? dz_as<W3D_DTYPE_F32>(a, gated, st) : dtype == W3D_DTYPE_BF16 ? dz_as<W3D_DTYPE_BF16>(a, gated, st) : dz_as<W3D_DTYPE_F16>(a, gated, st);
            strips = join_strips(R);
        } else {
            const Cut c = cut_of(R, gated ? b.pad : N, K, dtype, gated, aligned16(dy, N * eb), 1);          // (the tiles write the padding columns too)
            rc = run_product(a, prod, dtype, c, 1, st);
            strips = strips_of(c, R);
        }
        if (rc != W3D_OK) return rc;
        dz = dz_buf; ld_dz = b.ld_dz;
    } else if (R > 0 && db) {
        rc = w3d_column_sums(dy, R, N, dtype, colsum, b.colsum_ld, st);
        if (rc != W3D_OK) return rc;
        strips = b.strips;
    }
    if (db) { rc = w3d_fold_columns(colsum, (int)strips, b.colsum_ld, N, db, bias_dtype, st); if (rc != W3D_OK) return rc; }
    if (db2) { rc = w3d_fold_columns(colsum + b.colsum_ld / 2, (int)strips, b.colsum_ld, N, db2, bias_dtype, st); if (rc != W3D_OK) return rc; }
    if (dx && R > 0) {
        GemmArgs a = {};
        a.x = dz; a.ldx = ld_dz; a.w = W; a.w2 = W2; a.ldw = ldw;
        a.M = R; a.N = K; a.K = gated ? 2 * b.pad : N; a.k_split = gated ? b.pad : 0; a.w_rows = N;
        a.out = (uint8_t *)dx; a.ld_out = K * eb; a.out_dt = dtype; a.part = part;
        rc = run_product(a, PROD_DX, dtype, cut_of(R, K, a.K, dtype, false, aligned16(dx, K * eb), 1), 1, st);
        if (rc != W3D_OK) return rc;
    }
    // weight gradients: the two halves of a gated layer are one launch (blockIdx.z) when both are wanted
    const bool both = dw && dw2;
    for (int h = 0; h < 2; ++h) {
        void *o = h ? dw2 : dw;
        if (!o || (both && h && R > 0)) continue;
        if (R == 0) {
            rc = w3d_fold_columns(nullptr, 0, 0, N * K, o, dtype, st);
            if (rc != W3D_OK) return rc;
            continue;
        }
        GemmArgs a = {};
        a.x = dz + (h ? b.pad * eb : 0); a.ldx = ld_dz; a.w = X; a.ldw = ldx;
        a.M = N; a.N = K; a.K = R; a.w_rows = R; a.z_x = b.pad * eb;
        a.out = (uint8_t *)o; a.out2 = (uint8_t *)dw2; a.ld_out = K * eb; a.out_dt = dtype; a.part = part;
        const bool vec = aligned16(o, K * eb) && aligned16(both ? dw2 : nullptr, 0);
        rc = run_product(a, PROD_DW, dtype, cut_of(N, K, R, dtype, false, vec, parts, DW), both ? 2 : 1, st);
        if (rc != W3D_OK) return rc;
    }
    return W3D_OK;
}
}  // namespace

extern "C" size_t w3d_linear_workspace_bytes(int64_t R, int64_t K, int64_t N, int dtype, int gated, int views) { return R < 1 ? 0 : forward_bytes(R, K, N, dtype, gated != 0, views != 0); }
extern "C" size_t w3d_linear_bwd_workspace_bytes(int64_t R, int64_t K, int64_t N, int dtype, int act, int gated, int kept, int views) {
    if (R < 1 || K < 1 || N < 1) return 0;
    const bool no_act = !gated && act == ACT_NONE, ck = views || K * eb_of(dtype) % 16, cn = views || N * eb_of(dtype) % 16;
    const Bwd b = bwd_plan(R, K, N, dtype, gated != 0, no_act, kept != 0, ck, ck, no_act && cn);
    return (size_t)(b.copies + b.dz_bytes + b.colsum_bytes + b.part);
}
extern "C" int64_t w3d_linear_z_stride(int64_t N, int gated) { return N < 1 ? 0 : z_stride(N, gated != 0); }
extern "C" int w3d_linear_fwd(const void *x, const void *w, const void *bias, int bias_dtype, const void *residual, int64_t R, int64_t K, int64_t N, int dtype, int act, void *y,
                              float *z, void *workspace, size_t workspace_bytes, w3d_stream_t stream) {
    if (!float_dtype(dtype)) return W3D_ERR_ARG;
    return forward(x, nullptr, w, nullptr, nullptr, nullptr, bias, nullptr, bias_dtype, residual, R, K, N, dtype, dtype, act, false, y, z, workspace, workspace_bytes, w3d_s(stream));
}
extern "C" int w3d_linear_fp8_fwd(const void *x, const int32_t *x_scale, const void *w, const int32_t *w_scale, const void *bias, int bias_dtype, const void *residual, int64_t R,
                                  int64_t K, int64_t N, int out_dtype, int act, void *y, void *workspace, size_t workspace_bytes, w3d_stream_t stream) {
    if ((out_dtype != W3D_DTYPE_BF16 && out_dtype != W3D_DTYPE_F16) || (R > 0 && (!x_scale || !w_scale))) return W3D_ERR_ARG;
    return forward(x, x_scale, w, w_scale, nullptr, nullptr, bias, nullptr, bias_dtype, residual, R, K, N, W3D_DTYPE_FP8_E4M3, out_dtype, act, false, y, nullptr, workspace, workspace_bytes,
                   w3d_s(stream));
}
extern "C" int w3d_gated_linear_fwd(const void *x, const void *w_gate, const void *w_up, const void *b_gate, const void *b_up, int bias_dtype, int64_t R, int64_t K, int64_t N, int dtype,
                                    int act, void *y, float *z, void *workspace, size_t workspace_bytes, w3d_stream_t stream) {
    if (!float_dtype(dtype)) return W3D_ERR_ARG;
    return forward(x, nullptr, w_gate, nullptr, w_up, nullptr, b_gate, b_up, bias_dtype, nullptr, R, K, N, dtype, dtype, act, true, y, z, workspace, workspace_bytes, w3d_s(stream));
}
extern "C" int w3d_gated_linear_fp8_fwd(const void *x, const int32_t *x_scale, const void *w_gate, const int32_t *gate_scale, const void *w_up, const int32_t *up_scale,
                                        const void *b_gate, const void *b_up, int bias_dtype, int64_t R, int64_t K, int64_t N, int out_dtype, int act, void *y, void *workspace,
                                        size_t workspace_bytes, w3d_stream_t stream) {
    if ((out_dtype != W3D_DTYPE_BF16 && out_dtype != W3D_DTYPE_F16) || (R > 0 && (!x_scale || !gate_scale || !up_scale))) return W3D_ERR_ARG;
    return forward(x, x_scale, w_gate, gate_scale, w_up, up_scale, b_gate, b_up, bias_dtype, nullptr, R, K, N, W3D_DTYPE_FP8_E4M3, out_dtype, act, true, y, nullptr, workspace, workspace_bytes,
                   w3d_s(stream));
}
extern "C" int w3d_linear_bwd(const void *x, const void *w, const void *bias, int bias_dtype, const void *dy, const float *z, int64_t R, int64_t K, int64_t N, int dtype, int act, void *dx,
                              void *dw, void *dbias, void *workspace, size_t workspace_bytes, w3d_stream_t stream) {
    return backward(x, w, nullptr, bias, nullptr, bias_dtype, dy, z, R, K, N, dtype, act, false, dx, dw, nullptr, dbias, nullptr, workspace, workspace_bytes, w3d_s(stream));
}
extern "C" int w3d_gated_linear_bwd(const void *x, const void *w_gate, const void *w_up, const void *b_gate, const void *b_up, int bias_dtype, const void *dy, const float *z, int64_t R,
                                    int64_t K, int64_t N, int dtype, int act, void *dx, void *dw_gate, void *dw_up, void *db_gate, void *db_up, void *workspace, size_t workspace_bytes,
                                    w3d_stream_t stream) {
    return backward(x, w_gate, w_up, b_gate, b_up, bias_dtype, dy, z, R, K, N, dtype, act, true, dx, dw_gate, dw_up, db_gate, db_up, workspace, workspace_bytes, w3d_s(stream));
}
#endif
