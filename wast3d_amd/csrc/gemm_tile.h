// One output tile of C[m][n] = sum over k of X(m, k) W(n, k) on the matrix cores of gfx950, for the linear layers (linear.hip) and their gradients.
//
// Operands.  Each side is held in one of two orders: K_ROWS, rows m (n) of contiguous k, or M_ROWS, rows k of contiguous m (n).  The three products of a layer are
//   z  = x W^T        X: x [R][K] K_ROWS,    W: W [N][K] K_ROWS
//   dx = dz W         X: dz [R][N] K_ROWS,   W: W [N][K] M_ROWS   (contraction over N)
//   dW = dz^T x       X: dz [R][N] M_ROWS,   W: x [R][K] M_ROWS   (contraction over R)
// so no transposed copy of anything is ever made: M_ROWS fragments are formed by the transposing LDS read (16 bits) or single-element reads (f32).
//
// Slabs.  The contraction advances in slabs of 128 bytes of k (32 f32, 64 16-bit, 128 fp8 elements).  A K_ROWS slab is [rows][128 B], an M_ROWS slab [k of the slab][rows x element];
// 16-byte chunks are permuted inside a row (XOR with bits of the row) so that the fragment reads of 8 (16) neighbouring lanes touch all LDS banks.
//
// Matrix instructions.  W is the A operand and X the B operand: a lane then holds, for ONE row m, runs of consecutive n of the output.  Which row of W sits in which row of the operand is
// free, and is chosen so that a lane's runs join to 8 or 16 elements (K_ROWS; the M_ROWS read fixes it to 4).
//
// Sums are f32 in the accumulators, over the whole contraction or over one slice of it (slices > 1: partial tiles go to a workspace and are added in slice order by a second launch).
#pragma once
#include <type_traits>
#include "rows16.h"

namespace w3d_lin {
struct GemmArgs {
    const uint8_t *x, *w, *w2;          // operands; w2: the second weight matrix of a gated layer
    int64_t ldx, ldw;                   // bytes from storage row to storage row
    int64_t M, N, K;                    // C is M x N (gated: N of each half), contraction over K elements
    int64_t k_split;                    // > 0: contraction indices >= k_split take their W rows from w2 (dx of a gated layer: k_split = the padded N, W rows n and n - k_split)
    int64_t w_rows;                     // M_ROWS W: storage rows of w (and of w2): zeros beyond
    int64_t z_x, z_out;                 // blockIdx.z == 1 (second half of a gated dW): byte offset into x, and out2 instead of out
    // epilogue
    const uint8_t *bias, *bias2;        // [N] or NULL
    const uint8_t *res;                 // residual [M][N] or NULL
    const uint8_t *dy;                  // [M][N]: upstream gradient (BWD)
    const int32_t *xs, *ws, *ws2;       // fp8: E8M0 exponents of the rows of x, w, w2
    uint8_t *out, *out2;                // [M][N] (BWD: dz [M][ld_out bytes], gated: two halves half_out bytes apart)
    int64_t ld_out, half_out;
    float *colsum;                      // BWD: [row strips][colsum_ld] partial column sums of dz, or NULL
    int64_t colsum_ld;
    float *part;                        // slices > 1: [slice][M][part_ld] f32
    int64_t part_ld;
    int bias_f32, act, slices, tiles_m, tiles_n, vec_io, out_dt;
};
}  // namespace w3d_lin
using w3d_lin::GemmArgs;

namespace {

enum { K_ROWS = 0, M_ROWS = 1 };
enum { ACT_NONE = W3D_ACT_NONE, ACT_RELU = W3D_ACT_RELU, ACT_GELU = W3D_ACT_GELU, ACT_SILU = W3D_ACT_SILU, ACT_SIGMOID = W3D_ACT_SIGMOID };
enum { EPI_LINEAR = 0, EPI_GATED = 1, EPI_LINEAR_BWD = 2, EPI_GATED_BWD = 3, EPI_STORE = 4 };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t *lds_t;
typedef __attribute__((address_space(3))) void *lds_void_t;

constexpr int SLAB = 128;                        // bytes of contraction per slab
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;   // buffer offset past num_records: the load returns zeros

// ---- activations.  a = act(z), d = act'(z).
// gelu(z) = z Phi(z); Phi(-|z|) = exp(-z^2 / 2) p(t) / 2, t = 1 / (1 + 0.3275911 |z| / sqrt 2), p the degree-5 polynomial of Abramowitz & Stegun 7.1.26 (|error of erf| <= 1.5e-7): one exponential
// serves Phi and the density in the derivative, and the tail has no cancellation.
template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;                       // (a NaN stays)
    if (ACT == ACT_GELU) {
        const float h = fabsf(z);
        const float t = __builtin_amdgcn_rcpf(fmaf(h, 0.3275911f * 0.70710678f, 1.0f));
        const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        const float tail = 0.5f * p * __expf(-0.5f * z * z);
        return z * (z < 0.f ? tail : 1.0f - tail);
    }
    if (ACT == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    if (ACT == ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    return z;
}
template <int ACT>
__device__ __forceinline__ void act_both(float z, float &a, float &d) {
    if (ACT == ACT_NONE) { a = z; d = 1.f; }
    else if (ACT == ACT_RELU) { a = z < 0.f ? 0.f : z; d = z > 0.f ? 1.f : 0.f; }
    else if (ACT == ACT_GELU) {
        const float h = fabsf(z);
        const float t = __builtin_amdgcn_rcpf(fmaf(h, 0.3275911f * 0.70710678f, 1.0f));
        const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        const float e = __expf(-0.5f * z * z), tail = 0.5f * p * e, cdf = z < 0.f ? tail : 1.0f - tail;
        a = z * cdf;
        d = fmaf(z * 0.39894228f, e, cdf);
    } else {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
        if (ACT == ACT_SILU) { a = z * s; d = s * fmaf(z, 1.0f - s, 1.0f); }
        else { a = s; d = s * (1.0f - s); }
    }
}
// calls f with the activation as a compile-time value
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
    switch (act) {
        case ACT_RELU: f(std::integral_constant<int, ACT_RELU>()); break;
        case ACT_GELU: f(std::integral_constant<int, ACT_GELU>()); break;
        case ACT_SILU: f(std::integral_constant<int, ACT_SILU>()); break;
        case ACT_SIGMOID: f(std::integral_constant<int, ACT_SIGMOID>()); break;
        default: f(std::integral_constant<int, ACT_NONE>()); break;
    }
}

// ---- runs of CNT (4, 8 or 16) consecutive elements of a row, `n` of them inside; vec: the row is 16-byte aligned at 8-element steps
template <int DT, int CNT>
__device__ __forceinline__ void load_run(const uint8_t *p, int64_t n, bool vec, float (&v)[CNT]) {
    constexpr int EB = Elem<DT>::B;
    if (vec && n >= CNT) {
        uint32_t w[CNT * EB / 4];
        if (CNT * EB >= 16) {
#pragma unroll
            for (int i = 0; i < CNT * EB / 16; ++i) { const i32x4 t = reinterpret_cast<const i32x4 *>(p)[i]; __builtin_memcpy(&w[4 * i], &t, 16); }
        } else { const uint2 t = *reinterpret_cast<const uint2 *>(p); w[0] = t.x; w[1] = t.y; }
#pragma unroll
        for (int i = 0; i < CNT; ++i) {
            if (DT == W3D_DTYPE_F32) v[i] = __uint_as_float(w[i]);
            else if (DT == W3D_DTYPE_BF16) v[i] = (i & 1) ? __uint_as_float(w[i / 2] & 0xffff0000u) : __uint_as_float(w[i / 2] << 16);
            else v[i] = f16_to_f32((uint16_t)(w[i / 2] >> (16 * (i & 1))));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < CNT; ++i) v[i] = i < n ? load1<DT>(p + i * EB) : 0.f;
}
template <int DT, int CNT>
__device__ __forceinline__ void store_run(uint8_t *p, int64_t n, bool vec, const float (&v)[CNT]) {
    constexpr int EB = Elem<DT>::B;
    if (vec && n >= CNT) {
        uint32_t w[CNT * EB / 4];
#pragma unroll
        for (int i = 0; i < CNT * EB / 4; ++i) {
            if (DT == W3D_DTYPE_F32) w[i] = __float_as_uint(v[i]);
            else {
                const uint16_t a = DT == W3D_DTYPE_BF16 ? f32_to_bf16(v[2 * i]) : f32_to_f16(v[2 * i]);
                const uint16_t b = DT == W3D_DTYPE_BF16 ? f32_to_bf16(v[2 * i + 1]) : f32_to_f16(v[2 * i + 1]);
                w[i] = (uint32_t)a | ((uint32_t)b << 16);
            }
        }
        if (CNT * EB >= 16) {
#pragma unroll
            for (int i = 0; i < CNT * EB / 16; ++i) { i32x4 t; __builtin_memcpy(&t, &w[4 * i], 16); reinterpret_cast<i32x4 *>(p)[i] = t; }
        } else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        return;
    }
#pragma unroll
    for (int i = 0; i < CNT; ++i)
        if (i < n) store1<DT>(p + i * EB, v[i]);
}
template <int DT>
__device__ __forceinline__ float bias_at(const uint8_t *b, int bias_f32, int64_t n, int64_t N) {
    if (!b || n >= N) return 0.f;
    return bias_f32 ? load1<W3D_DTYPE_F32>(b + n * 4) : load1<DT>(b + n * Elem<DT>::B);
}

// ---- one side's slabs: global -> LDS.  ROWS rows of the output tile, NT threads.
template <int LAY, int ROWS, int EB, int NT, int HASH_BIT>
struct Stage {
    static constexpr int BYTES = ROWS * SLAB, PIECES = BYTES / 16 / NT, KPS = SLAB / EB;      // KPS: contraction elements per slab
    static constexpr int CPR = LAY == K_ROWS ? SLAB / 16 : ROWS * EB / 16;                     // chunks per LDS row
    static_assert(BYTES % (16 * NT) == 0, "whole pieces");

    // permutation of the 16-byte chunks of an LDS row.  K_ROWS: neighbouring operand rows r = 0..7 sit in tile rows (r & 3) + (4 * group stride) * (r >> 2): HASH_BIT is log2 of
    // that stride (2 where operand rows are tile rows).  M_ROWS, 16 bits: four consecutive k share a transposing read of 16 lanes; f32: k and k + 4 share the 64-lane read's halves.
    static __device__ __forceinline__ int swizzle(int row) {
        if (LAY == K_ROWS) return (row & 3) | (((row >> HASH_BIT) & 1) << 2);
        return EB == 4 ? ((row >> 2) & 1) << 2 : (row & 3) << 1;
    }
    static __device__ __forceinline__ void place(int tid, int i, int &row, int &chunk) {      // storage row inside the slab and source chunk of piece i
        const int p = i * NT + tid;
        row = p / CPR;
        chunk = (p % CPR) ^ swizzle(row);
    }
};

// MFMA over one slab of fragments: xf/wf [step] of 16 B a lane, two steps a slab
template <int DT>
__device__ __forceinline__ f32x4 mfma_step(const i32x4 (&w)[2], const i32x4 (&x)[2], int s, f32x4 c) {
    if (DT == W3D_DTYPE_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[s]), __builtin_bit_cast(bf16x8, x[s]), c, 0, 0, 0);
    if (DT == W3D_DTYPE_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w[s]), __builtin_bit_cast(f16x8, x[s]), c, 0, 0, 0);
    if (DT == W3D_DTYPE_F32) {
        const f32x4 a = __builtin_bit_cast(f32x4, w[s]), b = __builtin_bit_cast(f32x4, x[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    // fp8: both chunks of the slab are one operand of 32 bytes a lane; the rows' scales are applied to the f32 sums in the epilogue, the instruction's own are 1
    if (s) return c;
    i32x8 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = w[0][i]; a[4 + i] = w[1][i]; b[i] = x[0][i]; b[4 + i] = x[1][i]; }
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 127, 0, 127);
}

template <int DT, int LX, int LW, int EPI, int BM, int BN, int WM, int WN, bool ALIGNED>
struct Gemm {
    static constexpr int NT = WM * WN * 64, EB = Elem<DT>::B, KPS = SLAB / EB;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    static constexpr bool GATED = EPI == EPI_GATED || EPI == EPI_GATED_BWD;
    static constexpr int PARTS = GATED ? 2 : 1, FP = FN / PARTS, BNP = BN / PARTS;             // a gated tile is BN / 2 columns of each half: rows [0, BN/2) of the W slab gate, the rest up
    static constexpr int CG = LW == M_ROWS ? 1 : (FP < 4 ? FP : 4);                           // fragments whose runs of 4 join in one lane
    static constexpr int RUN = 4 * CG, GROUPS = FP / CG;
    static constexpr int HASH_W = CG == 4 ? 4 : CG == 2 ? 3 : 2;
    typedef Stage<LX, BM, EB, NT, 2> SX;
    typedef Stage<LW, BN, EB, NT, HASH_W> SW;
    static constexpr int BUF = SX::BYTES + SW::BYTES, LDS_BYTES = 2 * BUF;
    static_assert(!GATED || LW == K_ROWS, "gated products read the weights by rows");
    static_assert(!GATED || SW::PIECES % 2 == 0, "a piece of the W slab belongs to one half");

    // byte address (inside the slab) of a lane's first K_ROWS chunk: step s adds XOR 64
    static __device__ __forceinline__ int x_row(int wm, int f, int lane) { return wm * (BM / WM) + 16 * f + (lane & 15); }
    static __device__ __forceinline__ int w_row(int wn, int f, int lane) {                     // tile row of operand row r = lane & 15 of fragment f
        const int r = lane & 15, part = f / FP, fp = f % FP;
        return part * BNP + wn * (BNP / WN) + 16 * CG * (fp / CG) + 4 * CG * (r >> 2) + 4 * (fp % CG) + (r & 3);
    }
    template <typename S, int LAY>
    static __device__ __forceinline__ void frag(const uint8_t *slab, int row_of_lane, int base16, int lane, i32x4 (&v)[2]) {
        const int q = lane >> 4;
        if (LAY == K_ROWS) {
            const int sw = S::swizzle(row_of_lane);
#pragma unroll
            for (int s = 0; s < 2; ++s) v[s] = *reinterpret_cast<const i32x4 *>(slab + row_of_lane * SLAB + (((4 * s + q) ^ sw) << 4));
        } else if (EB == 2) {
            // rows k = 32 s + 8 q + 4 h + (0..3) of 16 elements each are transposed by 16 lanes: lane j gives the address of elements 4 (j & 3) .. +3 of row k + (j >> 2) and receives element
            // j of the four rows
            const int j = lane & 15;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int k = 32 * s + 8 * q + 4 * h + (j >> 2);
                    const int chunk = ((base16 * 2 + ((j & 3) >> 1)) ^ S::swizzle(k));
                    typedef __attribute__((address_space(3))) s16x4 *lp;
                    const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds_t)(slab + k * (S::CPR * 16) + chunk * 16 + (j & 1) * 8));
                    int2 u;
                    __builtin_memcpy(&u, &t, 8);
                    v[s][2 * h] = u.x; v[s][2 * h + 1] = u.y;
                }
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = 16 * s + 4 * q + e, m = base16 * 16 + (lane & 15);
                    v[s][e] = *reinterpret_cast<const int *>(slab + k * (S::CPR * 16) + (((m >> 2) ^ S::swizzle(k)) << 4) + (m & 3) * 4);
                }
        }
    }

    // a chunk of 16 bytes whose first n elements exist (register staging: any alignment)
    static __device__ __forceinline__ i32x4 chunk_of(const uint8_t *p, int64_t n) {
        i32x4 v = {0, 0, 0, 0};
        if (n >= 16 / EB) { __builtin_memcpy(&v, p, 16); return v; }
        if (n <= 0) return v;
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16 / EB; ++i)
            if (i < n) {
                uint32_t b = 0;
                __builtin_memcpy(&b, p + i * EB, EB);
                w[i * EB / 4] |= b << (8 * ((i * EB) & 3));
            }
        __builtin_memcpy(&v, w, 16);
        return v;
    }

    // address and extent of piece i of a side's slab
    struct Side {
        const uint8_t *base;      // first byte of the tile's operand (K_ROWS: row 0 of the tile; M_ROWS: column 0 of the tile, contraction row 0)
        int64_t ld;
        int64_t rows;             // K_ROWS: rows of the tile that exist; M_ROWS: columns that exist from the tile's first
        int64_t k;                // contraction elements that exist
    };
    template <typename S, int LAY>
    static __device__ __forceinline__ void load_dma(const Side &sd, int64_t k0, uint8_t *slab, int tid, int i) {
        int row, chunk;
        S::place(tid, i, row, chunk);
        const int64_t kleft = sd.k - k0;
        const bool ok = LAY == K_ROWS ? row < sd.rows && (int64_t)chunk * (16 / EB) < kleft : row < kleft && (int64_t)chunk * (16 / EB) < sd.rows;
        const uint32_t off = ok ? (uint32_t)row * (uint32_t)sd.ld + (uint32_t)chunk * 16u : OUT_OF_RANGE;
        const uint8_t *base = sd.base + (LAY == K_ROWS ? k0 * EB : k0 * sd.ld);
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, 0x7fffffff, 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t)(lds_t)(slab + (i * NT + wave * 64) * 16), 16, (int)off, 0, 0, 0);
    }
    template <typename S, int LAY>
    static __device__ __forceinline__ i32x4 load_reg(const Side &sd, int64_t k0, int tid, int i) {
        int row, chunk;
        S::place(tid, i, row, chunk);
        const int64_t kleft = sd.k - k0, e = (int64_t)chunk * (16 / EB);
        const bool ok = LAY == K_ROWS ? row < sd.rows : row < kleft;
        const int64_t n = ok ? (LAY == K_ROWS ? kleft : sd.rows) - e : 0;
        return chunk_of(sd.base + (LAY == K_ROWS ? row * sd.ld + k0 * EB : (k0 + row) * sd.ld) + e * EB, n);
    }

    static __device__ __forceinline__ void run(const GemmArgs &a, uint8_t *smem) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
        // tile of this block: consecutive blocks go round the 8 XCDs, so block b works on place (b % 8) * (tiles / 8) + b / 8 of an order in which neighbours share operand rows (each
        // XCD's L2 then serves a compact patch of C); the order runs down groups of 8 tile rows
        const int tiles = a.tiles_m * a.tiles_n, total = tiles * a.slices;
        int id = blockIdx.x;
        {
            const int q = total / 8, r = total % 8, xcd = id % 8, at = id / 8;
            id = xcd * q + min(xcd, r) + at;
        }
        const int slice = id / tiles;
        id -= slice * tiles;
        int tm, tn;
        {
            const int span = 8 * a.tiles_n, g = id / span, first = g * 8, rows = min(8, a.tiles_m - first), in = id - g * span;
            tm = first + in % rows;
            tn = in / rows;
        }
        const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BNP;
        const int64_t slabs = (a.K + KPS - 1) / KPS;
        const int64_t s_begin = slabs * slice / a.slices, s_end = slabs * (slice + 1) / a.slices;
        const bool z1 = blockIdx.z != 0;

        Side sx, sw, sw2;
        sx.base = a.x + (z1 ? a.z_x : 0) + (LX == K_ROWS ? m0 * a.ldx : m0 * EB);
        sx.ld = a.ldx; sx.rows = a.M - m0; sx.k = a.K;
        const int64_t w_at = LW == K_ROWS ? n0 * a.ldw : n0 * EB;
        sw.base = a.w + w_at; sw.ld = a.ldw; sw.rows = a.N - n0; sw.k = LW == M_ROWS ? a.w_rows : a.K;
        sw2 = sw;
        if (GATED) sw2.base = a.w2 + w_at;
        else if (a.k_split > 0) { sw2.base = a.w2 + w_at - a.k_split * a.ldw; sw2.k = a.k_split + a.w_rows; }

        f32x4 acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        // the half of a gated tile a piece of the W slab belongs to: its rows are shifted back to the half's first
        auto w_side = [&](int64_t k0, int i, Side &s) {
            if (GATED) {
                s = i < SW::PIECES / 2 ? sw : sw2;
                if (i >= SW::PIECES / 2) { s.base -= (int64_t)BNP * s.ld; s.rows += BNP; }
                else s.rows = s.rows < BNP ? s.rows : BNP;
            } else s = a.k_split > 0 && k0 >= a.k_split ? sw2 : sw;
        };
        auto dma = [&](int64_t t, uint8_t *buf) {
            const int64_t k0 = t * KPS;
#pragma unroll
            for (int i = 0; i < SX::PIECES; ++i) load_dma<SX, LX>(sx, k0, buf, tid, i);
#pragma unroll
            for (int i = 0; i < SW::PIECES; ++i) { Side s; w_side(k0, i, s); load_dma<SW, LW>(s, k0, buf + SX::BYTES, tid, i); }
        };
        i32x4 rx[ALIGNED ? 1 : SX::PIECES], rw[ALIGNED ? 1 : SW::PIECES];
        auto fetch = [&](int64_t t) {
            const int64_t k0 = t * KPS;
#pragma unroll
            for (int i = 0; i < SX::PIECES; ++i) rx[ALIGNED ? 0 : i] = load_reg<SX, LX>(sx, k0, tid, i);
#pragma unroll
            for (int i = 0; i < SW::PIECES; ++i) { Side s; w_side(k0, i, s); rw[ALIGNED ? 0 : i] = load_reg<SW, LW>(s, k0, tid, i); }
        };
        auto put = [&](uint8_t *buf) {
#pragma unroll
            for (int i = 0; i < SX::PIECES; ++i) *reinterpret_cast<i32x4 *>(buf + (i * NT + tid) * 16) = rx[ALIGNED ? 0 : i];
#pragma unroll
            for (int i = 0; i < SW::PIECES; ++i) *reinterpret_cast<i32x4 *>(buf + SX::BYTES + (i * NT + tid) * 16) = rw[ALIGNED ? 0 : i];
        };
        if (s_begin < s_end) {
            if (ALIGNED) dma(s_begin, smem);
            else { fetch(s_begin); put(smem); }
        }
        int cur = 0;
        for (int64_t t = s_begin; t < s_end; ++t, cur ^= 1) {
            __syncthreads();                             // slab t has landed (every wave drains its own LDS-DMA), and nobody reads the other buffer any more
            const uint8_t *bx = smem + cur * BUF, *bw = bx + SX::BYTES;
            i32x4 xf[FM][2], wf[FN][2];
#pragma unroll
            for (int j = 0; j < FN; ++j) frag<SW, LW>(bw, w_row(wn, j, lane), wn * FN + j, lane, wf[j]);
#pragma unroll
            for (int i = 0; i < FM; ++i) frag<SX, LX>(bx, x_row(wm, i, lane), wm * FM + i, lane, xf[i]);
            const bool more = t + 1 < s_end;
            if (more) {
                if (ALIGNED) dma(t + 1, smem + (cur ^ 1) * BUF);
                else fetch(t + 1);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mfma_step<DT>(wf[j], xf[i], s, acc[i][j]);
            if (!ALIGNED && more) put(smem + (cur ^ 1) * BUF);
        }
        epilogue(a, acc, m0, n0, slice, tm, wm, wn, lane, z1);
    }

    // first column (inside the output) of group g of a lane
    static __device__ __forceinline__ int64_t col_of(int64_t n0, int wn, int g, int lane) { return n0 + wn * (BNP / WN) + 16 * CG * g + RUN * (lane >> 4); }
    static __device__ __forceinline__ void gather(const f32x4 (&acc)[FM][FN], int i, int part, int g, float (&v)[RUN]) {
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * c + e] = acc[i][part * FP + g * CG + c][e];
    }

    static __device__ __forceinline__ void epilogue(const GemmArgs &a, f32x4 (&acc)[FM][FN], int64_t m0, int64_t n0, int slice, int tm, int wm, int wn, int lane, bool z1) {
        const int64_t mr = m0 + wm * (BM / WM) + (lane & 15);
        if (a.slices > 1) {
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const int64_t n = col_of(n0, wn, g, lane);
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        const int64_t m = mr + 16 * i;
                        if (m >= a.M) continue;
                        float v[RUN];
                        gather(acc, i, p, g, v);
                        const int64_t z = (int64_t)(z1 ? a.slices : 0) + slice;
                        store_run<W3D_DTYPE_F32, RUN>((uint8_t *)(a.part + (z * a.M + m) * a.part_ld + p * (a.part_ld / 2) + n), a.N - n, true, v);
                    }
                }
            return;
        }
        // (fp8 rows: the output is bf16 or f16)
        if (DT == W3D_DTYPE_FP8_E4M3) {
            if (a.out_dt == W3D_DTYPE_BF16) finish<W3D_DTYPE_BF16>(a, acc, mr, n0, tm, wm, wn, lane, z1);
            else finish<W3D_DTYPE_F16>(a, acc, mr, n0, tm, wm, wn, lane, z1);
        } else finish<DT == W3D_DTYPE_FP8_E4M3 ? W3D_DTYPE_BF16 : DT>(a, acc, mr, n0, tm, wm, wn, lane, z1);
    }

    template <int OT>
    static __device__ __forceinline__ void finish(const GemmArgs &a, f32x4 (&acc)[FM][FN], int64_t mr, int64_t n0, int tm, int wm, int wn, int lane, bool z1) {
        constexpr int OB = Elem<OT>::B;
        const bool vec = a.vec_io != 0;
        if (EPI == EPI_STORE) {
            uint8_t *out = z1 ? a.out2 : a.out;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int64_t n = col_of(n0, wn, g, lane);
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const int64_t m = mr + 16 * i;
                    if (m >= a.M) continue;
                    float v[RUN];
                    gather(acc, i, 0, g, v);
                    store_run<OT, RUN>(out + m * a.ld_out + n * OB, a.N - n, vec, v);
                }
            }
            return;
        }
        with_act(a.act, [&](auto act_c) {
            constexpr int ACT = decltype(act_c)::value;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int64_t n = col_of(n0, wn, g, lane);
                float b0[RUN], b1[RUN], c0[RUN], c1[RUN];
#pragma unroll
                for (int e = 0; e < RUN; ++e) {
                    b0[e] = bias_at<OT>(a.bias, a.bias_f32, n + e, a.N);
                    if (GATED) b1[e] = bias_at<OT>(a.bias2, a.bias_f32, n + e, a.N);
                    c0[e] = c1[e] = 0.f;
                }
                int s0[RUN], s1[RUN];                    // fp8: the sums are scaled by 2^(row exponent of x + row exponent of w), exactly
                if (DT == W3D_DTYPE_FP8_E4M3) {
#pragma unroll
                    for (int e = 0; e < RUN; ++e) {
                        s0[e] = n + e < a.N ? a.ws[n + e] - 254 : 0;
                        if (GATED) s1[e] = n + e < a.N ? a.ws2[n + e] - 254 : 0;
                    }
                }
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const int64_t m = mr + 16 * i;
                    const bool live = m < a.M;
                    float v[RUN], u[RUN], t[RUN];
                    gather(acc, i, 0, g, v);
                    if (GATED) gather(acc, i, 1, g, u);
                    if (DT == W3D_DTYPE_FP8_E4M3) {
                        const int xs = live ? a.xs[m] : 0;
#pragma unroll
                        for (int e = 0; e < RUN; ++e) { v[e] = __builtin_ldexpf(v[e], xs + s0[e]); if (GATED) u[e] = __builtin_ldexpf(u[e], xs + s1[e]); }
                    }
#pragma unroll
                    for (int e = 0; e < RUN; ++e) { v[e] += b0[e]; if (GATED) u[e] += b1[e]; }
                    if (EPI == EPI_LINEAR || EPI == EPI_GATED) {
                        if (!live) continue;
                        if (EPI == EPI_LINEAR && a.res) load_run<OT, RUN>(a.res + (m * a.N + n) * OB, a.N - n, vec, t);
#pragma unroll
                        for (int e = 0; e < RUN; ++e) {
                            v[e] = act_fwd<ACT>(v[e]);
                            if (EPI == EPI_GATED) v[e] *= u[e];
                            else if (a.res) v[e] += t[e];
                        }
                        store_run<OT, RUN>(a.out + m * a.ld_out + n * OB, a.N - n, vec, v);
                    } else {
                        // dz of the rows and columns that exist, zeros in the padding columns (they are part of the contraction of dx); column sums in f32 before the rounding
                        if (live) load_run<OT, RUN>(a.dy + (m * a.N + n) * OB, a.N - n, vec, t);
#pragma unroll
                        for (int e = 0; e < RUN; ++e) {
                            float act, der;
                            act_both<ACT>(v[e], act, der);
                            const bool in = live && n + e < a.N;
                            if (EPI == EPI_LINEAR_BWD) v[e] = in ? t[e] * der : 0.f;
                            else { v[e] = in ? t[e] * (u[e] * der) : 0.f; u[e] = in ? t[e] * act : 0.f; c1[e] += u[e]; }
                            c0[e] += v[e];
                        }
                        if (!live) continue;
                        const int64_t pad = (EPI == EPI_GATED_BWD ? a.half_out : a.ld_out) / OB - n;      // columns of the padded row from here: a multiple of 8 (16 bits) or 4
                        uint8_t *o = a.out + m * a.ld_out + n * OB;
                        constexpr int CH = 16 / OB;
#pragma unroll
                        for (int c = 0; c < RUN / CH; ++c) {
                            float h[CH];
                            if (c * CH < pad) {
#pragma unroll
                                for (int e = 0; e < CH; ++e) h[e] = v[c * CH + e];
                                store_run<OT, CH>(o + c * 16, CH, true, h);
                                if (EPI == EPI_GATED_BWD) {
#pragma unroll
                                    for (int e = 0; e < CH; ++e) h[e] = u[c * CH + e];
                                    store_run<OT, CH>(o + a.half_out + c * 16, CH, true, h);
                                }
                            }
                        }
                    }
                }
                if ((EPI == EPI_LINEAR_BWD || EPI == EPI_GATED_BWD) && a.colsum) {
                    // the 16 lanes of a DPP row hold 16 rows of the same columns: their sum ends in the row's last lane
#pragma unroll
                    for (int e = 0; e < RUN; ++e) {
                        c0[e] = row_sum(c0[e]);
                        if (GATED) c1[e] = row_sum(c1[e]);
                    }
                    if ((lane & 15) == 15) {
                        float *o = a.colsum + ((int64_t)tm * WM + wm) * a.colsum_ld + n;
#pragma unroll
                        for (int e = 0; e < RUN; ++e)
                            if (n + e < a.N) { o[e] = c0[e]; if (GATED) o[a.colsum_ld / 2 + e] = c1[e]; }
                    }
                }
            }
        });
    }
    static __device__ __forceinline__ float row_sum(float v) {
        v = dpp_add_step<0x111, 0xf>(v);
        v = dpp_add_step<0x112, 0xf>(v);
        v = dpp_add_step<0x114, 0xf>(v);
        return dpp_add_step<0x118, 0xf>(v);
    }
};

template <int DT, int LX, int LW, int EPI, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64, 1) void gemm_kernel(GemmArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    Gemm<DT, LX, LW, EPI, BM, BN, WM, WN, ALIGNED>::run(a, smem);
}

}  // namespace
