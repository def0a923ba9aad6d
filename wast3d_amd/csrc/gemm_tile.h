// One output tile of C[m][n] = sum over k of X(m, k) W(n, k) on the matrix cores of gfx950, for the linear layers (linear.hip) and their gradients.
//
// Operands.  Each side is held in one of two orders: K_ROWS, rows m (n) of contiguous k, or M_ROWS, rows k of contiguous m (n).  The three products of a layer are
//   z  = x W^T        X: x [R][K] K_ROWS,    W: W [N][K] K_ROWS
//   dx = dz W         X: dz [R][N] K_ROWS,   W: W [N][K] M_ROWS   (contraction over N)
//   dW = dz^T x       X: dz [R][N] M_ROWS,   W: x [R][K] M_ROWS   (contraction over R)
// so no transposed copy of anything is ever made: M_ROWS fragments are formed by the transposing LDS read (16 bits) or single-element reads (f32).  Storage rows of operands are 16-byte
// aligned (linear.hip copies the ones that are not).
//
// Slabs.  The contraction advances in slabs of 128 bytes of k (32 f32, 64 16-bit, 128 fp8 elements).  A K_ROWS slab is [rows][128 B], an M_ROWS slab [k of the slab][rows x element];
// 16-byte chunks are permuted inside a row (XOR with bits of the row) so that the fragment reads of 8 (16) neighbouring lanes touch all LDS banks.
//
// Matrix instructions.  W is the A operand and X the B operand: a lane then holds, for ONE row m, groups of four consecutive n of the output.
//
// Tiles of 128 x 128 and 64 x 64: two slabs in LDS, the next one's transfers under the products of this one; several blocks on a CU fill each other's waits.  They are for products with few
// 256 x 256 tiles, for f32, and for outputs that are not aligned.  Measured: bf16 784 rows 512 -> 512 6.8 us (64 x 64), 2048 rows 4096 -> 2048 dW 38 us (128 x 128, 0.9 PFLOP/s; 64 x 64 58, 256 x 256 57);
// f32 2048 rows 1024 -> 1024 46 us (64 x 64, 94 of the 132 TFLOP/s of a large product).
//
// Sums are f32 in the accumulators (fp8: with the instruction's own cut inside groups of eight, see mfma_step), over the whole contraction or over one slice of it (slices > 1: partial tiles go to a workspace and are added in slice order by a second launch).
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
    float *z;                           // forward: where the values before the activation go, [M][part_ld] (gated: the second half part_ld / 2 further), or NULL
    int64_t strip;                      // rows of one partial column sum of the joining launch
    int bias_f32, act, slices, tiles_m, tiles_n, out_dt;
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
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t *lds_t;
typedef __attribute__((address_space(3))) void *lds_void_t;

constexpr int SLAB = 128;                        // bytes of contraction per slab
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;   // buffer offset past num_records: the load returns zeros

// ---- activations.  a = act(z), d = act'(z).
// gelu(z) = z Phi(z) = max(z, 0) - h Phi(-h), h = |z|, with Phi(-h) to a relative bound: a gated layer multiplies the tail by what it likes.  Two forms of it:
//   Phi(-h) = e t P(t), e = exp(-h^2 / 2), t = 1 / (1 + 0.3 h): P of degree 7, fitted on [0, 14.3] to the smallest maximum of the relative error, 1.4e-7; in f32 2^-21 and the argument's rounding (h^2 2^-24), which
//     z's own last place costs too.  For f32 layers.
//   log2 Phi(-h) by a polynomial of degree 7, for 16-bit layers, where the epilogue is what a short contraction waits for (us at 65 536 x 256 -> 1 024, gated: degree 7 in either type 123 - 124,
//     degree 8 in bf16 126; linear, degree 10 for both: 88 in bf16 and 90 in f16 instead of 82 and 79).  bf16: fitted on [0, 10.5] to h |error of Phi| <= 1.9e-7 and 2.1e-3 of Phi (half a step is 3.9e-3); f16: on
//     [0, 8], 2.3e-7 and 2.1e-4 (4.9e-4).  Past its range, where Phi is below 5e-26 (7e-16), either falls a little faster than Phi.
//     (The first form in their derivatives: 65 536 x 256 -> 1 024 f16 in training 276 us instead of 270, bf16 the same.)
// Past 13.2 (14.4 in the first form) the exponential is below 2^-126 and becomes 0.
__device__ __forceinline__ float exp_half_square(float h) { return __builtin_amdgcn_exp2f(h * h * -0.72134752f); }
template <int OT> constexpr float FAR_TAIL = OT == W3D_DTYPE_F32 ? 16.0f : 13.2f;               // (Phi is 0 there: below 2^-126)
template <int OT>
__device__ __forceinline__ float normal_tail(float h, float e) {
    if (OT == W3D_DTYPE_F32) {
        const float t = __builtin_amdgcn_rcpf(fmaf(h, 0.3f, 1.0f));
        const float p = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 3.5531368e-2f, -1.5657105e-1f), 2.0520240e-1f), -5.2566256e-2f), 1.2794091e-1f), 1.0010950e-1f), 1.2072159e-1f), 1.1963145e-1f);
        return e * (t * p);
    }
    const float p = OT == W3D_DTYPE_F16
        ? fmaf(h, fmaf(h, fmaf(h, fmaf(h, fmaf(h, fmaf(h, fmaf(h, -1.4817135e-06f, 5.4606211e-05f), -0.000879072f), 0.0083331997f), -0.05368023f), -0.45865902f), -1.1512053f), -0.99999714f)
        : fmaf(h, fmaf(h, fmaf(h, fmaf(h, fmaf(h, fmaf(h, fmaf(h, -1.2373911e-06f, 4.9450155e-05f), -0.00084103353f), 0.0082123438f), -0.053499933f), -0.45878318f), -1.1511714f), -0.99999928f);
    return __builtin_amdgcn_exp2f(p);
}
// e = exp(-|z|), s = 1 / (1 + exp(-z)) and q = 1 - s without the cancellation (1 - s is 0 past z = 17, and wrong by 2^-24 before it).  The exponential's argument is rounded in 16-bit layers: |z| 2^-24 of the value.
template <int OT>
__device__ __forceinline__ void sigmoid_pair(float z, float &s, float &q) {
    const float e = OT == W3D_DTYPE_F32 ? expf(-fabsf(z)) : __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    s = z < 0.f ? er : r;
    q = z < 0.f ? r : er;
}
// OT: the layer's output type
template <int ACT, int OT>
__device__ __forceinline__ float act_fwd(float z) {
    if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;                       // (a NaN stays)
    if (ACT == ACT_GELU) {
        const float h = fminf(fabsf(z), FAR_TAIL<OT>), tail = normal_tail<OT>(h, exp_half_square(h));
        return fmaf(-h, tail, __builtin_elementwise_maximum(z, 0.f));    // (a NaN stays)
    }
    if (OT == W3D_DTYPE_F32 && (ACT == ACT_SILU || ACT == ACT_SIGMOID)) {
        float s, q;
        sigmoid_pair<OT>(z, s, q);
        return ACT == ACT_SILU ? z * s : s;
    }
    if (ACT == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    if (ACT == ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    return z;
}
template <int ACT, int OT>
__device__ __forceinline__ void act_both(float z, float &a, float &d) {
    if (ACT == ACT_NONE) { a = z; d = 1.f; }
    else if (ACT == ACT_RELU) { a = z < 0.f ? 0.f : z; d = z > 0.f ? 1.f : 0.f; }
    else if (ACT == ACT_GELU) {
        const float h = fminf(fabsf(z), FAR_TAIL<OT>), e = exp_half_square(z), tail = normal_tail<OT>(h, e);
        a = fmaf(-h, tail, z < 0.f ? 0.f : z);
        d = fmaf(z * 0.39894228f, e, z < 0.f ? tail : 1.0f - tail);
    } else {
        float s, q;
        sigmoid_pair<OT>(z, s, q);
        if (ACT == ACT_SILU) { a = z * s; d = s * fmaf(z, q, 1.0f); }
        else { a = s; d = s * q; }
    }
}
// The gradient that passes the activation: dy d, of a gated layer's gate dy (u d).  relu is a choice and no product: where it is off, nothing passes, whatever dy is (infinity, NaN); where z is
// not a number, dy does (as torch's relu).
template <int ACT>
__device__ __forceinline__ float through(float dy, float z, float d) {
    if (ACT == ACT_RELU) return z <= 0.f ? 0.f : dy;
    return dy * d;
}
template <int ACT>
__device__ __forceinline__ float through(float dy, float z, float d, float u) {
    if (ACT == ACT_RELU) return z <= 0.f ? 0.f : dy * u;
    return dy * (u * d);
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

// ---- runs of CNT (4, 8 or 16) consecutive elements of a row, `n` of them inside, at any alignment (global memory takes vector accesses at any element; element
// by element the four products of 4 999 x 999 -> 515 f16 in training took 14 us more of 110)
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef int i32x2_any __attribute__((ext_vector_type(2), aligned(2)));
template <int DT, int CNT>
__device__ __forceinline__ void load_run(const uint8_t *p, int64_t n, float (&v)[CNT]) {
    constexpr int EB = Elem<DT>::B;
    if (n >= CNT) {
        uint32_t w[CNT * EB / 4];
        if (CNT * EB >= 16) {
#pragma unroll
            for (int i = 0; i < CNT * EB / 16; ++i) { const i32x4 t = reinterpret_cast<const i32x4_any *>(p)[i]; __builtin_memcpy(&w[4 * i], &t, 16); }
        } else { const i32x2_any t = *reinterpret_cast<const i32x2_any *>(p); w[0] = t.x; w[1] = t.y; }
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
template <int DT>
__device__ __forceinline__ void unpack8(const i32x4 (&r)[Elem<DT>::B / 2], float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (DT == W3D_DTYPE_F32) v[i] = __int_as_float(r[i / 4 * (Elem<DT>::B / 4)][i % 4]);
        else {
            const uint32_t w = (uint32_t)r[0][i / 2];
            if (DT == W3D_DTYPE_BF16) v[i] = (i & 1) ? __uint_as_float(w & 0xffff0000u) : __uint_as_float(w << 16);
            else v[i] = f16_to_f32((uint16_t)(w >> (16 * (i & 1))));
        }
    }
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {                                  // two 16-bit elements, round to nearest even, in one instruction
    const f32x2 v = {a, b};
    if (DT == W3D_DTYPE_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int DT, int CNT>
__device__ __forceinline__ void store_run(uint8_t *p, int64_t n, const float (&v)[CNT]) {
    constexpr int EB = Elem<DT>::B;
    if (n >= CNT) {
        uint32_t w[CNT * EB / 4];
#pragma unroll
        for (int i = 0; i < CNT * EB / 4; ++i) {
            if (DT == W3D_DTYPE_F32) w[i] = __float_as_uint(v[i]);
            else w[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
        }
        if (CNT * EB >= 16) {
#pragma unroll
            for (int i = 0; i < CNT * EB / 16; ++i) { i32x4 t; __builtin_memcpy(&t, &w[4 * i], 16); reinterpret_cast<i32x4_any *>(p)[i] = t; }
        } else *reinterpret_cast<i32x2_any *>(p) = i32x2_any{(int)w[0], (int)w[1]};
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
template <int LAY, int ROWS, int EB, int NT>
struct Stage {
    static constexpr int BYTES = ROWS * SLAB, PIECES = BYTES / 16 / NT, KPS = SLAB / EB;      // KPS: contraction elements per slab
    static constexpr int CPR = LAY == K_ROWS ? SLAB / 16 : ROWS * EB / 16;                     // chunks per LDS row
    static_assert(BYTES % (16 * NT) == 0, "whole pieces");

    // permutation of the 16-byte chunks of an LDS row.  K_ROWS: 8 lanes read the same chunk of 8 neighbouring rows.  M_ROWS, 16 bits: a transposing read takes four
    // consecutive k per 16 lanes and parts 8 k apart; f32: k and k + 4 share a read's halves.
    static __device__ __forceinline__ int swizzle(int row) {
        if (LAY == K_ROWS) return row & 7;
        if (EB == 4) return ((row >> 2) & 1) << 2;
        return ((row & 3) | (CPR >= 16 ? ((row >> 3) & 1) << 2 : 0)) << 1;                      // (rows of 64 elements are 8 chunks)
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
    // fp8: both chunks of the slab are one operand of 32 bytes a lane; the rows' scales are applied to the f32 sums in the epilogue, the instruction's own are 1.  The instruction cuts the products of eight
    // consecutive contraction elements, towards zero, at 2^-13 of 2^(the largest sum of two exponents; a subnormal's is -6) before it adds them (in f32 from there on): at most 7 2^-13 of that for every eight, 2^-16 .. 2^-20 of the sum of magnitudes
    // for normal rows of 64 .. 16 384, up to 2^-10 for rows that span e4m3's whole range.  The price of twice the 16-bit rate: products as bf16 ones would be whole.
    if (s) return c;
    i32x8 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = w[0][i]; a[4 + i] = w[1][i]; b[i] = x[0][i]; b[4 + i] = x[1][i]; }
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 127, 0, 127);
}

// ---- what becomes of a wave's accumulators.  MS: rows of the matrix instruction (16 or 32): a lane holds groups of four consecutive n of one row m.  They go through a patch of LDS that the
// wave has to itself, ROWS rows at a time and in f32, and come back as runs of 8 n: 8 (gated: 4) lanes hold a row's 64 (32) columns, so that every load and store of the epilogue is whole
// 128-byte (64-byte) pieces of a row.  (Straight from the accumulators a store writes 16-byte pieces of 16 rows: 14 us per 256 x 256 tile instead of 8.)
// 16 rows at a time, unrolled (the accumulators cannot be indexed at run time): 55 us for 65536 x 256 -> 1024 where 64 rows and a loop take 64.  Gradients take up to 64 rows and loop over
// them a few passes at a time: unrolled as a whole, derivative, dy and column sums spill.
// What the epilogue reads (residual, dy) is loaded AHEAD passes early: a pass is a fraction of the memory's latency.
// VEC: rows of C (and of residual and dy) are whole, aligned runs of 8: a run is inside or outside, and there is no path by element (unrolled as often as here it costs registers: spills).
template <int DT, int EPI, int BM, int BN, int WM, int WN, int MS, bool VEC>
struct Out {
    static constexpr int EB = Elem<DT>::B;
    static constexpr bool GATED = EPI == EPI_GATED || EPI == EPI_GATED_BWD, BWD = EPI == EPI_LINEAR_BWD || EPI == EPI_GATED_BWD;
    static constexpr int PARTS = GATED ? 2 : 1, BNP = BN / PARTS;                              // a gated tile is BN / 2 columns of each half: rows [0, BN/2) of the W slab gate, the rest up
    static constexpr int FM = BM / WM / MS, FN = BN / WN / MS, FP = FN / PARTS;
    static constexpr int COLS = BN / WN, PCOLS = COLS / PARTS, LPR = PCOLS / 8, RPP = 64 / LPR;      // lanes per row, rows per pass
    static constexpr int ROWS = !BWD ? 16 : BM / WM < 64 ? BM / WM : 64, CHUNKS = BM / WM / ROWS, PASSES = ROWS / RPP, ALL = CHUNKS * PASSES, AHEAD = PASSES < 2 ? 1 : ALL < 4 || GATED ? 2 : 4;
    static constexpr int TURN = BWD ? AHEAD : PASSES;                                          // passes unrolled at a time
    static constexpr int PATCH = ROWS * COLS * 4;
    static_assert(COLS == 64 && BM / WM % ROWS == 0 && ROWS % 16 == 0 && PASSES % TURN == 0 && TURN % AHEAD == 0 || !BWD, "a patch row is 16 chunks");
    typedef typename std::conditional<MS == 32, f32x16, f32x4>::type acc_t;
    typedef acc_t Acc[FM][FN];

    static __device__ __forceinline__ int w_row(int wn, int f, int lane) { return (f / FP) * BNP + wn * PCOLS + MS * (f % FP) + (lane & (MS - 1)); }     // tile row of the lane's operand row
    static __device__ __forceinline__ int x_row(int wm, int f, int lane) { return wm * (BM / WM) + MS * f + (lane & (MS - 1)); }

    // 16 rows of the wave (step 0, 1, ..) into the patch; chunks of 16 bytes are permuted by XOR with the row: lanes that write (read) neighbouring rows touch different banks
    static __device__ __forceinline__ void put(const Acc &acc, int step, int lane, uint8_t *patch) {
        const int row = lane & 15;
        if (MS == 32 && ((lane >> 4) & 1) != (step & 1)) return;                               // half of a 32-row fragment
        const int i = step / (MS / 16);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int b = 0; b < MS * MS / 256; ++b) {
                const int chunk = MS == 32 ? 8 * j + 2 * b + (lane >> 5) : 4 * j + (lane >> 4);
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * b + e];
                *reinterpret_cast<f32x4 *>(patch + (16 * (step % (ROWS / 16)) + row) * (COLS * 4) + ((chunk ^ row) << 4)) = v;
            }
    }
    static __device__ __forceinline__ void get(const uint8_t *patch, int pass, int part, int lane, float (&v)[8]) {
        const int row = pass * RPP + lane / LPR, first = part * (PCOLS / 4) + 2 * (lane % LPR);
        f32x4 t[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) t[c] = *reinterpret_cast<const f32x4 *>(patch + row * (COLS * 4) + (((first + c) ^ (row & 15)) << 4));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = t[e / 4][e % 4];
    }
    // f(pass of the patch, row of the wave, is the row inside C, 8 elements of src, byte offset of the row's run past the wave's first row of dst) for every row this lane finishes.
    // SRC: there is a src, [M][N] of type OT; n: the lane's first column, c0: the wave's; ld: bytes from row to row of dst, DB: bytes of its elements.  (SRC at compile time: a load that may
    // be in flight makes the passes of a tile without one wait for their own stores.)
    template <int OT, int DB, bool SRC, typename F>
    static __device__ __forceinline__ void each_row(const GemmArgs &a, const Acc &acc, const uint8_t *src, int64_t ld, int64_t m0, int64_t n, int64_t c0, int wm, int lane, uint8_t *patch, F f) {
        constexpr int OB = Elem<OT>::B, RAW = OB * 8 / 16;
        const int64_t mw = m0 + wm * (BM / WM), left64 = a.M - mw - lane / LPR;
        const int left = (int)(left64 < BM ? left64 < -BM ? -BM : left64 : BM);                // rows from the lane's first that exist (<= 0: none)
        const bool any = a.M > mw && a.N > c0;                                                 // the wave's corner is inside C (uniform)
        const bool fast = VEC || n + 8 <= a.N;
        i32x4 ring[AHEAD][RAW];                                                                // src of the next passes (indexed at compile time: a rotation would wait for the loads)
        const uint32_t src_ld = (uint32_t)(a.N * OB);
        const uint8_t *from = src + mw * a.N * OB + c0 * OB;                                   // the wave's corner: uniform, lanes add 32 bits
        // VEC: loads are unconditional (the compiler counts them): rows and columns outside C read the tile's last row and the wave's first columns
        const uint32_t col = VEC && n >= a.N ? 0u : (uint32_t)(n - c0) * OB;
        auto fetch = [&](int q, int slot) {
            const int r = VEC ? (q * RPP < left ? q * RPP : left - 1) : q * RPP;
            if (VEC ? any : fast && r < left)
#pragma unroll
                for (int k = 0; k < RAW; ++k) ring[slot][k] = reinterpret_cast<const i32x4_any *>(from + (uint32_t)(lane / LPR + r) * src_ld + col)[k];
        };
        if (SRC)
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) fetch(k, k);
        uint32_t off = (uint32_t)(lane / LPR) * (uint32_t)ld + (uint32_t)(n - c0) * DB;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
            for (int s = 0; s < ROWS / 16; ++s) put(acc, c * (ROWS / 16) + s, lane, patch);
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int p0 = 0; p0 < PASSES; p0 += TURN)
#pragma unroll
                for (int k = 0; k < TURN; ++k) {
                    const int p = p0 + k, q = c * PASSES + p, row = q * RPP;
                    float t[8] = {};
                    if (SRC) {
                        if (fast) unpack8<OT>(ring[(c * PASSES + k) % AHEAD], t);
                        else if (!VEC && row < left) load_run<OT, 8>(from + (uint32_t)(lane / LPR + row) * src_ld + (uint32_t)(n - c0) * OB, a.N - n, t);
                        if (q + AHEAD < ALL) fetch(q + AHEAD, (c * PASSES + k) % AHEAD);
                    }
                    f(p, row, row < left, t, off);
                    off += RPP * (uint32_t)ld;
                }
            __builtin_amdgcn_wave_barrier();
        }
    }

    static __device__ __forceinline__ void epilogue(const GemmArgs &a, const Acc &acc, int64_t m0, int64_t n0, int slice, int tm, int wm, int wn, int lane, bool z1, uint8_t *patch) {
        const int64_t c0 = n0 + wn * PCOLS, n = c0 + 8 * (lane % LPR);
        if (a.slices > 1) {
            const int64_t z = (int64_t)(z1 ? a.slices : 0) + slice, ld = a.part_ld * 4;
            uint8_t *out = (uint8_t *)a.part + (z * a.M + m0 + wm * (BM / WM)) * ld + c0 * 4;
            each_row<W3D_DTYPE_F32, 4, false>(a, acc, nullptr, ld, m0, n, c0, wm, lane, patch, [&](int pass, int, bool live, float (&)[8], uint32_t off) {
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    float v[8];
                    get(patch, pass, p, lane, v);
                    if (live && n < a.N) store_run<W3D_DTYPE_F32, 8>(out + off + p * (ld / 2), VEC ? 8 : a.N - n, v);
                }
            });
            return;
        }
        // (fp8 rows: the output is bf16 or f16)
        if constexpr (DT == W3D_DTYPE_FP8_E4M3) {
            if (a.out_dt == W3D_DTYPE_BF16) finish<W3D_DTYPE_BF16>(a, acc, m0, n, c0, tm, wm, lane, z1, patch);
            else finish<W3D_DTYPE_F16>(a, acc, m0, n, c0, tm, wm, lane, z1, patch);
        } else finish<DT>(a, acc, m0, n, c0, tm, wm, lane, z1, patch);
    }

    template <int OT>
    static __device__ __forceinline__ void finish(const GemmArgs &a, const Acc &acc, int64_t m0, int64_t n, int64_t col0, int tm, int wm, int lane, bool z1, uint8_t *patch) {
        constexpr int OB = Elem<OT>::B;
        const int64_t mw = m0 + wm * (BM / WM);
        uint8_t *out = (EPI == EPI_STORE && z1 ? a.out2 : a.out) + mw * a.ld_out + col0 * OB;
        if constexpr (EPI == EPI_STORE) {
            each_row<OT, OB, false>(a, acc, nullptr, a.ld_out, m0, n, col0, wm, lane, patch, [&](int pass, int, bool live, float (&)[8], uint32_t off) {
                float v[8];
                get(patch, pass, 0, lane, v);
                if (live && n < a.N) store_run<OT, 8>(out + off, VEC ? 8 : a.N - n, v);
            });
            return;
        }
        float b0[8], b1[8], c0[8], c1[8];
        int s0[8], s1[8];                                // fp8: the sums are scaled by 2^(row exponent of x + row exponent of w), exactly
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            b0[e] = bias_at<OT>(a.bias, a.bias_f32, n + e, a.N);
            b1[e] = GATED ? bias_at<OT>(a.bias2, a.bias_f32, n + e, a.N) : 0.f;
            c0[e] = c1[e] = 0.f;
            s0[e] = s1[e] = 0;
            if (DT == W3D_DTYPE_FP8_E4M3 && n + e < a.N) { s0[e] = a.ws[n + e] - 254; if (GATED) s1[e] = a.ws2[n + e] - 254; }
        }
        const int64_t pad = (EPI == EPI_GATED_BWD ? a.half_out : a.ld_out) / OB - n;           // BWD: columns of the padded row from here, a multiple of 8 (16 bits) or 4
        auto row = [&](auto act_c, auto src_c, int pass, int r, bool live, float (&t)[8], uint32_t off) {
            float v[8], u[8];
            get(patch, pass, 0, lane, v);
            if (GATED) get(patch, pass, 1, lane, u);
            if (DT == W3D_DTYPE_FP8_E4M3) {
                const int xs = live ? a.xs[mw + lane / LPR + r] : 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) { v[e] = __builtin_ldexpf(v[e], xs + s0[e]); if (GATED) u[e] = __builtin_ldexpf(u[e], xs + s1[e]); }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[e] += b0[e]; if (GATED) u[e] += b1[e]; }
            if (DT != W3D_DTYPE_FP8_E4M3 && !BWD && a.z && live && n < a.N) {
                float *z = a.z + (mw + lane / LPR + r) * a.part_ld + n;
                store_run<W3D_DTYPE_F32, 8>((uint8_t *)z, a.N - n, v);
                if (GATED) store_run<W3D_DTYPE_F32, 8>((uint8_t *)(z + a.part_ld / 2), a.N - n, u);
            }
            auto apply = [&](auto act) {
                constexpr int ACT = decltype(act)::value;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (!BWD) {
                        v[e] = act_fwd<ACT, OT>(v[e]);
                        if (EPI == EPI_GATED) v[e] *= u[e];
                        else if (decltype(src_c)::value) v[e] += t[e];
                    } else {
                        float f, d;
                        act_both<ACT, OT>(v[e], f, d);
                        if (EPI == EPI_LINEAR_BWD) v[e] = through<ACT>(t[e], v[e], d);
                        else { v[e] = through<ACT>(t[e], v[e], d, u[e]); u[e] = t[e] * f; }
                    }
                }
            };
            if constexpr (BWD) with_act(a.act, apply);                                         // (per row: five copies of the whole would spill)
            else apply(act_c);
            // the padding columns of dz are part of the contraction of dx: zeros, also where the row's z or dy is not finite (VEC: a run is inside or outside as a whole, and linear rows have none)
            if constexpr (BWD && (GATED || !VEC))
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool in = n + (VEC ? 0 : e) < a.N;
                    v[e] = in ? v[e] : 0.f;
                    if (GATED) u[e] = in ? u[e] : 0.f;
                }
            if (BWD)
#pragma unroll
                for (int e = 0; e < 8; ++e) { c0[e] += live ? v[e] : 0.f; if (GATED) c1[e] += live ? u[e] : 0.f; }      // column sums in f32, before the rounding
            if (live && (BWD ? pad > 0 : n < a.N)) {
                store_run<OT, 8>(out + off, VEC ? 8 : BWD ? pad : a.N - n, v);
                if (EPI == EPI_GATED_BWD) store_run<OT, 8>(out + off + a.half_out, VEC ? 8 : pad, u);
            }
        };
        auto rows = [&](auto act_c, auto src_c) {
            each_row<OT, OB, decltype(src_c)::value>(a, acc, BWD ? a.dy : a.res, a.ld_out, m0, n, col0, wm, lane, patch,
                                                     [&](int pass, int r, bool live, float (&t)[8], uint32_t off) { row(act_c, src_c, pass, r, live, t, off); });
        };
        if constexpr (BWD) rows(std::integral_constant<int, ACT_NONE>(), std::true_type());
        else if (EPI == EPI_LINEAR && a.res) with_act(a.act, [&](auto act_c) { rows(act_c, std::true_type()); });
        else with_act(a.act, [&](auto act_c) { rows(act_c, std::false_type()); });
        if (BWD && a.colsum) {
            // lanes l, l + LPR, ... hold the same columns
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int o = LPR; o < 64; o *= 2) {
                    c0[e] += __shfl_xor(c0[e], o, 64);
                    if (GATED) c1[e] += __shfl_xor(c1[e], o, 64);
                }
            if (lane < LPR) {
                float *o = a.colsum + ((int64_t)tm * WM + wm) * a.colsum_ld + n;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n + e < a.N) { o[e] = c0[e]; if (GATED) o[a.colsum_ld / 2 + e] = c1[e]; }
            }
        }
    }
};

// tile of a block: consecutive blocks go round the 8 XCDs, so block b works on place (b % 8) * (tiles / 8) + b / 8 of an order in which neighbours share operand rows (each XCD's L2 then
// serves a compact patch of C); the order runs down groups of 8 tile rows
__device__ __forceinline__ void tile_of_block(const GemmArgs &a, int &slice, int &tm, int &tn) {
    const int tiles = a.tiles_m * a.tiles_n, total = tiles * a.slices;
    const int q = total / 8, r = total % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    int id = xcd * q + min(xcd, r) + at;
    slice = id / tiles;
    id -= slice * tiles;
    const int span = 8 * a.tiles_n, g = id / span, first = g * 8, rows = min(8, a.tiles_m - first), in = id - g * span;
    tm = first + in % rows;
    tn = in / rows;
}

template <int DT, int LX, int LW, int EPI, int BM, int BN, int WM, int WN>
struct Gemm {
    static constexpr int NT = WM * WN * 64, EB = Elem<DT>::B, KPS = SLAB / EB;
    typedef Out<DT, EPI, BM, BN, WM, WN, 16, false> O;
    static constexpr int FM = O::FM, FN = O::FN, BNP = O::BNP;
    static constexpr bool GATED = O::GATED;
    typedef Stage<LX, BM, EB, NT> SX;
    typedef Stage<LW, BN, EB, NT> SW;
    static constexpr int BUF = SX::BYTES + SW::BYTES, LDS_BYTES = 2 * BUF;
    static_assert(!GATED || LW == K_ROWS, "gated products read the weights by rows");
    static_assert(!GATED || SW::PIECES % 2 == 0, "a piece of the W slab belongs to one half");

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
    static __device__ __forceinline__ void run(const GemmArgs &a, uint8_t *smem) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
        int slice, tm, tn;
        tile_of_block(a, slice, tm, tn);
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

        typename O::Acc acc;
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
        if (s_begin < s_end) dma(s_begin, smem);
        int cur = 0;
        for (int64_t t = s_begin; t < s_end; ++t, cur ^= 1) {
            __syncthreads();                             // slab t has landed (every wave drains its own LDS-DMA), and nobody reads the other buffer any more
            const uint8_t *bx = smem + cur * BUF, *bw = bx + SX::BYTES;
            i32x4 xf[FM][2], wf[FN][2];
#pragma unroll
            for (int j = 0; j < FN; ++j) frag<SW, LW>(bw, O::w_row(wn, j, lane), wn * FN + j, lane, wf[j]);
#pragma unroll
            for (int i = 0; i < FM; ++i) frag<SX, LX>(bx, O::x_row(wm, i, lane), wm * FM + i, lane, xf[i]);
            if (t + 1 < s_end) dma(t + 1, smem + (cur ^ 1) * BUF);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mfma_step<DT>(wf[j], xf[i], s, acc[i][j]);
        }
        __syncthreads();                                 // the slabs' LDS becomes the waves' patches
        O::epilogue(a, acc, m0, n0, slice, tm, wm, wn, lane, z1, smem + wave * O::PATCH);
    }
};

template <int DT, int LX, int LW, int EPI, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 1) void gemm_kernel(GemmArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    Gemm<DT, LX, LW, EPI, BM, BN, WM, WN>::run(a, smem);
}

}  // namespace
