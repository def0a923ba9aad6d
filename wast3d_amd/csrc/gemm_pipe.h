// The large tile: 256 x 256 outputs, 8 waves, 16-bit or fp8 operands and outputs whose rows are aligned multiples of 16 bytes.  (gemm_tile.h: operand orders, output layout, epilogues.)
//
// Why this shape.  A 256 x 256 tile moves 32 KB from L2 per 64 bytes of contraction, 32 B per clock and CU at the full matrix rate; 128 x 128 tiles would need twice that, more than the
// L2s give (8192^3 forward with 128 x 128: 0.66 PFLOP/s).  Measured at 8192^3, bf16: forward 843 us (1.30 PFLOP/s), dx 792 (1.39), dW 878 (1.25); fp8, 8192 rows 4096 -> 8192: 2.28 PFLOP/s.
// At short contractions the start and the epilogue of a tile (9 - 13 us for 256 blocks in step, HBM writes) are not hidden: 16384 rows 1024 -> 4096 143 us against 101 of products.  A wave owns 128 x 64 outputs: 128 accumulator registers, 12 KB of fragments from LDS for 512 cycles of matrix instructions.
//
// Schedule.  The two waves of a SIMD belong to two groups that run half a turn apart: while one group issues its 32 matrix instructions, the other reads its next fragments from LDS; s_barrier
// swaps them.  So the matrix unit always has one wave that only computes, and LDS latency is never waited for by it.  The transfers of a slab three ahead are issued between the matrix
// instructions (their issue takes as long as the LDS reads and would be added to them: 909 -> 813 us at 8192^3, dx).  Ring of four slabs of 64 bytes of contraction (4 x 32 KB).
//   turn t of a wave:  read fragments of slab t | wait until its own part of slab t + 1 has landed | barrier |
//                      matrix instructions of slab t, transfers of slab t + 3 (into the buffer of t - 1, which both groups have read) | barrier
// The LDS reads are one asm block that ends with its own wait: as compiler-visible loads they would be made to wait for the transfers in flight (which might alias), and an output register
// must not be free before its data arrives.
#pragma once
#include "gemm_tile.h"

namespace {

constexpr int PIPE_SLAB = 64, PIPE_RING = 4;
#define W3D_WAIT_VM(n) (((n) & 15) | (((n) >> 4) << 14) | 0x0f70)      // s_waitcnt vmcnt(n), the other counters unwaited

template <int DT, int LX, int LW, int EPI>
struct Pipe {
    static constexpr int BM = 256, BN = 256, WM = 2, WN = 4, NT = 512, EB = Elem<DT>::B, KPS = PIPE_SLAB / EB, MS = DT == W3D_DTYPE_FP8_E4M3 ? 32 : 16;
    static_assert(EB <= 2 && (EB == 2 || (LX == K_ROWS && LW == K_ROWS)), "16-bit operands in any order, fp8 rows of contiguous k");
    typedef Out<DT, EPI, BM, BN, WM, WN, MS, true> O;
    static constexpr int FM = O::FM, FN = O::FN, BNP = O::BNP, SIDE = 256 * PIPE_SLAB, BUF = 2 * SIDE, LDS_BYTES = PIPE_RING * BUF;
    static_assert(LDS_BYTES >= WM * WN * O::PATCH, "the slabs' LDS becomes the waves' patches");
    static constexpr bool GATED = O::GATED;

    // 16-byte chunk permutation inside an LDS row.  K_ROWS (64-byte rows): 8 neighbouring lanes read 8 rows, two of which share the banks of 128 bytes.  M_ROWS (512-byte rows of one k):
    // the four k of one 16-lane part of a transposing read, and those of two parts (8 k apart), go to different 32-byte pieces of 256 bytes.
    static __device__ __forceinline__ int swizzle_k(int row) { return (row >> 1) & 3; }

    struct Mover {                            // one side's transfers: two 16-byte pieces per lane and slab
        const uint8_t *base, *base2;          // base2: from slab `swap` on (dx of a gated layer)
        int64_t step;                         // bytes per slab
        uint32_t off[2];
        int k_of[2];                          // first contraction element of the piece inside the slab
    };
    template <int LAY>
    static __device__ __forceinline__ void init(Mover &m, const uint8_t *base, int64_t ld, int64_t rows, int tid) {
        m.base = m.base2 = base;
        m.step = LAY == K_ROWS ? PIPE_SLAB : KPS * ld;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int p = i * NT + tid;
            if (LAY == K_ROWS) {
                const int row = p >> 2, chunk = (p & 3) ^ swizzle_k(row);
                m.k_of[i] = chunk * (16 / EB);
                m.off[i] = row < rows ? (uint32_t)row * (uint32_t)ld + (uint32_t)chunk * 16u : OUT_OF_RANGE;
            } else {
                const int row = p >> 5, chunk = (p & 31) ^ (((row & 3) | ((row >> 3) & 1) << 2) << 1);
                m.k_of[i] = row;
                m.off[i] = (int64_t)chunk * 8 < rows ? (uint32_t)row * (uint32_t)ld + (uint32_t)chunk * 16u : OUT_OF_RANGE;
            }
        }
    }
    static __device__ __forceinline__ void issue(const uint8_t *base, uint32_t off, uint8_t *lds) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, 0x7fffffff, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t)(lds_t)lds, 16, (int)off, 0, 0, 0);
    }

    static __device__ __forceinline__ uint32_t lds_offset(const void *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p; }

    static __device__ __forceinline__ void run(const GemmArgs &a, uint8_t *smem) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave >> 2;          // waves w and w + 4 share a SIMD
        const int wm = wave >> 2, wn = wave & 3;
        int slice, tm, tn;
        tile_of_block(a, slice, tm, tn);
        const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BNP;
        const int64_t slabs = (a.K + KPS - 1) / KPS;
        const int64_t t0 = slabs * slice / a.slices, t1 = slabs * (slice + 1) / a.slices;
        const bool z1 = blockIdx.z != 0;

        Mover mx, mw;
        init<LX>(mx, a.x + (z1 ? a.z_x : 0) + (LX == K_ROWS ? m0 * a.ldx : m0 * EB), a.ldx, a.M - m0, tid);
        const int64_t w_at = LW == K_ROWS ? n0 * a.ldw : n0 * EB;
        init<LW>(mw, a.w + w_at, a.ldw, GATED ? min(a.N - n0, (int64_t)BNP) : a.N - n0, tid);
        if (GATED) {                                                                           // rows 128.. of the slab are the second half's: pieces i = 1
            mw.base2 = a.w2 + w_at;
            const int row = (NT + tid) >> 2;
            mw.off[1] = row - BNP < a.N - n0 ? (uint32_t)(row - BNP) * (uint32_t)a.ldw + (uint32_t)((tid & 3) ^ swizzle_k(row)) * 16u : OUT_OF_RANGE;
        } else if (a.k_split > 0) mw.base2 = a.w2 + w_at - a.k_split * a.ldw;
        const int64_t wk = LW == M_ROWS ? a.w_rows : a.K;                                      // contraction elements of W that exist (per stacked matrix)
        const bool split = LW == M_ROWS && !GATED && a.k_split > 0;

        // transfers of slab t: addresses, then the four issues.  Slabs past the contraction's end are all out of range (nothing is read), so that every turn is alike.
        const uint8_t *bx, *bw, *bw1;
        uint32_t off[4];
        uint8_t *to;
        auto prepare = [&](int64_t t) {
            const int64_t k0 = t * KPS;
            const bool second = split && k0 >= a.k_split;
            const int64_t xl64 = a.K - k0, wl64 = (second ? a.k_split + wk : wk) - k0;
            const int xl = (int)(xl64 < KPS ? xl64 : KPS), wl = (int)(wl64 < KPS ? wl64 : KPS);
            bx = mx.base + t * mx.step;
            bw = (second ? mw.base2 : mw.base) + t * mw.step;
            bw1 = GATED ? mw.base2 + t * mw.step : bw;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                off[i] = mx.k_of[i] < xl ? mx.off[i] : OUT_OF_RANGE;
                off[2 + i] = mw.k_of[i] < wl ? mw.off[i] : OUT_OF_RANGE;
            }
            to = smem + (int)(t & (PIPE_RING - 1)) * BUF + wave * 1024;
        };
        auto fire = [&]() {
            issue(bx, off[0], to);
            issue(bx, off[1], to + NT * 16);
            issue(bw, off[2], to + SIDE);
            issue(bw1, off[3], to + SIDE + NT * 16);
        };

        typename O::Acc acc;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < MS * MS / 64; ++e) acc[i][j][e] = 0.f;

        // a lane's read addresses inside a buffer
        const uint32_t lds0 = lds_offset(smem);
        uint32_t ax[4], aw[4];
        {
            const int j = lane & 15, q = lane >> 4;
            if (LX == K_ROWS) {
                const int row = O::x_row(wm, 0, lane), sw = swizzle_k(row);
                if (MS == 16) ax[0] = lds0 + row * PIPE_SLAB + ((q ^ sw) << 4);
                else { ax[0] = lds0 + row * PIPE_SLAB + (((lane >> 5) ^ sw) << 4); ax[1] = ax[0] ^ 32u; }
            } else {
#pragma unroll
                for (int f = 0; f < 4; ++f) ax[f] = lds0 + (8 * q + (j >> 2)) * 512 + wm * 256 + ((q & 1) << 7) + (((f ^ (j >> 2)) & 3) << 5) + (j & 3) * 8;
            }
            if (LW == K_ROWS) {
                const int row = O::w_row(wn, 0, lane), sw = swizzle_k(row);
                if (MS == 16) aw[0] = lds0 + SIDE + row * PIPE_SLAB + ((q ^ sw) << 4);
                else { aw[0] = lds0 + SIDE + row * PIPE_SLAB + (((lane >> 5) ^ sw) << 4); aw[1] = aw[0] ^ 32u; }
            } else {
#pragma unroll
                for (int f = 0; f < 4; ++f) aw[f] = lds0 + SIDE + (8 * q + (j >> 2)) * 512 + (wn >> 1) * 256 + (((wn ^ q) & 1) << 7) + (((f ^ (j >> 2)) & 3) << 5) + (j & 3) * 8;
            }
        }

#pragma unroll
        for (int i = 0; i < 3; ++i) { prepare(t0 + i); fire(); }
        __builtin_amdgcn_s_waitcnt(W3D_WAIT_VM(8));
        __builtin_amdgcn_s_barrier();
        if (group == 1) __builtin_amdgcn_s_barrier();                                          // half a turn behind
        for (int64_t t = t0; t < t1; ++t) {
            const uint32_t at = (uint32_t)(t & (PIPE_RING - 1)) * BUF;
            i32x4 xf[8], wf[4];                                                                // fp8: pairs of them are one operand
            read_side<LX, 8>(ax, at, xf);
            read_side<LW, 4>(aw, at, wf);
            prepare(t + 3);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(W3D_WAIT_VM(4));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            fire();
            if constexpr (MS == 16) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        if (DT == W3D_DTYPE_BF16)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wf[j]), __builtin_bit_cast(bf16x8, xf[i]), acc[i][j], 0, 0, 0);
                        else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, wf[j]), __builtin_bit_cast(f16x8, xf[i]), acc[i][j], 0, 0, 0);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join8(wf[2 * j], wf[2 * j + 1]), join8(xf[2 * i], xf[2 * i + 1]), acc[i][j], 0, 0, 0, 127, 0, 127);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, MS == 16 ? 6 : 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, MS == 16 ? 8 : 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_s_barrier();
        }
        __builtin_amdgcn_s_waitcnt(W3D_WAIT_VM(0));
        __builtin_amdgcn_s_barrier();                                                          // nothing is in flight into the slabs' LDS, which becomes the waves' patches
        if (group == 0) __builtin_amdgcn_s_barrier();                                          // as many barriers as the other group
        O::epilogue(a, acc, m0, n0, slice, tm, wm, wn, lane, z1, smem + wave * O::PATCH);
    }
    static __device__ __forceinline__ i32x8 join8(i32x4 a, i32x4 b) {
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }

    // N fragments of a side: K_ROWS, 16 x 16: 16 tile rows apart; 32 x 32: two chunks per fragment, fragments 32 rows apart; M_ROWS: two transposing reads
    template <int LAY, int N>
    static __device__ __forceinline__ void read_side(const uint32_t (&a)[4], uint32_t at, i32x4 (&v)[N]) {
        if constexpr (LAY == K_ROWS && MS == 16 && N == 8) {
            asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:1024\n\tds_read_b128 %2, %8 offset:2048\n\tds_read_b128 %3, %8 offset:0xc00\n\t"
                         "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %8 offset:5120\n\tds_read_b128 %6, %8 offset:6144\n\tds_read_b128 %7, %8 offset:7168\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]) : "v"(a[0] + at) : "memory");
        } else if constexpr (LAY == K_ROWS && MS == 16) {
            constexpr int D1 = 1024, D2 = GATED ? O::BNP * PIPE_SLAB : 2048, D3 = D1 + D2;         // gated: fragments 2, 3 are the second half's
            asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(a[0] + at), "n"(D1), "n"(D2), "n"(D3) : "memory");
        } else if constexpr (LAY == K_ROWS && N == 8) {
            asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %8 offset:2048\n\tds_read_b128 %3, %9 offset:2048\n\t"
                         "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %8 offset:6144\n\tds_read_b128 %7, %9 offset:6144\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]) : "v"(a[0] + at), "v"(a[1] + at) : "memory");
        } else if constexpr (LAY == K_ROWS) {
            constexpr int D = GATED ? O::BNP * PIPE_SLAB : 2048;
            asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(a[0] + at), "v"(a[1] + at), "n"(D) : "memory");
        } else {
            typedef int i32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int g = 0; g < N / 4; ++g) {                                                  // fragments 4 g .. + 3: the other 128 bytes of a 256-byte piece of the row
                const uint32_t flip = g << 7;
                i32x2 l[4], h[4];
                asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\tds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                             "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\tds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                             "s_waitcnt lgkmcnt(0)"
                             : "=&v"(l[0]), "=&v"(h[0]), "=&v"(l[1]), "=&v"(h[1]), "=&v"(l[2]), "=&v"(h[2]), "=&v"(l[3]), "=&v"(h[3])
                             : "v"((a[0] + at) ^ flip), "v"((a[1] + at) ^ flip), "v"((a[2] + at) ^ flip), "v"((a[3] + at) ^ flip), "n"(0), "n"(2048) : "memory");
#pragma unroll
                for (int f = 0; f < 4; ++f) v[4 * g + f] = __builtin_shufflevector(l[f], h[f], 0, 1, 2, 3);
            }
        }
    }
};

template <int DT, int LX, int LW, int EPI>
__global__ __launch_bounds__(512, 1) void gemm_pipe_kernel(GemmArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    Pipe<DT, LX, LW, EPI>::run(a, smem);
}

}  // namespace
