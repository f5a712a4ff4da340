// gemm_direct.hpp -- the bf16 product's direct-to-LDS kernel on 256 x 256 tiles: its
// device code, shared by gemm.hip's C (+)= op(A) op(B) and the products of other
// files that take the accumulators with an epilogue of their own.
#pragma once

#include "gemm_common.hpp"

namespace agk_gemm {

constexpr int BM = 256, BN = 256;
constexpr int WM = 128, WN = 64;            // the registers an epilogue takes at a time
constexpr int TM = WM / 32, TN = WN / 32;   // as MFMA tiles
constexpr int kStageElems = (BM + BN) * kStride;

// ---- direct-to-LDS kernel -----------------------------------------------------
// Staging without registers: buffer_load_dwordx4 ... lds writes lane l's 16
// bytes to LDS at (wave-uniform base) + 16 * l, so one wave instruction fills
// a contiguous kilobyte of LDS; each lane fetches the global chunk that belongs
// at its position of the swizzled layout.  Rows past M or N are fetched from
// the last valid row (never stored).  The epilogue (store_block behind StoreC, or another
// one) takes the wave's block of C.  K % 64 k at the end of K are staged through registers with
// zeros past K (stage_k_tail) and multiplied before the whole k-tiles.
//
// The same 256 x 256 tile, over 4 waves of 128 x 128 (2 x 2; 4 x 4 MFMA tiles
// per wave, whose 256 accumulator registers live in AGPRs).  K is walked in
// 64-deep tiles through two LDS stages of 64 KiB (32 KiB per operand), filled by
// `buffer_load_dwordx4 ... lds`, so staging takes no registers.  Each operand is
// staged in the layout it has in memory:
// - k-contiguous ([rows][K]): 256 LDS rows of 64 k (128 bytes, 8 XOR-swizzled
//   16-byte chunks: lds_off above); a fragment is one 16-byte read.
// - k-strided (TR; [K][cols], the columns contiguous): 64 LDS rows of one k
//   each, 256 columns (512 bytes, 32 chunks whose 64-byte groups are XOR-
//   swizzled by k % 4: tr_off); a fragment is two ds_read_b64_tr_b16.  Within
//   each 16 lanes that instruction hands lane 4a + b, for e = 0..3, the element
//   at offset b from the address of lane 4e + a (checked on MI355X), so lane s
//   pointing at k0 + s / 4, column c0 + 4 (s % 4) gives lane j the four k
//   k0 .. k0 + 3 of column c0 + j: the MFMA operand layout.  No transposed copy
//   of the operand is made.
// Either way one load instruction moves 1 KiB of whole 128-byte lines, and the
// LDS destination of load j of wave w is the same kilobyte.
//
// Why this shape (measured on MI355X, c5 products):
// - Whole 128-byte rows per load: 32-deep tiles (64 bytes per row) asked L2 for
//   each line twice, half at a time, and the L1's queue of pending misses, not
//   HBM, set the pace (twice hipBLASLt's L2 request count for the same bytes,
//   TCP_TCC_READ_REQ).
// - One wave per SIMD with a 128 x 128 block reads a third fewer LDS bytes per
//   MFMA than two waves of 128 x 64, and its stream of 64 MFMAs per tile has
//   the loads and fragment reads interleaved between them; it was 4-6 % faster
//   than eight waves of 128 x 64 with the same stages.
//
// Schedule of tile t (after the barrier that makes tile t visible and frees the
// other stage): the 16 loads of tile t + 1 go into the other stage, one per
// two MFMAs of the first two substeps; the fragments run one 16-deep substep
// ahead of the MFMAs, so the substep that straddles the barrier (the last of
// tile t - 1) multiplies while tile t's first fragments are read.  At the end
// of the tile each wave waits for its own loads and reads, then the barrier.
constexpr int kDirectThreads = 256;
constexpr int kTrRow = 256;               // bf16 per LDS row of a k-strided operand

// Element offset of column col (a multiple of 4) of k-row k in a k-strided stage.
__device__ __forceinline__ int tr_off(int k, int col) {
    return k * kTrRow + ((((col >> 3) ^ ((k & 3) << 2))) << 3) + (col & 7);
}

struct DirectStage {
    __amdgpu_buffer_rsrc_t ra, rb;  // the tile's A and B (base and size in SGPRs)
    uint32_t oa[8], ob[8];          // byte offset of each lane's chunk, per load
    int step_a, step_b;             // bytes from one 64-deep k-tile to the next
};

// Load j of a wave (j = 0..7) fills kilobyte wave * 8 + j of one operand's half
// of `stage`; the tile's data starts `at` bytes into the operand.
__device__ __forceinline__ void direct_issue_a(const DirectStage& d, uint16_t* stage, int at,
                                               int wave) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(d.ra, (lds_ptr_t)(stage + (wave * 8 + j) * 512),
                                                 16, d.oa[j], at, 0, 0);
}
__device__ __forceinline__ void direct_issue_b(const DirectStage& d, uint16_t* stage, int at,
                                               int wave) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            d.rb, (lds_ptr_t)(stage + BM * BK + (wave * 8 + j) * 512), 16, d.ob[j], at,
            0, 0);
}

// Per-lane byte offsets of one operand's loads.  rows: valid rows (k-contiguous)
// or columns (k-strided) of the tile; ld: leading dimension in elements.
template <bool TR>
__device__ __forceinline__ void direct_offsets(uint32_t (&o)[8], int wave, int lane, int rows,
                                               int64_t ld) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (!TR) {
            const int row = wave * 64 + j * 8 + (lane >> 3);
            const int c = (lane & 7) ^ (row & 7) ^ ((row >> 3) & 7);  // chunk of slot lane % 8
            const int r = row < rows ? row : rows - 1;  // rows past M or N: the last valid row
            o[j] = (static_cast<uint32_t>(r) * static_cast<uint32_t>(ld) + c * 8) * 2;
        } else {
            const int k = wave * 16 + j * 2 + (lane >> 5);
            const int c = (lane & 31) ^ ((k & 3) << 2);  // chunk of slot lane % 32
            const int col = c * 8 < rows ? c * 8 : rows - 8;  // columns past M or N: the last 8
            o[j] = (static_cast<uint32_t>(k) * static_cast<uint32_t>(ld) + col) * 2;
        }
    }
}

// The fragments of one 16-deep substep s (0..3) of a wave: 4 of A (128 rows),
// NB of B (32 NB columns: 4 for the 256 x 256 tile, 2 for the 256 x 128 half
// tiles of a last round).
template <int NB>
struct Frags {
    bf16x8 a[TM], b[NB];
};

// MFMA operand lane l (row or column l % 32, k 8 (l / 32) .. + 7) of block
// column base c0, substep s, from a k-strided stage: two transposing reads of
// four k each.
__device__ __forceinline__ bf16x8 tr_frag(const uint16_t* lds, int c0, int s, int lane) {
    const int g = lane >> 4, sl = lane & 15;
    const int k = s * 16 + (g >> 1) * 8 + (sl >> 2);
    const int col = c0 + (g & 1) * 16 + 4 * (sl & 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(lds + tr_off(k, col)));
    const s16x4 hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(lds + tr_off(k + 4, col)));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// bc: the wave's first B column within the stage.
template <bool A_TR, bool B_TR, int NB>
__device__ __forceinline__ void read_frags(Frags<NB>& f, const uint16_t* stage, int s, int wm,
                                           int bc, int frow, int fk, int lane) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if constexpr (A_TR) f.a[i] = tr_frag(stage, wm * WM + i * 32, s, lane);
        else f.a[i] = lds_frag(stage, wm * WM + i * 32 + frow, s * 16 + fk);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        if constexpr (B_TR) f.b[j] = tr_frag(stage + BM * BK, bc + j * 32, s, lane);
        else f.b[j] = lds_frag(stage + BM * kStride, bc + j * 32 + frow, s * 16 + fk);
    }
}

template <bool F16, int NB>
__device__ __forceinline__ void mfma_sub(const Frags<NB>& f, f32x16 (&acc)[TM][NB]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
            acc[i][j] = mfma16<F16>(f.a[i], f.b[j], acc[i][j]);
}

// Scheduling groups: one load, one fragment read, two MFMAs (AGK_LRM); one
// fragment read, two MFMAs (AGK_RM).  Eight of them cover a substep's 16 MFMAs.
#define AGK_LRM                                         \
    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); \
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); \
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#define AGK_RM                                          \
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); \
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#define AGK_X8(g) g g g g g g g g

// Tile t of nk.  FIRST (tile 0) has no straddling substep; every step loads
// tile t + 1 (the last tile again at the end, into the stage nothing reads
// again).  Entering, f1 holds substep 3 of tile t - 1.  NB = 4: the 256 x 256
// tile, whose substeps interleave one load, one fragment read and two MFMAs;
// NB = 2 (half tiles): the same loads and reads around half the MFMAs, left to
// the compiler's schedule.
#define AGK_SUBSTEP_LRM    \
    if constexpr (NB == 4) { \
        AGK_X8(AGK_LRM)    \
    }
#define AGK_SUBSTEP_RM     \
    if constexpr (NB == 4) { \
        AGK_X8(AGK_RM)     \
    }
template <bool FIRST, bool A_TR, bool B_TR, int NB, class KM>
__device__ __forceinline__ void direct_step(const DirectStage& d, const KM& km,
                                            const uint16_t* cur,
                                            uint16_t* other, int t, int nk,
                                            f32x16 (&acc)[TM][NB], Frags<NB>& f0, Frags<NB>& f1,
                                            int wm, int bc, int frow, int fk, int lane,
                                            int wave) {
    const int tn = t + 1 < nk ? t + 1 : nk - 1;
    direct_issue_a(d, other, km.a(tn, d.step_a), wave);
    read_frags<A_TR, B_TR>(f0, cur, 0, wm, bc, frow, fk, lane);
    if constexpr (!FIRST) {
        mfma_sub<KM::kF16>(f1, acc);
        AGK_SUBSTEP_LRM
    }
    __builtin_amdgcn_sched_barrier(0);
    direct_issue_b(d, other, km.b(tn, d.step_b), wave);
    read_frags<A_TR, B_TR>(f1, cur, 1, wm, bc, frow, fk, lane);
    mfma_sub<KM::kF16>(f0, acc);
    AGK_SUBSTEP_LRM
    __builtin_amdgcn_sched_barrier(0);
    read_frags<A_TR, B_TR>(f0, cur, 2, wm, bc, frow, fk, lane);
    mfma_sub<KM::kF16>(f1, acc);
    AGK_SUBSTEP_RM
    __builtin_amdgcn_sched_barrier(0);
    read_frags<A_TR, B_TR>(f1, cur, 3, wm, bc, frow, fk, lane);
    mfma_sub<KM::kF16>(f0, acc);
    AGK_SUBSTEP_RM
    __builtin_amdgcn_sched_barrier(0);
    // This wave's loads of tile t + 1 have landed and its reads of tile t are
    // done; after the barrier every wave's are.  A bare barrier:
    // __syncthreads()'s fence adds nothing here (vmcnt and lgkmcnt are zero).
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Hands columns [64 H, 64 H + 64) of a wave's 128 x 128 block, whose first column
// is col0 of C, to the epilogue.  H is a template argument, not a loop's: a loop
// over the halves is too large for the compiler to unroll, and acc, indexed by a
// variable, moves to scratch memory.
template <int H, class Epi>
__device__ __forceinline__ void store_half(const f32x16 (&acc)[TM][2 * TN], const Epi& epi,
                                           int row0, int col0, int lane) {
    f32x16 part[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) part[i][j] = acc[i][H * TN + j];
    epi(part, row0, col0, lane);
}

// One tile's k loop and store.  NB = 4: the 256 x 256 tile at (m0, n0), wave
// (wm, wn) owning its 128 x 128 block; NB = 2: the 256 x 128 half of that tile
// starting at column n0 + half_off, wave (wm, wn) owning a 128 x 64 block.
// Both stage the tile's full 256 B columns (the same loads).  TAIL: K is not a
// multiple of 64; the last K % 64 k are multiplied first, staged through
// registers into st1 (which tile 1's loads fill only after it).
template <bool A_TR, bool B_TR, int NB, bool TAIL, class Epi, class KM>
__device__ __forceinline__ void direct_tile(const DirectStage& d, const KM& km, int nk,
                                            uint16_t* st0, uint16_t* st1,
                                            const uint16_t* __restrict__ a0, int64_t lda,
                                            int rows_a, const uint16_t* __restrict__ b0,
                                            int64_t ldb, int rows_b, int K, int m0, int n0,
                                            int half_off, int wm, int wn, int lane, int wave,
                                            const Epi& epi) {
    f32x16 acc[TM][NB];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    const int whole = K / BK;  // >= 1
    const int frow = lane & 31;
    const int fk = (lane >> 5) * 8;  // MFMA operand lanes 32..63 hold k 8..15
    const int bc = half_off + wn * (NB * 32);  // the wave's first B column in the stage
    if constexpr (TAIL) {
        stage_k_tail<A_TR, BM>(st1, a0, lda, rows_a, whole * BK, K);
        stage_k_tail<B_TR, BN>(st1 + BM * BK, b0, ldb, rows_b, whole * BK, K);
    }
    direct_issue_a(d, st0, km.a(0, d.step_a), wave);
    direct_issue_b(d, st0, km.b(0, d.step_b), wave);
    if constexpr (TAIL) {
        stage_barrier<16>();  // the tail's LDS writes, every wave (tile 0 still in flight)
        for (int s = 0; s * 16 < K - whole * BK; ++s) {
            Frags<NB> f;
            read_frags<A_TR, B_TR>(f, st1, s, wm, bc, frow, fk, lane);
            mfma_sub<KM::kF16>(f, acc);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Frags<NB> f0, f1;
    direct_step<true, A_TR, B_TR>(d, km, st0, st1, 0, nk, acc, f0, f1, wm, bc, frow, fk, lane, wave);
    int t = 1;
    for (; t + 1 < nk; t += 2) {
        direct_step<false, A_TR, B_TR>(d, km, st1, st0, t, nk, acc, f0, f1, wm, bc, frow, fk, lane,
                                       wave);
        direct_step<false, A_TR, B_TR>(d, km, st0, st1, t + 1, nk, acc, f0, f1, wm, bc, frow, fk,
                                       lane, wave);
    }
    if (t < nk)
        direct_step<false, A_TR, B_TR>(d, km, st1, st0, t, nk, acc, f0, f1, wm, bc, frow, fk, lane,
                                       wave);
    mfma_sub<KM::kF16>(f1, acc);  // substep 3 of the last tile

    if constexpr (NB == 4) {
        // the wave's 128 x 128 block leaves as two 128 x 64 halves
        store_half<0>(acc, epi, m0 + wm * WM, n0 + 2 * wn * WN, lane);
        store_half<1>(acc, epi, m0 + wm * WM, n0 + (2 * wn + 1) * WN, lane);
    } else {
        epi(acc, m0 + wm * WM, n0 + half_off + wn * WN, lane);
    }
}

// A_TR: A stored [K][lda] (its m contiguous); B_TR: B stored [K][ldb] (its n
// contiguous).  Otherwise the operand is [rows][ld] with k contiguous.
// Workgroups below full_tiles compute whole 256 x 256 tiles (tile_of's order);
// the ones after them split each remaining tile into two 256 x 128 halves
// (workgroup full_tiles + 2 h + q: half q of tile full_tiles + h), so that a
// last round of few tiles runs on twice as many CUs for half as long.  Every
// output element is summed in the same k order either way (bit-identical).
template <bool A_TR, bool B_TR, bool TAIL, class Epi, class KM = LinearK>
__device__ __forceinline__ void direct_body(const uint16_t* __restrict__ A, int64_t lda,
                                            const uint16_t* __restrict__ B, int64_t ldb, int M,
                                            int N, int K, int tiles_m, int tiles_n, int group_m,
                                            int full_tiles, uint16_t* st0, uint16_t* st1,
                                            const Epi& epi, KM km = {}) {
    const int nk = km.start(K / BK);
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    // wave-uniform, so kept in scalar registers (LDS destinations of the loads)
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1;
    const int wn = wave & 1;
    const int L = static_cast<int>(blockIdx.x);
    const bool halves = L >= full_tiles;
    const int tile = halves ? full_tiles + ((L - full_tiles) >> 1) : L;
    int tm, tn;
    tile_of(tile, tiles_m, tiles_n, group_m, tm, tn);
    const int m0 = tm * BM;
    const int n0 = tn * BN;

    const int rows_a = M - m0 < BM ? M - m0 : BM;
    const int rows_b = N - n0 < BN ? N - n0 : BN;
    const uint16_t* a0 = A_TR ? A + m0 : A + static_cast<int64_t>(m0) * lda;
    const uint16_t* b0 = B_TR ? B + n0 : B + static_cast<int64_t>(n0) * ldb;
    DirectStage d;
    // the resources span the bytes the tile's loads can address (their k
    // position is the scalar offset, always inside the operand)
    d.ra = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a0), static_cast<short>(0),
        static_cast<int>(A_TR ? ((K - 1) * lda + rows_a) * 2 : ((rows_a - 1) * lda + K) * 2) +
            km.more_a(),
        0x00020000);
    d.rb = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(b0), static_cast<short>(0),
        static_cast<int>(B_TR ? ((K - 1) * ldb + rows_b) * 2 : ((rows_b - 1) * ldb + K) * 2) +
            km.more_b(),
        0x00020000);
    d.step_a = A_TR ? static_cast<int>(BK * lda * 2) : BK * 2;
    d.step_b = B_TR ? static_cast<int>(BK * ldb * 2) : BK * 2;
    direct_offsets<A_TR>(d.oa, wave, lane, rows_a, lda);
    direct_offsets<B_TR>(d.ob, wave, lane, rows_b, ldb);

    if (!halves)
        direct_tile<A_TR, B_TR, 4, TAIL>(d, km, nk, st0, st1, a0, lda, rows_a, b0, ldb, rows_b, K, m0, n0,
                                         0, wm, wn, lane, wave, epi);
    else
        direct_tile<A_TR, B_TR, 2, TAIL>(d, km, nk, st0, st1, a0, lda, rows_a, b0, ldb, rows_b, K, m0, n0,
                                         ((L - full_tiles) & 1) * (BN / 2), wm, wn, lane, wave,
                                         epi);
}

// How many tiles the direct kernel computes whole: all of them, unless the
// last round (tiles beyond a multiple of the CU count) would fill at most half
// of the CUs; those tiles then run as two 256 x 128 halves each.
inline int direct_full_tiles(int tiles, int cus) {
    const int rem = tiles % cus;
    return (rem != 0 && 2 * rem <= cus) ? tiles - rem : tiles;
}

}  // namespace agk_gemm
