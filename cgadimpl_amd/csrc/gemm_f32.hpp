// gemm_f32.hpp -- the tiled fp32 product of gemm_f32.hip (its comment has the layouts), with
// its epilogue as a functor.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "gemm_common.hpp"
#include "rowcommon.hpp"

namespace agk_sgemm {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));  // in memory, at any float

constexpr int BK = 32;

// Float offset of 16-byte chunk c (0..7) of LDS row `row`: two rows share 256
// bytes (all 64 banks), whose 16 chunks are XOR-swizzled by the row pair.  The
// 16 lanes a 16-byte access serves at a time (rows 0-7 and 24-31 of one chunk,
// or 8 row quads of two chunks) then touch every bank once.
__device__ __forceinline__ int chunk_off(int row, int c) {
    return (row >> 1) * (2 * BK) + (((((row & 1) << 3) | c) ^ ((row >> 1) & 15)) << 2);
}

// One operand's 32-deep step of ROWS rows, as a lane holds it between its
// loads and its LDS writes: ROWS / 32 quads.
template <int ROWS>
struct Step {
    f32x4 v[ROWS / 32];
};

// What lane t of 256 loads of the operand whose rows r0 .. start at p, fixed for
// all steps.  KC: quad i holds k (t % 8) * 4 .. + 3 of row t / 8 + 32 i.
// Otherwise quad i holds four rows at k + i; 8 lanes cover 32 rows (128 bytes).
template <bool KC, int ROWS>
struct Place {
    const float* p;    // the quad's address at k = 0, quad 0
    int64_t ld;
    int rows;          // valid rows of the tile
    int r, k;          // first row and first k of the lane's quads, as staged
    int from;          // !KC: the first row loaded (below r by `shift` at the matrix's edge)
    int shift;
    bool edge;         // !KC: some lane of the workgroup has a shift
};

template <bool KC, int ROWS>
__device__ __forceinline__ Place<KC, ROWS> place(const float* __restrict__ src, int64_t ld, int r0,
                                                 int rows_total, int t) {
    Place<KC, ROWS> q;
    q.ld = ld;
    q.rows = rows_total - r0 < ROWS ? rows_total - r0 : ROWS;
    q.shift = 0;
    q.edge = false;
    if constexpr (KC) {
        q.r = q.from = t >> 3;
        q.k = (t & 7) * 4;
        q.p = src + static_cast<int64_t>(r0) * ld;
    } else {
        constexpr int kKb = 32 / (ROWS / 32);  // k groups of a step
        q.r = ((t & 7) + 8 * ((t >> 3) / kKb)) * 4;
        q.k = ((t >> 3) % kKb) * (ROWS / 32);
        q.p = src + r0;
        // rows_total >= 4: the quad stays inside the matrix (perhaps in the
        // tile before this one)
        q.from = q.r <= q.rows - 4 ? q.r : q.rows - 4;
        q.shift = q.r - q.from < 4 ? q.r - q.from : 0;
        q.edge = (q.rows & 3) != 0;
    }
    return q;
}

// Loads the whole step at k0 (k0 + 32 <= K).
template <bool KC, int ROWS>
__device__ __forceinline__ void load_step(Step<ROWS>& s, const Place<KC, ROWS>& q, int k0) {
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i) {
        if constexpr (KC) {
            const int row = q.r + 32 * i < q.rows ? q.r + 32 * i : q.rows - 1;
            s.v[i] = *reinterpret_cast<const f32x4_a4*>(q.p + static_cast<int64_t>(row) * q.ld + k0 +
                                                        q.k);
        } else {
            s.v[i] = *reinterpret_cast<const f32x4_a4*>(
                q.p + static_cast<int64_t>(k0 + q.k + i) * q.ld + q.from);
        }
    }
}

// The last K % 32 k, at k0: element by element, zeros past K.
template <bool KC, int ROWS>
__device__ __forceinline__ void load_tail(Step<ROWS>& s, const Place<KC, ROWS>& q, int k0, int K) {
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = k0 + q.k + (KC ? e : i);
            int row = KC ? q.r + 32 * i : q.from + e;
            row = row < q.rows ? row : q.rows - 1;
            s.v[i][e] = k >= K ? 0.0f
                               : KC ? q.p[static_cast<int64_t>(row) * q.ld + k]
                                    : q.p[static_cast<int64_t>(k) * q.ld + row];
        }
}

template <bool KC, int ROWS>
__device__ __forceinline__ void store_step(const Step<ROWS>& s, const Place<KC, ROWS>& q,
                                           float* lds) {
    if constexpr (KC) {
#pragma unroll
        for (int i = 0; i < ROWS / 32; ++i)
            *reinterpret_cast<f32x4*>(lds + chunk_off(q.r + 32 * i, q.k >> 2)) = s.v[i];
    } else {
        Step<ROWS> w = s;
        if (q.edge) {  // a quad moved down by `shift` rows holds row r + e at e + shift
#pragma unroll
            for (int i = 0; i < ROWS / 32; ++i)
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    float x = s.v[i][e];
                    x = q.shift == 1 ? s.v[i][e + 1] : x;
                    x = q.shift == 2 ? s.v[i][e + 2 < 4 ? e + 2 : 3] : x;
                    x = q.shift == 3 ? s.v[i][3] : x;
                    w.v[i][e] = x;
                }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float* at = lds + chunk_off(q.r + e, q.k >> 2) + (q.k & 3);
            if constexpr (ROWS == 32) *at = w.v[0][e];
            else if constexpr (ROWS == 64)
                *reinterpret_cast<f32x2*>(at) = f32x2{w.v[0][e], w.v[1][e]};
            else
                *reinterpret_cast<f32x4*>(at) =
                    f32x4{w.v[0][e], w.v[1][e], w.v[2][e], w.v[3][e]};
        }
    }
}

template <int NT>
struct Quads {
    f32x4 v[NT];
};

// The quads of substep s for NT blocks of 32 rows from row0.
template <int NT>
__device__ __forceinline__ void read_quads(Quads<NT>& f, const float* lds, int row0, int s,
                                           int lane) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
        f.v[i] = *reinterpret_cast<const f32x4*>(
            lds + chunk_off(row0 + i * 32 + (lane & 31), 2 * s + (lane >> 5)));
}

template <int TM, int TN>
__device__ __forceinline__ void mfma_quads(const Quads<TM>& a, const Quads<TN>& b,
                                           f32x16 (&acc)[TM][TN]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i][e], b.v[j][e], acc[i][j],
                                                                 0, 0, 0);
}

// One BM x BN tile by four waves, WVM of them along M; the epilogue takes a wave's accumulators,
// their first row and column, and the lane.  A_KC: A is [M][lda] (k contiguous), else A^T
// [K][lda]; B_KC: B is given as B^T [N][ldb] (k contiguous), else B [K][ldb].
template <int BM, int BN, int WVM, bool A_KC, bool B_KC, class Epi>
__device__ __forceinline__ void f32_body(const float* __restrict__ A, int64_t lda,
                                         const float* __restrict__ B, int64_t ldb, int M, int N,
                                         int K, int tiles_m, int tiles_n, const Epi& epi) {
    constexpr int kStage = (BM + BN) * BK;
    __shared__ __attribute__((aligned(16))) float l0[kStage];
    __shared__ __attribute__((aligned(16))) float l1[kStage];

    constexpr int WVN = 4 / WVM;
    constexpr int TM = BM / WVM / 32, TN = BN / WVN / 32;  // 32 x 32 MFMA blocks per wave
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = tid >> 6;
    const int wm = wave / WVN, wn = wave % WVN;
    int tm, tn;
    agk_gemm::tile_of(blockIdx.x, tiles_m, tiles_n, agk_gemm::kGroupM, tm, tn);
    const int m0 = tm * BM;
    const int n0 = tn * BN;

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    const Place<A_KC, BM> pa = place<A_KC, BM>(A, lda, m0, M, tid);
    const Place<B_KC, BN> pb = place<B_KC, BN>(B, ldb, n0, N, tid);
    const int nk = K / BK;  // whole steps
    Quads<TM> fa[2];
    Quads<TN> fb[2];
    auto read = [&](int f, const float* stage, int s) {
        read_quads(fa[f], stage, wm * (TM * 32), s, lane);
        read_quads(fb[f], stage + BM * BK, wn * (TN * 32), s, lane);
    };
    if (K % BK) {  // the ragged end of K first
        Step<BM> ta;
        Step<BN> tb;
        load_tail(ta, pa, nk * BK, K);
        load_tail(tb, pb, nk * BK, K);
        store_step(ta, pa, l1);
        store_step(tb, pb, l1 + BM * BK);
        __syncthreads();
        for (int s = 0; s * 8 < K % BK; ++s) {
            read(0, l1, s);
            mfma_quads(fa[0], fb[0], acc);
        }
    }
    if (nk > 0) {
        Step<BM> a0, a1;
        Step<BN> b0, b1;
        // step u, or the last one again: the loop below loads and stores
        // without conditions, so that the compiler can count the loads in
        // flight (behind a condition it waited for all of them each step)
        auto load = [&](Step<BM>& a, Step<BN>& b, int u) {
            const int k0 = (u < nk ? u : nk - 1) * BK;
            load_step(a, pa, k0);
            load_step(b, pb, k0);
        };
        auto store = [&](const Step<BM>& a, const Step<BN>& b, float* stage) {
            store_step(a, pa, stage);
            store_step(b, pb, stage + BM * BK);
        };
        load(a0, b0, 0);
        load(a1, b1, 1);
        store(a0, b0, l0);
        __syncthreads();
        // Step t out of `cur`.  (na, nb) are free and take step t + 2; (wa, wb)
        // hold step t + 1, for `nxt`.  The fragments run one substep ahead of
        // the MFMAs, across the barrier.
#define AGK_F32_STEP(FIRST, t, cur, nxt, na, nb, wa, wb) \
    load(na, nb, (t) + 2);                               \
    read(0, cur, 0);                                     \
    if (!FIRST) mfma_quads(fa[1], fb[1], acc);           \
    read(1, cur, 1);                                     \
    mfma_quads(fa[0], fb[0], acc);                       \
    read(0, cur, 2);                                     \
    mfma_quads(fa[1], fb[1], acc);                       \
    read(1, cur, 3);                                     \
    store(wa, wb, nxt);                                  \
    mfma_quads(fa[0], fb[0], acc);                       \
    __syncthreads();
        AGK_F32_STEP(true, 0, l0, l1, a0, b0, a1, b1)
        int t = 1;
        for (; t + 1 < nk; t += 2) {
            AGK_F32_STEP(false, t, l1, l0, a1, b1, a0, b0)
            AGK_F32_STEP(false, t + 1, l0, l1, a0, b0, a1, b1)
        }
        if (t < nk) {
            AGK_F32_STEP(false, t, l1, l0, a1, b1, a0, b0)
        }
#undef AGK_F32_STEP
        mfma_quads(fa[1], fb[1], acc);  // the last step's substep 3
    }

    epi(acc, m0 + wm * (TM * 32), n0 + wn * (TN * 32), lane);
}

}  // namespace agk_sgemm
