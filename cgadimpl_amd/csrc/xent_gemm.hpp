// xent_gemm.hpp -- the products of the vocabulary head's loss (xent.hip), of bf16 operands and
// of fp32 ones as fp16 planes: the direct and ring kernels of gemm_direct.hpp /
// gemm_ring.hpp with epilogues that take the logits while they are in registers, and a
// kernel for few k.  One translation unit per product instantiates its kernels
// (AGK_XENT_KERNELS and AGK_RING_KERNELS), to compile side by side.
//
// Every product has the vocabulary along M and the tokens along N where it makes or
// takes logits (z^T = w x^T): an accumulator tile then holds, in each lane, 16
// vocabulary rows of one token per 32 x 32 block, so a token's maximum and sum of
// exponentials are sums within a lane and one exchange between the wave's halves, where
// tokens along M would take a 5-step exchange over 32 lanes for every row of the tile.
#pragma once

#include <type_traits>

#include "gemm_common.hpp"
#include "gemm_direct.hpp"
#include "gemm_ring.hpp"

namespace agk_xent {

using agk_gemm::f32x16;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kLine = 64;  // bf16 of a 128-byte line

// fp32 operands.  A matrix (the forward: a row) is stored scaled by a power of two that
// brings its largest value to 2^14 .. 2^15, each value as two fp16 whose sum it is to 2^-22
// of it: x = a + b, a = fp16(x), b = fp16(x - a), in two planes side by side in each row.  A
// product of two is aa' + ab' + ba', three fp16 products summed in fp32 by walking K three
// times over different planes.  What is left out (bb' and the two remainders) is at most 3 *
// 2^-22 of each product, 12 times an fp32 rounding and of random sign: below the error of an
// fp32 sum of some dozens of products, and nothing next to one of thousands.  Values 2^-28 of
// the largest and below lose relative bits (fp16's smallest is 2^-24), at 2^-39 of the
// largest.  Three fp16 matrix instructions at 1250 TFLOP/s are 416 TFLOP/s of fp32; the fp32
// matrix instruction gives 113-135 (of 157).  In three bf16 planes (2^-25) it is six walks.
// 1000 tokens x 1000 x 32000, forward + backward on MI355X: fp32 instruction 2.47 ms, bf16
// planes 1.59, fp16 planes 0.96; relative error of dx 6e-7 (fp32 products of the BLAS
// library: 3e-6).
struct PlanesK {
    static constexpr bool kF16 = true, kStream = false;
    static constexpr int kWalks = 3;
    int plane_a, plane_b;  // bytes from one plane to the next
    int n;                 // k-tiles of a plane

    __device__ __forceinline__ int start(int tiles) {
        n = tiles;
        return kWalks * tiles;
    }
    __device__ __forceinline__ int walk(int t) const { return (t >= n) + (t >= 2 * n); }
    __device__ __forceinline__ int a(int t, int step) const {
        const int s = walk(t);
        return (t - s * n) * step + (s == 2 ? plane_a : 0);
    }
    __device__ __forceinline__ int b(int t, int step) const {
        const int s = walk(t);
        return (t - s * n) * step + (s == 1 ? plane_b : 0);
    }
    __device__ __forceinline__ int more_a() const { return plane_a; }
    __device__ __forceinline__ int more_b() const { return plane_b; }
};
constexpr float kTop = 16384.0f;  // 2^14
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// The two planes of two neighbouring (scaled) values.
__device__ __forceinline__ void split2(float x, float y, uint32_t (&plane)[2]) {
    const f16x2 a = {static_cast<_Float16>(x), static_cast<_Float16>(y)};
    const f16x2 b = {static_cast<_Float16>(x - static_cast<float>(a.x)),
                     static_cast<_Float16>(y - static_cast<float>(a.y))};
    plane[0] = __builtin_bit_cast(uint32_t, a);
    plane[1] = __builtin_bit_cast(uint32_t, b);
}

// Few tokens, one column of tiles: the time is the read of w, each row by one workgroup, so
// its loads are non-temporal.  Workgroups that walk K in step read the same offsets of rows
// that lie, as a rule, a power of two apart, which are in a few of the memory's channels; so
// each starts at a k-tile of its own.  Forward on MI355X, w not in the caches, in step /
// turned (us): 16 tokens x 4096 x 32000 55 / 48 (of it the join and two launches' gaps 8; 262
// MB at 6.6 TB/s), x 2048 x 50257 50 / 41, 64 x 8192 x 32000 108 / 96.  It does not pay with
// few tiles, which are bound by latency (16 x 4096 x 8000, 125 tiles: 24 / 27), nor where
// rows are not whole 128-byte lines, two k-tiles sharing one (16 x 1000 x 100000: 55 / 63);
// deeper rings gain nothing (4 or 7 stages of 128 x 32: the same).
struct TurnedK {
    static constexpr bool kF16 = false, kStream = true;
    int n, first;

    __device__ __forceinline__ int start(int tiles) {
        n = tiles;
        first = tiles ? static_cast<int>(blockIdx.x % static_cast<unsigned>(tiles)) : 0;
        return tiles;
    }
    __device__ __forceinline__ int a(int t, int step) const {
        return (t + first >= n ? t + first - n : t + first) * step;
    }
    __device__ __forceinline__ int b(int t, int step) const { return a(t, step); }
    __device__ __forceinline__ int more_a() const { return 0; }
    __device__ __forceinline__ int more_b() const { return 0; }
};

// exp(x) on v_exp_f32; see fast_exp in rowops.hip for its error.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// One v_max_f32 (fmaxf first quiets both operands).  It drops a NaN, which reaches
// the result through exp(z - max).
__device__ __forceinline__ float max_of(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// Row of element e of a wave block's 32-row group i, from its first row.
__device__ __forceinline__ int acc_row(int i, int e, int half) {
    return i * 32 + 8 * (e >> 2) + 4 * half + (e & 3);
}

// Where a token's label lies in the block of `rows` vocabulary rows from row0 (-1:
// elsewhere).
__device__ __forceinline__ int label_row(int64_t label, int64_t row0, int rows) {
    const int64_t r = label - row0;
    return r >= 0 && r < rows ? static_cast<int>(r) : -1;
}

// max(a, b, c) in one instruction.
__device__ __forceinline__ float max3_of(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Forward: the block's maximum and sum of exponentials of each token, and the logit
// of its label.  part[(row0 / block rows) * tokens + token] = {max, sum of exp(z - max)}.
//
// One wave per SIMD runs this while the matrix cores wait, so it is kept short: two
// maxima per instruction, one fma, one exponential and one addition per logit, in four
// chains.  The fma takes z log2(e) - t, t = m log2(e) rounded; the rounding, exact as
// another fma, goes into the sum as a factor.  SCALED: the accumulators are the logits over
// row_scale[row] * token_scale[token] (powers of two; row_scale has whole tiles' rows).
template <bool SCALED>
struct LseEpi {
    float2* part;
    float* picked;
    const int64_t* labels;
    int64_t v0;  // the first vocabulary row of the operand, which has `vocab` of them
    int vocab, tokens;
    const float* row_scale;
    const float* token_scale;

    // at(i, e): the logit in element e of group i, or the smallest value past the vocabulary
    template <int TMW, class At>
    __device__ __forceinline__ float2 reduce(At at) const {
        constexpr float kNone = -__builtin_inff();
        float m4[4] = {kNone, kNone, kNone, kNone};
#pragma unroll
        for (int i = 0; i < TMW; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 2)
                m4[(e / 2) & 3] = max3_of(m4[(e / 2) & 3], at(i, e), at(i, e + 1));
        float m = max_of(max_of(m4[0], m4[1]), max_of(m4[2], m4[3]));
        m = max_of(m, other_half(m));
        const float t = m == kNone ? 0.0f : m * kLog2e;  // no -inf - -inf
        float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < TMW; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                s4[e & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(at(i, e), kLog2e, -t));
        float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        s += other_half(s);
        if (m != kNone) s *= __builtin_amdgcn_exp2f(-__builtin_fmaf(m, kLog2e, -t));
        return make_float2(m, s);
    }

    template <int TMW, int TNW>
    __device__ __forceinline__ void operator()(const f32x16 (&acc)[TMW][TNW], int row0, int col0,
                                               int lane) const {
        if (row0 >= vocab) return;
        const int half = lane >> 5;
        const bool inner = row0 + TMW * 32 <= vocab;
        float2* const out = part + static_cast<int64_t>(row0 / (TMW * 32)) * tokens;
#pragma unroll
        for (int j = 0; j < TNW; ++j) {
            const int col = col0 + j * 32 + (lane & 31);
            const bool in = col < tokens;
            const int label = in ? label_row(labels[col], v0 + row0, TMW * 32) : -1;
            f32x16 z[TMW];
#pragma unroll
            for (int i = 0; i < TMW; ++i) {
                z[i] = acc[i][j];
                if constexpr (SCALED) {
                    const float ts = in ? token_scale[col] : 1.0f;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 rs = *reinterpret_cast<const float4*>(
                            row_scale + row0 + acc_row(i, q * 4, half));
                        z[i][q * 4] *= rs.x * ts;
                        z[i][q * 4 + 1] *= rs.y * ts;
                        z[i][q * 4 + 2] *= rs.z * ts;
                        z[i][q * 4 + 3] *= rs.w * ts;
                    }
                }
            }
            const int left = vocab - row0;
            const float2 v =
                inner ? reduce<TMW>([&](int i, int e) -> float { return z[i][e]; })
                      : reduce<TMW>([&](int i, int e) -> float {
                            return acc_row(i, e, half) < left ? z[i][e] : -__builtin_inff();
                        });
            if (in && half == 0) out[col] = v;
            if (__any(label >= 0)) {
#pragma unroll
                for (int i = 0; i < TMW; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (label == acc_row(i, e, half) && label < left) picked[col] = z[i][e];
            }
        }
    }
};

// Backward: G^T, weight * (softmax - [label]), rows v0 .. of the vocabulary as rows of ldg
// tokens, zeros in the columns from `tokens` to ldg (the padding of G's rows) and in the rows
// from `rows` to padded_rows: what the products that follow read of them.  PLANES = 1: rounded
// to bf16; 2: G 2^14's two fp16 planes, ldg apart, from accumulators that are the logits over
// *scale.
//
// One fma, one exponential and one product per logit.  Lanes c and c + 1 exchange rows e
// and e + 1, so that a store is 4 bytes of two neighbouring tokens.
template <int PLANES>
struct GradEpi {
    uint16_t* G;
    const float2* stats;
    const float* weight;  // 0: a token that is left out
    const int64_t* labels;
    int64_t v0;
    int ldg, rows, padded_rows, tokens;
    const float* scale;

    template <int TMW, int TNW>
    __device__ __forceinline__ void operator()(const f32x16 (&acc)[TMW][TNW], int row0, int col0,
                                               int lane) const {
        if (row0 >= padded_rows) return;
        const int half = lane >> 5, odd = lane & 1;
        const bool inner = row0 + TMW * 32 <= rows;
        // even lanes: {own low, neighbour's low}; odd lanes: {neighbour's high, own high}
        const uint32_t pick = odd ? 0x07060302u : 0x01000504u;
        const float sc = PLANES == 1 ? 1.0f : *scale;
        float w[TNW], m[TNW], shift[TNW];
        int at[TNW];
        bool hit = false, some_out = false;
#pragma unroll
        for (int j = 0; j < TNW; ++j) {
            const int col = col0 + j * 32 + (lane & 31);
            const bool in = col < tokens;
            const float2 st = in ? stats[col] : make_float2(0.0f, 0.0f);
            w[j] = in ? (PLANES == 1 ? weight[col] : weight[col] * kTop) : 0.0f;
            at[j] = in ? label_row(labels[col], v0 + row0, TMW * 32) : -1;
            hit = hit || at[j] >= 0;
            some_out = some_out || w[j] == 0.0f;
            // bf16: exp(z - (m + l)), m + l rounded once (2^-24 of its size: far below G's
            // rounding); fp32: the difference z - m first
            m[j] = PLANES == 1 ? 0.0f : st.x;
            shift[j] = (PLANES == 1 ? st.x + st.y : st.y) * kLog2e;
        }
        hit = __any(hit);
        some_out = __any(some_out);
        uint16_t* const out =
            G + col0 + (lane & 30) + static_cast<int64_t>(row0 + odd) * (PLANES * ldg);
        const int left = ldg - col0 - (lane & 30);  // ldg is even: a pair is in or out
        // a row's tokens together: its lines are written whole
#pragma unroll
        for (int i = 0; i < TMW; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const int r = acc_row(i, e, half);
                uint16_t* const row = out + static_cast<int64_t>(r) * (PLANES * ldg);
                const bool store = inner || row0 + r + odd < padded_rows;
#pragma unroll
                for (int j = 0; j < TNW; ++j) {
                    float g[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float z = PLANES == 1 ? acc[i][j][e + u]
                                                    : __builtin_fmaf(acc[i][j][e + u], sc, -m[j]);
                        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, -shift[j]));
                        if (hit) p -= at[j] == r + u ? 1.0f : 0.0f;
                        g[u] = w[j] * p;
                        if (some_out) g[u] = w[j] != 0.0f ? g[u] : 0.0f;  // z may be NaN there
                        if (!inner) g[u] = row0 + r + u < rows ? g[u] : 0.0f;
                    }
                    uint32_t own[2];
                    if constexpr (PLANES == 1) own[0] = agk_gemm::pack_bf16(g[0], g[1]);
                    else split2(g[0], g[1], own);
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                        const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(
                            static_cast<int>(own[q]), 0xb1, 0xf, 0xf, true));
                        const uint32_t v = __builtin_amdgcn_perm(own[q], other, pick);
                        if (store && j * 32 < left)
                            *reinterpret_cast<uint32_t*>(row + j * 32 + q * ldg) = v;
                    }
                }
            }
    }
};

// The same in fp32, from logits in fp32: rows of ldg tokens, zeros from `tokens` on.
struct GradEpiF32 {
    float* G;
    const float2* stats;
    const float* weight;
    const int64_t* labels;
    int64_t v0;
    int ldg, rows, tokens;

    template <int TMW, int TNW>
    __device__ __forceinline__ void operator()(const f32x16 (&acc)[TMW][TNW], int row0, int col0,
                                               int lane) const {
        const int half = lane >> 5;
#pragma unroll
        for (int j = 0; j < TNW; ++j) {
            const int col = col0 + j * 32 + (lane & 31);
            if (col >= ldg) continue;
            const bool in = col < tokens;
            const float2 st = in ? stats[col] : make_float2(0.0f, 0.0f);
            const float w = in ? weight[col] : 0.0f;
            const int at = in ? label_row(labels[col], v0 + row0, TMW * 32) : -1;
            const float shift = st.y * kLog2e;
#pragma unroll
            for (int i = 0; i < TMW; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = acc_row(i, e, half);
                    float p = __builtin_amdgcn_exp2f(
                        __builtin_fmaf(acc[i][j][e] - st.x, kLog2e, -shift));
                    p -= at == r ? 1.0f : 0.0f;
                    if (row0 + r < rows)
                        G[static_cast<int64_t>(row0 + r) * ldg + col] = w != 0.0f ? w * p : 0.0f;
                }
        }
    }
};

// C (+)= alpha * product (alpha NULL: 1), that in fp32 and rounded to C's type once.  The
// old values of a 32-row group are loaded together: one wait for 16 TNW loads.  A bf16 C that
// is not added to is stored 4 bytes at a time, as G is (ldc and N are even there): dw of 4099
// tokens x 2048 x 50257 802 -> 739 us on MI355X, of 16 tokens x 4096 x 32000 (all stores) 74 -> 67.
template <bool OUT_F32>
struct AddEpi {
    void* C;
    int64_t ldc;
    int64_t slice;  // elements between the K slices' outputs
    const float* alpha;
    int M, N, accumulate;

    template <int TMW, int TNW>
    __device__ __forceinline__ void operator()(const f32x16 (&acc)[TMW][TNW], int row0, int col0,
                                               int lane) const {
        using T = typename std::conditional<OUT_F32, float, uint16_t>::type;
        if (row0 >= M || col0 >= N) return;
        const int half = lane >> 5;
        const float a = alpha ? *alpha : 1.0f;
        T* const c0 = static_cast<T*>(C) + static_cast<int64_t>(blockIdx.y) * slice;
        const bool inner = row0 + TMW * 32 <= M && col0 + TNW * 32 <= N;
        if constexpr (!OUT_F32) {
            if (!accumulate) {
                const int odd = lane & 1, col = lane & 30;
                const uint32_t pick = odd ? 0x07060302u : 0x01000504u;
#pragma unroll
                for (int i = 0; i < TMW; ++i)
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const int r = row0 + acc_row(i, e, half) + odd;
                        uint16_t* const p = c0 + static_cast<int64_t>(r) * ldc + col0 + col;
#pragma unroll
                        for (int j = 0; j < TNW; ++j) {
                            const uint32_t own =
                                agk_gemm::pack_bf16(acc[i][j][e] * a, acc[i][j][e + 1] * a);
                            const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(
                                static_cast<int>(own), 0xb1, 0xf, 0xf, true));
                            if (inner || (r < M && col0 + j * 32 + col < N))
                                *reinterpret_cast<uint32_t*>(p + j * 32) =
                                    __builtin_amdgcn_perm(own, other, pick);
                        }
                    }
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < TMW; ++i) {
            T* const p0 = c0 + static_cast<int64_t>(row0 + i * 32 + 4 * half) * ldc + col0 +
                          (lane & 31);
            const int rows_left = M - (row0 + i * 32 + 4 * half);
            const int cols_left = N - (col0 + (lane & 31));
            T old[TNW][16] = {};
            if (accumulate) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
#pragma unroll
                    for (int j = 0; j < TNW; ++j)
                        if (inner || (8 * (e >> 2) + (e & 3) < rows_left && j * 32 < cols_left))
                            old[j][e] = p0[static_cast<int64_t>(8 * (e >> 2) + (e & 3)) * ldc + j * 32];
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int j = 0; j < TNW; ++j) {
                    float v = acc[i][j][e] * a;
                    if (accumulate) {
                        float o;
                        if constexpr (OUT_F32) o = old[j][e];
                        else o = __uint_as_float(static_cast<uint32_t>(old[j][e]) << 16);
                        v = agk::acc_add(o, v);
                    }
                    if (inner || (8 * (e >> 2) + (e & 3) < rows_left && j * 32 < cols_left)) {
                        T* const p = p0 + static_cast<int64_t>(8 * (e >> 2) + (e & 3)) * ldc + j * 32;
                        if constexpr (OUT_F32) *p = v;
                        else *p = static_cast<uint16_t>(agk_gemm::f32_to_bf16_bits(v));
                    }
                }
        }
    }
};

// One product: M, N as staged (an operand with rows contiguous needs them to be
// multiples of 8), the epilogue's own bounds what is stored.  slices > 1: K cut into
// that many parts of k_slice (a multiple of 64; the last takes the rest), one per
// grid row, each with its own output.
struct Product {
    const uint16_t* A;
    int64_t lda;
    const uint16_t* B;
    int64_t ldb;
    int M, N, K, slices, k_slice;
    hipStream_t st;
};

// The same of fp32 operands as they lie (xent_f32.hip); a k-strided one has at least four rows.
struct ProductF32 {
    const float* A;
    int64_t lda;
    const float* B;
    int64_t ldb;
    int M, N, K, slices, k_slice;
    hipStream_t st;
};

int launch_lse(const ProductF32& p, const LseEpi<false>& e);
int launch_grad(const ProductF32& p, const GradEpiF32& e);
int launch_dx(const ProductF32& p, const AddEpi<true>& e);
int launch_dw(const ProductF32& p, const AddEpi<true>& e);

// bf16 operands, and fp32 ones as planes (their leading dimension: two planes' worth).
int launch_lse(int shape, const Product& p, const LseEpi<false>& e);
int launch_lse(int shape, const Product& p, const LseEpi<true>& e, const PlanesK& k);
int launch_grad(int shape, const Product& p, const GradEpi<1>& e);
int launch_grad(int shape, const Product& p, const GradEpi<2>& e, const PlanesK& k);
int launch_dx(int shape, const Product& p, const AddEpi<true>& e);
int launch_dx(int shape, const Product& p, const AddEpi<true>& e, const PlanesK& k);
int launch_dw(int shape, const Product& p, const AddEpi<true>& e);
int launch_dw(int shape, const Product& p, const AddEpi<false>& e);
int launch_dw(int shape, const Product& p, const AddEpi<true>& e, const PlanesK& k);

}  // namespace agk_xent

#ifdef AGK_XENT_KERNELS

namespace agk_xent {

// Moves the operands to this grid row's K slice; its length.  (A kernel built for a K tail
// that the last slice alone has stages it for the others too, from the k that follow
// them, as zeros.)
template <bool A_TR, bool B_TR>
__device__ __forceinline__ int slice_of(const uint16_t* __restrict__& A, int64_t lda,
                                        const uint16_t* __restrict__& B, int64_t ldb, int K,
                                        int k_slice) {
    const int k0 = static_cast<int>(blockIdx.y) * k_slice;
    A += A_TR ? static_cast<int64_t>(k0) * lda : k0;
    B += B_TR ? static_cast<int64_t>(k0) * ldb : k0;
    return blockIdx.y + 1 < gridDim.y ? k_slice : K - k0;
}

template <bool A_TR, bool B_TR, bool TAIL, class Epi, class KM>
__global__ __launch_bounds__(agk_gemm::kDirectThreads) void xent_direct_kernel(
    const uint16_t* __restrict__ A, int64_t lda, const uint16_t* __restrict__ B, int64_t ldb, int M,
    int N, int K, int k_slice, const Epi epi, const KM km, int tiles_m, int tiles_n, int full_tiles) {
    __shared__ __attribute__((aligned(16))) uint16_t st0[agk_gemm::kStageElems];
    __shared__ __attribute__((aligned(16))) uint16_t st1[agk_gemm::kStageElems];
    const int k = slice_of<A_TR, B_TR>(A, lda, B, ldb, K, k_slice);
    agk_gemm::direct_body<A_TR, B_TR, TAIL>(A, lda, B, ldb, M, N, k, tiles_m, tiles_n,
                                            agk_gemm::kGroupM, full_tiles, st0, st1, epi, km);
}

template <bool A_TR, bool B_TR, class SH, class Epi, class KM>
__global__ __launch_bounds__(256, SH::kPerCu) void xent_ring_kernel(
    const uint16_t* __restrict__ A, int64_t lda, const uint16_t* __restrict__ B, int64_t ldb, int M,
    int N, int K, int k_slice, const Epi epi, const KM km, int tiles_m, int tiles_n) {
    const int k = slice_of<A_TR, B_TR>(A, lda, B, ldb, K, k_slice);
    agk_gemm::ring_body<A_TR, B_TR, SH>(A, lda, B, ldb, M, N, k, tiles_m, tiles_n,
                                        agk_gemm::kGroupM, epi, km);
}

// A product of few k (dw of few tokens: an outer product, whose time is its stores): all of K
// staged at once, one barrier, no ring.  A tile's stages (NKT tiles of 64 k) then take 24 KiB, or
// 48, instead of 64-72, so that six or three workgroups share a CU, and a workgroup's loads and
// stores hide behind the others'.  dw in bf16, 4096 x 32000 on MI355X, the shape pick_shape takes
// / this: 16 tokens 171 / 67 us (4.0 TB/s of stores), 128 tokens 150 / 110.  A row-by-row order of
// the tiles changes little (62-76, 119).
constexpr int kShortM = 64, kShortN = 128, kShortK = 128;

template <bool A_TR, bool B_TR, int NKT, class Epi>
__global__ __launch_bounds__(256, NKT == 1 ? 6 : 3) void xent_short_kernel(
    const uint16_t* __restrict__ A, int64_t lda, const uint16_t* __restrict__ B, int64_t ldb, int M,
    int N, int K, const Epi epi, int tiles_m, int tiles_n) {
    using namespace agk_gemm;
    using SH = RingShape<kShortM, kShortN, 2, 3>;
    __shared__ __attribute__((aligned(16))) uint16_t lds[NKT][SH::kElems];
    const int lane = static_cast<int>(threadIdx.x & 63);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int wm = wave / SH::kWvn, wn = wave % SH::kWvn;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, kGroupM, tm, tn);
    const int m0 = tm * kShortM, n0 = tn * kShortN;
    const int rows_a = M - m0 < kShortM ? M - m0 : kShortM;
    const int rows_b = N - n0 < kShortN ? N - n0 : kShortN;
    const uint16_t* const a0 = A_TR ? A + m0 : A + static_cast<int64_t>(m0) * lda;
    const uint16_t* const b0 = B_TR ? B + n0 : B + static_cast<int64_t>(n0) * ldb;
#pragma unroll
    for (int t = 0; t < NKT; ++t) {
        if (t * BK >= K) break;
        stage_k_tail<A_TR, kShortM>(lds[t], a0, lda, rows_a, t * BK, K);
        stage_k_tail<B_TR, kShortN>(lds[t] + kShortM * BK, b0, ldb, rows_b, t * BK, K);
    }
    f32x16 acc[SH::kTm][SH::kTn];
#pragma unroll
    for (int i = 0; i < SH::kTm; ++i)
#pragma unroll
        for (int j = 0; j < SH::kTn; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NKT; ++t) {
        const uint16_t* const sa = lds[t];
        const uint16_t* const sb = sa + kShortM * BK;
        const int left = K - t * BK;
        for (int s = 0; s * 16 < left && s < BK / 16; ++s) {
            RingFrags<SH::kTm, SH::kTn> f;
#pragma unroll
            for (int i = 0; i < SH::kTm; ++i)
                f.a[i] = ring_frag<A_TR, kShortM>(sa, (wm * SH::kTm + i) * 32, s, lane);
#pragma unroll
            for (int j = 0; j < SH::kTn; ++j)
                f.b[j] = ring_frag<B_TR, kShortN>(sb, (wn * SH::kTn + j) * 32, s, lane);
            ring_mfma<false>(f, acc);
        }
    }
    epi(acc, m0 + wm * SH::kTm * 32, n0 + wn * SH::kTn * 32, lane);
}

// K at most kShortK.
template <bool A_TR, bool B_TR, class Epi>
int launch_short(const Product& p, const Epi& e) {
    const int tiles_m = (p.M + kShortM - 1) / kShortM, tiles_n = (p.N + kShortN - 1) / kShortN;
    const dim3 grid(tiles_m * tiles_n), block(256);
    if (p.K <= agk_gemm::BK)
        hipLaunchKernelGGL((xent_short_kernel<A_TR, B_TR, 1, Epi>), grid, block, 0, p.st, p.A,
                           p.lda, p.B, p.ldb, p.M, p.N, p.K, e, tiles_m, tiles_n);
    else
        hipLaunchKernelGGL((xent_short_kernel<A_TR, B_TR, 2, Epi>), grid, block, 0, p.st, p.A,
                           p.lda, p.B, p.ldb, p.M, p.N, p.K, e, tiles_m, tiles_n);
    return agk::check_launch();
}

template <bool A_TR, bool B_TR, class Epi, class KM = agk_gemm::LinearK>
int launch_product(int shape, const Product& p, const Epi& e, const KM& km = {}) {
    using namespace agk_gemm;
    if (shape == 0) {
        const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
        const int tiles = tiles_m * tiles_n;
        const int full = p.slices > 1 ? tiles : direct_full_tiles(tiles, device_cus());
        const dim3 grid(full + 2 * (tiles - full), p.slices), block(kDirectThreads);
#define AGK_XENT_DIRECT(TAIL)                                                                    \
    hipLaunchKernelGGL((xent_direct_kernel<A_TR, B_TR, TAIL, Epi, KM>), grid, block, 0, p.st,    \
                       p.A, p.lda, p.B, p.ldb, p.M, p.N, p.K, p.k_slice, e, km, tiles_m, tiles_n, \
                       full)
        if constexpr (std::is_same<KM, LinearK>::value) {  // planes have no K tail
            if (p.K % BK != 0) AGK_XENT_DIRECT(true);
            else AGK_XENT_DIRECT(false);
        } else {
            AGK_XENT_DIRECT(false);
        }
#undef AGK_XENT_DIRECT
        return agk::check_launch();
    }
#define AGK_XENT_CASE(ID, BM_, BN_, WVM, NST)                                                    \
    case ID: {                                                                                   \
        using SH = RingShape<BM_, BN_, WVM, NST>;                                                \
        const int tiles_m = (p.M + BM_ - 1) / BM_, tiles_n = (p.N + BN_ - 1) / BN_;              \
        hipLaunchKernelGGL((xent_ring_kernel<A_TR, B_TR, SH, Epi, KM>),                          \
                           dim3(tiles_m * tiles_n, p.slices), dim3(256), 0, p.st, p.A, p.lda,    \
                           p.B, p.ldb, p.M, p.N, p.K, p.k_slice, e, km, tiles_m, tiles_n);       \
        break;                                                                                   \
    }
    switch (shape) { AGK_RING_SHAPES(AGK_XENT_CASE) }
#undef AGK_XENT_CASE
    return agk::check_launch();
}

// A product of x and w, both k-contiguous: on TurnedK where one column of tiles holds the tokens
// and the tiles are enough to be bound by the read of w.
template <class Epi>
int launch_logits(int shape, const Product& p, const Epi& e) {
    using namespace agk_gemm;
    const int least = p.lda % kLine == 0 ? device_cus() * 3 / 4 : 0x7fffffff;
#define AGK_XENT_CASE(ID, BM_, BN_, WVM, NST)                                                    \
    if constexpr (BM_ <= 128 && BN_ <= 128) {                                                    \
        const int tiles_m = (p.M + BM_ - 1) / BM_;                                               \
        if (shape == ID && p.N <= BN_ && tiles_m >= least) {                                     \
            using SH = RingShape<BM_, BN_, WVM, NST>;                                            \
            hipLaunchKernelGGL((xent_ring_kernel<false, false, SH, Epi, TurnedK>),               \
                               dim3(tiles_m), dim3(256), 0, p.st, p.A, p.lda, p.B, p.ldb, p.M,   \
                               p.N, p.K, p.k_slice, e, TurnedK{}, tiles_m, 1);                   \
            return agk::check_launch();                                                          \
        }                                                                                        \
    }
    AGK_RING_SHAPES(AGK_XENT_CASE)
#undef AGK_XENT_CASE
    return launch_product<false, false>(shape, p, e);
}

}  // namespace agk_xent

#endif  // AGK_XENT_KERNELS
