// xent.hip -- softmax cross entropy of a vocabulary head without its logits in memory
// (agk_linear_xent_fwd, agk_linear_xent_bwd): z = x w^T, x [tokens][cols], w [vocab][cols],
//   m = max_v z,  l = log sum_v exp(z - m),  loss = (m - z[label]) + l
//   G = dloss (exp((z - m) - l) - [v = label]),  dx = G w,  dw = G^T x
//
// bf16.  The forward is one product whose epilogue reduces the logits where they are:
// each wave's block of z^T leaves as {max, sum of exponentials} per token, 8 bytes for 32 to
// 128 logits, and a second kernel joins a token's blocks.  The backward makes z
// again, a piece of the vocabulary at a time, leaving G's piece in bf16 (the matrix
// cores' operand), and takes the two products from it.  dw's rows belong to one piece;
// dx adds up in fp32 over the pieces.  8 tokens vocab cols flop a step, 2 of the forward and
// 6 of the backward (2 of them the logits again: the price of not keeping them).  The matrix
// cores bound them: 8192 x 4096 x 131072 forward 6.2 ms and backward 19.9 on MI355X, 1350
// TFLOP/s; a few tokens' forward is bound by the read of w (TurnedK).
//
// fp32.  The same kernels on operands split into two fp16 planes (PlanesK), x once a call
// and w a piece at a time; in the backward, whose products sum along every index, after a pass
// over them for their largest values.  G leaves its kernel split.  Few tokens, whose time is the
// traffic of w, take the fp32 instruction instead (xent_f32.hip).
//
// A token that is left out (a negative label, or a zero dloss) has a zero row of G
// whatever its logits are, and the product over tokens reads its row of x as zeros,
// so that a NaN in it reaches nothing.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "agk_losses.h"
#include "rowcommon.hpp"
#include "xent_gemm.hpp"

namespace agk_xent {

using agk::aligned16;
using agk::check_launch;

// ---- joining a token's blocks ----------------------------------------------------

// loss and stats from the blocks' {max, sum}: TX tokens per workgroup of 1024 lanes,
// the other 1024 / TX lanes of a token taking its blocks in turn, kJoin of them
// loaded before any is used (the loads miss the caches: the latency of a few, not
// their bytes, is what a call of few tokens waits for).  Joined in a fixed order.
constexpr int kJoin = 8;
constexpr int kJoinLanes = 1024;

__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = max_of(m, m2);
    // exp(-inf - -inf) would be NaN: an empty side has nothing to scale
    const float a = m == top ? s : s * exp_of(m - top);
    const float b = m2 == top ? s2 : s2 * exp_of(m2 - top);
    m = top;
    s = a + b;
}

template <int TX>
__global__ __launch_bounds__(kJoinLanes) void xent_join(
    const float2* __restrict__ part, int64_t blocks, const float* __restrict__ picked,
    const int64_t* __restrict__ labels, float* __restrict__ loss, float2* __restrict__ stats,
    int64_t tokens, int64_t vocab) {
    constexpr int TY = kJoinLanes / TX;
    __shared__ float2 red[TY][TX];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * TX + tx;
    const int64_t tc = t < tokens ? t : tokens - 1;
    float m = -__builtin_inff(), s = 0.0f;
    for (int64_t b = ty; b < blocks; b += TY * kJoin) {
        float2 v[kJoin];
#pragma unroll
        for (int u = 0; u < kJoin; ++u) {
            const int64_t at = b + u * TY;
            v[u] = part[(at < blocks ? at : blocks - 1) * tokens + tc];
            if (at >= blocks) v[u] = make_float2(-__builtin_inff(), 0.0f);
        }
#pragma unroll
        for (int u = 0; u < kJoin; ++u) join(m, s, v[u].x, v[u].y);
    }
    red[ty][tx] = make_float2(m, s);
    for (int h = TY / 2; h > 0; h /= 2) {
        __syncthreads();
        if (ty < h) {
            const float2 o = red[ty + h][tx];
            join(m, s, o.x, o.y);
            red[ty][tx] = make_float2(m, s);
        }
    }
    if (ty != 0 || t >= tokens) return;
    const float l = logf(s);
    stats[t] = make_float2(m, l);
    const int64_t label = labels[t];
    loss[t] = label < 0 ? 0.0f : label >= vocab ? __builtin_nanf("") : (m - picked[t]) + l;
}

// ---- the backward's weights ---------------------------------------------------------

// What the kernels of one call pass on in device memory.
struct Scalars {
    float alpha;  // the backward's weights are dloss / alpha
    float z;      // fp32: the logits, dx and dw as factors of their products (powers of two;
    float dx;     // dw's with alpha)
    float dw;
};

// This lane's share of the largest finite |value| of a row (and of m), a wave to a row.
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ float row_max(const float* __restrict__ p, int cols, int lane, float m) {
    auto take = [&](float v) {
        v = __builtin_fabsf(v);
        if (v < __builtin_inff()) m = v > m ? v : m;
    };
    int c = lane * 4;
    for (; c + 4 <= cols; c += 256) {
        const f32x4_a4 q = *reinterpret_cast<const f32x4_a4*>(p + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) take(q[e]);
    }
    for (int e = c; e < cols && e < c + 4; ++e) take(p[e]);
    return m;
}
// e of a largest value of 2^e ..; the matrix's scale is 2^(14 - e), and the factor that takes a
// product of two such matrices back, 2^(e - 28), has to be a normal number.
__device__ __forceinline__ int top_exponent(float m) {
    const int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
    return m > 0.0f ? (e < -98 ? -98 : e) : 0;
}
__device__ __forceinline__ float pow2(int e) {
    e = e < -126 ? -126 : e > 127 ? 127 : e;
    return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

constexpr int kMaxParts = 1024;  // workgroups of the maximum's pass, per matrix

// A call's matrices: x (NULL: not in this launch) by the first x_groups workgroups, w by the rest.
struct Matrices {
    const float* x;
    const float* w;
    int64_t ldx, ldw, rows, wrows;
    int cols, x_groups;
    const int64_t* labels;  // tokens that are left out are read as zeros and have no part in
    const float* dloss;     // the maxima; NULL in the forward
    __device__ __forceinline__ bool keep(int64_t t) const {
        return labels[t] >= 0 && (!dloss || dloss[t] != 0.0f);
    }
};
// parts[0 .. kMaxParts): x's maxima by workgroup, parts[kMaxParts ..): w's.
__global__ __launch_bounds__(256) void xent_max(const Matrices a, float* __restrict__ parts) {
    __shared__ float red[4];
    const int g = static_cast<int>(blockIdx.x);
    const bool is_x = g < a.x_groups;
    const int k = is_x ? g : g - a.x_groups;
    const int64_t groups = is_x ? a.x_groups : static_cast<int>(gridDim.x) - a.x_groups;
    const int64_t first = static_cast<int64_t>(k) * 4 + (threadIdx.x >> 6);
    const int lane = static_cast<int>(threadIdx.x & 63);
    float m = 0.0f;
    for (int64_t r = first; r < (is_x ? a.rows : a.wrows); r += groups * 4)
        if (!is_x || a.keep(r))
            m = row_max(is_x ? a.x + r * a.ldx : a.w + r * a.ldw, a.cols, lane, m);
    for (int h = 32; h > 0; h /= 2) m = fmaxf(m, __shfl_xor(m, h));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0)
        parts[(is_x ? 0 : kMaxParts) + k] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// Row of an fp32 matrix (NULL: zeros) times s as two fp16 planes of kp values, by one wave;
// zeros past cols.
__device__ __forceinline__ void split_row(const float* __restrict__ src, int cols, int kp, float s,
                                          uint16_t* __restrict__ dst, int lane) {
    for (int c = lane * 4; c < kp; c += 256) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (src && c + 4 <= cols) {
            const f32x4_a4 q = *reinterpret_cast<const f32x4_a4*>(src + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = q[e] * s;
        } else if (src) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < cols) v[e] = src[c + e] * s;
        }
        uint32_t lo[2], hi[2];
        split2(v[0], v[1], lo);
        split2(v[2], v[3], hi);
#pragma unroll
        for (int q = 0; q < 2; ++q)
            *reinterpret_cast<uint2*>(dst + q * kp + c) = make_uint2(lo[q], hi[q]);
    }
}

// The forward's planes, each row by a scale of its own: the product is summed along the rows, so
// its factors are one per logit's row and column (scales: x's, then w's), and no pass over the
// matrices for their largest value goes before.
__global__ __launch_bounds__(256) void xent_split_rows(const Matrices a, int kp,
                                                       uint16_t* __restrict__ x2,
                                                       uint16_t* __restrict__ w2,
                                                       float* __restrict__ x_scales,
                                                       float* __restrict__ w_scales) {
    const int wave = static_cast<int>(threadIdx.x >> 6), lane = static_cast<int>(threadIdx.x & 63);
    const bool is_x = static_cast<int>(blockIdx.x) < a.x_groups;
    const int64_t g = is_x ? blockIdx.x : blockIdx.x - a.x_groups;
    const int64_t groups = is_x ? a.x_groups : static_cast<int>(gridDim.x) - a.x_groups;
    for (int64_t r = g * 4 + wave; r < (is_x ? a.rows : a.wrows); r += groups * 4) {
        const float* p = is_x ? a.x + r * a.ldx : a.w + r * a.ldw;
        if (is_x && !a.keep(r)) p = nullptr;
        float m = p ? row_max(p, a.cols, lane, 0.0f) : 0.0f;
        for (int h = 32; h > 0; h /= 2) m = fmaxf(m, __shfl_xor(m, h));
        const int e = top_exponent(m);
        split_row(p, a.cols, kp, pow2(14 - e), (is_x ? x2 : w2) + r * 2 * static_cast<int64_t>(kp),
                  lane);
        if (lane == 0) (is_x ? x_scales : w_scales)[r] = pow2(e - 14);
    }
}

// The planes of x (rows to x_padded, zeros past the last and for tokens left out) and of w (rows
// to w_padded), from the maxima of xent_max's x_parts and w_parts workgroups; four rows per
// workgroup at a time.  The first workgroup leaves the products' factors.
__global__ __launch_bounds__(256) void xent_split(const Matrices a, const float* __restrict__ parts,
                                                  int x_parts, int w_parts, int kp,
                                                  int64_t x_padded, int64_t w_padded,
                                                  uint16_t* __restrict__ x2,
                                                  uint16_t* __restrict__ w2,
                                                  Scalars* __restrict__ sc) {
    __shared__ float red[2][4];
    float mx = 0.0f, mw = 0.0f;
    for (int i = threadIdx.x; i < x_parts; i += 256) mx = fmaxf(mx, parts[i]);
    for (int i = threadIdx.x; i < w_parts; i += 256) mw = fmaxf(mw, parts[kMaxParts + i]);
    for (int h = 32; h > 0; h /= 2) {
        mx = fmaxf(mx, __shfl_xor(mx, h));
        mw = fmaxf(mw, __shfl_xor(mw, h));
    }
    const int wave = static_cast<int>(threadIdx.x >> 6), lane = static_cast<int>(threadIdx.x & 63);
    if (lane == 0) {
        red[0][wave] = mx;
        red[1][wave] = mw;
    }
    __syncthreads();
    mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    mw = fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3]));
    const int ex = top_exponent(mx), ew = top_exponent(mw);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        sc->z = pow2(ex + ew - 28);
        sc->dx = pow2(ew - 28);
        sc->dw = sc->alpha * pow2(ex - 28);
    }
    const int64_t pitch = 2 * static_cast<int64_t>(kp);
    if (static_cast<int>(blockIdx.x) < a.x_groups) {
        for (int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave; t < x_padded;
             t += static_cast<int64_t>(a.x_groups) * 4)
            split_row(t < a.rows && a.keep(t) ? a.x + t * a.ldx : nullptr, a.cols, kp, pow2(14 - ex),
                      x2 + t * pitch, lane);
    } else {
        const int64_t groups = static_cast<int>(gridDim.x) - a.x_groups;
        for (int64_t v = (static_cast<int64_t>(blockIdx.x) - a.x_groups) * 4 + wave; v < w_padded;
             v += groups * 4)
            split_row(v < a.wrows ? a.w + v * a.ldw : nullptr, a.cols, kp, pow2(14 - ew),
                      w2 + v * pitch, lane);
    }
}

// The first workgroup: weight[t] = dloss[t] / alpha for a token with a label, 0 for one
// without, NaN for one whose label is past the vocabulary; zeros to padded.  alpha: the
// largest finite |dloss| of the tokens with a label (1 where that is 0).
// The others: a token's row each, dst[t] = x[t], or zeros for one that is left out.
template <class T>
__global__ __launch_bounds__(1024) void xent_tokens(const float* __restrict__ dloss,
                                                    const int64_t* __restrict__ labels,
                                                    float* __restrict__ weight,
                                                    Scalars* __restrict__ sc, int64_t tokens,
                                                    int64_t padded, int64_t vocab,
                                                    const T* __restrict__ x, int64_t ldx,
                                                    T* __restrict__ dst, int cols) {
    if (blockIdx.x > 0) {
        for (int64_t t = (static_cast<int64_t>(blockIdx.x) - 1) * 4 + (threadIdx.x >> 8);
             t < tokens; t += (static_cast<int64_t>(gridDim.x) - 1) * 4) {
            const bool keep = labels[t] >= 0 && dloss[t] != 0.0f;
            if constexpr (sizeof(T) == 2) {
                const agk::u32x4* const from = reinterpret_cast<const agk::u32x4*>(x + t * ldx);
                agk::u32x4* const to = reinterpret_cast<agk::u32x4*>(dst + t * cols);
                for (int c = static_cast<int>(threadIdx.x & 255); c < cols / 8; c += 256)
                    to[c] = keep ? from[c] : agk::u32x4{0u, 0u, 0u, 0u};
            } else {
                for (int c = static_cast<int>(threadIdx.x & 255); c < cols; c += 256)
                    dst[t * cols + c] = keep ? x[t * ldx + c] : 0.0f;
            }
        }
        return;
    }
    __shared__ float red[16];
    float m = 0.0f;
    for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
        const float d = fabsf(dloss[t]);
        if (labels[t] >= 0 && d < __builtin_inff()) m = fmaxf(m, d);
    }
    for (int h = 32; h > 0; h /= 2) m = fmaxf(m, __shfl_xor(m, h));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int w = 0; w < 16; ++w) m = fmaxf(m, red[w]);
    const float c = m > 0.0f ? m : 1.0f;
    for (int64_t t = threadIdx.x; t < padded; t += 1024) {
        float w = 0.0f;
        if (t < tokens) {
            const int64_t label = labels[t];
            if (label >= vocab) w = __builtin_nanf("");
            else if (label >= 0) w = dloss[t] / c;
        }
        weight[t] = w;
    }
    if (threadIdx.x == 0) sc->alpha = c;
}

// dx (+)= alpha * (the K slices' sums, added in order), rounded to bf16 once.
__global__ __launch_bounds__(256) void xent_dx_out(const float* __restrict__ acc, int slices,
                                                   int64_t slice, const Scalars* __restrict__ sc,
                                                   const float* __restrict__ weight,
                                                   uint16_t* __restrict__ dx, int64_t n8, int cols8,
                                                   int accumulate) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n8) return;
    const float a = sc->alpha;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < slices; s0 += 4) {  // four slices' loads before they are added
        float u[4][8];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float4* q = reinterpret_cast<const float4*>(
                acc + (s0 + s < slices ? s0 + s : slices - 1) * slice + i * 8);
            *reinterpret_cast<float4*>(u[s]) = q[0];
            *reinterpret_cast<float4*>(u[s] + 4) = q[1];
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s0 + s < slices)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += u[s][e];
    }
    const bool keep = weight[i / cols8] != 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = keep ? v[e] * a : 0.0f;
    agk::u32x4* const out = reinterpret_cast<agk::u32x4*>(dx) + i;
    if (accumulate) {
        float o[8];
        agk::BF16::unpack(*out, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = agk::acc_add(o[e], v[e]);
    }
    *out = agk::BF16::pack(v);
}

// The same for fp32 (rows of cols8), four columns per lane.
__global__ __launch_bounds__(256) void xent_dx_out32(const float* __restrict__ acc, int slices,
                                                     int64_t slice, const Scalars* __restrict__ sc,
                                                     const float* __restrict__ weight,
                                                     float* __restrict__ dx, int64_t rows, int cols,
                                                     int cols8, int accumulate) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / (cols8 / 4);
    const int c = static_cast<int>(i - row * (cols8 / 4)) * 4;
    if (row >= rows) return;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < slices; s0 += 4) {
        float4 u[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
            u[s] = *reinterpret_cast<const float4*>(
                acc + (s0 + s < slices ? s0 + s : slices - 1) * slice + i * 4);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            if (s0 + s < slices) {
                v[0] += u[s].x;
                v[1] += u[s].y;
                v[2] += u[s].z;
                v[3] += u[s].w;
            }
    }
    const bool keep = weight[row] != 0.0f;
    const float a = sc->alpha;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (c + e < cols) {
            float* const p = dx + row * cols + c + e;
            const float g = keep ? v[e] * a : 0.0f;
            *p = accumulate ? agk::acc_add(*p, g) : g;
        }
}

// out[0 .. n) = 0 (4-byte words)
__global__ __launch_bounds__(256) void xent_zero(uint32_t* __restrict__ out, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * 256)
        out[i] = 0u;
}

// ---- sizes -------------------------------------------------------------------------------

// G's piece.  Larger pieces cost dx fewer additions and leave fewer part-filled rounds of
// tiles; that G then no longer fits the Infinity Cache does not show, the products being
// bound by the matrix cores.  Backward on MI355X, us for pieces of 64 / 128 / 256 / 512 MiB /
// 1 GiB: 8192 tokens x 4096 x 131072 22842 / 21095 / 20474 / 20068 / 20073; 4099 x 2048 x
// 50257 (pieces of 8192 / 16384 / 32768 rows, one piece) 2843 / 2805 / 2698 / 2444.
constexpr int64_t kPieceBytes = 512LL << 20;
constexpr int64_t kMaxOperand = 1LL << 30;    // values a product's 31-bit offsets reach
constexpr int64_t kMaxTokens = 1LL << 24;     // a workgroup per token within a grid

// G's rows are padded to whole 128-byte lines of bf16: the products fetch 128 bytes of
// a row at a time, which at any other pitch straddle two lines (kLine).

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline size_t region(int64_t bytes) { return static_cast<size_t>(up(bytes, 256)); }

// The vocabulary rows of a piece: `asked`, or what fills kPieceBytes, cut to equal
// pieces of whole 256-row tiles that the products' offsets reach.  per_row: values of the
// operands' longest row (G's or w's, in all planes).
inline int64_t piece_rows(int64_t vocab, int64_t ldg, int64_t ldw, int planes, int64_t asked) {
    const int64_t most = kMaxOperand / (planes * std::max(ldg, ldw));
    int64_t p = asked > 0 ? up(std::min(asked, vocab), 256)
                          : kPieceBytes / (2 * planes * (planes == 1 ? ldg : std::max(ldg, ldw)));
    p = std::max<int64_t>(std::min(p, most) / 256 * 256, 256);
    if (p >= vocab) return vocab;
    const int64_t n = (vocab + p - 1) / p;
    return up((vocab + n - 1) / n, 256);
}

// The tile of the logits' products: by the general rule, but for one column of 64 tokens, whose
// time is the read of w: 64 x 64 tiles (id 8) as long as one round holds them, 128 x 64 beyond.
// Forward of 16 tokens, us, rule / this: 4096 x 12000 37 / 28, x 20000 43 / 39, x 28000 54 / 43,
// 64 x 8192 x 12000 69 / 52; 64 x 64 tiles in two rounds: 2048 x 50257 46, 128 x 64 41.
inline int logits_shape(int64_t rows, int64_t vocab, int64_t cols, int dtype) {
    using namespace agk_gemm;
    const int cus = device_cus();
    if (dtype == AGK_BF16 && rows <= 64 && cols >= BK) return vocab <= 128 * cus ? 8 : 6;
    return pick_shape(vocab, rows, cols, cus);
}
// The forward's: the 32-row wave blocks of the 64-row tiles (ids 7 and 8: four times the partials)
// for few tokens only.
constexpr int64_t kFewTokens = 128;
inline int lse_shape(int64_t rows, int64_t vocab, int64_t cols, int dtype) {
    using namespace agk_gemm;
    const int s = logits_shape(rows, vocab, cols, dtype);
    if ((s != 7 && s != 8) || rows <= kFewTokens) return s;
    return agk::grid_fits(((vocab + 127) / 128) * ((rows + 63) / 64), 256) ? 6 : kRingLargest;
}
constexpr int64_t kMaxSlices = 32, kMinSlice = 512;
constexpr double kRoundUs = 5.0;

// Vocabulary rows of one wave's block.
inline int lse_block(int shape) {
    switch (shape) {
        case 0: return 128;
#define AGK_XENT_ROWS(ID, BM_, BN_, WVM, NST) \
    case ID: return BM_ / WVM;
        AGK_RING_SHAPES(AGK_XENT_ROWS)
#undef AGK_XENT_ROWS
        default: return 32;
    }
}
// Blocks per token that the workspace holds, whatever tiles a device's compute units give.
inline int64_t max_blocks(int64_t rows, int64_t vocab, int64_t piece) {
    const int64_t least = rows > kFewTokens ? 64 : 32;
    return ((vocab + piece - 1) / piece) * ((piece + least - 1) / least);
}

// The tile and K slices of dx = G w.  K is the piece's vocabulary rows, far longer than
// the tokens by cols output is large: tiles that fill the last round of CUs badly are cut along K
// until they fill it, each slice with an fp32 output of its own (xent_dx_out adds
// them in order).  The cost: the tile rule's (pick_shape) per 64-deep step, plus what a
// round costs besides (its first loads and its stores) and the slices' traffic.
struct DxPlan {
    int shape, slices, k_slice;
};
// The plan for the last piece, of n rows: as many of the slices as leave each a whole k-tile.
inline DxPlan last_piece(const DxPlan& plan, int64_t n) {
    DxPlan d = plan;
    for (;; --d.slices) {
        d.k_slice = static_cast<int>(up((n + d.slices - 1) / d.slices, 64));
        d.slices = static_cast<int>((n + d.k_slice - 1) / d.k_slice);
        if (d.slices == 1 || n - (d.slices - 1) * static_cast<int64_t>(d.k_slice) >= 64) break;
    }
    if (n < 64) d.shape = agk_gemm::kRingSmallK;
    return d;
}

inline DxPlan dx_plan(int64_t rows8, int64_t cols, int64_t k, int walks, double* us = nullptr) {
    using namespace agk_gemm;
    const int64_t cus = device_cus();
    // Few tokens are bound by the read of w: 64 x 128 tiles, as many slices as give each CU
    // one. dx alone (with the logits again) on MI355X, us, the cost below / this: 16 x 4096 x
    // 32000 112 / 103, 64 x 2048 x 50257 104 / 95, 64 x 4096 x 131072 402 / 391; with 256
    // columns no slices are enough.
    const int64_t across = (cols + 127) / 128, cuts = cus / across;
    if (rows8 <= 64 && walks == 1 && cuts >= 1 && cuts <= kMaxSlices && k >= cuts * kMinSlice)
    {
        if (us) *us = static_cast<double>(k * cols) * 2 / 5e6 + 2 * kRoundUs;
        return last_piece(DxPlan{7, static_cast<int>(cuts), 0}, k);
    }
    DxPlan best{pick_shape(rows8, cols, k, device_cus()), 1, static_cast<int>(up(k, 64))};
    double best_cost = 1e30;
    for (const RingCost& s : kRingCosts) {
        const int64_t tiles = ((rows8 + s.bm - 1) / s.bm) * ((cols + s.bn - 1) / s.bn);
        const double slots = static_cast<double>(cus * s.per_cu);
        for (int64_t n = 1; n <= kMaxSlices && (n == 1 || n * kMinSlice <= k * walks); ++n) {
            if (k < BK || !agk::grid_fits(tiles, 256)) break;
            const int64_t ks = up((k + n - 1) / n, 64), m = (k + ks - 1) / ks;
            if (m != n || k - (n - 1) * ks < BK) continue;  // every slice has a whole k-tile
            const double load = static_cast<double>(tiles * n) / slots;
            const double rounds = static_cast<double>(static_cast<int64_t>(load));
            const double fill = load - rounds;
            const double steps = static_cast<double>(ks) / 64 * walks;
            // the 256 x 256 kernel on two k-strided operands and a long K: 1.36 us a step at 53 %
            // fill, 1.64-1.70 full
            const double light = s.id == 0 ? 1.25 : s.light, full = s.id == 0 ? 1.65 : s.full;
            const double step =
                rounds * full + (fill > 0 ? light + (full - light) * fill * fill : 0.0);
            const double cost = step * steps + (rounds + (fill > 0)) * kRoundUs +
                                static_cast<double>(n * rows8 * cols) * 8 / 5e6;
            if (cost < best_cost) {
                best_cost = cost;
                best = DxPlan{s.id, static_cast<int>(n), static_cast<int>(ks)};
            }
        }
    }
    if (us) *us = best_cost;
    return best;
}

// fp32 of few tokens on the fp32 instruction, which reads w as it lies (its 32-row blocks are
// what max_blocks counts for kFewTokens and less; its k-strided loads take four columns).
// Forward / backward on MI355X, us, planes / this: 16 tokens x 2048 x 32000 203, 389 / 63,
// 237; 64 x 1024 x 32000 92, 210 / 46, 155; 128 x 1024 x 20000 73, 179 / 59, 172; 129 x 1024
// x 32000 106, 302 / 110, 330.
inline bool on_instruction(int64_t rows, int64_t vocab, int64_t cols, int dtype) {
    return dtype == AGK_F32 && rows <= kFewTokens && cols >= 4 && vocab <= 1LL << 28;
}
// dx's slices there: two workgroups per CU, each slice with 256 k at least.
inline DxPlan dx_plan32(int64_t rows8, int64_t cols, int64_t k) {
    const int64_t tiles = rows8 <= 32 ? (cols + 127) / 128 : (rows8 + 63) / 64 * ((cols + 63) / 64);
    const int64_t n = std::max<int64_t>(
        std::min<int64_t>({2 * agk_gemm::device_cus() / tiles, k / 256, 64}), 1);
    const int64_t ks = up((k + n - 1) / n, 32);
    return DxPlan{0, static_cast<int>((k + ks - 1) / ks), static_cast<int>(ks)};
}

// The workspaces.  `cols` of the operands as staged: kp for planes (whole k-tiles).
struct FwdLayout {
    int64_t kp, piece;
    size_t scales, picked, part, x2, w2, total;
};
inline FwdLayout fwd_layout(int64_t rows, int64_t vocab, int64_t cols, int dtype) {
    FwdLayout o;
    const bool whole = dtype == AGK_BF16 || on_instruction(rows, vocab, cols, dtype);
    o.kp = up(cols, 64);
    o.piece = whole ? vocab : piece_rows(vocab, 64, o.kp, 2, 0);
    o.scales = 0;  // x's and w's; a wave's block of up to 128 rows can pass the last one
    o.picked = o.scales + (whole ? 0 : region((up(rows, 64) + o.piece + 128) * 4));
    o.part = o.picked + region(rows * 4);
    o.x2 = o.part + region(max_blocks(rows, vocab, o.piece) * rows * 8);
    o.w2 = o.x2 + (whole ? 0 : region(rows * o.kp * 4));
    o.total = o.w2 + (whole ? 0 : region(o.piece * o.kp * 4));
    return o;
}

struct BwdLayout {
    bool instr;  // on_instruction
    int planes;
    int64_t piece, padded;             // vocabulary rows of a piece, and of its operands
    int64_t rows8, rows64, ldg, kp, cols8;
    int64_t main;  // dx: rows of the first product, the others (bf16) by a second
    DxPlan dx, rest;
    // The fp32 sums of dx: every slice's rows of cols8.
    int64_t rest_acc() const { return static_cast<int64_t>(dx.slices) * main * cols8; }
    int64_t acc_values() const {
        return rest_acc() + (main < rows8 ? rest.slices * (rows8 - main) * cols8 : 0);
    }
    size_t weight, scalars, parts, x, w2, g, acc, total;
};
inline BwdLayout bwd_layout(int64_t rows, int64_t vocab, int64_t cols, int64_t ldw, int dtype,
                            int64_t piece) {
    BwdLayout o;
    const bool bf16 = dtype == AGK_BF16;
    o.instr = on_instruction(rows, vocab, cols, dtype);
    o.planes = bf16 ? 1 : 2;
    o.rows8 = up(rows, 8);
    o.rows64 = up(rows, 64);
    o.ldg = o.instr ? up(rows, 32) : up(rows, kLine);
    o.kp = up(cols, 64);
    o.cols8 = up(cols, 8);
    o.piece = piece_rows(vocab, o.ldg, bf16 ? ldw : o.kp, o.planes, piece);
    o.padded = bf16 || o.instr ? o.piece : up(o.piece, 64);
    double us = 0.0;
    o.main = o.rows8;
    o.dx = o.instr ? dx_plan32(o.rows8, cols, o.piece)
                   : dx_plan(o.rows8, o.cols8, o.padded, bf16 ? 1 : PlanesK::kWalks, &us);
    o.rest = o.dx;
    // A few tokens past whole 256-row tiles cost a row of tiles: by themselves they are one more
    // read of w (4099 tokens x 2048 x 50257 on MI355X 811 us, so 605 + 47).
    const int64_t whole = rows / 256 * 256;
    if (bf16 && whole >= 1024 && rows > whole && rows - whole <= 64) {
        double us_main = 0.0, us_rest = 0.0;
        const DxPlan a = dx_plan(whole, o.cols8, o.padded, 1, &us_main);
        const DxPlan b = dx_plan(o.rows8 - whole, o.cols8, o.padded, 1, &us_rest);
        if (us_main + us_rest < us) {
            o.main = whole;
            o.dx = a;
            o.rest = b;
        }
    }
    o.weight = 0;
    o.scalars = o.weight + region(o.rows8 * 4);
    o.parts = o.scalars + region(sizeof(Scalars));
    o.x = o.parts + (bf16 ? 0 : region(2 * kMaxParts * 4));
    o.w2 = o.x + region(bf16 ? rows * cols * 2 : o.rows64 * o.kp * 4);
    o.g = o.w2 + (bf16 || o.instr ? 0 : region(o.padded * o.kp * 4));
    o.acc = o.g + region(o.padded * o.ldg * 2 * o.planes);
    o.total = o.acc + region(o.acc_values() * 4);
    return o;
}

inline int check_args(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows,
                      int64_t vocab, int64_t cols, int dtype) {
    constexpr int64_t kMax = 0x7fffffffLL - 1024;  // tiles past an edge stay within an int
    if (!agk::valid_dtype(dtype)) return AGK_EDTYPE;
    if (rows < 0 || vocab < 1 || cols < 1 || rows >= kMaxTokens || vocab > kMax || cols > kMax)
        return AGK_EINVAL;
    // 256 x 256 tiles of all logits: one grid's worth
    if (rows > 0 && vocab > (kMaxTokens - 1) * 65536 / up(rows, 256) - 256) return AGK_EINVAL;
    if (dtype == AGK_BF16 && cols % 8) return AGK_EINVAL;
    if (rows == 0) return AGK_OK;
    if (!x || !w || ldx < cols || ldw < cols) return AGK_EINVAL;
    if (rows > INT64_MAX / 16 / ldx || vocab > INT64_MAX / 16 / ldw) return AGK_EINVAL;
    if (dtype == AGK_BF16) {
        if (ldx % 8 || ldw % 8 || !aligned16(x) || !aligned16(w)) return AGK_EINVAL;
        if (256 * ldw > kMaxOperand || 256 * ldx > kMaxOperand) return AGK_EINVAL;
    } else if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 3u) ||
               cols > kMaxOperand / 1024) {  // 256 rows of two planes
        return AGK_EINVAL;
    }
    return AGK_OK;
}

int launch_join(const float2* part, int64_t blocks, const float* picked, const int64_t* labels,
                float* loss, float2* stats, int64_t tokens, int64_t vocab, hipStream_t st) {
#define AGK_JOIN(TX)                                                                             \
    hipLaunchKernelGGL(xent_join<TX>, dim3(static_cast<unsigned>((tokens + TX - 1) / TX)),       \
                       dim3(kJoinLanes), 0, st, part, blocks, picked, labels, loss, stats, tokens, \
                       vocab)
    // few tokens: more lanes for each one's blocks
    if (tokens <= 8) AGK_JOIN(1);
    else AGK_JOIN(16);
#undef AGK_JOIN
    return check_launch();
}

// The forward's planes: x's (where a.x) and those of a piece of w.
int launch_planes_rows(Matrices a, int64_t kp, uint16_t* x2, uint16_t* w2, float* x_scales,
                       float* w_scales, hipStream_t st) {
    a.x_groups = a.x ? static_cast<int>(std::min<int64_t>((a.rows + 3) / 4, 4096)) : 0;
    const int w_groups = static_cast<int>(std::min<int64_t>((a.wrows + 3) / 4, 16384));
    hipLaunchKernelGGL(xent_split_rows, dim3(a.x_groups + w_groups), dim3(256), 0, st, a,
                       static_cast<int>(kp), x2, w2, x_scales, w_scales);
    return check_launch();
}

// The maxima's pass and the split of x (where a.x) and of a piece of w: rows to x_padded and
// w_padded.  x's maxima and planes stay for the pieces after the first.
int launch_planes(Matrices a, float* parts, int64_t kp, int64_t x_padded, int64_t w_padded,
                  uint16_t* x2, uint16_t* w2, Scalars* sc, int* x_parts, hipStream_t st) {
    auto groups = [](int64_t rows, int64_t most) {
        return static_cast<int>(std::min<int64_t>((rows + 3) / 4, most));
    };
    a.x_groups = a.x ? groups(a.rows, kMaxParts / 4) : 0;
    if (a.x) *x_parts = a.x_groups;
    const int w_parts = groups(a.wrows, kMaxParts);
    hipLaunchKernelGGL(xent_max, dim3(a.x_groups + w_parts), dim3(256), 0, st, a, parts);
    const int rc = check_launch();
    if (rc != AGK_OK) return rc;
    a.x_groups = a.x ? groups(x_padded, 4096) : 0;
    hipLaunchKernelGGL(xent_split, dim3(a.x_groups + groups(w_padded, 16384)), dim3(256), 0, st, a,
                       parts, *x_parts, w_parts, static_cast<int>(kp), x_padded, w_padded, x2, w2,
                       sc);
    return check_launch();
}

}  // namespace agk_xent

extern "C" {

size_t agk_linear_xent_fwd_workspace_bytes(int64_t rows, int64_t vocab, int64_t cols, int dtype) {
    using namespace agk_xent;
    if (rows <= 0 || vocab <= 0 || cols <= 0 || !agk::valid_dtype(dtype)) return 0;
    return fwd_layout(rows, vocab, cols, dtype).total;
}

int agk_linear_xent_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int64_t* labels, float* loss, float* stats, void* workspace,
                        size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t cols,
                        int dtype, agk_stream_t stream) {
    using namespace agk_xent;
    int rc = check_args(x, ldx, w, ldw, rows, vocab, cols, dtype);
    if (rc != AGK_OK || rows == 0) return rc;
    if (!labels || !loss || !stats || (reinterpret_cast<uintptr_t>(loss) & 3u) ||
        ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(labels)) & 7u))
        return AGK_EINVAL;
    const FwdLayout o = fwd_layout(rows, vocab, cols, dtype);
    if (!workspace || workspace_bytes < o.total) return AGK_EWORKSPACE;
    if (!aligned16(workspace)) return AGK_EINVAL;
    agk::clear_pending_error();
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    char* const ws = static_cast<char*>(workspace);
    float* const picked = reinterpret_cast<float*>(ws + o.picked);
    float2* const part = reinterpret_cast<float2*>(ws + o.part);
    uint16_t* const x2 = reinterpret_cast<uint16_t*>(ws + o.x2);
    uint16_t* const w2 = reinterpret_cast<uint16_t*>(ws + o.w2);
    float* const x_scales = reinterpret_cast<float*>(ws + o.scales);
    float* const w_scales = x_scales + up(rows, 64);
    const bool bf16 = dtype == AGK_BF16;
    const int m = static_cast<int>(rows), kp = static_cast<int>(o.kp);
    if (on_instruction(rows, vocab, cols, dtype)) {
        const int nv = static_cast<int>(vocab);
        rc = launch_lse(ProductF32{static_cast<const float*>(w), ldw, static_cast<const float*>(x),
                                   ldx, nv, m, static_cast<int>(cols), 1, 0, st},
                        LseEpi<false>{part, picked, labels, 0, nv, m, nullptr, nullptr});
        if (rc != AGK_OK) return rc;
        return launch_join(part, (vocab + 31) / 32, picked, labels, loss,
                           reinterpret_cast<float2*>(stats), rows, vocab, st);
    }
    int64_t blocks = 0;
    for (int64_t v0 = 0; v0 < vocab; v0 += o.piece) {
        const int64_t n = std::min(o.piece, vocab - v0);
        const int nv = static_cast<int>(n);
        const int shape = lse_shape(rows, n, bf16 ? cols : o.kp, dtype);
        float2* const to = part + blocks * rows;
        if (bf16) {
            rc = launch_lse(shape,
                            Product{static_cast<const uint16_t*>(w), ldw,
                                    static_cast<const uint16_t*>(x), ldx, nv, m,
                                    static_cast<int>(cols), 1, 0, st},
                            LseEpi<false>{to, picked, labels, v0, nv, m, nullptr, nullptr});
        } else {
            const Matrices a{v0 ? nullptr : static_cast<const float*>(x),
                             static_cast<const float*>(w) + v0 * ldw, ldx, ldw, rows, n,
                             static_cast<int>(cols), 0, labels, nullptr};
            rc = launch_planes_rows(a, kp, x2, w2, x_scales, w_scales, st);
            if (rc != AGK_OK) return rc;
            rc = launch_lse(shape, Product{w2, 2 * o.kp, x2, 2 * o.kp, nv, m, kp, 1, 0, st},
                            LseEpi<true>{to, picked, labels, v0, nv, m, w_scales, x_scales},
                            PlanesK{kp * 2, kp * 2, 0});
        }
        if (rc != AGK_OK) return rc;
        blocks += (n + lse_block(shape) - 1) / lse_block(shape);
    }
    return launch_join(part, blocks, picked, labels, loss, reinterpret_cast<float2*>(stats), rows,
                       vocab, st);
}

size_t agk_linear_xent_bwd_workspace_bytes(int64_t rows, int64_t vocab, int64_t cols, int dtype,
                                           int64_t piece) {
    using namespace agk_xent;
    if (rows <= 0 || vocab <= 0 || cols <= 0 || !agk::valid_dtype(dtype)) return 0;
    return bwd_layout(rows, vocab, cols, cols, dtype, piece).total;
}

int agk_linear_xent_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int64_t* labels, const float* stats, const float* dloss, void* dx,
                        void* dw, int dw_dtype, void* workspace, size_t workspace_bytes,
                        int64_t rows, int64_t vocab, int64_t cols, int64_t piece, int dtype,
                        int accumulate, agk_stream_t stream) {
    using namespace agk_xent;
    int rc = check_args(x, ldx, w, ldw, rows, vocab, cols, dtype);
    if (rc != AGK_OK) return rc;
    if (!agk::valid_dtype(dw_dtype) || (dtype == AGK_F32 && dw_dtype != AGK_F32)) return AGK_EDTYPE;
    if (accumulate & ~AGK_ACCUM_ALL || piece < 0) return AGK_EINVAL;
    const int acc_dx = accumulate & AGK_ACCUM_DX ? 1 : 0;
    const int acc_dw = accumulate & AGK_ACCUM_DGAMMA ? 1 : 0;
    const int dw_size = dw_dtype == AGK_F32 ? 4 : 2;
    if (dw && (reinterpret_cast<uintptr_t>(dw) & 3u)) return AGK_EINVAL;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (rows == 0) {
        if (!dw || acc_dw) return AGK_OK;
        if (vocab > INT64_MAX / 16 / cols) return AGK_EINVAL;
        agk::clear_pending_error();
        const int64_t n = vocab * cols * dw_size / 4;  // bf16: cols is even
        hipLaunchKernelGGL(xent_zero, dim3(agk::capped_blocks((n + 255) / 256, 256)), dim3(256), 0,
                           st, static_cast<uint32_t*>(dw), n);
        return check_launch();
    }
    if (!labels || !stats || !dloss || (reinterpret_cast<uintptr_t>(dloss) & 3u) ||
        ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(labels)) & 7u))
        return AGK_EINVAL;
    if (!dx && !dw) return AGK_OK;
    const bool bf16 = dtype == AGK_BF16;
    if (dx && (reinterpret_cast<uintptr_t>(dx) & (bf16 ? 15u : 3u))) return AGK_EINVAL;
    // 31-bit offsets of the products: over tokens, and over G's smallest piece
    if (up(rows, kLine) * (bf16 ? 1 : 2) > kMaxOperand / 256) return AGK_EINVAL;
    if (bf16 ? rows > kMaxOperand / ldx : up(rows, 64) > kMaxOperand / (2 * up(cols, 64)))
        return AGK_EINVAL;
    BwdLayout o = bwd_layout(rows, vocab, cols, cols, dtype, piece);
    if (!workspace || workspace_bytes < o.total) return AGK_EWORKSPACE;
    if (!aligned16(workspace)) return AGK_EINVAL;
    if (bf16) {  // a wider ldw may need smaller pieces than the workspace was sized for
        const int64_t p = piece_rows(vocab, o.ldg, ldw, 1, piece);
        if (p < o.piece) {
            o.piece = p;
            auto again = [&](int64_t rows, const DxPlan& had) {
                const DxPlan d = dx_plan(rows, o.cols8, p, 1);
                return d.slices > had.slices ? last_piece(DxPlan{d.shape, had.slices, 0}, p) : d;
            };
            o.dx = again(o.main, o.dx);
            o.rest = o.main < o.rows8 ? again(o.rows8 - o.main, o.rest) : o.dx;
        }
    }
    agk::clear_pending_error();
    char* const ws = static_cast<char*>(workspace);
    float* const weight = reinterpret_cast<float*>(ws + o.weight);
    Scalars* const sc = reinterpret_cast<Scalars*>(ws + o.scalars);
    float* const acc = reinterpret_cast<float*>(ws + o.acc);
    uint16_t* const xk = reinterpret_cast<uint16_t*>(ws + o.x);
    uint16_t* const w2 = reinterpret_cast<uint16_t*>(ws + o.w2);
    uint16_t* const g = reinterpret_cast<uint16_t*>(ws + o.g);
    const float2* const in = reinterpret_cast<const float2*>(stats);
    const int m = static_cast<int>(rows), m8 = static_cast<int>(o.rows8);
    const int ldg = static_cast<int>(o.ldg), kp = static_cast<int>(o.kp);
    const int c1 = static_cast<int>(cols), c8 = static_cast<int>(o.cols8);
    const int cus = agk_gemm::device_cus();
    const int64_t slice = o.main * o.cols8, left8 = o.rows8 - o.main;
    const int mm = static_cast<int>(o.main);
    float* const acc_rest = acc + o.rest_acc();
    const int64_t copied = (bf16 || o.instr) && dw ? rows : 0;
    const dim3 grid(1 + agk::capped_blocks((copied + 3) / 4, 1 << 20)), block(1024);
    if (bf16)
        hipLaunchKernelGGL(xent_tokens<uint16_t>, grid, block, 0, st, dloss, labels, weight, sc,
                           rows, o.rows8, vocab, static_cast<const uint16_t*>(x), ldx, xk, c1);
    else
        hipLaunchKernelGGL(xent_tokens<float>, grid, block, 0, st, dloss, labels, weight, sc, rows,
                           o.rows8, vocab, static_cast<const float*>(x), ldx,
                           reinterpret_cast<float*>(xk), c1);
    if ((rc = check_launch()) != AGK_OK) return rc;
    int x_parts = 0;
    for (int64_t v0 = 0; v0 < vocab; v0 += o.piece) {
        const int64_t n = std::min(o.piece, vocab - v0);
        const int nv = static_cast<int>(n), np = static_cast<int>(bf16 ? n : up(n, 64));
        if (o.instr) {
            const float* const wp = static_cast<const float*>(w) + v0 * ldw;
            float* const g32 = reinterpret_cast<float*>(g);
            const float* const x0 = reinterpret_cast<const float*>(xk);
            rc = launch_grad(ProductF32{wp, ldw, static_cast<const float*>(x), ldx, nv, m, c1, 1, 0,
                                        st},
                             GradEpiF32{g32, in, weight, labels, v0, ldg, nv, m});
            if (rc != AGK_OK) return rc;
            // the last piece is shorter: fewer slices, which the others' sums are left in
            const int slices = static_cast<int>((n + o.dx.k_slice - 1) / o.dx.k_slice);
            if (dx)
                rc = launch_dx(ProductF32{g32, ldg, wp, ldw, m8, c1, nv, slices, o.dx.k_slice, st},
                               AddEpi<true>{acc, c8, slice, nullptr, m8, c1, v0 > 0});
            if (rc != AGK_OK) return rc;
            if (dw)
                rc = launch_dw(ProductF32{g32, ldg, x0, cols, nv, c1, m, 1, 0, st},
                               AddEpi<true>{static_cast<float*>(dw) + v0 * cols, cols, 0,
                                            &sc->alpha, nv, c1, acc_dw});
            if (rc != AGK_OK) return rc;
            continue;
        }
        const DxPlan d = n == o.piece ? o.dx : last_piece(o.dx, np);
        const AddEpi<true> de{acc, c8, slice, bf16 ? nullptr : &sc->dx, mm, c8, v0 > 0};
        char* const out = static_cast<char*>(dw) + v0 * cols * dw_size;
        if (bf16) {
            const uint16_t* const wp = static_cast<const uint16_t*>(w) + v0 * ldw;
            rc = launch_grad(logits_shape(rows, n, cols, dtype),
                             Product{wp, ldw, static_cast<const uint16_t*>(x), ldx, nv, m, c1, 1, 0,
                                     st},
                             GradEpi<1>{g, in, weight, labels, v0, ldg, nv, nv, m, nullptr});
            if (rc != AGK_OK) return rc;
            if (dx)
                rc = launch_dx(d.shape,
                               Product{g, ldg, wp, ldw, mm, c1, nv, d.slices, d.k_slice, st}, de);
            if (rc != AGK_OK) return rc;
            if (dx && left8) {
                const DxPlan r = n == o.piece ? o.rest : last_piece(o.rest, n);
                const int ml = static_cast<int>(left8);
                rc = launch_dx(r.shape,
                               Product{g + mm, ldg, wp, ldw, ml, c1, nv, r.slices, r.k_slice, st},
                               AddEpi<true>{acc_rest, c8, left8 * o.cols8, nullptr, ml, c8, v0 > 0});
            }
            if (rc != AGK_OK) return rc;
            const Product wt{g, ldg, xk, cols, nv, c1, m, 1, 0, st};
            const int shape = agk_gemm::pick_shape(n, cols, rows, cus);
            if (dw && dw_dtype == AGK_F32)
                rc = launch_dw(shape, wt, AddEpi<true>{out, cols, 0, &sc->alpha, nv, c1, acc_dw});
            else if (dw)
                rc = launch_dw(shape, wt, AddEpi<false>{out, cols, 0, &sc->alpha, nv, c1, acc_dw});
        } else {
            const Matrices a{v0 ? nullptr : static_cast<const float*>(x),
                             static_cast<const float*>(w) + v0 * ldw, ldx, ldw, rows, n, c1, 0,
                             labels, dloss};
            rc = launch_planes(a, reinterpret_cast<float*>(ws + o.parts), kp, o.rows64, np, xk, w2,
                               sc, &x_parts, st);
            if (rc != AGK_OK) return rc;
            rc = launch_grad(agk_gemm::pick_shape(np, rows, kp, cus),
                             Product{w2, 2 * o.kp, xk, 2 * o.kp, np, m, kp, 1, 0, st},
                             GradEpi<2>{g, in, weight, labels, v0, ldg, nv, np, m, &sc->z},
                             PlanesK{kp * 2, kp * 2, 0});
            if (rc != AGK_OK) return rc;
            if (dx)
                rc = launch_dx(d.shape,
                               Product{g, 2 * o.ldg, w2, 2 * o.kp, m8, c8, np, d.slices, d.k_slice,
                                       st},
                               de, PlanesK{ldg * 2, kp * 2, 0});
            if (rc != AGK_OK) return rc;
            if (dw)
                rc = launch_dw(agk_gemm::pick_shape(np, c8, ldg, cus),
                               Product{g, 2 * o.ldg, xk, 2 * o.kp, np, c8, ldg, 1, 0, st},
                               AddEpi<true>{out, cols, 0, &sc->dw, nv, c1, acc_dw},
                               PlanesK{ldg * 2, kp * 2, 0});
        }
        if (rc != AGK_OK) return rc;
    }
    if (!dx) return AGK_OK;
    const int64_t first = std::min(rows, o.main);
    const int64_t lanes = first * o.cols8 / (bf16 ? 8 : 4);
    const dim3 out_grid(static_cast<unsigned>((lanes + 255) / 256));
    if (bf16) {
        uint16_t* const out = static_cast<uint16_t*>(dx);
        hipLaunchKernelGGL(xent_dx_out, out_grid, dim3(256), 0, st, acc, o.dx.slices, slice, sc,
                           weight, out, lanes, c8 / 8, acc_dx);
        if (left8) {
            if ((rc = check_launch()) != AGK_OK) return rc;
            const int64_t more = (rows - first) * o.cols8 / 8;
            hipLaunchKernelGGL(xent_dx_out, dim3(static_cast<unsigned>((more + 255) / 256)),
                               dim3(256), 0, st, acc_rest, o.rest.slices, left8 * o.cols8, sc,
                               weight + first, out + first * cols, more, c8 / 8, acc_dx);
        }
    } else
        hipLaunchKernelGGL(xent_dx_out32, out_grid, dim3(256), 0, st, acc, o.dx.slices, slice, sc,
                           weight, static_cast<float*>(dx), rows, c1, c8, acc_dx);
    return check_launch();
}

}  // extern "C"
