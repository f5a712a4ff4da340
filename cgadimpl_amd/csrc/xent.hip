// xent.hip -- softmax cross entropy of a vocabulary head without its logits in memory
// (agk_linear_xent_fwd, agk_linear_xent_bwd): z = x w^T, x [tokens][cols], w [vocab][cols],
//   m = max_v z,  l = log sum_v exp(z - m),  loss = (m - z[label]) + l
//   G = dloss (exp((z - m) - l) - [v = label]),  dx = G w,  dw = G^T x
//
// bf16.  The forward is one product whose epilogue reduces the logits where they are:
// each wave's block of z^T leaves as {max, sum of exponentials} per token, 8 bytes for 32 to
// 128 logits, and a second kernel joins a token's blocks.  The backward makes z
// again, a piece of the vocabulary at a time, leaving G's piece in bf16 (the matrix
// cores' operand), and takes the two products from it.  dw's rows belong to one piece; dx adds up in fp32 over the pieces.
// 8 tokens vocab cols flop a step, 2 of the forward and 6 of the backward (2 of them
// the logits again: the price of not keeping them).
//
// fp32.  The same pieces on the fp32 product of gemm_f32.hip, z^T's piece in memory.
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

// weight[t] = dloss[t] / *alpha for a token with a label, 0 for one without, NaN for
// one whose label is past the vocabulary; zeros to padded.  *alpha: the largest finite
// |dloss| of the tokens with a label (1 where that is 0), or 1 if !SCALE.  One workgroup: a few
// thousand values.
template <bool SCALE>
__global__ __launch_bounds__(1024) void xent_weights(const float* __restrict__ dloss,
                                                     const int64_t* __restrict__ labels,
                                                     float* __restrict__ weight,
                                                     float* __restrict__ alpha, int64_t tokens,
                                                     int64_t padded, int64_t vocab) {
    float c = 1.0f;
    if constexpr (SCALE) {
        __shared__ float red[1024];
        float m = 0.0f;
        for (int64_t t = threadIdx.x; t < tokens; t += 1024) {
            const float d = fabsf(dloss[t]);
            if (labels[t] >= 0 && d < __builtin_inff()) m = fmaxf(m, d);
        }
        red[threadIdx.x] = m;
        for (int h = 512; h > 0; h /= 2) {
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < h)
                red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + h]);
        }
        __syncthreads();
        c = red[0] > 0.0f ? red[0] : 1.0f;
    }
    for (int64_t t = threadIdx.x; t < padded; t += 1024) {
        float w = 0.0f;
        if (t < tokens) {
            const int64_t label = labels[t];
            if (label >= vocab) w = __builtin_nanf("");
            else if (label >= 0) w = dloss[t] / c;
        }
        weight[t] = w;
    }
    if (threadIdx.x == 0) *alpha = c;
}

// dst[t] = x[t], or zeros for a token that is left out; rows of cols (T: 16 bytes of
// bf16, or one float).
template <class T>
__global__ __launch_bounds__(256) void xent_keep_rows(const T* __restrict__ x, int64_t ldx,
                                                      const float* __restrict__ weight,
                                                      T* __restrict__ dst, int cols) {
    const int64_t t = blockIdx.x;
    const bool keep = weight[t] != 0.0f;
    for (int c = threadIdx.x; c < cols; c += 256)
        dst[t * cols + c] = keep ? x[t * ldx + c] : T{};
}

// dx (+)= alpha * (the K slices' sums, added in order), rounded to bf16 once.
__global__ __launch_bounds__(256) void xent_dx_out(const float* __restrict__ acc, int slices,
                                                   int64_t slice, const float* __restrict__ alpha,
                                                   const float* __restrict__ weight,
                                                   uint16_t* __restrict__ dx, int64_t n8, int cols8,
                                                   int accumulate) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n8) return;
    const float a = *alpha;
    float v[8];
    const float4* p = reinterpret_cast<const float4*>(acc + i * 8);
    *reinterpret_cast<float4*>(v) = p[0];
    *reinterpret_cast<float4*>(v + 4) = p[1];
    for (int s = 1; s < slices; ++s) {
        float u[8];
        const float4* q = reinterpret_cast<const float4*>(acc + s * slice + i * 8);
        *reinterpret_cast<float4*>(u) = q[0];
        *reinterpret_cast<float4*>(u + 4) = q[1];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += u[e];
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

// ---- fp32: z^T's piece in memory ------------------------------------------------------

// A piece's blocks of kZRows vocabulary rows: {max, sum} per token and the labels'
// logits, as LseEpi leaves them.
constexpr int kZRows = 32;
__global__ __launch_bounds__(256) void xent_piece_lse(const float* __restrict__ z, int rows,
                                                      int64_t v0, int64_t tokens,
                                                      const int64_t* __restrict__ labels,
                                                      float2* __restrict__ part,
                                                      float* __restrict__ picked) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (t >= tokens) return;
    const int r0 = static_cast<int>(blockIdx.y) * kZRows;
    float v[kZRows];
#pragma unroll
    for (int r = 0; r < kZRows; ++r)
        v[r] = r0 + r < rows ? z[static_cast<int64_t>(r0 + r) * tokens + t] : -__builtin_inff();
    float m = v[0];
#pragma unroll
    for (int r = 1; r < kZRows; ++r) m = max_of(m, v[r]);
    const float shift = m == -__builtin_inff() ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < kZRows; ++r) s += exp_of(v[r] - shift);
    part[(v0 / kZRows + blockIdx.y) * tokens + t] = make_float2(m, s);
    const int at = label_row(labels[t], v0 + r0, kZRows);
    if (at >= 0 && r0 + at < rows) picked[t] = z[static_cast<int64_t>(r0 + at) * tokens + t];
}

// z^T's piece becomes G^T's.
__global__ __launch_bounds__(256) void xent_piece_grad(float* __restrict__ z, int rows, int64_t v0,
                                                       int64_t tokens,
                                                       const int64_t* __restrict__ labels,
                                                       const float2* __restrict__ stats,
                                                       const float* __restrict__ weight) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (t >= tokens) return;
    const int r0 = static_cast<int>(blockIdx.y) * kZRows;
    const float2 st = stats[t];
    const float w = weight[t];
    const int at = label_row(labels[t], v0 + r0, kZRows);
    float v[kZRows];
#pragma unroll
    for (int r = 0; r < kZRows; ++r)
        if (r0 + r < rows) v[r] = z[static_cast<int64_t>(r0 + r) * tokens + t];
#pragma unroll
    for (int r = 0; r < kZRows; ++r)
        if (r0 + r < rows) {
            float p = exp_of((v[r] - st.x) - st.y);
            p -= at == r ? 1.0f : 0.0f;
            z[static_cast<int64_t>(r0 + r) * tokens + t] = w != 0.0f ? w * p : 0.0f;
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
// bound by the matrix cores.  Backward on MI355X, us for pieces of 64 / 128 / 256 / 512 MiB / 1 GiB: 8192
// tokens x 4096 x 131072 22842 / 21095 / 20474 / 20068 / 20073; 4099 x 2048 x 50257 (pieces of
// 8192 / 16384 / 32768 rows, one piece) 2843 / 2805 / 2698 / 2444.
constexpr int64_t kPieceBytes = 512LL << 20;
constexpr int64_t kMaxOperand = 1LL << 30;    // values a product's 31-bit offsets reach
constexpr int64_t kMaxPiece = 1LL << 20;      // vocabulary rows, 32 per grid row of the fp32 kernels
constexpr int64_t kMaxTokens = 1LL << 24;     // a workgroup per token within a grid

// G's rows are padded to whole 128-byte lines of bf16: the products fetch 128 bytes of
// a row at a time, which at any other pitch straddle two lines.
constexpr int64_t kLine = 64;

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
inline size_t region(int64_t bytes) { return static_cast<size_t>(up(bytes, 256)); }

// The vocabulary rows of a piece: `asked`, or what fills kPieceBytes, cut to equal
// pieces of whole 256-row tiles that the products' offsets reach.
inline int64_t piece_rows(int64_t rows, int64_t vocab, int64_t ldw, int size, int64_t asked) {
    const int64_t row_bytes = up(rows, kLine) * size;
    int64_t p = asked > 0 ? up(std::min(asked, vocab), 256) : kPieceBytes / row_bytes;
    p = std::min(p, kMaxPiece);
    if (size == 2) p = std::min(p, std::min(kMaxOperand / ldw, kMaxOperand / up(rows, kLine)));
    p = std::max<int64_t>(p / 256 * 256, 256);
    if (p >= vocab) return vocab;
    const int64_t n = (vocab + p - 1) / p;
    return up((vocab + n - 1) / n, 256);
}

// The forward's tile: by the general rule, with the 32-row wave blocks of the 64-row
// tiles (ids 7 and 8: four times the partials) for few tokens only.
constexpr int64_t kFewTokens = 128;
inline int lse_shape(int64_t rows, int64_t vocab, int64_t cols) {
    using namespace agk_gemm;
    const int s = pick_shape(vocab, rows, cols, device_cus());
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
// Blocks per token that the workspace holds, whatever tile a device's compute units give.
inline int64_t max_blocks(int64_t rows, int64_t vocab, int dtype) {
    const int64_t least = dtype == AGK_BF16 && rows > kFewTokens ? 64 : 32;
    return (vocab + least - 1) / least;
}

// The tile and K slices of dx = G w.  K is the piece's vocabulary rows, far longer than
// the tokens by cols output is large: tiles that fill the last round of CUs badly are cut along K
// until they fill it, each slice with an fp32 output of its own (xent_dx_out adds
// them in order).  The cost: the tile rule's (pick_shape) per 64-deep step, plus what a
// round costs besides (its first loads and its stores) and the slices' traffic.
struct DxPlan {
    int shape, slices, k_slice;
};
inline DxPlan dx_plan(int64_t rows8, int64_t cols, int64_t k) {
    using namespace agk_gemm;
    const int64_t cus = device_cus();
    DxPlan best{pick_shape(rows8, cols, k, device_cus()), 1, static_cast<int>(up(k, 64))};
    double best_cost = 1e30;
    for (const RingCost& s : kRingCosts) {
        const int64_t tiles = ((rows8 + s.bm - 1) / s.bm) * ((cols + s.bn - 1) / s.bn);
        const double slots = static_cast<double>(cus * s.per_cu);
        for (int64_t n = 1; n <= kMaxSlices && (n == 1 || n * kMinSlice <= k); ++n) {
            if (k < BK || !agk::grid_fits(tiles, 256)) break;
            const int64_t ks = up((k + n - 1) / n, 64), m = (k + ks - 1) / ks;
            if (m != n || k - (n - 1) * ks < BK) continue;  // every slice has a whole k-tile
            const double load = static_cast<double>(tiles * n) / slots;
            const double rounds = static_cast<double>(static_cast<int64_t>(load));
            const double fill = load - rounds;
            const double steps = static_cast<double>(ks) / 64;
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
    return best;
}

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

// The backward's workspace.
struct Layout {
    int64_t piece, rows8, ldg;
    size_t weight, alpha, keep, g, acc, total;
};
inline Layout bwd_layout(int64_t rows, int64_t vocab, int64_t cols, int64_t ldw, int dtype,
                         int64_t piece) {
    Layout o;
    const int size = dtype == AGK_F32 ? 4 : 2;
    o.rows8 = up(rows, 8);
    o.ldg = dtype == AGK_F32 ? rows : up(rows, kLine);
    o.piece = piece_rows(rows, vocab, ldw, size, piece);
    o.weight = 0;
    o.alpha = o.weight + region(o.rows8 * 4);
    o.keep = o.alpha + region(4);
    o.g = o.keep + region(rows * cols * size);
    o.acc = o.g + region(o.piece * o.ldg * size);
    o.total = o.acc;
    if (dtype == AGK_BF16) {
        const DxPlan d = dx_plan(o.rows8, cols, o.piece);
        o.total += region(static_cast<int64_t>(d.slices) * o.rows8 * cols * 4);
    }
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
    if (rows == 0) return AGK_OK;
    if (!x || !w || ldx < cols || ldw < cols) return AGK_EINVAL;
    if (rows > INT64_MAX / 16 / ldx || vocab > INT64_MAX / 16 / ldw) return AGK_EINVAL;
    if (dtype == AGK_BF16) {
        if (cols % 8 || ldx % 8 || ldw % 8 || !aligned16(x) || !aligned16(w)) return AGK_EINVAL;
        if (256 * ldw > kMaxOperand || 256 * ldx > kMaxOperand) return AGK_EINVAL;
    } else if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 3u) {
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

}  // namespace agk_xent

extern "C" {

size_t agk_linear_xent_fwd_workspace_bytes(int64_t rows, int64_t vocab, int64_t cols, int dtype) {
    using namespace agk_xent;
    if (rows <= 0 || vocab <= 0 || cols <= 0 || !agk::valid_dtype(dtype)) return 0;
    size_t b = region(rows * 4) + region(max_blocks(rows, vocab, dtype) * rows * 8);
    if (dtype == AGK_F32) b += region(piece_rows(rows, vocab, cols, 4, 0) * rows * 4);
    return b;
}

int agk_linear_xent_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const int64_t* labels, float* loss, float* stats, void* workspace,
                        size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t cols,
                        int dtype, agk_stream_t stream) {
    using namespace agk_xent;
    const int rc = check_args(x, ldx, w, ldw, rows, vocab, cols, dtype);
    if (rc != AGK_OK || rows == 0) return rc;
    if (!labels || !loss || !stats || ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(labels)) & 7u))
        return AGK_EINVAL;
    if (!workspace ||
        workspace_bytes < agk_linear_xent_fwd_workspace_bytes(rows, vocab, cols, dtype))
        return AGK_EWORKSPACE;
    if (!aligned16(workspace)) return AGK_EINVAL;
    agk::clear_pending_error();
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    char* const ws = static_cast<char*>(workspace);
    float* const picked = reinterpret_cast<float*>(ws);
    float2* const part = reinterpret_cast<float2*>(ws + region(rows * 4));
    float2* const out = reinterpret_cast<float2*>(stats);
    if (dtype == AGK_BF16) {
        const int shape = lse_shape(rows, vocab, cols);
        const int block = lse_block(shape);
        const Product p{static_cast<const uint16_t*>(w), ldw, static_cast<const uint16_t*>(x), ldx,
                        static_cast<int>(vocab), static_cast<int>(rows), static_cast<int>(cols), 1,
                        0, st};
        const LseEpi e{part, picked, labels, static_cast<int>(vocab), static_cast<int>(rows)};
        const int r = launch_lse(shape, p, e);
        if (r != AGK_OK) return r;
        return launch_join(part, (vocab + block - 1) / block, picked, labels, loss, out, rows,
                           vocab, st);
    }
    const int64_t piece = piece_rows(rows, vocab, cols, 4, 0);
    float* const z = reinterpret_cast<float*>(
        ws + region(rows * 4) + region(max_blocks(rows, vocab, dtype) * rows * 8));
    for (int64_t v0 = 0; v0 < vocab; v0 += piece) {
        const int64_t n = std::min(piece, vocab - v0);
        int r = agk_gemm_f32(static_cast<const float*>(w) + v0 * ldw, ldw, 0,
                             static_cast<const float*>(x), ldx, 1, z, rows, n, rows, cols, 0,
                             stream);
        if (r != AGK_OK) return r;
        hipLaunchKernelGGL(xent_piece_lse,
                           dim3(static_cast<unsigned>((rows + 255) / 256),
                                static_cast<unsigned>((n + kZRows - 1) / kZRows)),
                           dim3(256), 0, st, z, static_cast<int>(n), v0, rows, labels, part,
                           picked);
        r = check_launch();
        if (r != AGK_OK) return r;
    }
    return launch_join(part, (vocab + kZRows - 1) / kZRows, picked, labels, loss, out, rows, vocab,
                       st);
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
        const int64_t n = vocab * cols * dw_size / 4;
        hipLaunchKernelGGL(xent_zero, dim3(agk::capped_blocks((n + 255) / 256, 256)), dim3(256), 0,
                           st, static_cast<uint32_t*>(dw), n);
        return check_launch();
    }
    if (!labels || !stats || !dloss ||
        ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(labels)) & 7u))
        return AGK_EINVAL;
    if (!dx && !dw) return AGK_OK;
    if (dtype == AGK_BF16) {
        if (dx && !aligned16(dx)) return AGK_EINVAL;
        if (rows > kMaxOperand / std::max(ldx, cols)) return AGK_EINVAL;
    } else if (dx && (reinterpret_cast<uintptr_t>(dx) & 3u)) {
        return AGK_EINVAL;
    }
    Layout o = bwd_layout(rows, vocab, cols, cols, dtype, piece);
    if (!workspace || workspace_bytes < o.total) return AGK_EWORKSPACE;
    if (!aligned16(workspace)) return AGK_EINVAL;
    // a wider ldw may need smaller pieces than the workspace was sized for
    if (dtype == AGK_BF16) o.piece = std::min(o.piece, piece_rows(rows, vocab, ldw, 2, piece));
    agk::clear_pending_error();
    char* const ws = static_cast<char*>(workspace);
    float* const weight = reinterpret_cast<float*>(ws + o.weight);
    float* const alpha = reinterpret_cast<float*>(ws + o.alpha);
    float* const acc = reinterpret_cast<float*>(ws + o.acc);
    const float2* const in = reinterpret_cast<const float2*>(stats);
    const bool bf16 = dtype == AGK_BF16;
    if (bf16)
        hipLaunchKernelGGL(xent_weights<true>, dim3(1), dim3(1024), 0, st, dloss, labels, weight,
                           alpha, rows, o.rows8, vocab);
    else
        hipLaunchKernelGGL(xent_weights<false>, dim3(1), dim3(1024), 0, st, dloss, labels, weight,
                           alpha, rows, o.rows8, vocab);
    if ((rc = check_launch()) != AGK_OK) return rc;
    if (dw) {
        const dim3 grid(static_cast<unsigned>(rows));
        if (bf16)
            hipLaunchKernelGGL(xent_keep_rows<agk::u32x4>, grid, dim3(256), 0, st,
                               static_cast<const agk::u32x4*>(x), ldx / 8, weight,
                               reinterpret_cast<agk::u32x4*>(ws + o.keep),
                               static_cast<int>(cols / 8));
        else
            hipLaunchKernelGGL(xent_keep_rows<float>, grid, dim3(256), 0, st,
                               static_cast<const float*>(x), ldx, weight,
                               reinterpret_cast<float*>(ws + o.keep), static_cast<int>(cols));
        if ((rc = check_launch()) != AGK_OK) return rc;
    }
    const int cus = agk_gemm::device_cus();
    const int64_t slice = o.rows8 * cols;
    DxPlan plan{0, 1, 0};
    if (bf16) plan = dx_plan(o.rows8, cols, o.piece);
    for (int64_t v0 = 0; v0 < vocab; v0 += o.piece) {
        const int64_t n = std::min(o.piece, vocab - v0);
        if (!bf16) {
            float* const z = reinterpret_cast<float*>(ws + o.g);
            const float* const wp = static_cast<const float*>(w) + v0 * ldw;
            rc = agk_gemm_f32(wp, ldw, 0, static_cast<const float*>(x), ldx, 1, z, rows, n, rows,
                              cols, 0, stream);
            if (rc != AGK_OK) return rc;
            hipLaunchKernelGGL(xent_piece_grad,
                               dim3(static_cast<unsigned>((rows + 255) / 256),
                                    static_cast<unsigned>((n + kZRows - 1) / kZRows)),
                               dim3(256), 0, st, z, static_cast<int>(n), v0, rows, labels, in,
                               weight);
            if ((rc = check_launch()) != AGK_OK) return rc;
            if (dx) {
                rc = agk_gemm_f32(z, rows, 1, wp, ldw, 0, static_cast<float*>(dx), cols, rows,
                                  cols, n, acc_dx || v0 > 0, stream);
                if (rc != AGK_OK) return rc;
            }
            if (dw) {
                rc = agk_gemm_f32(z, rows, 0, reinterpret_cast<const float*>(ws + o.keep), cols, 0,
                                  static_cast<float*>(dw) + v0 * cols, cols, n, cols, rows, acc_dw,
                                  stream);
                if (rc != AGK_OK) return rc;
            }
            continue;
        }
        const uint16_t* const wp = static_cast<const uint16_t*>(w) + v0 * ldw;
        uint16_t* const g = reinterpret_cast<uint16_t*>(ws + o.g);
        const int ldg = static_cast<int>(o.ldg), m = static_cast<int>(n);
        const Product zp{wp, ldw, static_cast<const uint16_t*>(x), ldx, m, static_cast<int>(rows),
                         static_cast<int>(cols), 1, 0, st};
        const GradEpi ge{g, in, weight, labels, v0, ldg, m, static_cast<int>(rows)};
        rc = launch_grad(agk_gemm::pick_shape(n, rows, cols, cus), zp, ge);
        if (rc != AGK_OK) return rc;
        if (dx) {
            DxPlan d = plan;
            if (n != o.piece) d = last_piece(plan, n);
            const int m8 = static_cast<int>(o.rows8);
            const Product dp{g, ldg, wp, ldw, m8, static_cast<int>(cols), m, d.slices, d.k_slice,
                             st};
            const AddEpi<true> de{acc, cols, slice, nullptr, m8, static_cast<int>(cols), v0 > 0};
            if ((rc = launch_dx(d.shape, dp, de)) != AGK_OK) return rc;
        }
        if (dw) {
            const Product wpd{g, ldg, reinterpret_cast<const uint16_t*>(ws + o.keep), cols, m,
                              static_cast<int>(cols), static_cast<int>(rows), 1, 0, st};
            const int shape = agk_gemm::pick_shape(n, cols, rows, cus);
            char* const out = static_cast<char*>(dw) + v0 * cols * dw_size;
            if (dw_dtype == AGK_F32)
                rc = launch_dw(shape, wpd, AddEpi<true>{out, cols, 0, alpha, m,
                                                        static_cast<int>(cols), acc_dw});
            else
                rc = launch_dw(shape, wpd, AddEpi<false>{out, cols, 0, alpha, m,
                                                         static_cast<int>(cols), acc_dw});
            if (rc != AGK_OK) return rc;
        }
    }
    if (bf16 && dx) {
        const int64_t n8 = rows * cols / 8;
        hipLaunchKernelGGL(xent_dx_out, dim3(static_cast<unsigned>((n8 + 255) / 256)), dim3(256), 0,
                           st, acc, plan.slices, slice, alpha, weight, static_cast<uint16_t*>(dx), n8,
                           static_cast<int>(cols / 8), acc_dx);
        return check_launch();
    }
    return AGK_OK;
}

}  // extern "C"
