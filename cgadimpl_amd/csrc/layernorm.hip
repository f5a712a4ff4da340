// layernorm.hip -- backward of LayerNorm with weight and bias (agk_layernorm_affine_bwd;
// the forward is LnAffineFwd in rowops.hip):
//   xhat = (x - mean) * rstd,  h = dy * gamma
//   dx (+)= rstd * (h - sum(h)/cols - xhat * sum(h * xhat)/cols)
//   dgamma (+)= sum_rows dy * xhat,  dbeta (+)= sum_rows dy
//
// One pass: a workgroup of up to 1024 lanes takes every nblk-th group of G rows, each row held
// in registers by TPR lanes (NV 16-byte slots of x and of dy per lane), and the next
// rows' loads are issued before the current rows are reduced.  Each lane adds its
// columns' dgamma and dbeta terms in fp32 over its rows; the workgroup's sums are one
// partial row of each, and a second kernel adds the partial rows in fp64 in a fixed
// order (no atomics: bit-identical run to run).  HBM-bound: x and dy read once, dx
// written once; 16384 x 8192 bf16 137 us on MI355X (5.9 TB/s) and 4.6 for the second kernel.
// One workgroup per CU that loops, not one per group of rows: the partial rows are then
// 256 whatever the rows are, and their two writes and reads stay in the caches.  4099 x 1030
// f32: 13.8 + 3.9 us, bound by latency (5.4 groups of rows per workgroup).  Rows of less than
// one slot, or too wide for registers, take a looped kernel that reads x and dy twice.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "agk_rowops.h"
#include "rowcommon.hpp"

namespace agk {
namespace layernorm {

constexpr int kLanes = 1024;
constexpr int kBlocks = 256;  // workgroups, one per CU, and partial rows

// (TPR, NV): lanes of a row and 16-byte slots per lane; 1024 / TPR rows at a time.  Rows of
// more than a wave take the fewest whole waves that hold them, of the steps below: with
// powers of two 4099 f32 rows of 1030 columns (258 slots) left half of the lanes idle, and
// with 1024 lanes alone 8192 x 8193 bf16 took 172 us (640 lanes of two slots: 121), f32 200
// (158).
#define AGK_LN_SHAPES(X)                                                                 \
    X(1, 1) X(2, 1) X(4, 1) X(8, 1) X(16, 1) X(32, 1) X(64, 1) X(128, 1) X(192, 1)       \
    X(256, 1) X(320, 1) X(512, 1) X(640, 1) X(768, 1) X(1024, 1)                \
    X(640, 2) X(768, 2) X(1024, 2) X(640, 4) X(768, 4) X(1024, 4)

// The widest shape's 32 columns of bf16 a lane do not fit its registers.
template <class S>
constexpr bool enabled(int nv) {
    return !(std::is_same<S, BF16>::value && nv == 4);
}

// The widest shapes' sums of dgamma and dbeta (16 columns a lane, 128 KiB a workgroup) lie in LDS,
// each lane's own: in registers beside two rows they spilled (MI355X, us, so / now: 8192 x 16384
// f32 661 / 300, 5.4 TB/s; bf16 395 / 151).
template <class S>
constexpr bool lds_sums(int nv) {
    return nv * S::kVec >= 16;
}

template <class T>
struct Args {
    const T* x;
    const T* gamma;  // NULL: ones
    const float* mean;
    const float* rstd;
    const T* dy;
    T* dx;           // NULL: not wanted
    float* partial;  // [2][nblk][cols]: dgamma's rows, then dbeta's; NULL: not wanted
    int64_t rows;
    int cols;
    int accumulate;  // into dx
};

template <bool RAG, class S>
__device__ __forceinline__ u32x4 load_row(const typename S::T* p) {
    return RAG ? load16_any_stream<S>(p) : load16_stream<S>(p);
}

// Two row sums at once.
template <int TPR, int G>
__device__ __forceinline__ void row_sum2(float& a, float& b,
                                         float2 (*red)[TPR > 64 ? G * (TPR / 64) : 1], int parity) {
    a = group_sum<TPR>(a);
    b = group_sum<TPR>(b);
    if constexpr (TPR > 64) {
        constexpr int kW = TPR / 64;
        const int wave = static_cast<int>(threadIdx.x % TPR) >> 6, row = threadIdx.x / TPR;
        if ((threadIdx.x & 63) == 0) red[parity][row * kW + wave] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            const float2 v = red[parity][row * kW + w];
            a += v.x;
            b += v.y;
        }
    }
}

template <class S, int NV>
struct Set {
    u32x4 x[NV], dy[NV];
    float mean, rstd;
};

template <class S, int TPR, int NV, bool RAG>
__global__ __launch_bounds__(kLanes / TPR * TPR) void ln_bwd(const Args<typename S::T> p) {
    using T = typename S::T;
    constexpr int W = S::kVec;
    constexpr int G = kLanes / TPR;
    constexpr bool kLdsSums = lds_sums<S>(NV);
    constexpr int kQuads = NV * W / 4;  // of a lane's columns
    __shared__ float2 red[2][TPR > 64 ? G * (TPR / 64) : 1];
    __shared__ float4 sums[kLdsSums ? 2 * kQuads * TPR : 1];  // [dgamma, dbeta][quad][lane]
    extern __shared__ float part[];  // G > 1: [G][cols]
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int cols = p.cols;
    const float inv_cols = 1.0f / static_cast<float>(cols);

    int col[NV], dup[NV];  // dup: leading elements the slot before holds too
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (t + k * TPR) * W;
        col[k] = slot_col<RAG, W>(t + k * TPR, cols);
        dup[k] = RAG && col[k] < c ? c - col[k] : 0;
    }
    float gm[NV][W];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (p.gamma && col[k] < cols)
            S::unpack(RAG ? load16_any<S>(p.gamma + col[k]) : load16<S>(p.gamma + col[k]), gm[k]);
        else
#pragma unroll
            for (int e = 0; e < W; ++e) gm[k][e] = 1.0f;
    }
    float dg[NV][W], db[NV][W];  // kLdsSums: of one row
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e) dg[k][e] = db[k][e] = 0.0f;
    if constexpr (kLdsSums) {
#pragma unroll
        for (int q = 0; q < 2 * kQuads; ++q) sums[q * TPR + t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    auto add = [](float4& s, const float* v) {
        s.x += v[0];
        s.y += v[1];
        s.z += v[2];
        s.w += v[3];
    };

    const int64_t stride = static_cast<int64_t>(gridDim.x) * G;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * G;
    const int64_t steps = (p.rows - first + stride - 1) / stride;  // the grid has no idle workgroup
    // rows past the end: the last one again, which nothing is added from or stored to
    auto issue = [&](Set<S, NV>& s, int64_t step) {
        const int64_t r = first + grp + step * stride;
        const int64_t row = r < p.rows ? r : p.rows - 1;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t at = row * cols + (col[k] < cols ? col[k] : 0);
            s.x[k] = load_row<RAG, S>(p.x + at);
            s.dy[k] = load_row<RAG, S>(p.dy + at);
        }
        s.mean = p.mean[row];
        s.rstd = p.rstd[row];
    };
    auto process = [&](const Set<S, NV>& s, int64_t step, int parity) {
        const int64_t r = first + grp + step * stride;
        const bool active = r < p.rows;
        float sh = 0.0f, shx = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float fx[W], fd[W];
            S::unpack(s.x[k], fx);
            S::unpack(s.dy[k], fd);
            const bool in = active && col[k] < cols;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float xhat = (fx[e] - s.mean) * s.rstd;
                const bool take = in && (!RAG || e >= dup[k]);
                const float d = take ? fd[e] : 0.0f;
                const float h = d * gm[k][e];
                const float xh = take ? xhat : 0.0f;
                sh += h;
                shx += h * xh;
                if constexpr (kLdsSums) {
                    dg[k][e] = d * xh;
                    db[k][e] = d;
                } else {
                    dg[k][e] += d * xh;
                    db[k][e] += d;
                }
            }
            if constexpr (kLdsSums) {
#pragma unroll
                for (int q = 0; q < W / 4; ++q) {
                    add(sums[(k * (W / 4) + q) * TPR + t], dg[k] + q * 4);
                    add(sums[(kQuads + k * (W / 4) + q) * TPR + t], db[k] + q * 4);
                }
            }
        }
        row_sum2<TPR, G>(sh, shx, red, parity);
        if (!p.dx || !active) return;
        const float mh = sh * inv_cols, mhx = shx * inv_cols;
        T* const dx = p.dx + r * cols;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (col[k] >= cols) continue;
            float fx[W], fd[W], o[W];
            S::unpack(s.x[k], fx);
            S::unpack(s.dy[k], fd);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float xhat = (fx[e] - s.mean) * s.rstd;
                o[e] = s.rstd * (fd[e] * gm[k][e] - mh - xhat * mhx);
            }
            if (p.accumulate) {
                if (RAG && dup[k]) {  // the slot before adds the elements both hold
                    for (int e = 0; e < W; ++e)
                        if (e >= dup[k]) S::put(dx + col[k] + e, acc_add(S::get(dx + col[k] + e), o[e]));
                    continue;
                }
                float old[W];
                S::unpack(load_row<RAG, S>(dx + col[k]), old);
#pragma unroll
                for (int e = 0; e < W; ++e) o[e] = acc_add(old[e], o[e]);
            }
            if constexpr (RAG) store16_any_stream<S>(dx + col[k], S::pack(o));
            else store16_stream<S>(dx + col[k], S::pack(o));
        }
    };
    Set<S, NV> a, b;
    issue(a, 0);
    for (int64_t s = 0; s < steps; s += 2) {
        issue(b, s + 1);
        process(a, s, 0);
        issue(a, s + 2);
        if (s + 1 < steps) process(b, s + 1, 1);
    }

    if (!p.partial) return;
    if constexpr (kLdsSums) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int q = 0; q < W / 4; ++q) {
                const float4 g = sums[(k * (W / 4) + q) * TPR + t];
                const float4 b4 = sums[(kQuads + k * (W / 4) + q) * TPR + t];
                dg[k][q * 4] = g.x, dg[k][q * 4 + 1] = g.y;
                dg[k][q * 4 + 2] = g.z, dg[k][q * 4 + 3] = g.w;
                db[k][q * 4] = b4.x, db[k][q * 4 + 1] = b4.y;
                db[k][q * 4 + 2] = b4.z, db[k][q * 4 + 3] = b4.w;
            }
    }
    const int64_t nblk = gridDim.x;
    float* const out[2] = {p.partial + blockIdx.x * static_cast<int64_t>(cols),
                           p.partial + (nblk + blockIdx.x) * static_cast<int64_t>(cols)};
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (G == 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (col[k] < cols) {
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        if (e >= dup[k]) out[which][col[k] + e] = which ? db[k][e] : dg[k][e];
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (col[k] < cols) {
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        if (e >= dup[k]) part[grp * cols + col[k] + e] = which ? db[k][e] : dg[k][e];
                }
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += TPR * G) {  // in group order
                float v = part[c];
                for (int q = 1; q < G; ++q) v += part[q * cols + c];
                out[which][c] = v;
            }
        }
    }
}

// Any width and alignment: a row at a time per workgroup, each lane's own columns of
// the workgroup's partial rows summed in memory.
template <class S>
__global__ __launch_bounds__(256) void ln_bwd_looped(const Args<typename S::T> p) {
    using T = typename S::T;
    __shared__ float2 red[2][4];
    const int cols = p.cols;
    const float inv_cols = 1.0f / static_cast<float>(cols);
    const int64_t nblk = gridDim.x;
    float* const pg = p.partial ? p.partial + blockIdx.x * static_cast<int64_t>(cols) : nullptr;
    float* const pb = pg ? pg + nblk * cols : nullptr;
    int parity = 0;
    for (int64_t r = blockIdx.x; r < p.rows; r += nblk) {
        const T* const x = p.x + r * cols;
        const T* const dy = p.dy + r * cols;
        const float mean = p.mean[r], rstd = p.rstd[r];
        float sh = 0.0f, shx = 0.0f;
        for (int64_t c = threadIdx.x; c < cols; c += 256) {
            const float h = S::get(dy + c) * (p.gamma ? S::get(p.gamma + c) : 1.0f);
            sh += h;
            shx += h * ((S::get(x + c) - mean) * rstd);
        }
        row_sum2<256, 1>(sh, shx, red, parity);
        parity ^= 1;
        const float mh = sh * inv_cols, mhx = shx * inv_cols;
        for (int64_t c = threadIdx.x; c < cols; c += 256) {
            const float d = S::get(dy + c);
            const float h = d * (p.gamma ? S::get(p.gamma + c) : 1.0f);
            const float xhat = (S::get(x + c) - mean) * rstd;
            if (pg) {
                const bool fresh = r == blockIdx.x;
                pg[c] = (fresh ? 0.0f : pg[c]) + d * xhat;
                pb[c] = (fresh ? 0.0f : pb[c]) + d;
            }
            if (p.dx) {
                const float v = rstd * (h - mh - xhat * mhx);
                T* const o = p.dx + r * cols + c;
                S::put(o, p.accumulate ? acc_add(S::get(o), v) : v);
            }
        }
    }
}

// dgamma and dbeta (grid y) from the partial rows: 32 columns per workgroup, 32 lanes to
// a column's partial rows, kFinBatch of them loaded before any is added; fp64, in a
// fixed order.
constexpr int kFinCols = 32, kFinSplits = 32, kFinBatch = 8;
__global__ __launch_bounds__(kFinCols* kFinSplits) void ln_finalize(
    const float* __restrict__ partial, int64_t nblk, int cols, float* __restrict__ dgamma,
    float* __restrict__ dbeta, int acc_gamma, int acc_beta) {
    __shared__ double red[kFinSplits][kFinCols];
    float* const out = blockIdx.y ? dbeta : dgamma;
    if (!out) return;
    const int tx = threadIdx.x % kFinCols, ty = threadIdx.x / kFinCols;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kFinCols + tx;
    const float* const p = partial + blockIdx.y * nblk * cols + (c < cols ? c : cols - 1);
    double s = 0.0;
    for (int64_t b = ty; b < nblk; b += kFinSplits * kFinBatch) {
        float v[kFinBatch];
#pragma unroll
        for (int u = 0; u < kFinBatch; ++u) {
            const int64_t at = b + u * kFinSplits;
            v[u] = p[(at < nblk ? at : nblk - 1) * cols];
        }
#pragma unroll
        for (int u = 0; u < kFinBatch; ++u) s += b + u * kFinSplits < nblk ? v[u] : 0.0f;
    }
    red[ty][tx] = s;
    __syncthreads();
    if (ty != 0 || c >= cols) return;
    for (int y = 1; y < kFinSplits; ++y) s += red[y][tx];
    const float v = static_cast<float>(s);
    const int acc = blockIdx.y ? acc_beta : acc_gamma;
    out[c] = acc ? acc_add(out[c], v) : v;
}

__global__ __launch_bounds__(256) void ln_zero(float* __restrict__ a, float* __restrict__ b,
                                               int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        if (a) a[i] = 0.0f;
        if (b) b[i] = 0.0f;
    }
}

struct Shape {
    int tpr = 0, nv = 0;  // tpr == 0: the looped kernel
};
template <class S>
inline Shape pick(int64_t cols) {
    Shape s;
    const int64_t slots = row_slots(cols, S::kVec);
    if (cols < S::kVec || slots > 4096) return s;
    const int nv = slots <= 1024 ? 1 : slots <= 2048 ? 2 : 4;
    if (!enabled<S>(nv)) return s;
    constexpr int kTpr[] = {1, 2, 4, 8, 16, 32, 64, 128, 192, 256, 320, 512, 640, 768, 1024};
    s.nv = nv;
    s.tpr = 1024;
    for (int tpr : kTpr)
        if ((nv == 1 || tpr >= 640) && static_cast<int64_t>(tpr) * nv >= slots) {
            s.tpr = tpr;
            break;
        }
    return s;
}

// Workgroups: one per CU, none without a row.  The same bound for every path, so that the
// workspace depends on rows and cols alone.
inline int64_t blocks(int64_t rows, int g) {
    return std::min<int64_t>((rows + g - 1) / g, kBlocks);
}

template <class S>
int launch(const Args<typename S::T>& a, int64_t* nblk, hipStream_t st) {
    const bool vec = a.cols % S::kVec == 0 && aligned16(a.x) && aligned16(a.dy) &&
                     (!a.dx || aligned16(a.dx)) && (!a.gamma || aligned16(a.gamma));
    const Shape s = pick<S>(a.cols);
    if (s.tpr == 0) {
        *nblk = blocks(a.rows, 1);
        hipLaunchKernelGGL(ln_bwd_looped<S>, dim3(static_cast<unsigned>(*nblk)), dim3(256), 0, st,
                           a);
        return check_launch();
    }
    const int g = kLanes / s.tpr;
    *nblk = blocks(a.rows, g);
    // few groups of rows each: as many workgroups as have the same number of them, which is as
    // quick and leaves fewer partial rows (MI355X, us: 300 x 16384 f32 43 -> 35, 300 x 8192 22 -> 18)
    const int64_t groups = (a.rows + g - 1) / g, each = (groups + *nblk - 1) / *nblk;
    if (each <= 4) *nblk = (groups + each - 1) / each;
    const size_t lds = g > 1 && a.partial ? static_cast<size_t>(g) * a.cols * 4 : 0;
    const dim3 grid(static_cast<unsigned>(*nblk)), block(g * s.tpr);
#define AGK_X(TPR, NV)                                                                      \
    if constexpr (enabled<S>(NV)) {                                                         \
        if (s.tpr == TPR && s.nv == NV) {                                                   \
            if (vec) hipLaunchKernelGGL((ln_bwd<S, TPR, NV, false>), grid, block, lds, st, a); \
            else hipLaunchKernelGGL((ln_bwd<S, TPR, NV, true>), grid, block, lds, st, a);   \
            return check_launch();                                                          \
        }                                                                                   \
    }
    AGK_LN_SHAPES(AGK_X)
#undef AGK_X
    return AGK_EINVAL;
}

template <class S>
int run(const void* x, const void* gamma, const float* mean, const float* rstd, const void* dy,
        void* dx, float* dgamma, float* dbeta, float* partial, int64_t rows, int64_t cols,
        int accumulate, hipStream_t st) {
    using T = typename S::T;
    Args<T> a;
    a.x = static_cast<const T*>(x);
    a.gamma = static_cast<const T*>(gamma);
    a.mean = mean;
    a.rstd = rstd;
    a.dy = static_cast<const T*>(dy);
    a.dx = static_cast<T*>(dx);
    a.partial = dgamma || dbeta ? partial : nullptr;
    a.rows = rows;
    a.cols = static_cast<int>(cols);
    a.accumulate = accumulate & AGK_ACCUM_DX;
    int64_t nblk = 0;
    const int rc = launch<S>(a, &nblk, st);
    if (rc != AGK_OK || !a.partial) return rc;
    const int acc_g = (accumulate & AGK_ACCUM_DGAMMA) != 0;
    const int acc_b = (accumulate & AGK_ACCUM_DBETA) != 0;
    hipLaunchKernelGGL(ln_finalize,
                       dim3(static_cast<unsigned>((cols + kFinCols - 1) / kFinCols), 2),
                       dim3(kFinCols * kFinSplits), 0, st, partial, nblk, static_cast<int>(cols),
                       dgamma, dbeta, acc_g, acc_b);
    return check_launch();
}

}  // namespace layernorm
}  // namespace agk

extern "C" {

size_t agk_layernorm_affine_bwd_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || agk::check_sizes(rows, cols) != AGK_OK) return 0;
    return static_cast<size_t>(agk::layernorm::blocks(rows, 1)) * cols * 8;
}

int agk_layernorm_affine_bwd(const void* x, const void* gamma, const float* mean,
                             const float* rstd, const void* dy, void* dx, float* dgamma,
                             float* dbeta, void* workspace, size_t workspace_bytes, int64_t rows,
                             int64_t cols, int dtype, int accumulate, agk_stream_t stream) {
    using namespace agk;
    if (!valid_dtype(dtype)) return AGK_EDTYPE;
    const int rc = check_sizes(rows, cols);
    if (rc != AGK_OK) return rc;
    if (accumulate & ~(AGK_ACCUM_ALL | AGK_ACCUM_DBETA)) return AGK_EINVAL;
    if (cols == 0 || (!dx && !dgamma && !dbeta)) return AGK_OK;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (rows == 0) {
        float* const g = accumulate & AGK_ACCUM_DGAMMA ? nullptr : dgamma;
        float* const b = accumulate & AGK_ACCUM_DBETA ? nullptr : dbeta;
        if (!g && !b) return AGK_OK;
        clear_pending_error();
        hipLaunchKernelGGL(layernorm::ln_zero, dim3(capped_blocks((cols + 255) / 256, 256)),
                           dim3(256), 0, st, g, b, cols);
        return check_launch();
    }
    if (!x || !mean || !rstd || !dy) return AGK_EINVAL;
    if (dgamma || dbeta) {
        if (!workspace || workspace_bytes < agk_layernorm_affine_bwd_workspace_bytes(rows, cols))
            return AGK_EWORKSPACE;
        if (reinterpret_cast<uintptr_t>(workspace) & 3u) return AGK_EINVAL;
    }
    clear_pending_error();
    float* const partial = static_cast<float*>(workspace);
    return dtype == AGK_F32
               ? layernorm::run<F32>(x, gamma, mean, rstd, dy, dx, dgamma, dbeta, partial, rows,
                                     cols, accumulate, st)
               : layernorm::run<BF16>(x, gamma, mean, rstd, dy, dx, dgamma, dbeta, partial, rows,
                                      cols, accumulate, st);
}

}  // extern "C"
