// distill.hip -- distillation from a teacher's top logits (agk_distill_topk_fwd,
// agk_distill_topk_bwd).  Per row of student logits z, against the teacher's logits t_j
// of the columns i_j:
//   q = softmax(z / T),  p = softmax(t / T) over the entries,
//   loss = T^2 sum_j p_j (log p_j - log q[i_j]),   dz = dloss T (q - sum_{j: i_j = v} p_j)
//
// Both passes stream z: the forward reads it once, keeping a running maximum and sum
// per lane, the backward reads it once and writes dz.  The teacher's part is a few
// hundred values a row.  HBM bounds them.  A row is one workgroup's; rows too few to fill the chip are
// cut into segments, whose {max, sum} meet in a second kernel (forward), or which
// are independent, each computing the row's p again (backward).

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "agk_losses.h"
#include "rowcommon.hpp"

namespace agk {
namespace distill {

constexpr int kLanes = 256;
constexpr int kWaves = kLanes / 64;
constexpr int kMaxK = AGK_DISTILL_MAX_K;
constexpr int kPerLane = kMaxK / kLanes;  // entries of the teacher a lane holds
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float max_of(float a, float b) {  // one v_max_f32; drops a NaN
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// Reductions over the workgroup; every lane gets the result.  `red` is free again
// after the barrier of the next call, so calls alternate between two arrays.
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int h = 32; h > 0; h /= 2) v = max_of(v, __shfl_xor(v, h));
    return v;
}
__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = max_of(v, red[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += red[w];
    return v;
}

struct Args {
    const void* z;
    const int64_t* index;
    const void* t;
    int t_bf16;
    int64_t rows, cols;
    int k;
    int segs;          // segments per row
    int64_t seg_cols;  // columns of a segment (a multiple of 8; the last may have fewer)
    float temperature, scale;  // scale = log2(e) / T
};

// A row's teacher as the lanes hold it: entry j = lane + i * kLanes.
struct Teacher {
    int64_t index[kPerLane];  // < 0: no entry
    float p[kPerLane], logp[kPerLane];
    bool any, bad;  // an entry with a probability; a column past the last
};

// red: three arrays of kWaves floats.
__device__ __forceinline__ void load_teacher(const Args& a, int64_t row, Teacher& o,
                                             float (*red)[kWaves]) {
    float t[kPerLane];
    float top = -__builtin_inff();
    int flags = 0;
    const int64_t base = row * a.k;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int j = static_cast<int>(threadIdx.x) + i * kLanes;
        o.index[i] = -1;
        t[i] = -__builtin_inff();
        if (j < a.k) {
            o.index[i] = a.index[base + j];
            const float v = a.t_bf16 ? BF16::get(static_cast<const uint16_t*>(a.t) + base + j)
                                     : static_cast<const float*>(a.t)[base + j];
            if (o.index[i] >= 0) {
                t[i] = v;
                if (!(v == -__builtin_inff())) flags |= 1;
                if (o.index[i] >= a.cols) flags |= 2;
            }
        }
        top = max_of(top, t[i]);
    }
    const bool any = __syncthreads_or(flags & 1), bad = __syncthreads_or(flags & 2);
    o.any = any;
    o.bad = bad;
    top = block_max(top, red[0]);
    float e[kPerLane], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        e[i] = t[i] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((t[i] - top) * a.scale);
        sum += e[i];
    }
    sum = block_sum(sum, red[1]);
    const float logs = logf(sum);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        o.p[i] = e[i] / sum;
        o.logp[i] = (t[i] - top) / a.temperature - logs;
    }
}

template <class S>
__device__ __forceinline__ void seg_range(const Args& a, int seg, int64_t& c0, int& n) {
    c0 = static_cast<int64_t>(seg) * a.seg_cols;
    const int64_t left = a.cols - c0;
    n = static_cast<int>(left < a.seg_cols ? left : a.seg_cols);
}

// Running {max, sum of 2^((z - max) * scale)}.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float scale) {
    const float top = max_of(m, m2);
    const float x = m == top ? s : s * __builtin_amdgcn_exp2f((m - top) * scale);
    const float y = m2 == top ? s2 : s2 * __builtin_amdgcn_exp2f((m2 - top) * scale);
    m = top;
    s = x + y;
}

// {max, sum} of a segment, in lane 0.
constexpr int kBatch = 4;  // 16-byte loads in flight per lane
template <class S>
__device__ __forceinline__ void seg_lse(const Args& a, int64_t row, int seg, float& m, float& s,
                                        float2* red) {
    using T = typename S::T;
    constexpr int W = S::kVec;
    int64_t c0;
    int n;
    seg_range<S>(a, seg, c0, n);
    const T* const z = static_cast<const T*>(a.z) + row * a.cols + c0;
    m = -__builtin_inff();
    s = 0.0f;
    const int nvec = n / W;
    for (int v0 = threadIdx.x; v0 < nvec; v0 += kLanes * kBatch) {
        u32x4 raw[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int v = v0 + u * kLanes;
            raw[u] = load16_any_stream<S>(z + static_cast<int64_t>(v < nvec ? v : v0) * W);
        }
        float f[kBatch][W];
        float top = m;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            S::unpack(raw[u], f[u]);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                if (v0 + u * kLanes >= nvec) f[u][e] = -__builtin_inff();
                top = max_of(top, f[u][e]);
            }
        }
        const float shift = top == -__builtin_inff() ? 0.0f : top;
        // before the first finite value s is 0, or a NaN already met
        float sum = m == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f((m - shift) * a.scale);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int e = 0; e < W; ++e) sum += __builtin_amdgcn_exp2f((f[u][e] - shift) * a.scale);
        m = top;
        s = sum;
    }
    const int c = nvec * W + static_cast<int>(threadIdx.x);
    if (c < n) {
        const float v = S::get(z + c);
        const float top = max_of(m, v);
        const float shift = top == -__builtin_inff() ? 0.0f : top;
        s = (m == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f((m - shift) * a.scale)) +
            __builtin_amdgcn_exp2f((v - shift) * a.scale);
        m = top;
    }
#pragma unroll
    for (int h = 32; h > 0; h /= 2) {
        const float m2 = __shfl_xor(m, h), s2 = __shfl_xor(s, h);
        join(m, s, m2, s2, a.scale);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(m, s);
    __syncthreads();
    m = red[0].x;
    s = red[0].y;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) join(m, s, red[w].x, red[w].y, a.scale);
}

// The row's loss from its {max, sum}; called by the whole workgroup.
template <class S>
__device__ __forceinline__ void row_loss(const Args& a, int64_t row, float m, float s, float* loss,
                                         float2* stats, float (*red)[kWaves]) {
    using T = typename S::T;
    const T* const z = static_cast<const T*>(a.z) + row * a.cols;
    const float l = logf(s);
    Teacher t;
    load_teacher(a, row, t, red);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
        if (t.index[i] >= 0 && t.index[i] < a.cols && !(t.p[i] == 0.0f)) {
            const float logq = (S::get(z + t.index[i]) - m) / a.temperature - l;
            v += t.p[i] * (t.logp[i] - logq);
        }
    v = block_sum(v, red[2]);
    if (threadIdx.x == 0) {
        stats[row] = make_float2(m, l);
        loss[row] = t.bad ? __builtin_nanf("") : t.any ? a.temperature * a.temperature * v : 0.0f;
    }
}

// One workgroup per row (segs == 1), looping over what the grid leaves.
template <class S>
__global__ __launch_bounds__(kLanes) void distill_fwd(const Args a, float* __restrict__ loss,
                                                      float2* __restrict__ stats) {
    __shared__ float2 red2[kWaves];
    __shared__ float red[3][kWaves];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float m, s;
        seg_lse<S>(a, row, 0, m, s, red2);
        row_loss<S>(a, row, m, s, loss, stats, red);
        __syncthreads();
    }
}

// Segments: part[row * segs + seg].
template <class S>
__global__ __launch_bounds__(kLanes) void distill_part(const Args a, float2* __restrict__ part) {
    __shared__ float2 red2[kWaves];
    const int64_t row = blockIdx.x / static_cast<unsigned>(a.segs);
    const int seg = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.segs));
    float m, s;
    seg_lse<S>(a, row, seg, m, s, red2);
    if (threadIdx.x == 0) part[blockIdx.x] = make_float2(m, s);
}

template <class S>
__global__ __launch_bounds__(kLanes) void distill_join(const Args a, const float2* __restrict__ part,
                                                       float* __restrict__ loss,
                                                       float2* __restrict__ stats) {
    __shared__ float red[3][kWaves];
    const int64_t row = blockIdx.x;
    float m = -__builtin_inff(), s = 0.0f;
    for (int i = threadIdx.x & 63; i < a.segs; i += 64) {
        const float2 v = part[row * a.segs + i];
        join(m, s, v.x, v.y, a.scale);
    }
#pragma unroll
    for (int h = 32; h > 0; h /= 2) {
        const float m2 = __shfl_xor(m, h), s2 = __shfl_xor(s, h);
        join(m, s, m2, s2, a.scale);
    }
    row_loss<S>(a, row, m, s, loss, stats, red);
}

// dz of one segment of one row.
template <class S>
__global__ __launch_bounds__(kLanes) void distill_bwd(const Args a, const float2* __restrict__ stats,
                                                      const float* __restrict__ dloss, void* dz_,
                                                      int accumulate) {
    using T = typename S::T;
    constexpr int W = S::kVec;
    __shared__ float red[3][kWaves];
    __shared__ int at[kMaxK];   // column within the segment; -1: elsewhere
    __shared__ float prob[kMaxK];
    for (int64_t item = blockIdx.x; item < a.rows * a.segs; item += gridDim.x) {
        const int64_t row = item / a.segs;
        int64_t c0;
        int n;
        seg_range<S>(a, static_cast<int>(item - row * a.segs), c0, n);
        const int64_t base = row * a.cols + c0;
        const T* const z = static_cast<const T*>(a.z) + base;
        T* const dz = static_cast<T*>(dz_) + base;
        Teacher t;
        load_teacher(a, row, t, red);
        const float2 st = stats[row];
        const float c = t.bad ? __builtin_nanf("") : t.any ? dloss[row] * a.temperature : 0.0f;
        auto grad = [&](float v) {
            return c * __builtin_amdgcn_exp2f((v - st.x) * a.scale - st.y * kLog2e);
        };
        // The columns the teacher named: what they need of z and the old dz is read
        // before any of dz is written.
        float own_z[kPerLane], own_old[kPerLane];
        int own_at[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int j = static_cast<int>(threadIdx.x) + i * kLanes;
            const int64_t r = t.index[i] - c0;
            own_at[i] = t.index[i] >= 0 && r >= 0 && r < n ? static_cast<int>(r) : -1;
            own_z[i] = own_old[i] = 0.0f;
            if (own_at[i] >= 0) {
                own_z[i] = S::get(z + own_at[i]);
                if (accumulate) own_old[i] = S::get(dz + own_at[i]);
            }
            if (j < a.k) {
                at[j] = own_at[i];
                prob[j] = t.p[i];
            }
        }
        __syncthreads();
        const int nvec = n / W;
        if (c == 0.0f) {
            if (!accumulate) {
                const u32x4 zero = {0u, 0u, 0u, 0u};
                for (int v = threadIdx.x; v < nvec; v += kLanes)
                    store16_any_stream<S>(dz + static_cast<int64_t>(v) * W, zero);
                const int e = nvec * W + static_cast<int>(threadIdx.x);
                if (e < n) S::put(dz + e, 0.0f);
            }
        } else {
            for (int v0 = threadIdx.x; v0 < nvec; v0 += kLanes * kBatch) {
                u32x4 raw[kBatch], old[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int v = v0 + u * kLanes;
                    const int64_t e = static_cast<int64_t>(v < nvec ? v : v0) * W;
                    raw[u] = load16_any_stream<S>(z + e);
                    if (accumulate) old[u] = load16_any_stream<S>(dz + e);
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int v = v0 + u * kLanes;
                    if (v >= nvec) continue;
                    float f[W];
                    S::unpack(raw[u], f);
#pragma unroll
                    for (int e = 0; e < W; ++e) f[e] = grad(f[e]);
                    if (accumulate) {
                        float o[W];
                        S::unpack(old[u], o);
#pragma unroll
                        for (int e = 0; e < W; ++e) f[e] = acc_add(o[e], f[e]);
                    }
                    store16_any_stream<S>(dz + static_cast<int64_t>(v) * W, S::pack(f));
                }
            }
            const int e = nvec * W + static_cast<int>(threadIdx.x);
            if (e < n) {
                const float g = grad(S::get(z + e));
                S::put(dz + e, accumulate ? acc_add(S::get(dz + e), g) : g);
            }
            // The named columns again, after every store of the segment: q - sum of
            // their p.  Entries of one column all write the same value.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                if (own_at[i] < 0) continue;
                float p = 0.0f;
                for (int j = 0; j < a.k; ++j) p += at[j] == own_at[i] ? prob[j] : 0.0f;
                const float g = grad(own_z[i]) - c * p;
                S::put(dz + own_at[i], accumulate ? acc_add(own_old[i], g) : g);
            }
        }
        __syncthreads();
    }
}

// Segments of a row: enough workgroups to fill the chip (8 of 256 lanes per CU), of
// at least kMinSeg columns.
constexpr int64_t kFill = 2048;
constexpr int64_t kMinSeg = 2048;
inline int segments(int64_t rows, int64_t cols) {
    const int64_t want = (kFill + rows - 1) / rows, most = (cols + kMinSeg - 1) / kMinSeg;
    int64_t s = std::max<int64_t>(std::min(want, most), 1);
    const int64_t w = ((cols + s - 1) / s + 7) / 8 * 8;
    return static_cast<int>((cols + w - 1) / w);
}

inline int check(int64_t rows, int64_t cols, int64_t k, float temperature, int dtype, int t_dtype) {
    if (!valid_dtype(dtype) || !valid_dtype(t_dtype)) return AGK_EDTYPE;
    const int rc = check_sizes(rows, cols);
    if (rc != AGK_OK) return rc;
    if (k < 0 || k > kMaxK || !(temperature >= 1e-4f && temperature <= 1e4f)) return AGK_EINVAL;
    if (rows > 0 && cols == 0) return AGK_EINVAL;
    if (rows > INT64_MAX / 16 / std::max<int64_t>(k, 1)) return AGK_EINVAL;
    return AGK_OK;
}

inline Args args(const void* z, const int64_t* index, const void* t, int64_t rows, int64_t cols,
                 int64_t k, float temperature, int t_dtype) {
    Args a;
    a.z = z;
    a.index = index;
    a.t = t;
    a.t_bf16 = t_dtype == AGK_BF16;
    a.rows = rows;
    a.cols = cols;
    a.k = static_cast<int>(k);
    a.segs = segments(rows, cols);
    a.seg_cols = ((cols + a.segs - 1) / a.segs + 7) / 8 * 8;
    a.temperature = temperature;
    a.scale = static_cast<float>(1.4426950408889634 / temperature);
    return a;
}

template <class S>
int forward(const Args& a, float* loss, float2* stats, float2* part, hipStream_t st) {
    if (a.segs == 1) {
        hipLaunchKernelGGL(distill_fwd<S>, dim3(capped_blocks(a.rows, kLanes)), dim3(kLanes), 0, st,
                           a, loss, stats);
        return check_launch();
    }
    hipLaunchKernelGGL(distill_part<S>, dim3(static_cast<unsigned>(a.rows * a.segs)), dim3(kLanes),
                       0, st, a, part);
    const int rc = check_launch();
    if (rc != AGK_OK) return rc;
    hipLaunchKernelGGL(distill_join<S>, dim3(static_cast<unsigned>(a.rows)), dim3(kLanes), 0, st, a,
                       part, loss, stats);
    return check_launch();
}

}  // namespace distill
}  // namespace agk

extern "C" {

size_t agk_distill_topk_workspace_bytes(int64_t rows, int64_t cols) {
    using namespace agk::distill;
    if (rows <= 0 || cols <= 0 || agk::check_sizes(rows, cols) != AGK_OK) return 0;
    const int s = segments(rows, cols);
    return s > 1 ? static_cast<size_t>(rows) * s * sizeof(float2) : 0;
}

int agk_distill_topk_fwd(const void* z, const int64_t* index, const void* t, float* loss,
                         float* stats, void* workspace, size_t workspace_bytes, int64_t rows,
                         int64_t cols, int64_t k, float temperature, int dtype, int t_dtype,
                         agk_stream_t stream) {
    using namespace agk::distill;
    const int rc = check(rows, cols, k, temperature, dtype, t_dtype);
    if (rc != AGK_OK || rows == 0) return rc;
    if (!z || !loss || !stats || (k > 0 && (!index || !t))) return AGK_EINVAL;
    if ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(index)) & 7u)
        return AGK_EINVAL;
    const size_t need = agk_distill_topk_workspace_bytes(rows, cols);
    if (need && (!workspace || workspace_bytes < need)) return AGK_EWORKSPACE;
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 7u)) return AGK_EINVAL;
    agk::clear_pending_error();
    const Args a = args(z, index, t, rows, cols, k, temperature, t_dtype);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    float2* const out = reinterpret_cast<float2*>(stats);
    float2* const part = static_cast<float2*>(workspace);
    return dtype == AGK_F32 ? forward<agk::F32>(a, loss, out, part, st)
                            : forward<agk::BF16>(a, loss, out, part, st);
}

int agk_distill_topk_bwd(const void* z, const int64_t* index, const void* t, const float* stats,
                         const float* dloss, void* dz, int64_t rows, int64_t cols, int64_t k,
                         float temperature, int dtype, int t_dtype, int accumulate,
                         agk_stream_t stream) {
    using namespace agk::distill;
    const int rc = check(rows, cols, k, temperature, dtype, t_dtype);
    if (rc != AGK_OK) return rc;
    if (accumulate & ~AGK_ACCUM_DX) return AGK_EINVAL;
    if (rows == 0) return AGK_OK;
    if (!z || !stats || !dloss || !dz || (k > 0 && (!index || !t))) return AGK_EINVAL;
    if ((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(index)) & 7u)
        return AGK_EINVAL;
    const int64_t bytes = rows * cols * (dtype == AGK_F32 ? 4 : 2);
    if (dz != z && !agk::disjoint(dz, z, bytes)) return AGK_EINVAL;
    agk::clear_pending_error();
    const Args a = args(z, index, t, rows, cols, k, temperature, t_dtype);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const float2* const in = reinterpret_cast<const float2*>(stats);
    const dim3 grid(agk::capped_blocks(rows * a.segs, kLanes));
    const int acc = accumulate != 0;
    if (dtype == AGK_F32)
        hipLaunchKernelGGL(distill_bwd<agk::F32>, grid, dim3(kLanes), 0, st, a, in, dloss, dz, acc);
    else
        hipLaunchKernelGGL(distill_bwd<agk::BF16>, grid, dim3(kLanes), 0, st, a, in, dloss, dz,
                           acc);
    return agk::check_launch();
}

}  // extern "C"
