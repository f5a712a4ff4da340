// distill.hip -- distillation from a teacher's top logits (agk_distill_topk_fwd,
// agk_distill_topk_bwd).  Per row of student logits z, against the teacher's logits t_j
// of the columns i_j:
//   q = softmax(z / T),  p = softmax(t / T) over the entries,
//   loss = T^2 sum_j p_j (log p_j - log q[i_j]),   dz = dloss T (q - sum_{j: i_j = v} p_j)
//
// Both passes stream z: the forward reads it once, keeping a running maximum and sum
// per lane, the backward reads it once and writes dz.  The teacher's part is a few
// hundred values a row.  HBM bounds them: 8192 x 50257 bf16, k = 64, 135 us forward (6.1 TB/s) and
// 270 backward (6.1) on MI355X.  In the forward a row is one workgroup's; a few very wide rows
// are cut into segments, whose {max, sum} meet in a second kernel, and where rows are many each
// is a wave's; the backward takes a row in chunks always, each computing the row's p again.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "agk_losses.h"
#include "rowcommon.hpp"

namespace agk {
namespace distill {

constexpr int kLanes = 256;
constexpr int kWaves = kLanes / 64;
constexpr int kMaxK = AGK_DISTILL_MAX_K;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float max_of(float a, float b) {  // one v_max_f32; drops a NaN
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int h = 32; h > 0; h /= 2) v = max_of(v, __shfl_xor(v, h));
    return v;
}

struct Args {
    const void* z;
    const int64_t* index;
    const void* t;
    int t_bf16;
    int64_t rows, cols;
    int k;
    int segs;          // segments per row (the forward of very wide rows; else 1)
    int64_t seg_cols;  // columns of a segment (a multiple of 8; the last may have fewer)
    float temperature, scale;  // scale = log2(e) / T
};

// A row's teacher, held by one wave: PER entries per lane, entry j in lane j % 64.  A wave works
// it out by itself, without a barrier: two loads, a maximum and a sum over 64 lanes.
template <int PER>
struct Teacher {
    int64_t index[PER];  // as loaded
    int at[PER];         // column; -1: no entry
    float p[PER];        // t, after exponentials() exp((t - top) / T); p = that / sum
    float top, sum;
    bool any, bad;       // an entry with a probability; a column past the last

    __device__ __forceinline__ void load(const Args& a, int64_t row) {
        const int lane = static_cast<int>(threadIdx.x & 63);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int j = i * 64 + lane;
            index[i] = -1;
            p[i] = 0.0f;
            if (a.k) {  // uniform; lanes past the entries load the first one
                const int64_t e = row * a.k + (j < a.k ? j : 0);
                index[i] = a.index[e];
                p[i] = a.t_bf16 ? BF16::get(static_cast<const uint16_t*>(a.t) + e)
                                : static_cast<const float*>(a.t)[e];
            }
        }
    }
    __device__ __forceinline__ void place(const Args& a) {
        const int lane = static_cast<int>(threadIdx.x & 63);
        top = -__builtin_inff();
        any = bad = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool in = i * 64 + lane < a.k && index[i] >= 0;
            if (!in) p[i] = -__builtin_inff();
            any = any || !(p[i] == -__builtin_inff());
            bad = bad || (in && index[i] >= a.cols);
            at[i] = in && index[i] < a.cols ? static_cast<int>(index[i]) : -1;
            top = max_of(top, p[i]);
        }
        any = __any(any);
        bad = __any(bad);
        top = wave_max(top);
    }
    __device__ __forceinline__ void exponentials(const Args& a) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            p[i] = p[i] == -__builtin_inff() ? 0.0f
                                             : __builtin_amdgcn_exp2f((p[i] - top) * a.scale);
            sum += p[i];
        }
        sum = group_sum<64>(sum);
    }
};

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

// A segment as its elements before the first 16-byte boundary (at most W - 1), a body of
// whole 16-byte slots and the elements after it (at most W - 1): rows of odd widths start
// at any element, and 16-byte accesses off their boundary run at 5.8 of 6.4 TB/s.
struct Parts {
    int head, slots, tail0;  // tail0: the first element after the body
};
template <class S>
__device__ __forceinline__ Parts parts_of(const void* p, int n) {
    using T = typename S::T;
    constexpr int W = S::kVec;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
    Parts q;
    q.head = off ? W - off : 0;
    if (q.head > n) q.head = n;
    q.slots = (n - q.head) / W;
    q.tail0 = q.head + q.slots * W;
    return q;
}
// The element of head or tail that lane t has (-1: none).
__device__ __forceinline__ int edge(const Parts& q, int n, int t) {
    const int c = t < 8 ? (t < q.head ? t : -1) : t < 16 ? q.tail0 + t - 8 : -1;
    return c < n ? c : -1;
}

// A lane's running maximum m and sum s of 2^((z - m) scale).  The exponent is one fma,
// z scale - t with t = m scale rounded once; what the rounding left, d = m scale - t, is
// exact as an fma and goes into the sum as 2^-d, so that sums of different m add up as if
// t were exact.  Where m scale overflows (logits of 1e38, or masks of the type's lowest
// value and nothing else) the difference is formed first.
struct Lse {
    float m, s;
    template <int N>
    __device__ __forceinline__ void add(const float (&f)[N], float scale) {
        float top = m;
#pragma unroll
        for (int e = 0; e < N; ++e) top = max_of(top, f[e]);
        if (top == -__builtin_inff()) {  // s stays 0, or takes a NaN
#pragma unroll
            for (int e = 0; e < N; ++e) s += f[e] == f[e] ? 0.0f : f[e];
            return;
        }
        if (top != m) s = m == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f((m - top) * scale);
        m = top;
        const float t = top * scale;
        float sum = 0.0f;
        if (__builtin_fabsf(t) < 1e37f) {
#pragma unroll
            for (int e = 0; e < N; ++e)
                sum += __builtin_amdgcn_exp2f(__builtin_fmaf(f[e], scale, -t));
            s += sum * __builtin_amdgcn_exp2f(-__builtin_fmaf(top, scale, -t));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) s += __builtin_amdgcn_exp2f((f[e] - top) * scale);
        }
    }
};

// {max, sum} of a segment, in every lane of a workgroup of LANES, or of a wave (LANES = 64).
constexpr int kBatch = 4;  // 16-byte loads in flight per lane
template <class S, int LANES>
__device__ __forceinline__ void seg_lse(const Args& a, int64_t row, int seg, float& m, float& s,
                                        float2* red) {
    using T = typename S::T;
    constexpr int W = S::kVec;
    int64_t c0;
    int n;
    seg_range(a, seg, c0, n);
    const T* const z = static_cast<const T*>(a.z) + row * a.cols + c0;
    const Parts q = parts_of<S>(z, n);
    const u32x4* const body = reinterpret_cast<const u32x4*>(z + q.head);
    Lse r{-__builtin_inff(), 0.0f};
    const int lane = static_cast<int>(LANES == 64 ? threadIdx.x & 63 : threadIdx.x);
    int v = lane;
    for (; v + (kBatch - 1) * LANES < q.slots; v += LANES * kBatch) {
        u32x4 raw[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) raw[u] = __builtin_nontemporal_load(body + v + u * LANES);
        float f[kBatch * W];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            float g[W];
            S::unpack(raw[u], g);
#pragma unroll
            for (int e = 0; e < W; ++e) f[u * W + e] = g[e];
        }
        r.add(f, a.scale);
    }
    for (; v < q.slots; v += LANES) {
        float f[W];
        S::unpack(__builtin_nontemporal_load(body + v), f);
        r.add(f, a.scale);
    }
    if (const int c = edge(q, n, lane); c >= 0) {
        const float f[1] = {S::get(z + c)};
        r.add(f, a.scale);
    }
    m = r.m;
    s = r.s;
#pragma unroll
    for (int h = 32; h > 0; h /= 2) {
        const float m2 = __shfl_xor(m, h), s2 = __shfl_xor(s, h);
        join(m, s, m2, s2, a.scale);
    }
    if constexpr (LANES == 64) return;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(m, s);
    __syncthreads();
    m = red[0].x;
    s = red[0].y;
#pragma unroll
    for (int w = 1; w < LANES / 64; ++w) join(m, s, red[w].x, red[w].y, a.scale);
}

// The named columns' z, loaded before the row is streamed; then the row's loss from its
// {max, sum}.  Both by one wave.
template <class S, int PER>
__device__ __forceinline__ void named_z(const Args& a, int64_t row, const Teacher<PER>& t,
                                        float (&zt)[PER]) {
    const typename S::T* const z = static_cast<const typename S::T*>(a.z) + row * a.cols;
#pragma unroll
    for (int i = 0; i < PER; ++i) zt[i] = t.at[i] >= 0 ? S::get(z + t.at[i]) : 0.0f;
}
template <int PER>
__device__ __forceinline__ void row_loss(const Args& a, int64_t row, float m, float s,
                                         Teacher<PER>& t, const float (&zt)[PER], float* loss,
                                         float2* stats) {
    float logp[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) logp[i] = (t.p[i] - t.top) / a.temperature;
    t.exponentials(a);
    const float l = logf(s), logs = logf(t.sum);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float p = t.p[i] / t.sum;
        const float logq = (zt[i] - m) / a.temperature - l;
        v += t.at[i] >= 0 && !(p == 0.0f) ? p * (logp[i] - logs - logq) : 0.0f;
    }
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) {
        stats[row] = make_float2(m, l);
        loss[row] = t.bad ? __builtin_nanf("") : t.any ? a.temperature * a.temperature * v : 0.0f;
    }
}

// One workgroup per row, looping over what the grid leaves.  Its first wave has the
// teacher's part.
template <class S, int LANES, int PER>
__global__ __launch_bounds__(LANES) void distill_fwd(const Args a, float* __restrict__ loss,
                                                     float2* __restrict__ stats) {
    __shared__ float2 red[LANES / 64];
    const bool first = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)) == 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Teacher<PER> t;
        float zt[PER];
        if (first) {
            t.load(a, row);
            t.place(a);
            named_z<S, PER>(a, row, t, zt);
        }
        float m, s;
        seg_lse<S, LANES>(a, row, 0, m, s, red);
        if (first) row_loss<PER>(a, row, m, s, t, zt, loss, stats);
        __syncthreads();
    }
}

// One wave per row, four rows per workgroup.
template <class S, int PER>
__global__ __launch_bounds__(kLanes) void distill_fwd_wave(const Args a, float* __restrict__ loss,
                                                           float2* __restrict__ stats) {
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves +
                       __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
         row < a.rows; row += static_cast<int64_t>(gridDim.x) * kWaves) {
        Teacher<PER> t;
        float zt[PER], m, s;
        t.load(a, row);
        t.place(a);
        named_z<S, PER>(a, row, t, zt);
        seg_lse<S, 64>(a, row, 0, m, s, nullptr);
        row_loss<PER>(a, row, m, s, t, zt, loss, stats);
    }
}

// Segments: part[row * segs + seg].
template <class S>
__global__ __launch_bounds__(kLanes) void distill_part(const Args a, float2* __restrict__ part) {
    __shared__ float2 red[kWaves];
    const int64_t row = blockIdx.x / static_cast<unsigned>(a.segs);
    const int seg = static_cast<int>(blockIdx.x % static_cast<unsigned>(a.segs));
    float m, s;
    seg_lse<S, kLanes>(a, row, seg, m, s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = make_float2(m, s);
}

// A wave per row.
template <class S, int PER>
__global__ __launch_bounds__(64) void distill_join(const Args a, const float2* __restrict__ part,
                                                   float* __restrict__ loss,
                                                   float2* __restrict__ stats) {
    const int64_t row = blockIdx.x;
    Teacher<PER> t;
    float zt[PER];
    t.load(a, row);
    t.place(a);
    named_z<S, PER>(a, row, t, zt);
    float m = -__builtin_inff(), s = 0.0f;
    for (int i = threadIdx.x; i < a.segs; i += 64) {
        const float2 v = part[row * a.segs + i];
        join(m, s, v.x, v.y, a.scale);
    }
#pragma unroll
    for (int h = 32; h > 0; h /= 2) {
        const float m2 = __shfl_xor(m, h), s2 = __shfl_xor(s, h);
        join(m, s, m2, s2, a.scale);
    }
    row_loss<PER>(a, row, m, s, t, zt, loss, stats);
}

// ---- backward ------------------------------------------------------------------------
// One wave per chunk of kChunk 16-byte slots of a row, four chunks in a row per workgroup
// and no barrier: a stream of reads and writes runs fastest where the chip works through
// memory in one compact window (copies: 6.05 TB/s with 16 KiB per workgroup, 4.2-5.2 with
// workgroups that loop over long rows; this kernel so, 352 us where it takes 270 now).  The
// wave issues its loads of z behind those of the row's teacher and computes p for itself while
// they are in flight (PER entries per lane, a maximum and a sum over the wave).  The entries
// whose column lies in the chunk are then taken one by one, in order: the column's slot and
// element are the same for the whole wave, so that one lane's register takes - c p.  Columns
// named twice need nothing more.
constexpr int kSlots = 4;              // 16-byte slots per lane
constexpr int kChunk = 64 * kSlots;    // and per wave

// Orders a wave's LDS accesses among its lanes (the hardware takes them in order).
__device__ __forceinline__ void lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// DENSE: chunks of many entries (from kDense on).  One by one they would take longer than the
// chunk's bytes; so their probabilities are added into an LDS array of the chunk's columns, 64
// at a time: the lanes claim their columns' places in a small table (the lowest lane gets it,
// so that a column's entries are added in their order), the winners add, the others try again.
template <class S>
struct Dense {
    static constexpr int kEdge = kChunk * S::kVec;  // head, then tail, behind the chunk's columns
    float delta[kEdge + 16];
    unsigned claim[256];

    __device__ __forceinline__ void clear(int lane) {
#pragma unroll
        for (int u = 0; u < kSlots; ++u)
#pragma unroll
            for (int e = 0; e < S::kVec; e += 4)
                *reinterpret_cast<float4*>(delta + (u * 64 + lane) * S::kVec + e) =
                    make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (lane < 16) delta[kEdge + lane] = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; ++u) claim[u * 64 + lane] = ~0u;
        lds_order();
    }
    // delta[pos] += p for lanes whose pos is not negative
    __device__ __forceinline__ void add(int pos, float p, int lane) {
        bool left = pos >= 0;
        const int place = pos & 255;
        while (__any(left)) {
            if (left) atomicMin(&claim[place], static_cast<unsigned>(lane));
            lds_order();
            const bool won = left && *const_cast<volatile unsigned*>(&claim[place]) ==
                                         static_cast<unsigned>(lane);
            lds_order();
            if (won) {
                delta[pos] += p;
                claim[place] = ~0u;
            }
            lds_order();
            left = left && !won;
        }
    }
};

template <class S, int PER, bool ACC, bool DENSE>
__global__ __launch_bounds__(kLanes, DENSE ? 3 : PER == 1 && !ACC ? 8 : PER <= 4 ? 5 : 3) void
distill_bwd(
    const Args a, const float2* __restrict__ stats, const float* __restrict__ dloss, void* dz_,
    int chunks) {
    using T = typename S::T;
    constexpr int W = S::kVec;
    __shared__ typename std::conditional<DENSE, Dense<S>, char>::type dense[kWaves];
    const int lane = static_cast<int>(threadIdx.x & 63);
    const int64_t items = a.rows * chunks;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves +
                        __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
         item < items; item += static_cast<int64_t>(gridDim.x) * kWaves) {
        const int64_t row = item / chunks;
        const int chunk = static_cast<int>(item - row * chunks);
        const int cols = static_cast<int>(a.cols);
        const T* const z = static_cast<const T*>(a.z) + row * a.cols;
        T* const dz = static_cast<T*>(dz_) + row * a.cols;
        const Parts q = parts_of<S>(z, cols);
        const u32x4* const zb = reinterpret_cast<const u32x4*>(z + q.head);
        T* const db = dz + q.head;  // 16-byte aligned where z and dz start alike
        // loads return in order: those that are needed first, first
        Teacher<PER> t;
        t.load(a, row);
        const float2 st = stats[row];
        const float weight = dloss[row];
        __builtin_amdgcn_sched_barrier(0);

        // the chunk's slots, and the edges with the first and the last chunk
        u32x4 raw[kSlots], old[ACC ? kSlots : 1];
#pragma unroll
        for (int u = 0; u < kSlots; ++u) {
            const int v = chunk * kChunk + u * 64 + lane;
            const int vc = v < q.slots ? v : 0;
            raw[u] = q.slots ? __builtin_nontemporal_load(zb + vc) : u32x4{0u, 0u, 0u, 0u};
            if constexpr (ACC)
                old[u] = q.slots ? load16_any_stream<S>(db + static_cast<int64_t>(vc) * W) : u32x4{0u, 0u, 0u, 0u};
        }
        int ec = -1;
        if (chunk == 0 && lane < q.head) ec = lane;
        if (chunk == chunks - 1 && lane >= 8 && q.tail0 + lane - 8 < cols) ec = q.tail0 + lane - 8;
        float ez = 0.0f, eold = 0.0f;
        if (ec >= 0) {
            ez = S::get(z + ec);
            if constexpr (ACC) eold = S::get(dz + ec);
        }
        __builtin_amdgcn_sched_barrier(0);

        t.place(a);
        t.exponentials(a);
        const float sum = t.sum;
        const float c = t.bad ? __builtin_nanf("") : t.any ? weight * a.temperature : 0.0f;
        const float l2 = st.y * kLog2e;
        auto grad = [&](float v) {
            return c * __builtin_amdgcn_exp2f(__builtin_fmaf(v - st.x, a.scale, -l2));
        };
        float f[kSlots][W];
        float eg = grad(ez);
#pragma unroll
        for (int u = 0; u < kSlots; ++u) {
            S::unpack(raw[u], f[u]);
#pragma unroll
            for (int e = 0; e < W; ++e) f[u][e] = grad(f[u][e]);
        }
        const int first = q.head + chunk * kChunk * W;  // the chunk's columns but the edges
        if constexpr (DENSE) {
            Dense<S>& d = dense[threadIdx.x >> 6];
            d.clear(lane);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = t.at[i], r = at - first;
                int pos = -1;
                if (at >= 0 && at < q.head)
                    pos = chunk == 0 ? Dense<S>::kEdge + at : -1;
                else if (at >= q.tail0)
                    pos = chunk == chunks - 1 ? Dense<S>::kEdge + 8 + at - q.tail0 : -1;
                else if (at >= 0 && r >= 0 && r < kChunk * W)
                    pos = r;
                d.add(pos, t.p[i], lane);
            }
            const float inv = 1.0f / sum;
            // (an untouched column keeps its value where c is not finite too)
            auto less = [&](float g, float p) { return p == 0.0f ? g : g - c * (p * inv); };
#pragma unroll
            for (int u = 0; u < kSlots; ++u)
#pragma unroll
                for (int e = 0; e < W; ++e)
                    f[u][e] = less(f[u][e], d.delta[(u * 64 + lane) * W + e]);
            if (lane < 16) eg = less(eg, d.delta[Dense<S>::kEdge + lane]);
            lds_order();
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int r = t.at[i] - first;
                const bool mine = t.at[i] >= 0 && ((r >= 0 && r < kChunk * W) ||
                                                 (chunk == 0 && r < 0) ||
                                                 (chunk == chunks - 1 && t.at[i] >= q.tail0));
                unsigned long long todo = __ballot(mine);
                while (todo) {
                    const int l = __builtin_ctzll(todo);
                    todo &= todo - 1;
                    const int col = __builtin_amdgcn_readlane(t.at[i], l);
                    const float d =
                        c * (__int_as_float(__builtin_amdgcn_readlane(__float_as_int(t.p[i]), l)) / sum);
                    if (col == ec) eg -= d;
                    const int rel = col - first;
                    if (rel < 0 || col >= q.tail0) continue;
                    const int slot = rel / W, elem = rel % W;
                    const float mine_d = lane == (slot & 63) ? d : 0.0f;
#pragma unroll
                    for (int u = 0; u < kSlots; ++u)
                        if (u == slot / 64) {
#pragma unroll
                            for (int e = 0; e < W; ++e)
                                if (e == elem) f[u][e] -= mine_d;
                        }
                }
            }
        }
        // a row without a teacher or weight: zeros, whatever z holds
        const bool zero = c == 0.0f;
#pragma unroll
        for (int u = 0; u < kSlots; ++u) {
            const int v = chunk * kChunk + u * 64 + lane;
#pragma unroll
            for (int e = 0; e < W; ++e) f[u][e] = zero ? 0.0f : f[u][e];
            if constexpr (ACC) {
                float o[W];
                S::unpack(old[u], o);
#pragma unroll
                for (int e = 0; e < W; ++e) f[u][e] = acc_add(o[e], f[u][e]);
            }
            if (v < q.slots) store16_any_stream<S>(db + static_cast<int64_t>(v) * W, S::pack(f[u]));
        }
        if (ec >= 0) {
            eg = zero ? 0.0f : eg;
            S::put(dz + ec, ACC ? acc_add(eold, eg) : eg);
        }
    }
}

// Segments of a row in the forward.  A few rows of many columns are cut into kMinSeg columns and
// more, kFill workgroups of them; else a row is one workgroup's, which reads 40 bytes a ns
// on a CU of its own, and saves the second kernel.  MI355X, us, whole / cut: f32 32 x 32000 6.3 /
// 8.0, 1 x 151936 15.9 / 7.9, 4 x 262144 20.6 / 8.2, bf16 96 x 131072 (256 KiB) 13.8 / 14.3.
constexpr int64_t kFill = 2048;
constexpr int64_t kMinSeg = 2048;
constexpr int64_t kWholeBytes = 320 << 10;
inline int segments(int64_t rows, int64_t cols, int dtype) {
    if (rows >= 256 || cols * (dtype == AGK_F32 ? 4 : 2) <= kWholeBytes) return 1;
    const int64_t want = (kFill + rows - 1) / rows, most = (cols + kMinSeg - 1) / kMinSeg;
    const int64_t s = std::min(want, most);
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
                 int64_t k, float temperature, int dtype, int t_dtype) {
    Args a;
    a.z = z;
    a.index = index;
    a.t = t;
    a.t_bf16 = t_dtype == AGK_BF16;
    a.rows = rows;
    a.cols = cols;
    a.k = static_cast<int>(k);
    a.segs = segments(rows, cols, dtype);
    a.seg_cols = ((cols + a.segs - 1) / a.segs + 7) / 8 * 8;
    a.temperature = temperature;
    a.scale = static_cast<float>(1.4426950408889634 / temperature);
    return a;
}

// Lanes of a row in the forward, by how many rows share the chip: a wave each from seven
// waves per CU on (no barrier, and four loads in flight each are enough), looping on three
// workgroups per CU where rows are long, which keeps the chip's accesses together; then
// workgroups of 256 lanes, of 512 and, up to one per CU, of 1024.  MI355X, us, 256 lanes /
// this: 20000 x 2000 bf16 43 / 28, 16384 x 8000 bf16 (k = 256) 103 / 77, 2048 x 50257 f32 72
// / 63 (6.6 TB/s), 8192 x 50257 bf16 132 / 130 (uncapped 141), 500 x 32000 bf16 11.4 / 10.4
// (1024 lanes 15.2), 300 x 50257 f32 22 / 16 (1024 lanes 20).  Waves for fewer rows: 1500 x
// 100000 bf16 64, 256 lanes 54; 512 lanes: 1000 x 150000 bf16 59, 256 lanes 54.
constexpr int64_t kWaveRows = 7 * 256, kGroupRows = 3 * 256;
constexpr int64_t kShortSlots = 2048, kLongGroups = 3 * 256;

template <class S, int PER>
int forward_per(const Args& a, float* loss, float2* stats, float2* part, hipStream_t st) {
    if (a.segs > 1) {
        hipLaunchKernelGGL(distill_part<S>, dim3(static_cast<unsigned>(a.rows * a.segs)),
                           dim3(kLanes), 0, st, a, part);
        const int rc = check_launch();
        if (rc != AGK_OK) return rc;
        hipLaunchKernelGGL((distill_join<S, PER>), dim3(static_cast<unsigned>(a.rows)), dim3(64), 0,
                           st, a, part, loss, stats);
        return check_launch();
    }
    const int64_t slots = a.cols / S::kVec;
    if (a.rows >= kWaveRows) {
        int64_t groups = (a.rows + kWaves - 1) / kWaves;
        if (slots > kShortSlots) groups = std::min(groups, kLongGroups);
        hipLaunchKernelGGL((distill_fwd_wave<S, PER>), dim3(capped_blocks(groups, kLanes)),
                           dim3(kLanes), 0, st, a, loss, stats);
        return check_launch();
    }
#define AGK_FWD(LANES)                                                                     \
    hipLaunchKernelGGL((distill_fwd<S, LANES, PER>), dim3(capped_blocks(a.rows, LANES)),   \
                       dim3(LANES), 0, st, a, loss, stats)
    if (a.rows >= kGroupRows || slots <= 1024) AGK_FWD(kLanes);
    else if (a.rows > 256) AGK_FWD(512);
    else AGK_FWD(1024);
#undef AGK_FWD
    return check_launch();
}
template <class S>
int forward(const Args& a, float* loss, float2* stats, float2* part, hipStream_t st) {
    if (a.k <= 64) return forward_per<S, 1>(a, loss, stats, part, st);
    if (a.k <= 256) return forward_per<S, 4>(a, loss, stats, part, st);
    return forward_per<S, kMaxK / 64>(a, loss, stats, part, st);
}

// Entries per chunk, were the columns even, from which the chunk takes them through LDS.  MI355X,
// us, one by one / so: 10.4 entries (8192 x 50257 bf16, k = 256) 322 / 336, 16 (20000 x 2000 bf16)
// 36 / 31, 26 (8192 x 20000 bf16) 183 / 138, 66 (16384 x 8000 bf16) 291 / 115, 102 (20000 x 2000
// f32) 218 / 59.
constexpr int kDense = 12;

template <class S, int PER>
int backward_per(const Args& a, const float2* stats, const float* dloss, void* dz, bool acc,
                 hipStream_t st) {
    const int64_t n = a.cols / S::kVec;  // slots at most
    const int chunks = static_cast<int>(std::max<int64_t>((n + kChunk - 1) / kChunk, 1));
    const int64_t groups = (a.rows * chunks + kWaves - 1) / kWaves;
    const dim3 grid(capped_blocks(groups, kLanes)), block(kLanes);
    constexpr int64_t kCols = kChunk * S::kVec;
    const bool dense = a.k * kCols >= kDense * std::max(a.cols, kCols);
#define AGK_BWD(ACC, DENSE)                                                                     \
    hipLaunchKernelGGL((distill_bwd<S, PER, ACC, DENSE>), grid, block, 0, st, a, stats, dloss,  \
                       dz, chunks)
    if (dense && acc) AGK_BWD(true, true);
    else if (dense) AGK_BWD(false, true);
    else if (acc) AGK_BWD(true, false);
    else AGK_BWD(false, false);
#undef AGK_BWD
    return check_launch();
}
template <class S>
int backward(const Args& a, const float2* stats, const float* dloss, void* dz, bool acc,
             hipStream_t st) {
    if (a.k <= 64) return backward_per<S, 1>(a, stats, dloss, dz, acc, st);
    if (a.k <= 256) return backward_per<S, 4>(a, stats, dloss, dz, acc, st);
    return backward_per<S, kMaxK / 64>(a, stats, dloss, dz, acc, st);
}

}  // namespace distill
}  // namespace agk

extern "C" {

size_t agk_distill_topk_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
    using namespace agk::distill;
    if (rows <= 0 || cols <= 0 || agk::check_sizes(rows, cols) != AGK_OK) return 0;
    if (!agk::valid_dtype(dtype)) return 0;
    const int s = segments(rows, cols, dtype);
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
    const size_t need = agk_distill_topk_workspace_bytes(rows, cols, dtype);
    if (need && (!workspace || workspace_bytes < need)) return AGK_EWORKSPACE;
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 7u)) return AGK_EINVAL;
    agk::clear_pending_error();
    const Args a = args(z, index, t, rows, cols, k, temperature, dtype, t_dtype);
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
    const Args a = args(z, index, t, rows, cols, k, temperature, dtype, t_dtype);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const float2* const in = reinterpret_cast<const float2*>(stats);
    const bool acc = accumulate != 0;
    return dtype == AGK_F32 ? backward<agk::F32>(a, in, dloss, dz, acc, st)
                            : backward<agk::BF16>(a, in, dloss, dz, acc, st);
}

}  // extern "C"
