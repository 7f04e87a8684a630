// Tokens sorted by expert, and their rows there and back.
//
//   offsets[e]  = chosen places (t, k) with an expert below e;  offsets[E] = all that have one
//   row_of[t,k] = offsets[e] + places of the same expert e in front of (t, k), in the order of t, then k;  -1: no expert
//   source[r]   = t K + k of row r;  -1 from offsets[E] on
//   gather      rows[row_of[t,k]] = x[t]                 gradient  dx[t] = sum_k drows[row_of[t,k]]
//   combine     out[t] = sum_k w[t,k] rows[row_of[t,k]]  gradient  drows[row_of[t,k]] = w[t,k] dout[t],
//                                                                  dw[t,k] = <dout[t], rows[row_of[t,k]]>
// Every sum runs in the order of k in 32 bits and is rounded once; there are no atomics, so every call gives the same bits.
#pragma once

#include <cooperative_groups.h>

#include "ops_common.cuh"

namespace kleos {
namespace sorting {
using namespace ops;

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kCluster = 8;

// One cluster sorts: block c takes the c-th share of the places, warp w of it the w-th share of those, 32 at a time in
// order, so a place's rank is what the blocks, the warps and the turns in front of it counted, and its rank among
// the lanes.  Counters: hist[w][e].
__global__ void __launch_bounds__(kThreads) sort_kernel(const int* topk, int n, int E, int* offsets, int* row_of, int* source) {
    namespace cg = cooperative_groups;
    extern __shared__ int hist[];          // [kWarps][E]
    __shared__ int mine[ops::kMaxExperts];  // this block's places of every expert
    __shared__ int base[ops::kMaxExperts];  // row of the block's first place of every expert
    __shared__ int scan[kWarps];
    __shared__ int filled;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    int* count = hist + warp * E;
    for (int i = tid; i < kWarps * E; i += kThreads) hist[i] = 0;
    // turns of 32 places, an equal number for every warp
    const long long turns = ((long long)n + 31) / 32, per = (turns + blocks * kWarps - 1) / (blocks * kWarps);
    const long long first = ((long long)block * kWarps + warp) * per, last = min(first + per, turns);
    __syncthreads();
    auto expert_at = [&](long long turn) {
        const long long i = turn * 32 + lane;
        const int e = i < n ? topk[i] : -1;
        return e < 0 || e >= E ? -1 : e;
    };
    // the places of expert e in front of this one in the warp's own share
    auto rank = [&](int e) {
        const unsigned same = __match_any_sync(0xffffffffu, e);
        const int before = __popc(same & ((1u << lane) - 1));
        const int r = e < 0 ? 0 : count[e] + before;
        __syncwarp();
        if (e >= 0 && before == 0) count[e] = r + __popc(same);
        __syncwarp();
        return r;
    };
    for (long long t = first; t < last; ++t) rank(expert_at(t));
    __syncthreads();
    // a thread per expert: the warps' counts become the places in front of each warp
    int total = 0;
    if (tid < E) {
        for (int w = 0; w < kWarps; ++w) {
            const int c = hist[w * E + tid];
            hist[w * E + tid] = total;
            total += c;
        }
        mine[tid] = total;
    }
    cluster.sync();
    int before = 0, all = 0;
    if (tid < E)
        for (int b = 0; b < blocks; ++b) {
            const int c = cluster.map_shared_rank(mine, b)[tid];
            if (b < block) before += c;
            all += c;
        }
    // exclusive sums over the experts
    int upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    int front = 0;
    for (int w = 0; w < warp; ++w) front += scan[w];
    upto += front;
    if (tid < E) {
        base[tid] = upto - all + before;
        if (block == 0) {
            offsets[tid] = upto - all;
            if (tid == E - 1) offsets[E] = upto;
        }
    }
    if (tid == E - 1) filled = upto;
    __syncthreads();
    for (long long t = first; t < last; ++t) {
        const int e = expert_at(t), r = rank(e);
        const long long i = t * 32 + lane;
        if (i >= n) continue;
        const int row = e < 0 ? -1 : base[e] + r;
        row_of[i] = row;
        if (source && row >= 0) source[row] = (int)i;
    }
    if (source)
        for (long long i = (long long)filled + block * kThreads + tid; i < n; i += (long long)blocks * kThreads) source[i] = -1;
    cluster.sync();  // (no block leaves while another may still read its counts)
}

struct Move {
    const void *from, *other;  // `other`: the rows whose product with dout is wanted
    void* to;
    const int *row_of, *offsets;
    const float* weights;
    float* dweights;
    long long ld;  // of the token matrix
    int T, K, E, H, n;  // n = T * K rows
};

// Rows that no place leads to are zeros: the tail, from offsets[E] on.
template <typename T, int V>
__device__ __forceinline__ void clear_tail(const Move& m) {
    if (!m.offsets) return;
    const int filled = min(max(m.offsets[m.E], 0), m.n);
    Vec<T, V> zero;
#pragma unroll
    for (int k = 0; k < V; ++k) zero.v[k] = Elem<T>::from_f(0.f);
    for (long long r = filled + blockIdx.x; r < m.n; r += gridDim.x)
        for (int j = threadIdx.x * V; j < m.H; j += blockDim.x * V) store_vec<T, V>(static_cast<T*>(m.to) + r * m.H + j, zero);
}

// A block a token: its row is read once and stored K times.
template <typename T, int V>
__global__ void __launch_bounds__(256) gather_kernel(Move m) {
    pdl_wait();
    pdl_trigger();
    for (long long t = blockIdx.x; t < m.T; t += gridDim.x) {
        const T* x = static_cast<const T*>(m.from) + t * m.ld;
        for (int j = threadIdx.x * V; j < m.H; j += blockDim.x * V) {
            const auto v = load_vec<T, V>(x + j);
            for (int k = 0; k < m.K; ++k) {
                const int r = m.row_of[t * m.K + k];
                if (r >= 0 && r < m.n) store_vec<T, V>(static_cast<T*>(m.to) + (long long)r * m.H + j, v);
            }
        }
    }
    clear_tail<T, V>(m);
}

// A block a token.  Without weights: the gradient of gather.
template <typename T, int V>
__global__ void __launch_bounds__(256) combine_kernel(Move m) {
    pdl_wait();
    pdl_trigger();
    for (long long t = blockIdx.x; t < m.T; t += gridDim.x) {
        T* out = static_cast<T*>(m.to) + t * m.ld;
        for (int j = threadIdx.x * V; j < m.H; j += blockDim.x * V) {
            float s[V];
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] = 0.f;
            for (int k = 0; k < m.K; ++k) {
                const int r = m.row_of[t * m.K + k];
                if (r < 0 || r >= m.n) continue;
                const float w = m.weights ? m.weights[t * m.K + k] : 1.f;
                const auto v = load_vec<T, V>(static_cast<const T*>(m.from) + (long long)r * m.H + j);
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] = fmaf(w, Elem<T>::to_f(v.v[i]), s[i]);
            }
            Vec<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = Elem<T>::from_f(s[i]);
            store_vec<T, V>(out + j, o);
        }
    }
}

// A block a token: dout[t] is read once for all its K rows.
template <typename T, int V>
__global__ void __launch_bounds__(256) combine_back_kernel(Move m) {
    __shared__ float part[kMaxTopK][8];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (long long t = blockIdx.x; t < m.T; t += gridDim.x) {
        const T* dout = static_cast<const T*>(m.from) + t * m.ld;
        float dot[kMaxTopK];
#pragma unroll
        for (int k = 0; k < kMaxTopK; ++k) dot[k] = 0.f;
        for (int j = threadIdx.x * V; j < m.H; j += 256 * V) {
            const auto d = load_vec<T, V>(dout + j);
#pragma unroll
            for (int k = 0; k < kMaxTopK; ++k) {
                if (k >= m.K) break;
                const int r = m.row_of[t * m.K + k];
                if (r < 0 || r >= m.n) continue;
                const float w = m.weights ? m.weights[t * m.K + k] : 1.f;
                const auto v = load_vec<T, V>(static_cast<const T*>(m.other) + (long long)r * m.H + j);
                Vec<T, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float f = Elem<T>::to_f(d.v[i]);
                    dot[k] = fmaf(f, Elem<T>::to_f(v.v[i]), dot[k]);
                    o.v[i] = Elem<T>::from_f(w * f);
                }
                store_vec<T, V>(static_cast<T*>(m.to) + (long long)r * m.H + j, o);
            }
        }
        __syncthreads();  // (the sums of the token before have been read)
#pragma unroll
        for (int k = 0; k < kMaxTopK; ++k) {
            if (k >= m.K) break;
            const float v = warp_sum(dot[k]);
            if (lane == 0) part[k][warp] = v;
        }
        __syncthreads();
        if (threadIdx.x < m.K && m.dweights) {
            float v = part[threadIdx.x][0];
            for (int w = 1; w < 8; ++w) v += part[threadIdx.x][w];
            m.dweights[t * m.K + threadIdx.x] = v;
        }
    }
    clear_tail<T, V>(m);
}

}  // namespace sorting
}  // namespace kleos
