// Tokens sorted by expert, and their rows there and back.
//
//   offsets[e]  = chosen places (t, k) with an expert below e;  offsets[E] = all that have one
//   row_of[t,k] = offsets[e] + places of the same expert e in front of (t, k), in the order of t, then k;  -1: no expert
//   source[r]   = t K + k of row r;  -1 from offsets[E] on
//   gather      rows[row_of[t,k]] = x[t]                 gradient  dx[t] = sum_k drows[row_of[t,k]]
//   combine     out[t] = sum_k w[t,k] rows[row_of[t,k]]  gradient  drows[row_of[t,k]] = w[t,k] dout[t],
//                                                                  dw[t,k] = <dout[t], rows[row_of[t,k]]>
// Every sum runs in the order of k in 32 bits and is rounded once; there are no atomics, so every call gives the same bits.
//
// Moving rows is bound by HBM.  16384 tokens of 2048 bf16 on two experts each: gather 32 us and combine 34 for 201 MB (6.3 and 5.9
// TB/s), the gradients of combine 55 for 336 MB (6.1); sorting them 7 us, which is latency: one cluster of eight blocks,
// their counts exchanged once.  One token: 3.1, 1.7 and 1.6 us of launches.
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
// the lanes.  Counters: hist[w][e].  Lanes with the same expert find one another by a ballot per bit of it, which takes
// the same time whatever the experts (kBits: as many as E takes).  match.any takes longer the more of them there are: 32768
// places spread evenly over 64 experts 9.7 us, now 8.2; by Zipf over 128 6.4 and 7.0; one token 2.7 and 3.1.  kKept: every warp has at
// most kKeep turns, whose experts and ranks stay in its registers; otherwise it goes through its share twice, kKeep
// turns' loads at a time.
constexpr int kKeep = 8;
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
template <bool kKept, int kBits>
__global__ void __launch_bounds__(kThreads) sort_kernel(const int* topk, int n, int E, int* offsets, int* row_of, int* source) {
    namespace cg = cooperative_groups;
    extern __shared__ int hist[];          // [kWarps][E]
    __shared__ int mine[ops::kMaxExperts];  // this block's places of every expert
    __shared__ int base[ops::kMaxExperts];  // row of the block's first place of every expert
    __shared__ int scan[kWarps];
    __shared__ int filled;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    int* count = hist + warp * E;
    for (int i = lane; i < E; i += 32) count[i] = 0;
    // turns of 32 places, an equal number for every warp
    const long long turns = ((long long)n + 31) / 32, per = (turns + blocks * kWarps - 1) / (blocks * kWarps);
    const long long first = ((long long)block * kWarps + warp) * per, last = min(first + per, turns);
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    auto expert_at = [&](long long turn) {
        const long long i = turn * 32 + lane;
        const int e = i < n ? topk[i] : -1;
        return e < 0 || e >= E ? -1 : e;
    };
    // the places of expert e in front of this one in the warp's own share
    auto rank = [&](int e) {
        unsigned same = 0xffffffffu;
        const int id = e < 0 ? E : e;
#pragma unroll
        for (int b = 0; b < kBits; ++b) {
            const bool set = (id >> b) & 1;
            const unsigned with = __ballot_sync(0xffffffffu, set);
            same &= set ? with : ~with;
        }
        const int before = __popc(same & ((1u << lane) - 1));
        const int r = e < 0 ? 0 : count[e] + before;
        __syncwarp();
        if (e >= 0 && before == 0) count[e] = r + __popc(same);
        __syncwarp();
        return r;
    };
    int kept_e[kKeep], kept_r[kKeep];
    if constexpr (kKept) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k) kept_e[k] = k < per && first + k < last ? expert_at(first + k) : -1;
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
            if (k < per) kept_r[k] = rank(kept_e[k]);
    } else {
        for (long long t = first; t < last; t += kKeep) {
#pragma unroll
            for (int k = 0; k < kKeep; ++k) kept_e[k] = t + k < last ? expert_at(t + k) : -1;
#pragma unroll
            for (int k = 0; k < kKeep; ++k)
                if (t + k < last) rank(kept_e[k]);
        }
    }
    __syncthreads();
    // a thread per expert: the warps' counts become the places in front of each warp
    int total = 0;
    if (tid < E) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int c = hist[w * E + tid];
            hist[w * E + tid] = total;
            total += c;
        }
        mine[tid] = total;
    }
    int before = 0, all = total;
    if (blocks > 1) {
        cluster.sync();
        all = 0;
        if (tid < E) {
            int c[kCluster];
#pragma unroll
            for (int b = 0; b < kCluster; ++b) c[b] = cluster.map_shared_rank(mine, b)[tid];
#pragma unroll
            for (int b = 0; b < kCluster; ++b) {
                if (b < block) before += c[b];
                all += c[b];
            }
        }
        cluster_arrive();
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
    int front = lane < warp ? scan[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) front += __shfl_xor_sync(0xffffffffu, front, o);
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
    auto place = [&](long long t, int e, int r) {
        const long long i = t * 32 + lane;
        if (i >= n) return;
        const int row = e < 0 ? -1 : base[e] + r;
        row_of[i] = row;
        if (source && row >= 0) source[row] = (int)i;
    };
    if constexpr (kKept) {
        // (ranks were counted from the warp's own start; count[] now holds what is in front of the warp)
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
            if (k < per && first + k < last) place(first + k, kept_e[k], kept_r[k] + (kept_e[k] < 0 ? 0 : count[kept_e[k]]));
    } else {
        for (long long t = first; t < last; t += kKeep) {
#pragma unroll
            for (int k = 0; k < kKeep; ++k) kept_e[k] = t + k < last ? expert_at(t + k) : -1;
#pragma unroll
            for (int k = 0; k < kKeep; ++k)
                if (t + k < last) place(t + k, kept_e[k], rank(kept_e[k]));
        }
    }
    if (source)
        for (long long i = (long long)filled + block * kThreads + tid; i < n; i += (long long)blocks * kThreads) source[i] = -1;
    if (blocks > 1) cluster_wait();  // (no block leaves while another may still read its counts)
}

struct Move {
    const void *from, *other;  // `other`: the rows whose product with dout is wanted
    void* to;
    const int *row_of, *offsets;
    const float* weights;
    float* dweights;
    long long ld;  // of the token matrix
    int T, K, E, H, n;  // n = T * K rows
    int span;           // columns that a token's blocks take at a time
    int lanes;          // threads of a token: the block, or, where that is larger, a warp
};

// Rows that no place leads to are zeros: the tail, from offsets[E] on.
template <typename T, int V>
__device__ __forceinline__ void clear_tail(const Move& m) {
    const int filled = min(max(m.offsets[m.E], 0), m.n);
    Vec<T, V> zero;
#pragma unroll
    for (int k = 0; k < V; ++k) zero.v[k] = Elem<T>::from_f(0.f);
    for (long long r = filled + blockIdx.x; r < m.n; r += gridDim.x)
        for (int j = (blockIdx.y * blockDim.x + threadIdx.x) * V; j < m.H; j += gridDim.y * blockDim.x * V) store_vec<T, V>(static_cast<T*>(m.to) + r * m.H + j, zero);
}

// m.lanes threads take a token, a thread every m.lanes-th vector of it, kAhead vectors of each row at a time; KT
// >= K, so that all their loads are on their way before the first is needed.  The host chooses as many threads as
// have four vectors each (as many as have kAhead: 16384 tokens of 2048 bf16, top-2, combine 34 -> 40 us, its gradients 63 -> 73),
// or one where there are few tokens, and a token a block; eight where a warp is enough for one (200000 tokens of 64 bf16, a
// token a block 207 us, which is what the chip takes to start as many; eight 61), not where it is not (8192 tokens of 2048
// bf16, top-4, combine 29 -> 33).  Vectors are 16 bytes, or two elements, or one, as rows and pointers allow (4000 tokens of 1090
// bf16, top-8, combine one by one 64, in pairs 25 us).  Where there are few tokens the blocks of a column of the grid share one
// token's row, kAhead vectors a thread each (one token of 7270, top-8: combine in one block 33 us, in 15 2.0).
template <int V, int KT>
constexpr int kAhead = KT == 8 ? (V <= 2 ? 2 : 1) : KT == 4 ? (V <= 2 ? 4 : 2) : 4 / KT;
template <int KT>
constexpr int kAhead<2, KT> = KT == 8 ? 2 : 4;

struct Token {
    long long t;
    int group, lane;
    __device__ __forceinline__ explicit Token(const Move& m) {
        const bool several = (int)blockDim.x != m.lanes;  // (then of a warp each)
        group = several ? threadIdx.x >> 5 : 0;
        lane = several ? threadIdx.x & 31 : threadIdx.x;
        t = several ? (long long)blockIdx.x * (blockDim.x >> 5) + group : blockIdx.x;
    }
};
// The rows of a token, -1 where it has none.
template <int KT>
__device__ __forceinline__ void rows_of_token(const Move& m, long long t, int (&r)[KT]) {
#pragma unroll
    for (int k = 0; k < KT; ++k) {
        r[k] = k < m.K ? m.row_of[t * m.K + k] : -1;
        if (r[k] >= m.n) r[k] = -1;
    }
}

// The token's row is read once and stored K times.
template <typename T, int V, int KT>
__global__ void __launch_bounds__(256) gather_kernel(Move m) {
    constexpr int U = kAhead<V, 1>;
    pdl_wait();
    pdl_trigger();
    const Token token(m);
    const int step = m.lanes * V;
    if (token.t < m.T) {
        const T* x = static_cast<const T*>(m.from) + token.t * m.ld;
        int r[KT];
        rows_of_token<KT>(m, token.t, r);
        for (int j0 = blockIdx.y * U * step + token.lane * V; j0 < m.H; j0 += m.span) {
            Vec<T, V> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + u * step < m.H) v[u] = load_vec<T, V>(x + j0 + u * step);
#pragma unroll
            for (int k = 0; k < KT; ++k)
                if (r[k] >= 0)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (j0 + u * step < m.H) store_vec<T, V>(static_cast<T*>(m.to) + (long long)r[k] * m.H + j0 + u * step, v[u]);
        }
    }
    clear_tail<T, V>(m);
}

// V running sums, in pairs where there are two.
template <int V>
struct Sums {
    F2 s[V / 2];
    __device__ __forceinline__ Sums() {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) s[i] = both(0.f);
    }
    template <typename T>
    __device__ __forceinline__ void add(float w, const Vec<T, V>& v) {
        F2 p[V / 2];
        to_pairs<T, V>(v, p);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) s[i] = fma2(both(w), p[i], s[i]);
    }
    template <typename T>
    __device__ __forceinline__ Vec<T, V> rounded() const {
        return from_pairs<T, V>(s);
    }
};
template <>
struct Sums<1> {
    float s = 0.f;
    template <typename T>
    __device__ __forceinline__ void add(float w, const Vec<T, 1>& v) {
        s = fmaf(w, Elem<T>::to_f(v.v[0]), s);
    }
    template <typename T>
    __device__ __forceinline__ Vec<T, 1> rounded() const {
        return Vec<T, 1>{{Elem<T>::from_f(s)}};
    }
};

// Without weights: the gradient of gather.  Vectors of one or two elements are loaded without a condition, at row 0
// and the row's last vector where there is none (4000 tokens of 1087, top-8 64 -> 34 us); the bounds on registers are what wide
// rows took before a token could have several blocks (16384 tokens of 64, top-4: 7.9 us, without them 10.8); eight rows of 16-byte
// vectors spill 4 to 40 bytes under theirs.
template <typename T, int V, int KT>
__global__ void __launch_bounds__(256, V <= 2 ? (KT >= 4 ? 3 : 5) : KT >= 4 ? 3 : KT == 2 ? 5 : 6) combine_kernel(Move m) {
    constexpr int U = kAhead<V, KT>;
    pdl_wait();
    pdl_trigger();
    const Token token(m);
    if (token.t >= m.T) return;
    const int step = m.lanes * V;
    T* out = static_cast<T*>(m.to) + token.t * m.ld;
    int r[KT];
    float w[KT];
    rows_of_token<KT>(m, token.t, r);
#pragma unroll
    for (int k = 0; k < KT; ++k) w[k] = m.weights && r[k] >= 0 ? m.weights[token.t * m.K + k] : 1.f;
#pragma unroll 1
    for (int j0 = blockIdx.y * U * step + token.lane * V; j0 < m.H; j0 += m.span) {
        Vec<T, V> v[KT][U];
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if constexpr (V <= 2)
                    v[k][u] = load_vec<T, V>(static_cast<const T*>(m.from) + (long long)max(r[k], 0) * m.H + min(j0 + u * step, m.H - V));
                else if (r[k] >= 0 && j0 + u * step < m.H)
                    v[k][u] = load_vec<T, V>(static_cast<const T*>(m.from) + (long long)r[k] * m.H + j0 + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j0 + u * step >= m.H) continue;
            Sums<V> s;
#pragma unroll
            for (int k = 0; k < KT; ++k)
                if (r[k] >= 0) s.template add<T>(w[k], v[k][u]);
            store_vec<T, V>(out + j0 + u * step, s.template rounded<T>());
        }
    }
}

// dout[t] is read once for all its K rows.  Vectors past a row's end are its last one, those of no row the first row's: without
// a condition in front of them all loads are on their way at once (16384 tokens of 2048 bf16, top-2 63 -> 58 us; element by
// element it is the other way round, 16384 x 2047 108 -> 188, and for combine_kernel, 34.3 -> 35.7).
template <typename T, int V, int KT>
__global__ void __launch_bounds__(256) combine_back_kernel(Move m) {
    constexpr int U = kAhead<V, KT>;
    __shared__ float part[KT][8];
    pdl_wait();
    pdl_trigger();
    const Token token(m);
    const int warp = threadIdx.x >> 5, step = m.lanes * V;
    float dot[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) dot[k] = 0.f;
    if (token.t < m.T) {
        const T* dout = static_cast<const T*>(m.from) + token.t * m.ld;
        int r[KT];
        float w[KT];
        rows_of_token<KT>(m, token.t, r);
#pragma unroll
        for (int k = 0; k < KT; ++k) w[k] = m.weights && r[k] >= 0 ? m.weights[token.t * m.K + k] : 1.f;
        for (int j0 = token.lane * V; j0 < m.H; j0 += U * step) {
            Vec<T, V> d[U], v[KT][U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (V > 1 || j0 + u * step < m.H) d[u] = load_vec<T, V>(dout + (V > 1 ? min(j0 + u * step, m.H - V) : j0 + u * step));
            if (m.dweights)
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (V > 1 || (r[k] >= 0 && j0 + u * step < m.H))
                            v[k][u] = load_vec<T, V>(static_cast<const T*>(m.other) + (long long)max(r[k], 0) * m.H + (V > 1 ? min(j0 + u * step, m.H - V) : j0 + u * step));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j0 + u * step >= m.H) continue;
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = Elem<T>::to_f(d[u].v[i]);
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    if (r[k] < 0) continue;
                    Vec<T, V> o;
#pragma unroll
                    for (int i = 0; i < V; ++i) o.v[i] = Elem<T>::from_f(w[k] * f[i]);
                    store_vec<T, V>(static_cast<T*>(m.to) + (long long)r[k] * m.H + j0 + u * step, o);
                    if (m.dweights)
#pragma unroll
                        for (int i = 0; i < V; ++i) dot[k] = fmaf(f[i], Elem<T>::to_f(v[k][u].v[i]), dot[k]);
                }
            }
        }
    }
    if (m.dweights) {
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            dot[k] = warp_sum(dot[k]);
            if ((threadIdx.x & 31) == 0) part[k][warp] = dot[k];
        }
        __syncthreads();
        if (token.t < m.T && token.lane < m.K) {
            const int first = token.group * (m.lanes >> 5);
            float v = part[token.lane][first];
            for (int i = 1; i < m.lanes >> 5; ++i) v += part[token.lane][first + i];
            m.dweights[token.t * m.K + token.lane] = v;
        }
    }
    clear_tail<T, V>(m);
}

}  // namespace sorting
}  // namespace kleos
