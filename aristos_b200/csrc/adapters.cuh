// Low-rank adapters of many requests beside a projection that they share, with their gradients.
//
//   request i: rows offsets[i] .. offsets[i + 1] - 1, adapter l = adapter[i]
//   u = x A[l]^T            y  = base + s_l u B[l]^T       A [L, r, K], B [L, N, r]
//   v = s_l dy B[l]         dx = dbase + v A[l]
//   dA[l] = sum over its rows of v^T x                     dB[l] = s_l sum over its rows of dy^T u
//
// Rows without an adapter (a number outside 0 .. L - 1, rows before the first request or behind the last) keep base and dbase
// and have no part in the gradients; u is zero there.
//
// A cluster of blocks takes up to kTile rows of a request: it shares the sums of u (of v), meets, and shares the columns of y
// (of dx), so that u never leaves the chip between the two products.  Both passes over rows are one kernel: what differs is the
// direction in which the adapters are read.  Bound by HBM (x, base and y once), by latency for a few rows.
#pragma once

#include <cooperative_groups.h>

#include "ops_common.cuh"

namespace kleos {
namespace adapters {
using namespace ops;

constexpr int kMostRank = 128;
constexpr int kMostRequests = 1 << 16;

struct Args {
    const void* in;    // x, or dy
    const void* p;     // summed over first: A, or B
    const void* q;     // then: B, or A
    const void* base;  // null: zeros
    void* out;         // y, or dx
    float* u;          // u, or v; may be null
    const int *offsets, *adapter;
    const float* scale;  // null: ones
    long long ldi, ldb, ldo;
    int rows, R, L, r, len, cols;  // len of `in`, columns of `out`
};

struct Tile {
    int begin, end, adapter;  // adapter -1: rows without one
};

// Rows of request i; request -1 are the rows before the first, request R those behind the last.
__device__ __forceinline__ Group request_rows(const int* offsets, int R, int i, int rows) {
    Group g;
    g.begin = i < 0 ? 0 : min(max(offsets[i], 0), rows);
    g.end = i == R ? rows : max(g.begin, min(offsets[i + 1], rows));
    return g;
}

// The `index`-th tile of so many rows; false when there are fewer.  All threads of the block (256 at most) call it.
template <int kRows>
__device__ __forceinline__ bool find_tile(const Args& a, int index, Tile* tile) {
    __shared__ Tile found;
    __shared__ int sums[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) found.begin = -1;
    int before = 0;
    for (int i0 = -1; i0 <= a.R; i0 += blockDim.x) {
        const int i = i0 + (int)threadIdx.x;
        Group g{0, 0};
        if (i <= a.R) g = request_rows(a.offsets, a.R, i, a.rows);
        const int n = (g.end - g.begin + kRows - 1) / kRows;
        int up = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += v;
        }
        if (lane == 31) sums[warp] = up;
        __syncthreads();
        int first = before + up - n;
        for (int w = 0; w < (int)blockDim.x / 32; ++w) {
            first += w < warp ? sums[w] : 0;
            before += sums[w];
        }
        if (first <= index && index < first + n) {
            found.begin = g.begin + (index - first) * kRows;
            found.end = min(g.end, found.begin + kRows);
            const int l = i < 0 || i == a.R ? -1 : a.adapter[i];
            found.adapter = l >= 0 && l < a.L ? l : -1;
        }
        __syncthreads();
        if (before > index) break;
    }
    *tile = found;
    return found.begin >= 0;
}

// out = base (zeros without one) for the columns [c0, c1) of a tile's rows, V elements at once.
template <typename T, int V>
__device__ __forceinline__ void copy_base(const Args& a, const Tile& t, int c0, int c1) {
    const T* base = static_cast<const T*>(a.base);
    T* out = static_cast<T*>(a.out);
    if (base == out) return;
    constexpr int U = 8;  // of a thread on their way
    const int across = (c1 - c0 + V - 1) / V, n = (t.end - t.begin) * across;
    for (int i0 = threadIdx.x; i0 < n; i0 += U * blockDim.x) {
        Vec<T, V> v[U] = {};
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * (int)blockDim.x;
            if (base && i < n) v[k] = load_vec<T, V>(base + (long long)(t.begin + i / across) * a.ldb + c0 + i % across * V);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int i = i0 + k * (int)blockDim.x;
            if (i < n) store_vec<T, V>(out + (long long)(t.begin + i / across) * a.ldo + c0 + i % across * V, v[k]);
        }
    }
}

// ---------------------------------------------------------------- rows, any element type and alignment
constexpr int kRowsSimt = 8;

// V elements of `in` (and of p, forward) at once.
template <typename T, int V, bool kBack>
__global__ void __launch_bounds__(256) rows_kernel(Args a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int M = kRowsSimt, J = 2;
    __shared__ float u[M][kMostRank];
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_trigger();
    Tile t;
    if (!find_tile<M>(a, blockIdx.x / blocks, &t)) return;  // (all blocks of the cluster)
    const int n = t.end - t.begin, share = (a.cols + blocks - 1) / blocks, c0 = min(a.cols, block * share), c1 = min(a.cols, c0 + share);
    if (t.adapter < 0) {
        copy_base<T, 1>(a, t, c0, c1);
        if (a.u && block == 0)
            for (int i = threadIdx.x; i < n * a.r; i += 256) a.u[(long long)t.begin * a.r + i] = 0.f;
        return;
    }
    const float scale = a.scale ? a.scale[t.adapter] : 1.f;
    const T* p = static_cast<const T*>(a.p) + (size_t)t.adapter * a.r * a.len;
    const T* q = static_cast<const T*>(a.q) + (size_t)t.adapter * a.r * a.cols;
    const T* in[M];
#pragma unroll
    for (int m = 0; m < M; ++m) in[m] = static_cast<const T*>(a.in) + (long long)(t.begin + min(m, n - 1)) * a.ldi;
    cluster.sync();  // (every block of the cluster is there to be written to)
    // the cluster's warps share the columns of u, two at a time
    for (int j0 = (block * 8 + warp) * J; j0 < a.r; j0 += blocks * 8 * J) {
        float s[M][J];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int j = 0; j < J; ++j) s[m][j] = 0.f;
#pragma unroll 2
        for (int k = lane * V; k < a.len; k += 32 * V) {
            Vec<T, V> w[J], x[M];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int jj = min(j0 + j, a.r - 1);
                if constexpr (!kBack) {
                    w[j] = load_vec<T, V>(p + (size_t)jj * a.len + k);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) w[j].v[v] = p[(size_t)(k + v) * a.r + jj];
                }
            }
#pragma unroll
            for (int m = 0; m < M; ++m) x[m] = load_vec<T, V>(in[m] + k);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int v = 0; v < V; ++v) s[m][j] = fmaf(Elem<T>::to_f(x[m].v[v]), Elem<T>::to_f(w[j].v[v]), s[m][j]);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float v = warp_sum(s[m][j]) * (kBack ? scale : 1.f);
                if (j0 + j >= a.r) continue;
                if (lane < blocks) *cluster.map_shared_rank(&u[m][j0 + j], lane) = v;
                if (lane == 0 && a.u && m < n) a.u[(long long)(t.begin + m) * a.r + j0 + j] = v;
            }
    }
    cluster.sync();
    const T* base = static_cast<const T*>(a.base);
    T* out = static_cast<T*>(a.out);
    for (int c = c0 + (int)threadIdx.x; c < c1; c += 256) {
        float s[M];
#pragma unroll
        for (int m = 0; m < M; ++m) s[m] = 0.f;
#pragma unroll 4
        for (int j = 0; j < a.r; ++j) {
            const float w = Elem<T>::to_f(kBack ? q[(size_t)j * a.cols + c] : q[(size_t)c * a.r + j]);
#pragma unroll
            for (int m = 0; m < M; ++m) s[m] = fmaf(u[m][j], w, s[m]);
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if (m >= n) break;
            const float before = base ? Elem<T>::to_f(base[(long long)(t.begin + m) * a.ldb + c]) : 0.f;
            out[(long long)(t.begin + m) * a.ldo + c] = Elem<T>::from_f(fmaf(kBack ? 1.f : scale, s[m], before));
        }
    }
}

// ---------------------------------------------------------------- gradients of the adapters
struct Grads {
    const void* in;      // x, or dy
    const float* c;      // v, or u
    void* out;           // dA [L, r, cols], or dB [L, cols, r]
    const int *offsets, *adapter;
    const float* scale;  // null: ones (dA: v has it already)
    long long ldi;
    int rows, R, L, r, cols;
    bool wide_out;       // results are floats
};

// dA (kDb false) or dB: a block takes 32 columns of one adapter, eight groups of warps its rows in turn.
template <typename T, bool kDb>
__global__ void __launch_bounds__(256) grads_kernel(Grads a) {
    constexpr int J = 16;
    __shared__ float part[8][J][33];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = blockIdx.y, j0 = blockIdx.z * J, n = min(J, a.r - j0);
    const int c = blockIdx.x * 32 + lane;
    float s[J];
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = 0.f;
    for (int i = 0; i < a.R; ++i) {
        if (a.adapter[i] != l) continue;
        const Group g = group_rows(a.offsets, i, a.rows);
        for (int row = g.begin + warp; row < g.end; row += 8) {
            const float x = c < a.cols ? Elem<T>::to_f(static_cast<const T*>(a.in)[row * a.ldi + c]) : 0.f;
            const float* f = a.c + (long long)row * a.r + j0;
#pragma unroll
            for (int j = 0; j < J; ++j) s[j] = fmaf(f[min(j, n - 1)], x, s[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) part[warp][j][lane] = s[j];
    __syncthreads();
    const float scale = a.scale ? a.scale[l] : 1.f;
    for (int i = threadIdx.x; i < n * 32; i += 256) {
        const int j = kDb ? i % n : i / 32, cc = kDb ? i / n : i % 32, col = blockIdx.x * 32 + cc;
        if (col >= a.cols) continue;
        float v = 0.f;
        for (int w = 0; w < 8; ++w) v += part[w][j][cc];
        v *= scale;
        const size_t at = kDb ? ((size_t)l * a.cols + col) * a.r + j0 + j : ((size_t)l * a.r + j0 + j) * a.cols + col;
        if (a.wide_out) static_cast<float*>(a.out)[at] = v;
        else static_cast<T*>(a.out)[at] = Elem<T>::from_f(v);
    }
}

}  // namespace adapters
}  // namespace kleos
