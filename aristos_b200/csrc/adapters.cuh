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
// A cluster of blocks takes some rows of a request: it shares the sums of u (of v), meets, and shares the columns of y
// (of dx), so that u never leaves the chip between the two products.  Both passes over rows are one kernel: what differs is the
// direction in which the adapters are read.  The kernels here take any element type and alignment, on the FP32 pipes, and are bound by
// issue and latency (2943 rows, N = 1087, K = 1090, rank 12, floats: 46 us each way, both gradients 35); those of adapters_mma.cuh take 16-bit rows on
// 16-byte boundaries.
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
    bool quads;                    // whether the adapters' elements can be read four at a time along the rank
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
// Sums of N values over a warp, N / 32 of them a lane: half of the values go to the other lane at every step, N - 1 exchanges instead of 5 N.
// Lane l ends with those from index sum of (l >> 4 - k & 1) N / 2^(k + 1) on.
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N]) {
    const int lane = threadIdx.x & 31;
    int n = N / 2;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1, n /= 2) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            if (i >= n) break;
            const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
}
template <int N>
__device__ __forceinline__ int warp_sums_index() {
    const int lane = threadIdx.x & 31;
    return (lane >> 4 & 1) * (N / 2) + (lane >> 3 & 1) * (N / 4) + (lane >> 2 & 1) * (N / 8) + (lane >> 1 & 1) * (N / 16) + (lane & 1) * (N / 32);
}

constexpr int kRowsSimt = 8;

// FP32 multiply-adds: two groups of four warps have four rows each; a group's warps (times the cluster's blocks) take the sums' elements in turn,
// a lane for 8 or 16 columns of u at once.  V elements of `in` (and of p, forward) at once.
template <typename T, int V, bool kBack>
__global__ void __launch_bounds__(256, 2) rows_kernel(Args a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int M = kRowsSimt, MW = 4, J = V > 1 ? 8 : 16, KS = 4;
    __shared__ float part[KS][M][kMostRank + 1];
    __shared__ float u[M][kMostRank];
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rg = warp & 1, ks = warp >> 1;
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
    const T* in[MW];  // rows past the last are the last; nobody takes their sums
#pragma unroll
    for (int m = 0; m < MW; ++m) in[m] = static_cast<const T*>(a.in) + (long long)(t.begin + min(rg * MW + m, n - 1)) * a.ldi;
    for (int j0 = 0; j0 < a.r; j0 += J) {
        float s[MW * J];
#pragma unroll
        for (int i = 0; i < MW * J; ++i) s[i] = 0.f;
#pragma unroll 1
        for (int k = ((block * KS + ks) * 32 + lane) * V; k < a.len; k += blocks * KS * 32 * V) {
            Vec<T, V> w[J], x[MW];
#pragma unroll
            for (int m = 0; m < MW; ++m) x[m] = load_vec<T, V>(in[m] + k);
            if (kBack && a.quads) {
#pragma unroll
                for (int j = 0; j < J; j += 4)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const Vec<T, 4> l = load_vec<T, 4>(p + (size_t)(k + v) * a.r + min(j0 + j, a.r - 4));
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[j + i].v[v] = l.v[i];
                    }
            } else {
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
            }
#pragma unroll
            for (int m = 0; m < MW; ++m)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int v = 0; v < V; ++v) s[m * J + j] = fmaf(Elem<T>::to_f(x[m].v[v]), Elem<T>::to_f(w[j].v[v]), s[m * J + j]);
        }
        warp_sums<MW * J>(s);
        const int first = warp_sums_index<MW * J>();
#pragma unroll
        for (int i = 0; i < MW * J / 32; ++i)
            if (j0 + (first + i) % J < a.r) part[ks][rg * MW + (first + i) / J][j0 + (first + i) % J] = s[i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.r; i += 256) {
        const int m = i / a.r, j = i % a.r;
        float v = part[0][m][j];
#pragma unroll
        for (int k = 1; k < KS; ++k) v += part[k][m][j];
        part[0][m][j] = kBack ? v * scale : v;
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    for (int i = threadIdx.x; i < n * a.r; i += 256) {
        const int m = i / a.r, j = i % a.r;
        float v = 0.f;
        if (blocks == 1) v = part[0][m][j];
        else
            for (int k = 0; k < blocks; ++k) v += *cluster.map_shared_rank(&part[0][m][j], k);
        u[m][j] = v;
        if (a.u && block == 0) a.u[(long long)t.begin * a.r + i] = v;
    }
    if (blocks > 1) cluster.sync();  // (no block leaves while its sums may still be read)
    else __syncthreads();
    const T* base = static_cast<const T*>(a.base);
    T* out = static_cast<T*>(a.out);
    for (int c = c0 + (int)threadIdx.x; c < c1; c += 256) {
        float s[M], before[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            s[m] = 0.f;
            before[m] = base && m < n ? Elem<T>::to_f(base[(long long)(t.begin + m) * a.ldb + c]) : 0.f;
        }
        if (!kBack && a.quads) {
#pragma unroll 4
            for (int j = 0; j < a.r; j += 4) {
                const Vec<T, 4> l = load_vec<T, 4>(q + (size_t)c * a.r + j);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int m = 0; m < M; ++m) s[m] = fmaf(u[m][j + i], Elem<T>::to_f(l.v[i]), s[m]);
            }
        } else
#pragma unroll 8
        for (int j = 0; j < a.r; ++j) {
            const float w = Elem<T>::to_f(kBack ? q[(size_t)j * a.cols + c] : q[(size_t)c * a.r + j]);
#pragma unroll
            for (int m = 0; m < M; ++m) s[m] = fmaf(u[m][j], w, s[m]);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
            if (m < n) out[(long long)(t.begin + m) * a.ldo + c] = Elem<T>::from_f(fmaf(kBack ? 1.f : scale, s[m], before[m]));
    }
}

// ---------------------------------------------------------------- gradients of the adapters
// One of the two, or none (no strips).  Both are one launch where one kernel takes both.
struct Grads {
    const void* in;      // x, or dy
    const float* c;      // v, or u
    void* out;           // dA [L, r, cols], or dB [L, cols, r]
    bool db;             // which
    int strips;          // of columns, a cluster each
    const int *offsets, *adapter;
    const float* scale;  // null: ones (dA: v has it already)
    long long ldi;
    int rows, R, L, r, cols;
    bool wide_out;       // results are floats
};

// dA and dB: a cluster takes 32 columns and 16 ranks of one adapter; its blocks take 64 rows of a request in turn, whose factors
// are in shared memory, and a warp every eighth of those.
template <typename T>
__global__ void __launch_bounds__(256) grads_kernel(Grads first_of_two, Grads second_of_two) {
    namespace cg = cooperative_groups;
    constexpr int J = 16, kRows = 64, kMine = kRows / 8;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ __align__(16) float c[2][kRows][J];
    __shared__ float part[8][J][33];
    __shared__ float sums[J][33];
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    pdl_wait();
    pdl_trigger();
    const int strip = blockIdx.x / blocks;
    const bool second = strip >= first_of_two.strips;
    const Grads a = second ? second_of_two : first_of_two;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = blockIdx.y, j0 = blockIdx.z * J, n = min(J, a.r - j0);
    const int first = (strip - (second ? first_of_two.strips : 0)) * 32, col = first + lane;
    const bool there = col < a.cols;
    const T* in = static_cast<const T*>(a.in) + (there ? col : 0);
    float s[J];
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = 0.f;
    int count = 0, turn = 0;
    for (int i0 = 0; i0 < a.R; i0 += 32) {
        const int i = i0 + lane;
        unsigned of = __ballot_sync(0xffffffffu, i < a.R && a.adapter[i] == l);
        for (; of; of &= of - 1) {
            const Group g = group_rows(a.offsets, i0 + __ffs(of) - 1, a.rows);
            for (int row0 = g.begin; row0 < g.end; row0 += kRows) {
                if (count++ % blocks != block) continue;
                const int rows = min(kRows, g.end - row0);
                float x[kMine];
#pragma unroll
                for (int k = 0; k < kMine; ++k) x[k] = there && warp + 8 * k < rows ? Elem<T>::to_f(in[(long long)(row0 + warp + 8 * k) * a.ldi]) : 0.f;
                turn ^= 1;  // (two buffers in turn: one meeting a step)
                for (int k = threadIdx.x; k < kRows * J; k += 256) {
                    const int row = k / J, j = k % J;
                    c[turn][row][j] = row < rows && j < n ? a.c[(long long)(row0 + row) * a.r + j0 + j] : 0.f;
                }
                __syncthreads();
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    if (warp + 8 * k >= rows) break;
#pragma unroll
                    for (int j = 0; j < J; j += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&c[turn][warp + 8 * k][j]);
                        s[j] = fmaf(f.x, x[k], s[j]);
                        s[j + 1] = fmaf(f.y, x[k], s[j + 1]);
                        s[j + 2] = fmaf(f.z, x[k], s[j + 2]);
                        s[j + 3] = fmaf(f.w, x[k], s[j + 3]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j) part[warp][j][lane] = s[j];
    __syncthreads();
    const float scale = a.scale ? a.scale[l] : 1.f;
    for (int i = threadIdx.x; i < J * 32; i += 256) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += part[w][i / 32][i % 32];
        sums[i / 32][i % 32] = v * scale;
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    for (int i = block * 256 + threadIdx.x; i < n * 32; i += blocks * 256) {
        const int j = a.db ? i % n : i / 32, cc = a.db ? i / n : i % 32;
        if (first + cc >= a.cols) continue;
        float v = 0.f;
        for (int k = 0; k < blocks; ++k) v += *cluster.map_shared_rank(&sums[j][cc], k);
        const size_t at = a.db ? ((size_t)l * a.cols + first + cc) * a.r + j0 + j : ((size_t)l * a.r + j0 + j) * a.cols + first + cc;
        if (a.wide_out) static_cast<float*>(a.out)[at] = v;
        else static_cast<T*>(a.out)[at] = Elem<T>::from_f(v);
    }
    if (blocks > 1) cluster.sync();
}

}  // namespace adapters
}  // namespace kleos
