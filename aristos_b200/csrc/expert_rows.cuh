// The experts' products of a few rows, a token or some in serving: the weights of the experts that have a row are
// streamed once for every four of its rows (two where rows are fewer than two an expert), from as many blocks as there are columns
// to share out.
//
//   forward_rows_kernel  y[r]  = x[r] W[e]^T + b[e]   a warp takes two or four columns and goes along the weights' rows
//   dx_rows_kernel       dx[r] = dy[r] W[e]           a thread takes a vector of columns and goes down the weights' rows; a
//                                                     cluster shares those rows where columns make few blocks
//
// Sums are fp32, in a fixed order: along a lane, then over the lanes (over the warps, over the blocks).
//
// Bound by the latency of a launch and its loads, then by HBM and L2 (5.9 to 6.4 TB/s of weights).  bf16, N = K = 2048, one row 5.1 us,
// two rows of two experts 5.8 (16.8 MB; tensor cores 8.9 and 10.9).  Floats, N = K = 2048: one row 6 us forward and 8 dx; 32 rows of
// 16 experts 50 and 46, of one expert 23 and 22 (with its rows one after the other in a block 154 and 120); 8 rows, N = 5176, K = 1792
// 19 and 32 (38 and 71).  Loads without a condition, all on their way before the first is used: 16 of the weights for dx, 8 forward.
#pragma once

#include "expert_simt.cuh"

namespace kleos {
namespace experts {
namespace few {

// The expert of which `row` is the first, or the first after so many times kRows: those rows of it, E for a row of nobody, -1 for one
// in between.  All threads of the block call it.
template <int kRows>
__device__ __forceinline__ int group_begun_by(const Args& a, int row, Group* rows) {
    __shared__ int found;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        const Group g = group_rows(a.offsets, e, a.rows);
        if (g.begin <= row && row < g.end && (row - g.begin) % kRows == 0) atomicMax(&found, e);  // (one, if the offsets ascend)
    }
    __syncthreads();
    const int e = found;
    if (e < 0) return row >= min(max(a.offsets[a.E], 0), a.rows) ? a.E : -1;
    *rows = group_rows(a.offsets, e, a.rows);
    rows->begin = row;
    rows->end = min(rows->end, row + kRows);
    return e;
}

// kRows of an expert at a time by C columns a warp: each row's elements are fetched (from L1) once for C products.
template <typename T, int V, int kRows, int C>
__global__ void __launch_bounds__(256) forward_rows_kernel(Args a) {
    constexpr int P = V > 1 ? V / 2 : 1;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, n0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * C;
    Group g;
    const int e = group_begun_by<kRows>(a, blockIdx.y, &g);
    T* y = static_cast<T*>(a.out);
    if (e < 0 || n0 >= a.N) return;
    const int cols = min(C, a.N - n0);
    if (e == a.E) {
        if (lane < cols) y[(long long)blockIdx.y * a.ldo + n0 + lane] = Elem<T>::from_f(0.f);
        return;
    }
    const T* w = static_cast<const T*>(a.w) + ((size_t)e * a.N + n0) * a.K;
    const int r0 = g.begin, rows = g.end - g.begin;
    const T* x = static_cast<const T*>(a.x) + (long long)r0 * a.ldx;
    F2 s2[kRows][C];
    float s1[kRows][C];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) s2[r][c] = both(0.f), s1[r][c] = 0.f;
    constexpr int U = 8 / C;  // vectors of a column on their way
    for (int k0 = lane * V; k0 < a.K; k0 += U * 32 * V) {
        // columns and rows past the last are the last: without a condition all loads are on their way at once
        Vec<T, V> u[C][U];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (k0 + i * 32 * V < a.K) u[c][i] = load_vec<T, V>(w + (size_t)min(c, cols - 1) * a.K + k0 + i * 32 * V);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int k = k0 + i * 32 * V;
            if (k >= a.K) break;
            Vec<T, V> f[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) f[r] = load_vec<T, V>(x + (long long)min(r, rows - 1) * a.ldx + k);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if constexpr (V > 1) {
                        F2 p[P], q[P];
                        to_pairs<T, V>(f[r], p);
                        to_pairs<T, V>(u[c][i], q);
#pragma unroll
                        for (int j = 0; j < P; ++j) s2[r][c] = fma2(p[j], q[j], s2[r][c]);
                    } else {
                        s1[r][c] = fmaf(Elem<T>::to_f(f[r].v[0]), Elem<T>::to_f(u[c][i].v[0]), s1[r][c]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (r >= rows || c >= cols) continue;
            float v = warp_sum(V > 1 ? sum2(s2[r][c]) : s1[r][c]);
            if (lane == 0) {
                if (a.bias) v += Elem<T>::to_f(static_cast<const T*>(a.bias)[(size_t)e * a.N + n0 + c]);
                y[(long long)(r0 + r) * a.ldo + n0 + c] = Elem<T>::from_f(v);
            }
        }
}

constexpr int kDxWarps = 16;
template <typename T, int V>
__global__ void __launch_bounds__(32 * kDxWarps) dx_rows_kernel(Args a) {
    constexpr int kWarps = kDxWarps, kRows = 4;
    extern __shared__ float part[];                  // [kWarps][32 * V + 1]
    __shared__ __align__(16) float f[kWarps][32][kRows];  // dy of 32 rows of the weights, a warp's own
    __shared__ float sums[kRows][32 * V];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k0 = blockIdx.x / blocks * 32 * V, k = k0 + lane * V;
    Group g;
    const int e = group_begun_by<kRows>(a, blockIdx.y, &g);
    T* dx = static_cast<T*>(a.out);
    if (e < 0) return;
    if (e == a.E) {
        for (int j = threadIdx.x; block == 0 && j < 32 * V && k0 + j < a.K; j += 32 * kWarps) dx[(long long)blockIdx.y * a.ldo + k0 + j] = Elem<T>::from_f(0.f);
        return;
    }
    const T* w = static_cast<const T*>(a.w) + (size_t)e * a.N * a.K + k;
    const int r0 = g.begin, rows = g.end - g.begin;
    const T* dy = static_cast<const T*>(a.dy) + (long long)r0 * a.ldy;
    float s[kRows][V];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) s[r][j] = 0.f;
    for (int n0 = (block * kWarps + warp) * 32; n0 < a.N; n0 += blocks * kWarps * 32) {
        constexpr int U = 16;  // rows of the weights on their way; past the last they are the last
        const int end = min(32, a.N - n0);
        Vec<T, V> u[U];
        auto fetch = [&](int i0) {
            if (k >= a.K) return;
#pragma unroll
            for (int i = 0; i < U; ++i) u[i] = load_vec<T, V>(w + (size_t)min(n0 + i0 + i, a.N - 1) * a.K);
        };
        auto add = [&](int i0) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (i0 + i >= end) break;
                const float4 q = *reinterpret_cast<const float4*>(f[warp][i0 + i]);
                const float d[kRows] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int r = 0; r < kRows; ++r)
#pragma unroll
                    for (int j = 0; j < V; ++j) s[r][j] = fmaf(d[r], Elem<T>::to_f(u[i].v[j]), s[r][j]);
            }
        };
        fetch(0);
        float d[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) d[r] = r < rows && n0 + lane < a.N ? Elem<T>::to_f(dy[r * a.ldy + n0 + lane]) : 0.f;
        __syncwarp();  // (all lanes are through with the rows before)
#pragma unroll
        for (int r = 0; r < kRows; ++r) f[warp][lane][r] = d[r];
        __syncwarp();
        if (k >= a.K) continue;
        add(0);
        fetch(U);
        add(U);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r >= rows) break;
        __syncthreads();  // (the row before has been added up)
#pragma unroll
        for (int j = 0; j < V; ++j) part[warp * (32 * V + 1) + lane * V + j] = s[r][j];
        __syncthreads();
        // a warp adds up a column in sixteen, a lane per partial sum
        for (int c = warp; c < 32 * V; c += kWarps) {
            const float v = warp_sum(lane < kWarps ? part[lane * (32 * V + 1) + c] : 0.f);
            if (lane != 0) continue;
            if (blocks > 1) sums[r][c] = v;
            else if (k0 + c < a.K) dx[(long long)(r0 + r) * a.ldo + k0 + c] = Elem<T>::from_f(v);
        }
    }
    if (blocks == 1) return;
    cluster.sync();
    for (int i = block * 32 * kWarps + threadIdx.x; i < rows * 32 * V; i += blocks * 32 * kWarps) {
        const int r = i / (32 * V), c = i % (32 * V);
        float v = 0.f;
        for (int b = 0; b < blocks; ++b) v += cluster.map_shared_rank(&sums[0][0], b)[i];
        if (k0 + c < a.K) dx[(long long)(r0 + r) * a.ldo + k0 + c] = Elem<T>::from_f(v);
    }
    cluster.sync();  // (no block leaves while its sums may still be read)
}

}  // namespace few
}  // namespace experts
}  // namespace kleos
