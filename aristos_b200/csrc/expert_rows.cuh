// The experts' products of a few rows, a token or some in serving: the weights of the experts that have a row are
// streamed once for up to eight of its rows, from as many blocks as there are columns to share out.
//
//   forward_rows_kernel  y[r]  = x[r] W[e]^T + b[e]   a warp takes two or four columns and goes along the weights' rows
//   dx_rows_kernel       dx[r] = dy[r] W[e]           a thread takes a vector of columns and goes down the weights' rows
//
// Sums are fp32, in a fixed order: along a lane, then over the lanes (over the warps).
//
// Bound by the latency of a launch and its loads, then by HBM: bf16, N = K = 2048, one row 5.2 us, two rows of two experts 5.9 (16.8
// MB) where the tensor cores' sixteen tiles take 13.4 and 13.8; four rows 13.0 and 14.0, or of one expert 15.3 and 11.5;
// more columns fill the chip with tiles (N = 14336, K = 4096, one row 32 and 25).  Floats: one row 7 us forward and 14 dx,
// 32 rows of 27 experts 105 and 80, where the kernel of many rows takes 236 and 270 for 64 of 64; 32 rows of one expert,
// each vector of whose x is fetched for four columns only, 153 and 120 (75 and 84 for 16 such experts).
#pragma once

#include "expert_simt.cuh"

namespace kleos {
namespace experts {
namespace few {

// The group that row `row` begins, E for a row of nobody, -1 for one inside a group.  All threads of the block call it.
__device__ __forceinline__ int group_begun_by(const Args& a, int row, Group* rows) {
    __shared__ int found;
    if (threadIdx.x == 0) found = row >= min(max(a.offsets[a.E], 0), a.rows) ? a.E : -1;
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
        const Group g = group_rows(a.offsets, e, a.rows);
        if (g.begin == row && g.end > row) found = e;
    }
    __syncthreads();
    const int e = found;
    if (e >= 0 && e < a.E) *rows = group_rows(a.offsets, e, a.rows);
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
    const int e = group_begun_by(a, blockIdx.y, &g);
    T* y = static_cast<T*>(a.out);
    if (e < 0 || n0 >= a.N) return;
    const int cols = min(C, a.N - n0);
    if (e == a.E) {
        if (lane < cols) y[(long long)blockIdx.y * a.ldo + n0 + lane] = Elem<T>::from_f(0.f);
        return;
    }
    const T* w = static_cast<const T*>(a.w) + ((size_t)e * a.N + n0) * a.K;
    for (int r0 = g.begin; r0 < g.end; r0 += kRows) {
        const T* x = static_cast<const T*>(a.x) + (long long)r0 * a.ldx;
        const int rows = min(kRows, g.end - r0);
        F2 s2[kRows][C];
        float s1[kRows][C];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) s2[r][c] = both(0.f), s1[r][c] = 0.f;
        constexpr int U = 8 / C;  // vectors of a column on their way
        for (int k0 = lane * V; k0 < a.K; k0 += U * 32 * V) {
            Vec<T, V> u[C][U];
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (c < cols && k0 + i * 32 * V < a.K) u[c][i] = load_vec<T, V>(w + (size_t)c * a.K + k0 + i * 32 * V);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int k = k0 + i * 32 * V;
                if (k >= a.K) break;
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    if (r >= rows) break;
                    const Vec<T, V> f = load_vec<T, V>(x + r * a.ldx + k);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        if (c >= cols) break;
                        if constexpr (V > 1) {
                            F2 p[P], q[P];
                            to_pairs<T, V>(f, p);
                            to_pairs<T, V>(u[c][i], q);
#pragma unroll
                            for (int j = 0; j < P; ++j) s2[r][c] = fma2(p[j], q[j], s2[r][c]);
                        } else {
                            s1[r][c] = fmaf(Elem<T>::to_f(f.v[0]), Elem<T>::to_f(u[c][i].v[0]), s1[r][c]);
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
}

template <typename T, int V>
__global__ void __launch_bounds__(1024) dx_rows_kernel(Args a) {
    constexpr int kWarps = 32, kRows = 4;
    extern __shared__ float part[];                  // [kWarps][32 * V + 1]
    __shared__ __align__(16) float f[kWarps][32][kRows];  // dy of 32 rows of the weights, a warp's own
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k0 = blockIdx.x * 32 * V, k = k0 + lane * V;
    Group g;
    const int e = group_begun_by(a, blockIdx.y, &g);
    T* dx = static_cast<T*>(a.out);
    if (e < 0) return;
    if (e == a.E) {
        for (int j = threadIdx.x; j < 32 * V && k0 + j < a.K; j += 1024) dx[(long long)blockIdx.y * a.ldo + k0 + j] = Elem<T>::from_f(0.f);
        return;
    }
    const T* w = static_cast<const T*>(a.w) + (size_t)e * a.N * a.K + k;
    for (int r0 = g.begin; r0 < g.end; r0 += kRows) {
        const T* dy = static_cast<const T*>(a.dy) + (long long)r0 * a.ldy;
        const int rows = min(kRows, g.end - r0);
        float s[kRows][V];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) s[r][j] = 0.f;
        for (int n0 = warp * 32; n0 < a.N; n0 += kWarps * 32) {
            __syncwarp();
#pragma unroll
            for (int r = 0; r < kRows; ++r) f[warp][lane][r] = r < rows && n0 + lane < a.N ? Elem<T>::to_f(dy[r * a.ldy + n0 + lane]) : 0.f;
            __syncwarp();
            if (k >= a.K) continue;
            constexpr int U = 4;  // rows of the weights on their way
            const int end = min(32, a.N - n0);
            for (int i0 = 0; i0 < end; i0 += U) {
                Vec<T, V> u[U];
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (i0 + i < end) u[i] = load_vec<T, V>(w + (size_t)(n0 + i0 + i) * a.K);
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
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (r >= rows) break;
            __syncthreads();  // (the row before has been added up)
#pragma unroll
            for (int j = 0; j < V; ++j) part[warp * (32 * V + 1) + lane * V + j] = s[r][j];
            __syncthreads();
            // a warp adds up V columns, a lane per partial sum
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = warp * V + j;
                const float v = warp_sum(part[lane * (32 * V + 1) + c]);
                if (lane == 0 && k0 + c < a.K) dx[(long long)(r0 + r) * a.ldo + k0 + c] = Elem<T>::from_f(v);
            }
        }
    }
}

}  // namespace few
}  // namespace experts
}  // namespace kleos
