// Layer norm and its gradients.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), h = (x - m) r, y = h w + b            (per row)
//   g = dy w, dx = r (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum over rows of dy
//
// HBM bounds both: 2 and 3 elements moved per value.  A row is held in the registers of its threads, read once; the
// squares are of differences from the mean (a difference of two sums would lose what a large mean takes).  All of it is
// in 32 bits and rounded once, when it is stored.
#pragma once

#include <type_traits>

#include "ops_common.cuh"

namespace kleos {
namespace norm {
using namespace ops;

constexpr int kMaxPartials = 296;  // blocks that add up dw and db; their sums go through the workspace

struct Args {
    const void *x, *dy, *weight, *bias;
    void *y, *dx, *dweight, *dbias;
    float *mean, *rstd, *partial;
    long long ldx, lddy, ldy, lddx;
    int rows, H;
    bool wide;  // parameters are floats, whatever the element type
    float eps;
};

template <typename T>
__device__ __forceinline__ float param(const void* p, int j, bool wide, float otherwise) {
    return !p ? otherwise : wide ? static_cast<const float*>(p)[j] : Elem<T>::to_f(static_cast<const T*>(p)[j]);
}
template <typename T>
__device__ __forceinline__ void put_param(void* p, int j, bool wide, float v) {
    if (wide) static_cast<float*>(p)[j] = v;
    else static_cast<T*>(p)[j] = Elem<T>::from_f(v);
}

// Sum of (a, b) over the G threads of a row, the same in all of them: a warp, or a whole block of G threads.
template <int G>
__device__ __forceinline__ float2 row_sum(float a, float b, float2* shared) {
    a = warp_sum(a);
    b = warp_sum(b);
    if constexpr (G > 32) {
        constexpr int W = G / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        __syncthreads();  // (the sums of the row before have been read)
        if (lane == 0) shared[warp] = make_float2(a, b);
        __syncthreads();
        const float2 v = lane < W ? shared[lane] : make_float2(0.f, 0.f);
        a = warp_sum(v.x);
        b = warp_sum(v.y);
    }
    return make_float2(a, b);
}

template <typename T, int V, int N>
__device__ __forceinline__ void load_row(const T* row, int H, int G, int at, Vec<T, V> (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = (at + i * G) * V;
        if (j < H) v[i] = load_vec<T, V>(row + j);
    }
}

// G threads a row, N vectors of V elements each; rows / block = blockDim / G.
template <typename T, int V, int G, int N>
__global__ void __launch_bounds__(G > 256 ? G : 256) forward_kernel(Args a) {
    __shared__ float2 shared[32];
    pdl_wait();
    pdl_trigger();
    const int at = threadIdx.x % G, per = blockDim.x / G, H = a.H;
    const float inv = 1.f / (float)H;
    for (long long r = (long long)blockIdx.x * per + threadIdx.x / G; r < a.rows; r += (long long)gridDim.x * per) {
        Vec<T, V> x[N];
        load_row<T, V, N>(static_cast<const T*>(a.x) + r * a.ldx, H, G, at, x);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((at + i * G) * V < H)
#pragma unroll
                for (int k = 0; k < V; ++k) s += Elem<T>::to_f(x[i].v[k]);
        const float m = row_sum<G>(s, 0.f, shared).x * inv;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((at + i * G) * V < H)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = Elem<T>::to_f(x[i].v[k]) - m;
                    s = fmaf(d, d, s);
                }
        const float rs = 1.f / sqrtf(row_sum<G>(s, 0.f, shared).x * inv + a.eps);
        T* y = static_cast<T*>(a.y) + r * a.ldy;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (at + i * G) * V;
            if (j >= H) continue;
            Vec<T, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k)
                o.v[k] = Elem<T>::from_f(fmaf((Elem<T>::to_f(x[i].v[k]) - m) * rs, param<T>(a.weight, j + k, a.wide, 1.f),
                                              param<T>(a.bias, j + k, a.wide, 0.f)));
            store_vec<T, V>(y + j, o);
        }
        if (at == 0) {
            if (a.mean) a.mean[r] = m;
            if (a.rstd) a.rstd[r] = rs;
        }
    }
}

// Rows too long for registers: a block reads its row three times.
template <typename T>
__global__ void __launch_bounds__(1024) forward_long_kernel(Args a) {
    __shared__ float2 shared[32];
    pdl_wait();
    pdl_trigger();
    const float inv = 1.f / (float)a.H;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        T* y = static_cast<T*>(a.y) + r * a.ldy;
        float s = 0.f;
        for (int j = threadIdx.x; j < a.H; j += 1024) s += Elem<T>::to_f(x[j]);
        const float m = row_sum<1024>(s, 0.f, shared).x * inv;
        s = 0.f;
        for (int j = threadIdx.x; j < a.H; j += 1024) {
            const float d = Elem<T>::to_f(x[j]) - m;
            s = fmaf(d, d, s);
        }
        const float rs = 1.f / sqrtf(row_sum<1024>(s, 0.f, shared).x * inv + a.eps);
        for (int j = threadIdx.x; j < a.H; j += 1024)
            y[j] = Elem<T>::from_f(fmaf((Elem<T>::to_f(x[j]) - m) * rs, param<T>(a.weight, j, a.wide, 1.f), param<T>(a.bias, j, a.wide, 0.f)));
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = m;
            if (a.rstd) a.rstd[r] = rs;
        }
    }
}

// dx of the block's rows, and its sums over them for dw and db: partial[block][0] and [1].
template <typename T, int V, int G, int N>
__global__ void __launch_bounds__(G > 256 ? G : 256) backward_kernel(Args a) {
    extern __shared__ float sums[];  // G == 32: [2 * H]
    __shared__ float2 shared[32];
    pdl_wait();
    pdl_trigger();
    const int at = threadIdx.x % G, per = blockDim.x / G, H = a.H;
    const float inv = 1.f / (float)H;
    float dw[N][V], db[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.f;
    for (long long r = (long long)blockIdx.x * per + threadIdx.x / G; r < a.rows; r += (long long)gridDim.x * per) {
        Vec<T, V> x[N], dy[N];
        load_row<T, V, N>(static_cast<const T*>(a.x) + r * a.ldx, H, G, at, x);
        load_row<T, V, N>(static_cast<const T*>(a.dy) + r * a.lddy, H, G, at, dy);
        const float m = a.mean[r], rs = a.rstd[r];
        float sg = 0.f, sgh = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (at + i * G) * V;
            if (j >= H) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = Elem<T>::to_f(dy[i].v[k]), h = (Elem<T>::to_f(x[i].v[k]) - m) * rs;
                const float g = d * param<T>(a.weight, j + k, a.wide, 1.f);
                sg += g;
                sgh = fmaf(g, h, sgh);
                dw[i][k] = fmaf(d, h, dw[i][k]);
                db[i][k] += d;
            }
        }
        const float2 s = row_sum<G>(sg, sgh, shared);
        const float mg = s.x * inv, mgh = s.y * inv;
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (at + i * G) * V;
            if (j >= H) continue;
            Vec<T, V> o;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float h = (Elem<T>::to_f(x[i].v[k]) - m) * rs;
                const float g = Elem<T>::to_f(dy[i].v[k]) * param<T>(a.weight, j + k, a.wide, 1.f);
                o.v[k] = Elem<T>::from_f(rs * (g - mg - h * mgh));
            }
            store_vec<T, V>(dx + j, o);
        }
    }
    if (!a.partial) return;
    float* mine = a.partial + (size_t)blockIdx.x * 2 * H;
    if constexpr (G == 32) {
        // a warp's rows are its own: the warps' sums are added in their order
        for (int warp = 0; warp < per; ++warp) {
            if ((int)threadIdx.x >> 5 == warp)
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int j = (at + i * G) * V + k;
                        if (j < H) {
                            sums[j] = warp ? sums[j] + dw[i][k] : dw[i][k];
                            sums[H + j] = warp ? sums[H + j] + db[i][k] : db[i][k];
                        }
                    }
            __syncthreads();
        }
        for (int j = threadIdx.x; j < 2 * H; j += blockDim.x) mine[j] = sums[j];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int j = (at + i * G) * V + k;
                if (j < H) {
                    mine[j] = dw[i][k];
                    mine[H + j] = db[i][k];
                }
            }
    }
}

// Rows too long for registers: dx, a block a row; dw and db by column_kernel.
template <typename T>
__global__ void __launch_bounds__(1024) backward_long_kernel(Args a) {
    __shared__ float2 shared[32];
    pdl_wait();
    pdl_trigger();
    const float inv = 1.f / (float)a.H;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T*>(a.x) + r * a.ldx, *dy = static_cast<const T*>(a.dy) + r * a.lddy;
        const float m = a.mean[r], rs = a.rstd[r];
        float sg = 0.f, sgh = 0.f;
        for (int j = threadIdx.x; j < a.H; j += 1024) {
            const float g = Elem<T>::to_f(dy[j]) * param<T>(a.weight, j, a.wide, 1.f);
            sg += g;
            sgh = fmaf(g, (Elem<T>::to_f(x[j]) - m) * rs, sgh);
        }
        const float2 s = row_sum<1024>(sg, sgh, shared);
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
        for (int j = threadIdx.x; j < a.H; j += 1024) {
            const float g = Elem<T>::to_f(dy[j]) * param<T>(a.weight, j, a.wide, 1.f), h = (Elem<T>::to_f(x[j]) - m) * rs;
            dx[j] = Elem<T>::from_f(rs * (g - s.x * inv - h * s.y * inv));
        }
    }
}
// ... sums over a block's share of the rows, a thread a column
template <typename T>
__global__ void __launch_bounds__(256) column_kernel(Args a) {
    pdl_wait();
    pdl_trigger();
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= a.H) return;
    float dw = 0.f, db = 0.f;
    for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float d = Elem<T>::to_f(static_cast<const T*>(a.dy)[r * a.lddy + j]);
        dw = fmaf(d, (Elem<T>::to_f(static_cast<const T*>(a.x)[r * a.ldx + j]) - a.mean[r]) * a.rstd[r], dw);
        db += d;
    }
    float* mine = a.partial + (size_t)blockIdx.y * 2 * a.H;
    mine[j] = dw;
    mine[a.H + j] = db;
}

// dw and db: the blocks' sums, added up eight at a time by 8 threads a column in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(Args a, int partials) {
    __shared__ float s[8][33];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (j < 2 * a.H)
        for (int p = part; p < partials; p += 8) v += a.partial[(size_t)p * 2 * a.H + j];
    s[part][lane] = v;
    __syncthreads();
    if (part == 0 && j < 2 * a.H) {
#pragma unroll
        for (int k = 1; k < 8; ++k) v += s[k][lane];
        if (j < a.H) {
            if (a.dweight) put_param<T>(a.dweight, j, a.wide, v);
        } else if (a.dbias) {
            put_param<T>(a.dbias, j - a.H, a.wide, v);
        }
    }
}

// Calls f with threads a row and vectors a thread for H elements in vectors of V: a warp where four vectors a lane hold
// the row, else a block of 256 or 512 threads.  False where a row is too long for their registers.
template <int V, typename F>
bool with_shape(int H, F f) {
    constexpr int kMost = V == 1 ? 16 : 4;
    const int n = (H + V - 1) / V;
    auto shape = [&](auto g, auto k) {
        f(g, k);
        return true;
    };
    using std::integral_constant;
    if (n <= 32) return shape(integral_constant<int, 32>(), integral_constant<int, 1>());
    if (n <= 64) return shape(integral_constant<int, 32>(), integral_constant<int, 2>());
    if (n <= 128) return shape(integral_constant<int, 32>(), integral_constant<int, 4>());
    if (n <= 256) return shape(integral_constant<int, 256>(), integral_constant<int, 1>());
    if (n <= 512) return shape(integral_constant<int, 256>(), integral_constant<int, 2>());
    if (n <= 1024) return shape(integral_constant<int, 256>(), integral_constant<int, 4>());
    if (n <= 512 * kMost) return shape(integral_constant<int, 512>(), integral_constant<int, kMost>());
    return false;
}

}  // namespace norm
}  // namespace kleos
