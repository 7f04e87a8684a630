// The experts' products on the FP32 pipes, for what the tensor-core kernels cannot load (sizes, strides or addresses that are
// no multiples of 16 bytes) and for the weight gradients of a few float rows.
//
//   kForward  y[r]  = x[r] W[e]^T + b[e]      for the rows r of expert e, offsets[e] <= r < offsets[e + 1]
//   kDx       dx[r] = dy[r] W[e]
//   kDw       dW[e] = sum over r of dy[r]^T x[r]
//
// A block computes a 128 x 128 tile of one expert, a thread 8 x 8 of it, over slices of 16 that are loaded into registers
// while the slice before them is multiplied.  Operands are converted when they are loaded, so products and sums are
// fp32 multiply-adds whatever the type, two at a time (fma.rn.f32x2: half the instructions, the same rounding).
// Bound by the FP32 pipes: 4096 float rows of 16 experts, N = K = 2048, 34.4 GFLOP: 1014, 965 and 734 us (34, 36 and 47 TFLOP/s of
// 74); the few rows of many experts by the stores of dW (128 experts, N = 4424, K = 384, 128 rows: 870 MB in 199 us).
#pragma once

#include <cooperative_groups.h>

#include "ops_common.cuh"

namespace kleos {
namespace experts {
using namespace ops;

enum Mode { kForward, kDx, kDw };

struct Args {
    const void *x, *dy, *w, *bias;  // rows [rows][K] and [rows][N], weights [E][N][K]
    void* out;
    const int* offsets;
    long long ldx, ldy, ldo;
    int rows, E, N, K;
    bool wide_out;  // dW as floats
};

// first[e] = tiles of `tile` rows of the experts before e, for e <= E; rows of nobody count as those of expert E, and
// first[E + 1] is the total.  All threads of the block call it.
__device__ __forceinline__ void tiles_of_groups(int* first, const int* offsets, int E, int rows, int tile) {
    if (threadIdx.x < 32) {
        int at = 0;
        for (int e0 = 0; e0 <= E; e0 += 32) {
            const int e = e0 + (int)threadIdx.x;
            int n = 0;
            if (e < E) {
                const Group g = group_rows(offsets, e, rows);
                n = (g.end - g.begin + tile - 1) / tile;
            } else if (e == E) {
                n = (rows - min(max(offsets[E], 0), rows) + tile - 1) / tile;
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if ((int)threadIdx.x >= o) upto += v;
            }
            if (e <= E) {
                first[e] = at + upto - n;
                if (e == E) first[E + 1] = at + upto;
            }
            at += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    __syncthreads();
}
// The group that tile t belongs to: the last one that begins at or before it.
__device__ __forceinline__ int group_of_tile(const int* first, int E, int t) {
    int lo = 0, hi = E;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

constexpr int kTile = 128, kSlice = 16, kPitch = kTile + 4;

// Where line l of step k of a slice lies: eights of lines change places every four steps, so that neither the stores of
// operands that are contiguous along the steps nor the reads of four lines at once meet a bank conflict.
__device__ __forceinline__ int place(int k, int l) { return l ^ ((k & 12) << 1); }

// Eight elements of an operand for a thread.  kAlong: the slice's direction is the contiguous one in memory (thread t
// holds four steps of lines t / 4 and 64 + t / 4), else the tile's is (thread t holds lines 8 (t % 16).. of step t / 16).
template <typename T, bool kAlong, int V>
struct Operand {
    const T* p;      // line 0 of the tile, step 0
    long long ld;
    int lines, steps;  // that exist
    float v[8];
    __device__ __forceinline__ void load(int step0) {
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            const int line = kAlong ? (threadIdx.x >> 2) + (i >> 2) * 64 : (threadIdx.x & 15) * 8 + i;
            const int step = step0 + (kAlong ? (threadIdx.x & 3) * 4 + (i & 3) : threadIdx.x >> 4);
            const bool in = kAlong ? line < lines && step + V <= steps : step < steps && line + V <= lines;
            Vec<T, V> u;
            if (in) u = load_vec<T, V>(p + (kAlong ? line * ld + step : step * ld + line));
#pragma unroll
            for (int k = 0; k < V; ++k) v[i + k] = in ? Elem<T>::to_f(u.v[k]) : 0.f;
        }
    }
    __device__ __forceinline__ void put(float (*s)[kPitch]) const {
        if constexpr (kAlong) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = (threadIdx.x & 3) * 4 + (i & 3);
                s[k][place(k, (threadIdx.x >> 2) + (i >> 2) * 64)] = v[i];
            }
        } else {
            const int k = threadIdx.x >> 4;
            float4* d = reinterpret_cast<float4*>(&s[k][place(k, (threadIdx.x & 15) * 8)]);
            d[0] = make_float4(v[0], v[1], v[2], v[3]);
            d[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
};

// V: elements of a load, four where every row begins on a 16-byte boundary and is a multiple of it, else 1.
template <typename T, int kMode, int V>
__global__ void __launch_bounds__(256, 2) product_kernel(Args a) {
    __shared__ __align__(16) float sa[2][kSlice][kPitch], sb[2][kSlice][kPitch];
    __shared__ int first[kMaxExperts + 2];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x;
    const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy), *w = static_cast<const T*>(a.w);
    const int cols = kMode == kForward ? a.N : a.K;  // of the result
    const int c0 = blockIdx.y * kTile;
    int e, m0, lines, steps;  // first line of the tile and how many it has; length of the sums
    long long row0 = 0;
    if constexpr (kMode == kDw) {
        e = blockIdx.z;
        const Group g = group_rows(a.offsets, e, a.rows);
        row0 = g.begin;
        steps = g.end - g.begin;
        m0 = blockIdx.x * kTile;
        lines = min(kTile, a.N - m0);
    } else {
        tiles_of_groups(first, a.offsets, a.E, a.rows, kTile);
        const int t = blockIdx.x;
        if (t >= first[a.E + 1]) return;
        e = group_of_tile(first, a.E, t);
        Group g;
        if (e < a.E) g = group_rows(a.offsets, e, a.rows);
        else g = Group{min(max(a.offsets[a.E], 0), a.rows), a.rows};
        m0 = g.begin + (t - first[e]) * kTile;
        lines = min(kTile, g.end - m0);
        steps = e == a.E ? 0 : kMode == kForward ? a.K : a.N;  // rows of nobody: zeros
    }
    const size_t we = (size_t)e * a.N * a.K;
    constexpr bool kA = kMode != kDw, kB = kMode == kForward;
    Operand<T, kA, V> A;
    Operand<T, kB, V> B;
    A.lines = lines;
    B.lines = min(kTile, cols - c0);
    A.steps = B.steps = steps;
    if constexpr (kMode == kForward) {
        A.p = x + m0 * a.ldx;
        A.ld = a.ldx;
        B.p = w + we + (size_t)c0 * a.K;
        B.ld = a.K;
    } else if constexpr (kMode == kDx) {
        A.p = dy + m0 * a.ldy;
        A.ld = a.ldy;
        B.p = w + we + c0;
        B.ld = a.K;
    } else {
        A.p = dy + row0 * a.ldy + m0;
        A.ld = a.ldy;
        B.p = x + row0 * a.ldx + c0;
        B.ld = a.ldx;
    }
    const int ty = tid >> 4, tx = tid & 15;  // lines 4 ty.. and 64 + 4 ty.., columns likewise
    F2 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = both(0.f);
    A.load(0);
    B.load(0);
    A.put(sa[0]);
    B.put(sb[0]);
    __syncthreads();
    int now = 0;
    for (int s = 0; s < steps; s += kSlice, now ^= 1) {
        const bool more = s + kSlice < steps;
        if (more) {
            A.load(s + kSlice);
            B.load(s + kSlice);
        }
#pragma unroll
        for (int k = 0; k < kSlice; ++k) {
            float4 u[2];
            ulonglong2 v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u[h] = *reinterpret_cast<const float4*>(&sa[now][k][place(k, 64 * h + 4 * ty)]);
                v[h] = *reinterpret_cast<const ulonglong2*>(&sb[now][k][place(k, 64 * h + 4 * tx)]);
            }
            const float f[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
            const F2 g[4] = {{v[0].x}, {v[0].y}, {v[1].x}, {v[1].y}};
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fma2(both(f[i]), g[j], acc[i][j]);
        }
        if (more) {
            A.put(sa[now ^ 1]);
            B.put(sb[now ^ 1]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int line = (i < 4 ? 0 : 60) + 4 * ty + i;
        if (line >= lines) continue;
        const size_t row = kMode == kDw ? we + (size_t)(m0 + line) * a.K : (size_t)(m0 + line) * a.ldo;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = c0 + 64 * h + 4 * tx;
            if (c >= cols) continue;
            const float2 p = split(acc[i][2 * h]), q = split(acc[i][2 * h + 1]);
            float v[4] = {p.x, p.y, q.x, q.y};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (kMode == kForward && a.bias && e < a.E && c + j < cols) v[j] += Elem<T>::to_f(static_cast<const T*>(a.bias)[(size_t)e * a.N + c + j]);
            if constexpr (V > 1 && sizeof(T) == 4) {  // whole vectors: the result's rows are such too
                *reinterpret_cast<float4*>(static_cast<float*>(a.out) + row + c) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (c + j >= cols) continue;
                    if (kMode == kDw && a.wide_out) static_cast<float*>(a.out)[row + c + j] = v[j];
                    else static_cast<T*>(a.out)[row + c + j] = Elem<T>::from_f(v[j]);
                }
            }
        }
    }
}

// db[e] = sum of the rows of dy of expert e.  A block sums sixteen vectors of V columns of an expert, 64 rows at a time and two
// of them a thread on their way; then over the 64 partial sums in a fixed order.  Bound by HBM and by the fullest
// expert's chain of loads: 11771 x 2880 fp16, 24 experts 24 us, 4096 x 2048 floats 12; with eight vectors a block 22 and
// 13, with 32 36 and 11.  Where the blocks leave multiprocessors idle, a cluster of up to eight shares an expert's rows, 64 at a
// time in turn, and its first block adds their sums in order: one expert's 4198 rows of 1056 bf16 120 -> 10 us, 8000 of 14336 286
// -> 63.
constexpr int kBiasLanes = 16;
template <typename T, int V>
__global__ void __launch_bounds__(1024, 2) bias_kernel(Args a) {
    constexpr int kLanes = kBiasLanes, kParts = 1024 / kLanes, kAhead = 2;
    __shared__ float s[kParts][kLanes * V + 1], sums[kLanes * V];
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank(), stride = kParts * blocks;
    pdl_wait();
    pdl_trigger();
    const int e = blockIdx.y, lane = threadIdx.x % kLanes, part = threadIdx.x / kLanes + kParts * block, c0 = blockIdx.x / blocks * kLanes * V, c = c0 + lane * V;
    const Group g = group_rows(a.offsets, e, a.rows);
    float v[V] = {};
    if (c < a.N) {
        const T* p = static_cast<const T*>(a.dy) + (long long)(g.begin + part) * a.ldy + c;
        for (int left = g.end - g.begin - part; left > 0; left -= stride * kAhead, p += stride * kAhead * a.ldy) {
            Vec<T, V> u[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (stride * k < left) u[k] = load_vec<T, V>(p + stride * k * a.ldy);
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (stride * k < left)
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] += Elem<T>::to_f(u[k].v[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s[threadIdx.x / kLanes][lane * V + i] = v[i];
    __syncthreads();
    auto store = [&](int j, float t) {
        const size_t at = (size_t)e * a.N + c0 + j;
        if (a.wide_out) static_cast<float*>(a.out)[at] = t;
        else static_cast<T*>(a.out)[at] = Elem<T>::from_f(t);
    };
    // a warp per column
    for (int j = threadIdx.x >> 5; j < kLanes * V && c0 + j < a.N; j += 32) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < kParts; k += 32) t += s[k + (threadIdx.x & 31)][j];
        t = warp_sum(t);
        if ((threadIdx.x & 31) != 0) continue;
        if (blocks == 1) store(j, t);
        else sums[j] = t;
    }
    if (blocks == 1) return;
    cluster.sync();
    if (block == 0 && threadIdx.x < kLanes * V && c0 + (int)threadIdx.x < a.N) {
        float t = sums[threadIdx.x];
        for (int b = 1; b < blocks; ++b) t += cluster.map_shared_rank(sums, b)[threadIdx.x];
        store(threadIdx.x, t);
    }
    cluster.sync();  // (no block leaves while its sums may still be read)
}

}  // namespace experts
}  // namespace kleos
