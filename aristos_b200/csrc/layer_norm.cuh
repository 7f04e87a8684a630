// Layer norm and its gradients.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), h = (x - m) r, y = h w + b            (per row)
//   g = dy w, dx = r (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum over rows of dy
//
// HBM bounds both: 2 and 3 elements moved per value.  A row is held in the registers of its threads, read once; the
// squares are of differences from the mean (a difference of two sums would lose what a large mean takes).  All of it is
// in 32 bits, two values an instruction, and rounded once, when it is stored.
//
// Measured (one call after the other, inputs larger than L2): 16384 x 4096 bf16 forward 45 us = 6.0 TB/s, gradients 73 us = 5.5
// TB/s with the sums over rows (a first form, rows loaded into registers and parameters one by one, 156 and 196);
// floats 5.2 and 5.5; 65536 x 512 bf16 5.3 and 3.6; rows that begin anywhere, 16384 x 4095 bf16, 2.7 and 3.1, floats 4.4 and 5.0.
// What is left is the issue of instructions in the gradients of 16-bit rows (two warps' worth a cycle on sixteen warps) and, in
// short rows, what a row costs beside its elements.
#pragma once

#include <type_traits>

#include "ops_common.cuh"
#include "tc_common.cuh"

namespace kleos {
namespace norm {
using namespace ops;

constexpr int kMaxPartials = 296;  // blocks that add up dw and db; their sums go through the workspace

struct Args {
    const void *x, *dy, *weight, *bias;
    void *y, *dx, *dweight, *dbias;
    float *mean, *rstd, *partial;
    long long ldx, lddy, ldy, lddx;
    int rows, H, depth;  // depth: stages of the ring
    long long wait_cycles;  // for a row's copies
    bool wide;       // parameters are floats, whatever the element type
    bool param_vec;  // ... and can be loaded as vectors
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

// V parameters from column j on, as floats.
template <typename T, int V>
__device__ __forceinline__ void load_params(const void* p, int j, bool wide, bool vec, float otherwise, float (&f)[V]) {
    if (p && vec) {
        if (wide) {
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const auto u = load_vec<float, (V < 4 ? V : 4)>(static_cast<const float*>(p) + j + k);
#pragma unroll
                for (int i = 0; i < (V < 4 ? V : 4); ++i) f[k + i] = u.v[i];
            }
        } else {
            const auto u = load_vec<T, V>(static_cast<const T*>(p) + j);
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = Elem<T>::to_f(u.v[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = param<T>(p, j + k, wide, otherwise);
    }
}

template <typename T, int V>
__device__ __forceinline__ void load_params(const void* p, int j, bool wide, bool vec, float otherwise, F2 (&f)[V / 2]) {
    float v[V];
    load_params<T, V>(p, j, wide, vec, otherwise, v);
#pragma unroll
    for (int k = 0; k < V / 2; ++k) f[k] = pair(v[2 * k], v[2 * k + 1]);
}

// Sum over the W lanes of a group of a warp (W a power of two), the same in all of them.
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum of (a, b) over the G threads of a row, the same in all of them: a warp, or a whole block of G threads, which
// meets once (`turn` alternates between the two halves of `shared`).
template <int G>
__device__ __forceinline__ float2 row_sum(float a, float b, float2 (*shared)[32], int turn) {
    a = warp_sum(a);
    b = warp_sum(b);
    if constexpr (G > 32) {
        constexpr int W = G / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) shared[turn & 1][warp] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 v = shared[turn & 1][w];
            a += v.x;
            b += v.y;
        }
    }
    return make_float2(a, b);
}

// Rows on their way to the shared memory of the threads that share a row: one row of one or two matrices a stage, `depth` of
// them in flight, filled by bulk copies that one thread issues.
constexpr int kMostDepth = 8;
template <typename T, int kMatrices>
struct Ring {
    T* rows;
    unsigned long long* full;  // [depth]
    const T* from[kMatrices];
    long long ld[kMatrices];
    int depth, H, total;  // total: rows of the matrices
    // One thread: row r to stage s.
    __device__ __forceinline__ void issue(long long r, int s) const {
        if (r >= total) return;
        const uint32_t bytes = (uint32_t)(H * sizeof(T));
        tc::mbar_expect_tx(&full[s], kMatrices * bytes);
#pragma unroll
        for (int m = 0; m < kMatrices; ++m) tc::bulk_load(rows + (s * kMatrices + m) * H, from[m] + r * ld[m], bytes, &full[s]);
    }
    __device__ __forceinline__ const T* row(int s, int m) const { return rows + (s * kMatrices + m) * H; }
    // False when the copies did not come in so many cycles.  The thread then gives up: what it owes becomes NaN, it waits for
    // no row after this one (its group's rows would each take as long again) and issues no copies.
    __device__ __forceinline__ bool wait(int s, uint32_t parity, long long cycles) const {
        if (tc::mbar_try_wait(&full[s], parity)) return true;
        const long long t0 = clock64();
        while (!tc::mbar_try_wait(&full[s], parity))
            if (clock64() - t0 > cycles) return false;
        return true;
    }
};
template <typename T, int kMatrices>
__device__ __forceinline__ Ring<T, kMatrices> make_ring(void* smem, unsigned long long* full, const Args& a, bool first) {
    Ring<T, kMatrices> r;
    r.rows = static_cast<T*>(smem);
    r.full = full;
    r.depth = a.depth;
    r.H = a.H;
    r.total = a.rows;
    r.from[0] = static_cast<const T*>(a.x);
    r.ld[0] = a.ldx;
    if constexpr (kMatrices == 2) {
        r.from[1] = static_cast<const T*>(a.dy);
        r.ld[1] = a.lddy;
    }
    if (first) {
        for (int i = 0; i < a.depth; ++i) tc::mbar_init(&full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    return r;
}

// What a thread has of a row: N vectors of V elements, G threads a row.
template <int V, int G, int N, typename F>
__device__ __forceinline__ void each_vector(int at, int H, F f) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        if ((at + i * G) * V < H) f(i, (at + i * G) * V);
}

// The G threads of a row meet: a warp, or as many as share the named barrier of their group.
template <int G>
__device__ __forceinline__ void meet(int group) {
    if constexpr (G == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(G) : "memory");
}

// Rows that can be copied in bulk.  G threads have a row, N vectors of V elements each; the block's groups of G threads go
// through rows of their own, each with a ring and a barrier.  A group meets once a row: every warp sums the squares
// around its own mean, and what the warps' means differ by from the row's is added when they meet (the same sum,
// without a second round).
template <int G>
constexpr int kForwardGroups = G < 256 ? 256 / G : 1;

template <typename T, int V, int G, int N>
__global__ void __launch_bounds__(G * kForwardGroups<G>, G > 256 ? 1 : 2) forward_kernel(Args a) {
    constexpr int P = kForwardGroups<G>, W = G / 32;
    static_assert(W == 1 || P < 16, "sixteen named barriers");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long full[P][kMostDepth];
    __shared__ float2 shared[P][2][W];
    __shared__ float share[P][W];  // values of a row that a warp holds
    const int at = threadIdx.x % G, group = threadIdx.x / G, H = a.H, warp = at >> 5, lane = threadIdx.x & 31;
    const auto ring = make_ring<T, 1>(smem + (size_t)group * a.depth * H * sizeof(T), full[group], a, at == 0);
    const long long step = (long long)gridDim.x * P, first = blockIdx.x + (long long)group * gridDim.x;
    pdl_wait();
    pdl_trigger();
    if (at == 0)
        for (int i = 0; i < a.depth; ++i) ring.issue(first + i * step, i);
    const float inv = 1.f / (float)H;
    F2 w[N][V / 2], b[N][V / 2];
    float mine = 0.f;
    each_vector<V, G, N>(at, H, [&](int i, int j) {
        mine += V;
        load_params<T, V>(a.weight, j, a.wide, a.param_vec, 1.f, w[i]);
        load_params<T, V>(a.bias, j, a.wide, a.param_vec, 0.f, b[i]);
    });
    const float n = warp_sum(mine), inv_n = n > 0.f ? 1.f / n : 0.f;
    if (lane == 0) share[group][warp] = n;
    __syncthreads();
    const float my_share = share[group][lane % W];  // of the warp that this lane answers for
    int stage = 0, turn = 0;
    uint32_t parity = 0;
    bool dead = false;
    for (long long r = first; r < a.rows; r += step, turn ^= 1) {
        if (!dead) dead = !ring.wait(stage, parity, a.wait_cycles);
        F2 x[N][V / 2], s = both(dead ? __uint_as_float(0x7fffffffu) : 0.f);  // (mean and deviation of the whole row with it)
        each_vector<V, G, N>(at, H, [&](int i, int j) {
            to_pairs<T, V>(load_vec<T, V>(ring.row(stage, 0) + j), x[i]);
#pragma unroll
            for (int k = 0; k < V / 2; ++k) s = add2(s, x[i][k]);
        });
        float m = warp_sum(sum2(s)) * inv_n;
        F2 q2 = both(0.f);
        const F2 minus = both(-m);
        each_vector<V, G, N>(at, H, [&](int i, int) {
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                const F2 d = add2(x[i][k], minus);
                q2 = fma2(d, d, q2);
            }
        });
        float q = warp_sum(sum2(q2));
        if (W > 1 && lane == 0) shared[group][turn][warp] = make_float2(m, q);
        meet<G>(group);  // ... and the row is in registers
        if (at == 0 && !dead) ring.issue(r + a.depth * step, stage);
        if (++stage == a.depth) stage = 0, parity ^= 1;
        if constexpr (W > 1) {
            const float2 v = shared[group][turn][lane % W];
            m = lanes_sum<W>(v.x * my_share) * inv;
            const float d = v.x - m;
            q = lanes_sum<W>(fmaf(my_share * d, d, v.y));
        }
        const float rs = rsqrtf(q * inv + a.eps);
        T* y = static_cast<T*>(a.y) + r * a.ldy;
        const F2 rs2 = both(rs), m2 = both(-m);
        each_vector<V, G, N>(at, H, [&](int i, int j) {
            F2 o[V / 2];
#pragma unroll
            for (int k = 0; k < V / 2; ++k) o[k] = fma2(mul2(add2(x[i][k], m2), rs2), w[i][k], b[i][k]);
            store_vec<T, V>(y + j, from_pairs<T, V>(o));
        });
        if (at == 0) {
            if (a.mean) a.mean[r] = m;
            if (a.rstd) a.rstd[r] = rs;
        }
    }
    if (dead) tc::settle_after_abort();
}

// Any other row, loaded element by element while the row before it is added up.  (16384 rows of 4092 bf16, whose rows begin on
// 8-byte boundaries: two elements at a time took 158 us forward and 165 back, one at a time 98 and 132.)
template <typename T, int G, int N>
struct Row {
    T v[N];
    __device__ __forceinline__ void fetch(const void* p, long long at_element, int at, int H) {
        const T* row = static_cast<const T*>(p) + at_element;
        each_vector<1, G, N>(at, H, [&](int i, int j) { v[i] = row[j]; });
    }
    __device__ __forceinline__ float operator[](int i) const { return Elem<T>::to_f(v[i]); }
};

template <typename T, int G, int N>
__global__ void __launch_bounds__(G * kForwardGroups<G>, G > 256 ? 1 : 2) forward_odd_kernel(Args a) {
    constexpr int P = kForwardGroups<G>, W = G / 32;
    __shared__ float2 shared[P][2][W];
    const int at = threadIdx.x % G, group = threadIdx.x / G, H = a.H, warp = at >> 5, lane = threadIdx.x & 31;
    const long long step = (long long)gridDim.x * P, first = blockIdx.x + (long long)group * gridDim.x;
    pdl_wait();
    pdl_trigger();
    const float inv = 1.f / (float)H;
    auto sum = [&](float v, int turn) {
        v = warp_sum(v);
        if constexpr (W > 1) {
            if (lane == 0) shared[group][turn][warp].x = v;
            meet<G>(group);
            v = lanes_sum<W>(shared[group][turn][lane % W].x);
        }
        return v;
    };
    float w[N], b[N];
    each_vector<1, G, N>(at, H, [&](int i, int j) {
        w[i] = param<T>(a.weight, j, a.wide, 1.f);
        b[i] = param<T>(a.bias, j, a.wide, 0.f);
    });
    Row<T, G, N> next;
    if (first < a.rows) next.fetch(a.x, first * a.ldx, at, H);
    for (long long r = first; r < a.rows; r += step) {
        float x[N], s = 0.f;
        each_vector<1, G, N>(at, H, [&](int i, int) {
            x[i] = next[i];
            s += x[i];
        });
        if (r + step < a.rows) next.fetch(a.x, (r + step) * a.ldx, at, H);
        const float m = sum(s, 0) * inv;
        s = 0.f;
        each_vector<1, G, N>(at, H, [&](int i, int) {
            const float d = x[i] - m;
            s = fmaf(d, d, s);
        });
        const float rs = rsqrtf(sum(s, 1) * inv + a.eps);
        T* y = static_cast<T*>(a.y) + r * a.ldy;
        each_vector<1, G, N>(at, H, [&](int i, int j) {
            y[j] = Elem<T>::from_f(fmaf((x[i] - m) * rs, w[i], b[i]));
        });
        if (at == 0) {
            if (a.mean) a.mean[r] = m;
            if (a.rstd) a.rstd[r] = rs;
        }
    }
}

// Rows too long for registers: a block reads its row three times.
template <typename T>
__global__ void __launch_bounds__(1024) forward_long_kernel(Args a) {
    __shared__ float2 shared[2][32];
    pdl_wait();
    pdl_trigger();
    const float inv = 1.f / (float)a.H;
    int turn = 0;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        T* y = static_cast<T*>(a.y) + r * a.ldy;
        float s = 0.f;
        for (int j = threadIdx.x; j < a.H; j += 1024) s += Elem<T>::to_f(x[j]);
        const float m = row_sum<1024>(s, 0.f, shared, turn++).x * inv;
        s = 0.f;
        for (int j = threadIdx.x; j < a.H; j += 1024) {
            const float d = Elem<T>::to_f(x[j]) - m;
            s = fmaf(d, d, s);
        }
        const float rs = rsqrtf(row_sum<1024>(s, 0.f, shared, turn++).x * inv + a.eps);
        for (int j = threadIdx.x; j < a.H; j += 1024)
            y[j] = Elem<T>::from_f(fmaf((Elem<T>::to_f(x[j]) - m) * rs, param<T>(a.weight, j, a.wide, 1.f), param<T>(a.bias, j, a.wide, 0.f)));
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = m;
            if (a.rstd) a.rstd[r] = rs;
        }
    }
}

// Sum over a warp of a (returned in lanes 0..15) and of b (in lanes 16..31).
__device__ __forceinline__ float warp_sums(float a, float b) {
    const bool high = threadIdx.x & 16;
    float v = (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// dx of the block's rows, and its sums over them for dw and db: partial[block][0] and [1].  G threads have a row, N
// vectors of V elements each, 32 elements where the row is long enough: what a row costs beside its elements (two sums
// over the group, a barrier, addresses) is as many instructions as 16 elements.  A thread's columns are the same
// in every row, so their sums stay in its registers; the weights, which would take as many again, are in shared
// memory.  The groups of G threads go through rows of their own, each with a ring and a barrier, and add up at the end.
// Above 8192 elements a row those sums are 64 registers a thread and about 440 bytes spill: 16384 x 16384 bf16 471 us = 3.4 TB/s, floats
// 769 = 4.2.
template <int G>
constexpr int kGroups = 512 / G;

// out[j] = sum of the groups' sums[p][j], in their order; all threads of the block call it.
template <int P>
__device__ __forceinline__ void add_groups(float* out, const float* sums, int n) {
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        float v = sums[j];
#pragma unroll
        for (int p = 1; p < P; ++p) v += sums[p * n + j];
        out[j] = v;
    }
}
// V floats of shared memory as pairs.
template <int V>
__device__ __forceinline__ void weights_at(const float* p, F2 (&w)[V / 2]) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
        const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(p + k);
        w[k / 2].v = u.x;
        w[k / 2 + 1].v = u.y;
    }
}
template <typename T, int V, int G, int N>
__global__ void __launch_bounds__(G * kGroups<G>, 1) backward_kernel(Args a) {
    constexpr int P = kGroups<G>, W = G / 32;
    static_assert(W == 1 || P < 16, "sixteen named barriers");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ unsigned long long full[P][kMostDepth];
    __shared__ float shared[P][2][2][W];
    const int at = threadIdx.x % G, group = threadIdx.x / G, H = a.H, warp = at >> 5, lane = threadIdx.x & 31;
    // weights as floats, then the groups' rings
    float* weight = reinterpret_cast<float*>(smem);
    unsigned char* rings = smem + (size_t)(H * 4 + 127) / 128 * 128;
    const auto ring = make_ring<T, 2>(rings + (size_t)group * a.depth * 2 * H * sizeof(T), full[group], a, at == 0);
    const long long step = (long long)gridDim.x * P, first = blockIdx.x + (long long)group * gridDim.x;
    pdl_wait();
    pdl_trigger();
    if (at == 0)
        for (int i = 0; i < a.depth; ++i) ring.issue(first + i * step, i);
    const float inv = 1.f / (float)H;
    F2 dw[N][V / 2], db[N][V / 2];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < V / 2; ++k) dw[i][k] = db[i][k] = both(0.f);
    for (int j = threadIdx.x; j < H; j += G * P) weight[j] = param<T>(a.weight, j, a.wide, 1.f);
    __syncthreads();
    float next_m = 0.f, next_rs = 0.f;
    if (first < a.rows) next_m = a.mean[first], next_rs = a.rstd[first];
    int stage = 0;
    uint32_t parity = 0;
    long long turn = 0;
    bool dead = false;
    for (long long r = first; r < a.rows; r += step, ++turn) {
        float m = next_m, rs = next_rs;
        if (r + step < a.rows) next_m = a.mean[r + step], next_rs = a.rstd[r + step];
        if (!dead) dead = !ring.wait(stage, parity, a.wait_cycles);
        if (dead) rs = __uint_as_float(0x7fffffffu);  // (dx of the whole row and this thread's dw with it; db below)
        const T *px = ring.row(stage, 0), *pdy = ring.row(stage, 1);
        const F2 rs2 = both(rs), m2 = both(-m);
        F2 h[N][V / 2], g[N][V / 2], sg2 = both(0.f), sgh2 = both(0.f);
        each_vector<V, G, N>(at, H, [&](int i, int j) {
            F2 d[V / 2], w[V / 2];
            to_pairs<T, V>(load_vec<T, V>(px + j), h[i]);
            to_pairs<T, V>(load_vec<T, V>(pdy + j), d);
            weights_at<V>(weight + j, w);
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                h[i][k] = mul2(add2(h[i][k], m2), rs2);
                g[i][k] = mul2(d[k], w[k]);
                sg2 = add2(sg2, g[i][k]);
                sgh2 = fma2(g[i][k], h[i][k], sgh2);
                dw[i][k] = fma2(d[k], h[i][k], dw[i][k]);
                db[i][k] = add2(db[i][k], d[k]);
            }
        });
        const float mine = warp_sums(sum2(sg2), sum2(sgh2));
        float sg, sgh;
        if constexpr (W > 1) {
            float (*s)[W] = shared[group][turn & 1];
            if ((lane & 15) == 0) s[lane >> 4][warp] = mine;
            meet<G>(group);
            sg = sgh = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                sg += s[0][i];
                sgh += s[1][i];
            }
        } else {
            meet<G>(group);
            sg = __shfl_sync(0xffffffffu, mine, 0);
            sgh = __shfl_sync(0xffffffffu, mine, 16);
        }
        if (at == 0 && !dead) ring.issue(r + a.depth * step, stage);  // (the group has met: the row is in registers)
        const F2 c0 = both(-rs * sg * inv), c1 = both(-rs * sgh * inv);
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
        each_vector<V, G, N>(at, H, [&](int i, int j) {
            F2 o[V / 2];
#pragma unroll
            for (int k = 0; k < V / 2; ++k) o[k] = fma2(h[i][k], c1, fma2(g[i][k], rs2, c0));
            store_vec<T, V>(dx + j, from_pairs<T, V>(o));
        });
        if (++stage == a.depth) stage = 0, parity ^= 1;
    }
    if (dead) {
        tc::settle_after_abort();
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int k = 0; k < V / 2; ++k) db[i][k] = both(__uint_as_float(0x7fffffffu));
    }
    if (!a.partial) return;
    // the groups' sums side by side in shared memory, then added in their order
    float *out = a.partial + (size_t)blockIdx.x * 2 * H, *to = out;
    float* sums = reinterpret_cast<float*>(rings);  // [P][2 * H]: every row has been read
    __syncthreads();
    if (P > 1) to = sums + (size_t)group * 2 * H;
    each_vector<V, G, N>(at, H, [&](int i, int j) {
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const float2 u = split(dw[i][c / 2]), v = split(db[i][c / 2]);
            to[j + c] = c & 1 ? u.y : u.x;
            to[H + j + c] = c & 1 ? v.y : v.x;
        }
    });
    if (P > 1) add_groups<P>(out, sums, 2 * H);
}

// ... of any other row
template <typename T, int G, int N>
__global__ void __launch_bounds__(G * kGroups<G>, 1) backward_odd_kernel(Args a) {
    constexpr int P = kGroups<G>, W = G / 32;
    extern __shared__ float sums[];  // [P][2 * H] where there are several groups
    __shared__ float2 shared[P][2][W];
    const int at = threadIdx.x % G, group = threadIdx.x / G, H = a.H, warp = at >> 5, lane = threadIdx.x & 31;
    const long long step = (long long)gridDim.x * P, first = blockIdx.x + (long long)group * gridDim.x;
    pdl_wait();
    pdl_trigger();
    const float inv = 1.f / (float)H;
    float w[N], dw[N], db[N];
#pragma unroll
    for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.f;
    each_vector<1, G, N>(at, H, [&](int i, int j) { w[i] = param<T>(a.weight, j, a.wide, 1.f); });
    Row<T, G, N> x, dy;
    float m = 0.f, rs = 0.f;
    auto fetch = [&](long long r) {
        x.fetch(a.x, r * a.ldx, at, H);
        dy.fetch(a.dy, r * a.lddy, at, H);
        m = a.mean[r];
        rs = a.rstd[r];
    };
    if (first < a.rows) fetch(first);
    int turn = 0;
    for (long long r = first; r < a.rows; r += step, turn ^= 1) {
        float h[N], g[N], sg = 0.f, sgh = 0.f;
        const float rs_now = rs;
        each_vector<1, G, N>(at, H, [&](int i, int) {
            const float d = dy[i];
            h[i] = (x[i] - m) * rs;
            g[i] = d * w[i];
            sg += g[i];
            sgh = fmaf(g[i], h[i], sgh);
            dw[i] = fmaf(d, h[i], dw[i]);
            db[i] += d;
        });
        if (r + step < a.rows) fetch(r + step);
        sg = warp_sum(sg);
        sgh = warp_sum(sgh);
        if constexpr (W > 1) {
            if (lane == 0) shared[group][turn][warp] = make_float2(sg, sgh);
            meet<G>(group);
            const float2 v = shared[group][turn][lane % W];
            sg = lanes_sum<W>(v.x);
            sgh = lanes_sum<W>(v.y);
        }
        const float c0 = -rs_now * sg * inv, c1 = -rs_now * sgh * inv;
        T* dx = static_cast<T*>(a.dx) + r * a.lddx;
        each_vector<1, G, N>(at, H, [&](int i, int j) { dx[j] = Elem<T>::from_f(fmaf(h[i], c1, fmaf(g[i], rs_now, c0))); });
    }
    if (!a.partial) return;
    float *out = a.partial + (size_t)blockIdx.x * 2 * H, *to = P > 1 ? sums + (size_t)group * 2 * H : out;
    each_vector<1, G, N>(at, H, [&](int i, int j) {
        to[j] = dw[i];
        to[H + j] = db[i];
    });
    if (P > 1) add_groups<P>(out, sums, 2 * H);
}

// Rows too long for registers: dx, a block a row; dw and db by column_kernel.
template <typename T>
__global__ void __launch_bounds__(1024) backward_long_kernel(Args a) {
    __shared__ float2 shared[2][32];
    pdl_wait();
    pdl_trigger();
    const float inv = 1.f / (float)a.H;
    int turn = 0;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T*>(a.x) + r * a.ldx, *dy = static_cast<const T*>(a.dy) + r * a.lddy;
        const float m = a.mean[r], rs = a.rstd[r];
        float sg = 0.f, sgh = 0.f;
        for (int j = threadIdx.x; j < a.H; j += 1024) {
            const float g = Elem<T>::to_f(dy[j]) * param<T>(a.weight, j, a.wide, 1.f);
            sg += g;
            sgh = fmaf(g, (Elem<T>::to_f(x[j]) - m) * rs, sgh);
        }
        const float2 s = row_sum<1024>(sg, sgh, shared, turn++);
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

// dw and db: the blocks' sums, a 32nd of them by each of 32 threads a column, then those, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) finish_kernel(Args a, int partials) {
    __shared__ float s[32][33];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (j < 2 * a.H)
#pragma unroll 10
        for (int p = part; p < partials; p += 32) v += a.partial[(size_t)p * 2 * a.H + j];
    s[part][lane] = v;
    __syncthreads();
    const float t = warp_sum(s[lane][part]);  // column `part` of the block
    const int c = blockIdx.x * 32 + part;
    if (lane == 0 && c < 2 * a.H) {
        if (c < a.H) {
            if (a.dweight) put_param<T>(a.dweight, c, a.wide, t);
        } else if (a.dbias) {
            put_param<T>(a.dbias, c - a.H, a.wide, t);
        }
    }
}

// Calls f with threads a row and vectors a thread for H elements in vectors of V: 16 elements a thread, 8 for short rows, 32
// for long ones; 24 where that leaves fewer idle and their instructions, not HBM, are the limit: of 16-bit rows (forward,
// 8192 x 5120 53 us with 16 and 33 with 24, 16384 x 1088 28 and 18; back 72 and 62, but 8192 x 1536 31 and 34; floats the
// same or slower).  False where a row is too long for registers.
template <int V, bool kBack, typename F>
bool with_shape(int H, F f) {
    constexpr int K = 8 / V;
    auto shape = [&](auto g, auto n) {
        f(g, n);
        return true;
    };
    using std::integral_constant;
    if (H <= 256) return shape(integral_constant<int, 32>(), integral_constant<int, K>());
    if (H <= 512) return shape(integral_constant<int, 32>(), integral_constant<int, 2 * K>());
    if constexpr (V == 8 && !kBack) {
        if (H <= 768) return shape(integral_constant<int, 32>(), integral_constant<int, 3>());
        if (H > 1024 && H <= 1536) return shape(integral_constant<int, 64>(), integral_constant<int, 3>());
        if (H > 2048 && H <= 128 * 24) return shape(integral_constant<int, 128>(), integral_constant<int, 3>());
    }
    if (H <= 1024) return shape(integral_constant<int, 64>(), integral_constant<int, 2 * K>());
    if (H <= 2048) return shape(integral_constant<int, 128>(), integral_constant<int, 2 * K>());
    if (H <= 4096) return shape(integral_constant<int, 256>(), integral_constant<int, 2 * K>());
    if constexpr (V == 8)
        if (H <= 6144) return shape(integral_constant<int, 256>(), integral_constant<int, 3>());
    if (H <= 8192) return shape(integral_constant<int, 512>(), integral_constant<int, 2 * K>());
    if (H <= 16384) return shape(integral_constant<int, 512>(), integral_constant<int, 4 * K>());
    return false;
}
// ... for rows that are loaded element by element: 8 a thread, 16 above 4096
template <typename F>
bool with_odd_shape(int H, F f) {
    auto shape = [&](auto g, auto n) {
        f(g, n);
        return true;
    };
    using std::integral_constant;
    if (H <= 256) return shape(integral_constant<int, 32>(), integral_constant<int, 8>());
    if (H <= 512) return shape(integral_constant<int, 64>(), integral_constant<int, 8>());
    if (H <= 1024) return shape(integral_constant<int, 128>(), integral_constant<int, 8>());
    if (H <= 2048) return shape(integral_constant<int, 256>(), integral_constant<int, 8>());
    if (H <= 4096) return shape(integral_constant<int, 512>(), integral_constant<int, 8>());
    if (H <= 8192) return shape(integral_constant<int, 512>(), integral_constant<int, 16>());
    return false;
}

}  // namespace norm
}  // namespace kleos
