// A whole MoE layer for the few tokens of a decode step: the router, the experts that it chose and the weighted sum of
// their results.
//
//   l = x Wg^T + bias;  e_1 .. e_K the K largest l (ties: the lower expert);  w_k = exp(l_k) / (exp(l_1) + .. + exp(l_K))
//   out = sum over k of w_k (W2[e_k] h_k + b2[e_k]),   h_k = f(z) or, gated, f(z) z',   z (and z') = W1[e_k] x + b1[e_k]
//
// Three launches: gate_kernel chooses, stream_kernel (moe_stream.cuh) makes h and then out.  A call reads the chosen experts' weights
// once and little else: bound by HBM, and by latency for one token.  The router is latency too: 8 us for one token alone, 14 for 128 (64 experts,
// H = 2048; with rows straight from memory 12 and 28, in 64-bit arithmetic 14 and 43).
//
// The logits are sums of 46 bits: which expert is chosen does not hang on the order of a sum.  An expert whose logit is
// minus infinity is never chosen: the place keeps -1 and a weight of 0, and a token all of whose experts are out gives zeros.
#pragma once

#include <cooperative_groups.h>

#include "activation.cuh"

namespace kleos {
namespace tokens {
using namespace ops;

constexpr int kMostTokens = 128;
constexpr int kMostPlaces = kMostTokens * kMaxTopK;

struct Args {
    const void *x, *gate, *w1, *b1, *w2, *b2;
    const float* gate_bias;
    void* out;
    int* topk;       // [T, K]
    float* weights;  // [T, K]
    void* h;         // [T * K] rows of ldh
    long long ldx, ldo, ldh;
    int T, H, I, E, K;
    int act;
    int group;  // tokens of a cluster of gate_kernel
};

// ---------------------------------------------------------------- the router
constexpr int kGateBlocks = 8, kGateWarps = 8, kGateTokens = 4;

// A sum that keeps what its additions round off (two floats at once): the total is exact to about 2^-46.  The multiprocessor's 64-bit
// additions and conversions would take ten times as long (128 tokens, 64 experts: 41 us).  Once an infinity is in it, or a product or a
// sum on the way is past the floats' range, the rest is no number: the kernel adds such a logit up anew in 64 bits.
struct Kept {
    F2 s, rest;
    __device__ __forceinline__ Kept() : s(both(0.f)), rest(both(0.f)) {}
    static __device__ __forceinline__ F2 minus(F2 a, F2 b) { return fma2(b, both(-1.f), a); }
    __device__ __forceinline__ void add(F2 p) {
        const F2 to = add2(s, p), b = minus(to, s);
        rest = add2(rest, add2(minus(s, minus(to, b)), minus(p, b)));
        s = to;
    }
    __device__ __forceinline__ double total() const {
        const float2 a = split(s), b = split(rest);
        return ((double)a.x + (double)a.y) + ((double)b.x + (double)b.y);
    }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A cluster takes up to kGateTokens tokens: its warps share the experts, its blocks the tokens that are then chosen for.  Rows on 16-byte
// boundaries (V above 1) come a kilobyte at a time through shared memory, kGateStages steps of it.
constexpr int kGateChunk = 1024, kGateStages = 5, kGateRows = kGateWarps + kGateTokens;
constexpr int kGateSmem = kGateStages * kGateRows * kGateChunk;  // (where V is above 1)

template <typename T, int V>
__global__ void __launch_bounds__(32 * kGateWarps) gate_kernel(Args a) {
    namespace cg = cooperative_groups;
    constexpr int P = V > 1 ? V / 2 : 1;
    typedef char Stage[kGateRows][kGateChunk];  // a row of every warp's expert, then the tokens
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double logits[kMaxExperts];
    extern __shared__ __align__(128) char memory[];
    Stage* const stage = reinterpret_cast<Stage*>(memory);
    const int block = (int)cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t0 = (int)(blockIdx.x / kGateBlocks) * a.group, n = min(a.group, a.T - t0);
    cluster.sync();  // (every block of the cluster is there to be written to)
    pdl_wait();
    pdl_trigger();
    const T* x = static_cast<const T*>(a.x) + t0 * a.ldx;
    auto add = [](Kept& s, F2 p, F2 q) {
        const F2 r = mul2(p, q);  // (of 16-bit factors: exact)
        s.add(r);
        if constexpr (sizeof(T) == 4) s.rest = add2(s.rest, fma2(p, q, mul2(r, both(-1.f))));
    };
    for (int e0 = block * kGateWarps; e0 < a.E; e0 += kGateBlocks * kGateWarps) {
        const int e = e0 + warp;
        const T* w = static_cast<const T*>(a.gate) + (size_t)min(e, a.E - 1) * a.H;
        Kept s[kGateTokens];
        if constexpr (V > 1) {
            const int row_bytes = a.H * (int)sizeof(T), steps = (row_bytes + kGateChunk - 1) / kGateChunk;
            auto copy = [&](int step) {
                if (step < steps)
#pragma unroll
                    for (int i = threadIdx.x; i < kGateRows * (kGateChunk / 16); i += 32 * kGateWarps) {
                        const int row = i / (kGateChunk / 16), piece = i % (kGateChunk / 16) * 16, at = step * kGateChunk + piece;
                        if (row >= kGateWarps + n) break;
                        const char* from = row < kGateWarps ? reinterpret_cast<const char*>(static_cast<const T*>(a.gate) + (size_t)min(e0 + row, a.E - 1) * a.H)
                                                            : reinterpret_cast<const char*>(x + (row - kGateWarps) * a.ldx);
                        const bool there = at < row_bytes;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(&stage[step % kGateStages][row][piece])),
                                     "l"(there ? from + at : from), "r"(there ? 16 : 0) : "memory");
                    }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            for (int i = 0; i < kGateStages - 1; ++i) copy(i);
            for (int step = 0; step < steps; ++step) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kGateStages - 2) : "memory");
                __syncthreads();
                copy(step + kGateStages - 1);
                const auto& rows = stage[step % kGateStages];
#pragma unroll
                for (int i = 0; i < kGateChunk / 512; ++i) {
                    const int at = i * 512 + lane * 16;
                    F2 p[P];
                    to_pairs<T, V>(load_vec<T, V>(reinterpret_cast<const T*>(&rows[warp][at])), p);
#pragma unroll
                    for (int t = 0; t < kGateTokens; ++t) {
                        if (t >= n) break;
                        F2 q[P];
                        to_pairs<T, V>(load_vec<T, V>(reinterpret_cast<const T*>(&rows[kGateWarps + t][at])), q);
#pragma unroll
                        for (int j = 0; j < P; ++j) add(s[t], p[j], q[j]);
                    }
                }
            }
            __syncthreads();  // (the next experts' rows come into the same places)
        } else {
#pragma unroll 4
            for (int k = lane; k < a.H; k += 32) {
                const F2 p = pair(Elem<T>::to_f(w[k]), 0.f);
#pragma unroll
                for (int t = 0; t < kGateTokens; ++t)
                    if (t < n) add(s[t], p, pair(Elem<T>::to_f(x[t * a.ldx + k]), 0.f));
            }
        }
        auto put = [&](int t, double v) {
            if (lane == 0 && e < a.E) *cluster.map_shared_rank(&logits[e], t) = a.gate_bias ? v + (double)a.gate_bias[e] : v;
        };
        unsigned anew = 0;  // tokens, the same for the whole warp
#pragma unroll
        for (int t = 0; t < kGateTokens; ++t) {
            if (t >= n) break;
            const double v = warp_sum(s[t].total());
            if (!isfinite(v)) anew |= 1u << t;
            put(t, v);
        }
#pragma unroll 1
        for (; anew; anew &= anew - 1) {
            const int t = __ffs(anew) - 1;
            double v = 0.0;
#pragma unroll 1
            for (int k = lane; k < a.H; k += 32) v += (double)Elem<T>::to_f(w[k]) * (double)Elem<T>::to_f(x[t * a.ldx + k]);
            put(t, warp_sum(v));
        }
    }
    cluster.sync();
    if (block >= n || warp != 0) return;
    const int t = t0 + block;
    // a logit as a number that grows with it, NaN above all; 0: minus infinity, or chosen already
    auto key_of = [](double v) {
        const unsigned long long b = __double_as_longlong(v == 0.0 ? 0.0 : v);
        return v != v ? ~0ull : v == -INFINITY ? 0ull : (b >> 63) ? ~b : b | 1ull << 63;
    };
    double mine = 0.0, top = 0.0;  // lane k: the k-th logit
    int id = -1;
    for (int k = 0; k < a.K; ++k) {
        unsigned long long best = 0;
        int at = kMaxExperts;
        for (int e = lane; e < a.E; e += 32) {
            const unsigned long long key = key_of(logits[e]);
            if (key > best) best = key, at = e;
        }
        const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32));
        const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32) == high ? (unsigned)best : 0u);
        if (high == 0 && low == 0) break;  // only experts that are out are left
        at = __reduce_min_sync(0xffffffffu, (unsigned)(best >> 32) == high && (unsigned)best == low ? at : kMaxExperts);
        const double v = logits[at];
        if (k == 0) top = v;
        if (lane == k) mine = v, id = at;
        __syncwarp();
        if (lane == 0) logits[at] = -INFINITY;
        __syncwarp();
    }
    const double p = id < 0 ? 0.0 : exp(mine - top), sum = warp_sum(p);
    if (lane < a.K) {
        a.topk[t * a.K + lane] = id;
        a.weights[t * a.K + lane] = id < 0 ? 0.f : (float)(p / sum);
    }
}

}  // namespace tokens
}  // namespace kleos
