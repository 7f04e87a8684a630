// The activation between an expert's two products, with its gradient.
//
//   h[r, i]  = f(z[r, i])                     or, gated, f(z[r, i]) z[r, I + i]
//   dz[r, i] = dh[r, i] f'(z[r, i])           or, gated, dh f'(z[r, i]) z[r, I + i] and dh f(z[r, i])
//
//   f: 0 ReLU max(z, 0), 1 GELU z N(z) with N the normal distribution's sum, 2 SiLU z s(z) with s(z) = 1 / (1 + e^-z)
//
// Each element is read once and each result written once, in 32 bits with one rounding.  16384 rows, I = 2048, one call after the other: ReLU and SiLU
// are bound by HBM (gated, bf16: 32 us forward, 60 backward, 6.2 and 5.6 TB/s; floats 61 and 105, 6.5 and 6.4), GELU's erfc and exp of 32 bits
// by issue (gated, bf16: 66 and 88 us, 3.0 and 3.8 TB/s; floats 86 and 107); so are rows that are loaded an element at a time (2943 x 1087
// floats, GELU: 14 and 16).
#pragma once

#include "ops_common.cuh"

namespace kleos {
namespace act {
using namespace ops;

constexpr int kKinds = 3;
constexpr char kWhich[] = "hidden_act must be 0 (ReLU), 1 (GELU) or 2 (SiLU)";

struct Args {
    const void* z;
    const void* dh;  // null: forward
    void* out;       // h, or dz
    long long ldz, ldh, ldo;
    long long rows;
    int I;
};

// N(z) from erfc, which keeps its relative accuracy where N is small (0.5 (1 + erf) is off by 5 % at z = -5).
__device__ __forceinline__ float normal_sum(float z) { return 0.5f * erfcf(-0.70710678118654752f * z); }
// s(z) and 1 - s(z), from e^-|z|, which cannot overflow.  16-bit results do not show the fast exponential's and quotient's
// last bits (relative 2^-20 up to |z| = 10, 2^-17 at 88).
template <bool kFast>
__device__ __forceinline__ float2 sigmoid(float z) {
    const float e = kFast ? __expf(-fabsf(z)) : expf(-fabsf(z));
    const float r = kFast ? __fdividef(1.f, 1.f + e) : 1.f / (1.f + e);
    return z >= 0.f ? make_float2(r, e * r) : make_float2(e * r, r);
}

template <int kKind, bool kFast>
__device__ __forceinline__ float value(float z) {
    if constexpr (kKind == 0) return z > 0.f ? z : z != z ? z : 0.f;
    if constexpr (kKind == 1) return z * normal_sum(z);
    return z * sigmoid<kFast>(z).x;
}

// Value and slope.  ReLU's slope at zero is 0.
template <int kKind, bool kFast>
__device__ __forceinline__ float2 both_of(float z) {
    if constexpr (kKind == 0) return make_float2(value<0, kFast>(z), z > 0.f ? 1.f : 0.f);
    if constexpr (kKind == 1) {
        const float n = normal_sum(z);
        return make_float2(z * n, fmaf(z, 0.3989422804014327f * expf(-0.5f * z * z), n));
    }
    const float2 p = sigmoid<kFast>(z);
    return make_float2(z * p.x, p.x * fmaf(z, p.y, 1.f));
}

// Calls f with the kind as a constant.
template <typename F>
auto with_kind(int kind, F f) {
    if (kind == 0) return f(std::integral_constant<int, 0>());
    if (kind == 1) return f(std::integral_constant<int, 1>());
    return f(std::integral_constant<int, 2>());
}

// A block takes blockDim.x vectors of columns of blockDim.y rows at a time; a thread has so many rows on their way that it is 16 bytes of each
// matrix or more.
template <typename T, int V, int kKind, bool kGated, bool kBack>
__global__ void __launch_bounds__(256) activation_kernel(Args a) {
    constexpr bool kFast = sizeof(T) == 2;
    constexpr int U = V * sizeof(T) >= 16 ? 1 : V * sizeof(T) >= 8 ? 2 : 4;
    pdl_wait();
    pdl_trigger();
    const int i = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    if (i >= a.I) return;
    const T* z = static_cast<const T*>(a.z) + i;
    T* out = static_cast<T*>(a.out) + i;
    const long long step = (long long)gridDim.y * blockDim.y;
    for (long long r0 = (long long)blockIdx.y * blockDim.y + threadIdx.y; r0 < a.rows; r0 += U * step) {
        Vec<T, V> g[U], u[U], d[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {  // (rows past the last are the last)
            const long long r = min(r0 + k * step, a.rows - 1);
            g[k] = load_vec<T, V>(z + r * a.ldz);
            if constexpr (kGated) u[k] = load_vec<T, V>(z + r * a.ldz + a.I);
            if constexpr (kBack) d[k] = load_vec<T, V>(static_cast<const T*>(a.dh) + r * a.ldh + i);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const long long r = r0 + k * step;
            if (r >= a.rows) break;
            Vec<T, V> first, second;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float x = Elem<T>::to_f(g[k].v[j]);
                if constexpr (!kBack) {
                    const float f = value<kKind, kFast>(x);
                    first.v[j] = Elem<T>::from_f(kGated ? f * Elem<T>::to_f(u[k].v[j]) : f);
                } else {
                    const float2 f = both_of<kKind, kFast>(x);
                    const float dh = Elem<T>::to_f(d[k].v[j]);
                    first.v[j] = Elem<T>::from_f(kGated ? dh * Elem<T>::to_f(u[k].v[j]) * f.y : dh * f.y);
                    if constexpr (kGated) second.v[j] = Elem<T>::from_f(dh * f.x);
                }
            }
            store_vec<T, V>(out + r * a.ldo, first);
            if constexpr (kGated && kBack) store_vec<T, V>(out + r * a.ldo + a.I, second);
        }
    }
}

}  // namespace act
}  // namespace kleos
