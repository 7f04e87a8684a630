// What the operators around the experts share (layer norm, sort by expert, rows there and back, products): vectors of
// elements, sums over a warp, launches, refusals.
#pragma once

#include <cstdio>

#include "common.cuh"

namespace kleos {
namespace ops {

constexpr int kMaxExperts = 1024;  // experts of a sort or of products

// N elements that are loaded and stored at once.
template <typename T, int N>
struct __align__(sizeof(T) * N) Vec {
    T v[N];
};

// No read-only path here either: the kernel in front may still be writing what its successor's blocks wait for.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
    return *reinterpret_cast<const Vec<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
    *reinterpret_cast<Vec<T, N>*>(p) = v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Two floats in a register pair: one instruction for both, each rounded as the scalar one would (add, mul, fma .f32x2).
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 pair(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ F2 both(float a) { return pair(a, a); }
__device__ __forceinline__ float2 split(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ float sum2(F2 a) {
    const float2 f = split(a);
    return f.x + f.y;
}

// A vector of elements as pairs of floats, and back (one rounding).
template <typename T, int V>
__device__ __forceinline__ void to_pairs(const Vec<T, V>& v, F2 (&p)[V / 2]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) p[i] = pair(v.v[2 * i], v.v[2 * i + 1]);
    } else {
        const auto* h = reinterpret_cast<const typename Pack2<T>::type*>(v.v);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = Pack2<T>::to_f2(h[i]);
            p[i] = pair(f.x, f.y);
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> from_pairs(const F2 (&p)[V / 2]) {
    Vec<T, V> v;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float2 f = split(p[i]);
        if constexpr (sizeof(T) == 4) {
            v.v[2 * i] = f.x;
            v.v[2 * i + 1] = f.y;
        } else {
            reinterpret_cast<typename Pack2<T>::type*>(v.v)[i] = Pack2<T>::from_f2(f.x, f.y);
        }
    }
    return v;
}

// Offsets come from the caller's device memory, so no kernel trusts them: rows outside [0, rows) do not exist.
struct Group {
    int begin, end;
};
__device__ __forceinline__ Group group_rows(const int* offsets, int e, int rows) {
    Group g;
    g.begin = min(max(offsets[e], 0), rows);
    g.end = max(min(offsets[e + 1], rows), g.begin);
    return g;
}

inline int refuse(const char* call, int code, const char* what) {
    std::fprintf(stderr, "[kleos_b200] %s: %s\n", call, what);
    return code;
}

inline bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline cudaStream_t stream_of(void* stream) { return stream ? static_cast<cudaStream_t>(stream) : cudaStreamPerThread; }

// Launched as the kernels of a forward are (see pdl_wait()): every kernel here calls pdl_wait() before it touches
// global memory.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t lc{};
    lc.gridDim = grid;
    lc.blockDim = dim3((unsigned)threads);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, kernel, args...);
}

inline int finish(const char* call, cudaError_t e) {
    if (e == cudaSuccess) return KLEOS_OK;
    cudaGetLastError();  // (a refused launch is reported here and not to a later call)
    std::fprintf(stderr, "[kleos_b200] %s: launch failed: %s\n", call, cudaGetErrorString(e));
    return KLEOS_E_CUDA;
}

// Multiprocessors of the current device, 0 when there is none.
inline int sm_count() {
    static int known[64] = {};
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 0;
    if (dev < 64 && known[dev]) return known[dev];
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < 64) known[dev] = n;
    return n;
}

// Lets a kernel have more than 48 KiB of dynamic shared memory, once per device.
template <typename... P>
cudaError_t allow_smem(void (*kernel)(P...), bool (&done)[64], int bytes) {
    int dev = -1;
    cudaError_t rc = cudaGetDevice(&dev);
    if (rc != cudaSuccess || (dev < 64 && done[dev])) return rc;
    rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (rc == cudaSuccess && dev < 64) done[dev] = true;
    return rc;
}

// Blocks of a kernel that all multiprocessors hold at once, which is what a kernel whose blocks share out their work
// evenly is launched with.
template <typename... P>
int resident_blocks(void (*kernel)(P...), int threads, size_t smem) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) return 0;
    return n * sm_count();
}

// Calls f with a null pointer of the element type of `torch_dtype` (0 float, 2 bf16, 3 fp16).
template <typename F>
int with_type(const char* call, int torch_dtype, F f) {
    switch (torch_dtype) {
        case 0: return f(static_cast<float*>(nullptr));
        case 2: return f(static_cast<__nv_bfloat16*>(nullptr));
        case 3: return f(static_cast<__half*>(nullptr));
        default: return refuse(call, KLEOS_E_UNSUPPORTED, "torch_dtype must be 0 (float), 2 (bf16) or 3 (fp16)");
    }
}

}  // namespace ops
}  // namespace kleos
