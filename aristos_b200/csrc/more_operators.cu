// C ABI of further operators around the experts: the activation between an expert's two products, and low-rank adapters of many
// requests, each with its gradients.  No counterpart in the reference.  None of them needs kleos_initialize, allocates, synchronises or
// keeps anything between calls.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "activation.cuh"
#include "adapters.cuh"
#include "adapters_mma.cuh"

namespace kleos {
namespace {
using namespace ops;

constexpr int kMostColumns = 1 << 22;

// ---------------------------------------------------------------- activation
template <bool kBack>
int activation(const char* call, const act::Args& a, int kind, bool gated, int torch_dtype, cudaStream_t st) {
    return with_type(call, torch_dtype, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        constexpr int W = 16 / sizeof(T);
        return act::with_kind(kind, [&](auto k) {
            auto run = [&](auto v, auto g) {
                constexpr int V = decltype(v)::value;
                const int vectors = (a.I + V - 1) / V;
                int lanes = 32;
                while (lanes < 256 && lanes < vectors) lanes *= 2;
                const int deep = 256 / lanes, across = (vectors + lanes - 1) / lanes;
                // every block a few rows, eight blocks a multiprocessor
                const long long want = std::max(1LL, 8LL * sm_count() / across), most = (a.rows + deep - 1) / deep;
                const dim3 grid(across, (unsigned)std::min<long long>(65535, std::min(most, std::max(want, (most + 15) / 16))));
                cudaLaunchConfig_t lc{};
                lc.gridDim = grid;
                lc.blockDim = dim3(lanes, deep);
                lc.stream = st;
                cudaLaunchAttribute at{};
                at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
                at.val.programmaticStreamSerializationAllowed = 1;
                lc.attrs = &at;
                lc.numAttrs = 1;
                return finish(call, cudaLaunchKernelEx(&lc, act::activation_kernel<T, V, decltype(k)::value, decltype(g)::value, kBack>, a));
            };
            auto with_v = [&](auto g) {
                using std::integral_constant;
                const std::initializer_list<long long> lds = {a.ldz, a.ldo, kBack ? a.ldh : 0, a.I};
                if (by(16, sizeof(T), {a.z, a.dh, a.out}, lds)) return run(integral_constant<int, W>(), g);
                if (by(2 * sizeof(T), sizeof(T), {a.z, a.dh, a.out}, lds)) return run(integral_constant<int, 2>(), g);
                return run(integral_constant<int, 1>(), g);
            };
            return gated ? with_v(std::true_type()) : with_v(std::false_type());
        });
    });
}

const char* bad_activation(long long rows, int I, int gated, long long ldz, long long ldh) {
    if (rows < 0 || rows > kMostRows || I < 1 || I > kMostColumns) return "rows must be from 0 to 2^31 - 2^16, I from 1 to 2^22";
    if (ldz < (gated ? 2LL * I : I) || ldh < I) return "no row may be longer than its stride";
    return nullptr;
}

// ---------------------------------------------------------------- adapters
const char* bad_adapters(int rows, int R, int L, int r, int N, int K) {
    if (rows < 0 || rows > kMostRows || R < 1 || R > adapters::kMostRequests) return "rows must be from 0 to 2^31 - 2^16, requests from 1 to 65536";
    if (L < 1 || L > 65535 || r < 1 || r > adapters::kMostRank) return "adapters must be from 1 to 65535, their rank from 1 to 128";
    if (N < 1 || K < 1 || N > kMostColumns || K > kMostColumns) return "N and K must be from 1 to 2^22";
    return nullptr;
}

// f with the smallest of the ranks that kernels are made for as a constant.
template <typename F>
cudaError_t with_rank(int r, F f) {
    using std::integral_constant;
    if (r <= 16) return f(integral_constant<int, 16>());
    if (r <= 32) return f(integral_constant<int, 32>());
    if (r <= 64) return f(integral_constant<int, 64>());
    return f(integral_constant<int, 128>());
}

template <typename T, bool kBack, int RT, int TR>
cudaError_t adapter_rows_mma(const adapters::Args& a, cudaStream_t st) {
    using namespace adapters;
    const long long tiles = a.rows / TR + a.R + 2;  // at most
    // blocks of a cluster: while every warp has 128 bytes of a row to sum, and until two blocks a multiprocessor are there
    int cluster = 1;
    while (cluster < 8 && tiles * cluster < 2LL * sm_count() && a.len * 2 > cluster * Shape<RT, TR>::KS * 128) cluster *= 2;
    if (tiles * cluster > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const auto kernel = rows_mma_kernel<T, kBack, RT, TR>;
    static bool allowed[64];
    cudaError_t rc = allow_smem(kernel, allowed, Shape<RT, TR>::kBytes);
    if (rc == cudaSuccess) rc = launch(kernel, dim3((unsigned)(tiles * cluster)), 256, Shape<RT, TR>::kBytes, cluster, st, a);
    return rc;
}

template <typename T, bool kBack>
cudaError_t adapter_rows(const adapters::Args& a, cudaStream_t st) {
    using namespace adapters;
    constexpr int W = 16 / sizeof(T);
    if constexpr (sizeof(T) == 2) {
        // (ranks up to 16 are read 8 bytes at a time)
        if ((a.r % 8 == 0 || (a.r % 4 == 0 && a.r < 16)) && by_16(2, {a.in, a.p, a.q, a.base, a.out}, {a.ldi, a.ldb, a.ldo, a.len, a.cols}))
            return with_rank(a.r, [&](auto rt) {
                constexpr int RT = decltype(rt)::value;
                // requests of few rows: tiles of as many as the tensor cores take
                if (a.rows < 24LL * a.R) return adapter_rows_mma<T, kBack, RT, 16>(a, st);
                if constexpr (RT <= 64)
                    if (a.r % 8 == 0 && a.rows / kPipeRows + a.R / 2 >= sm_count()) {  // (its copies are of 16 bytes)
                        const auto kernel = rows_pipe_kernel<T, kBack, RT>;
                        static bool allowed[64];
                        cudaError_t rc = allow_smem(kernel, allowed, PipeShape<RT>::kBytes);
                        if (rc == cudaSuccess) rc = launch(kernel, dim3((unsigned)(a.rows / kPipeRows + a.R + 2)), kPipeThreads, PipeShape<RT>::kBytes, 1, st, a);
                        return rc;
                    }
                return adapter_rows_mma<T, kBack, RT, 64>(a, st);
            });
    }
    const long long tiles = a.rows / kRowsSimt + a.R + 2;  // at most
    int cluster = 1;
    while (cluster < 8 && 2 * tiles * cluster <= 4LL * sm_count() && a.len > cluster * 256) cluster *= 2;
    if (tiles * cluster > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const bool wide = by_16(sizeof(T), {a.in, kBack ? nullptr : a.p}, {a.ldi, a.len});
    const auto kernel = wide ? rows_kernel<T, kBack ? 4 : W, kBack> : rows_kernel<T, 1, kBack>;
    Args g = a;
    g.quads = a.r % 4 == 0 && aligned(kBack ? a.p : a.q, 4 * sizeof(T));
    return launch(kernel, dim3((unsigned)(tiles * cluster)), 256, 0, cluster, st, g);
}

// Blocks of a cluster that share the rows of an adapter: until so many blocks a multiprocessor are there, while each has `rows` of them on average.
int grads_cluster(long long groups, long long blocks, long long all, long long rows) {
    int cluster = 1;
    while (cluster < 8 && 2 * groups * cluster <= blocks * sm_count() && all > cluster * rows) cluster *= 2;
    return cluster;
}

// One or both of them (no strips: not).
template <typename T>
cudaError_t adapter_grads(adapters::Grads a, adapters::Grads b, cudaStream_t st) {
    using namespace adapters;
    auto tensor = [](const Grads& g) { return !g.out || (sizeof(T) == 2 && g.r % 2 == 0 && by_16(2, {g.in}, {g.ldi, g.cols}) && aligned(g.c, 8)); };
    if (a.out && b.out && tensor(a) != tensor(b)) {
        const cudaError_t rc = adapter_grads<T>(a, Grads{}, st);
        return rc == cudaSuccess ? adapter_grads<T>(b, Grads{}, st) : rc;
    }
    if (!a.out) std::swap(a, b);
    if (!a.out) return cudaSuccess;
    auto cut = [&](int columns) {
        a.strips = (a.cols + columns - 1) / columns;
        b.strips = b.out ? (b.cols + columns - 1) / columns : 0;
        return (long long)a.strips + b.strips;
    };
    if constexpr (sizeof(T) == 2) {
        if (tensor(a))
            return with_rank(std::min(a.r, 64), [&](auto rt) {
                constexpr int RT = decltype(rt)::value <= 64 ? decltype(rt)::value : 64, kBytes = GradShape<T, RT>::kBytes;
                const long long strips = cut(kGradColumns), parts = (a.r + RT - 1) / RT;
                const int cluster = grads_cluster(strips * a.L * parts, 4, a.rows, kGradRows * 4LL);
                auto run = [&](auto wide, auto both) {
                    const auto kernel = grads_mma_kernel<T, RT, decltype(wide)::value, decltype(both)::value ? 2 : 1>;
                    static bool allowed[64];
                    cudaError_t rc = allow_smem(kernel, allowed, kBytes);
                    if (rc == cudaSuccess) rc = launch(kernel, dim3((unsigned)(strips * cluster), a.L, (unsigned)parts), 256, kBytes, cluster, st, a, b);
                    return rc;
                };
                if (a.wide_out) return run(std::true_type(), std::true_type());
                return a.rows <= kBothParts ? run(std::false_type(), std::true_type()) : run(std::false_type(), std::false_type());
            });
    }
    const long long strips = cut(32), parts = (a.r + 15) / 16;
    const int cluster = grads_cluster(strips * a.L * parts, 6, a.rows, 256);
    return launch(grads_kernel<T>, dim3((unsigned)(strips * cluster), a.L, (unsigned)parts), 256, 0, cluster, st, a, b);
}

}  // namespace
}  // namespace kleos

using namespace kleos;

extern "C" {

int kleos_activation(const void* z, long long ldz, long long rows, int I, int hidden_act, int gated, int torch_dtype, void* h, long long ldh,
                     void* stream) {
    const char* call = "kleos_activation";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (hidden_act < 0 || hidden_act >= act::kKinds) return refuse(call, KLEOS_E_ARG, act::kWhich);
    if (const char* bad = bad_activation(rows, I, gated, ldz, ldh)) return refuse(call, KLEOS_E_ARG, bad);
    if (rows == 0) return KLEOS_OK;
    if (!z || !h) return refuse(call, KLEOS_E_ARG, kNull);
    if (!whole(bytes_of(torch_dtype), {z, h})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, kNoDevice);
    act::Args a{};
    a.z = z; a.out = h; a.ldz = ldz; a.ldo = ldh; a.rows = rows; a.I = I;
    return activation<false>(call, a, hidden_act, gated != 0, torch_dtype, stream_of(stream));
}

int kleos_activation_backward(const void* dh, long long lddh, const void* z, long long ldz, long long rows, int I, int hidden_act, int gated,
                              int torch_dtype, void* dz, long long lddz, void* stream) {
    const char* call = "kleos_activation_backward";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (hidden_act < 0 || hidden_act >= act::kKinds) return refuse(call, KLEOS_E_ARG, act::kWhich);
    if (const char* bad = bad_activation(rows, I, gated, std::min(ldz, lddz), lddh)) return refuse(call, KLEOS_E_ARG, bad);
    if (rows == 0) return KLEOS_OK;
    if (!dh || !z || !dz) return refuse(call, KLEOS_E_ARG, kNull);
    if (!whole(bytes_of(torch_dtype), {dh, z, dz})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, kNoDevice);
    act::Args a{};
    a.z = z; a.dh = dh; a.out = dz; a.ldz = ldz; a.ldh = lddh; a.ldo = lddz; a.rows = rows; a.I = I;
    return activation<true>(call, a, hidden_act, gated != 0, torch_dtype, stream_of(stream));
}

int kleos_adapter_products(const void* x, long long ldx, const int32_t* offsets, const int32_t* adapter, const void* a, const void* b,
                           const float* scale, const void* base, long long ldb, int rows, int R, int L, int r, int N, int K,
                           int torch_dtype, void* y, long long ldy, float* u, void* stream) {
    const char* call = "kleos_adapter_products";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (const char* bad = bad_adapters(rows, R, L, r, N, K)) return refuse(call, KLEOS_E_ARG, bad);
    if (ldx < K || ldy < N || (base && ldb < N) || (base == y && ldb != ldy)) return refuse(call, KLEOS_E_ARG, "no row may be longer than its stride, and base in place has y's");
    if (rows == 0) return KLEOS_OK;
    if (!x || !offsets || !adapter || !a || !b || !y) return refuse(call, KLEOS_E_ARG, kNull);
    if (!whole(bytes_of(torch_dtype), {x, a, b, base, y}) || !whole(4, {offsets, adapter, scale, u})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, kNoDevice);
    adapters::Args g{};
    g.in = x; g.p = a; g.q = b; g.base = base; g.out = y; g.u = u; g.offsets = offsets; g.adapter = adapter; g.scale = scale;
    g.ldi = ldx; g.ldb = ldb; g.ldo = ldy; g.rows = rows; g.R = R; g.L = L; g.r = r; g.len = K; g.cols = N;
    return with_type(call, torch_dtype, [&](auto* null) {
        return finish(call, adapter_rows<std::remove_pointer_t<decltype(null)>, false>(g, stream_of(stream)));
    });
}

long long kleos_adapter_products_workspace(int rows, int r) {
    return rows < 0 || rows > kMostRows || r < 1 || r > adapters::kMostRank ? KLEOS_E_ARG : 4LL * rows * r;
}

int kleos_adapter_products_backward(const void* dy, long long lddy, const void* x, long long ldx, const float* u, const int32_t* offsets,
                                    const int32_t* adapter, const void* a, const void* b, const float* scale, const void* dbase,
                                    long long ldb, int rows, int R, int L, int r, int N, int K, int torch_dtype, int grad_dtype, void* dx,
                                    long long lddx, void* da, void* db, void* workspace, long long workspace_bytes, void* stream) {
    const char* call = "kleos_adapter_products_backward";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (grad_dtype != 0 && grad_dtype != torch_dtype) return refuse(call, KLEOS_E_UNSUPPORTED, "grad_dtype must be 0 (float) or the element type");
    if (const char* bad = bad_adapters(rows, R, L, r, N, K)) return refuse(call, KLEOS_E_ARG, bad);
    if (lddy < N || ldx < K || lddx < K || (dbase && ldb < K) || (dbase == dx && ldb != lddx))
        return refuse(call, KLEOS_E_ARG, "no row may be longer than its stride, and dbase in place has dx's");
    if (!offsets || !adapter || (rows > 0 && (!dy || !x || !u || !a || !b || !dx))) return refuse(call, KLEOS_E_ARG, kNull);
    if (da && rows > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < 4LL * rows * r))
        return refuse(call, KLEOS_E_ARG, "da needs a 16-byte aligned workspace of kleos_adapter_products_workspace(rows, r) bytes");
    if (!whole(bytes_of(torch_dtype), {dy, x, a, b, dbase, dx}) || !whole(bytes_of(grad_dtype), {da, db}) || !whole(4, {u, offsets, adapter, scale}))
        return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, kNoDevice);
    const cudaStream_t st = stream_of(stream);
    return with_type(call, torch_dtype, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        cudaError_t rc = cudaSuccess;
        if (rows > 0) {
            adapters::Args g{};
            g.in = dy; g.p = b; g.q = a; g.base = dbase; g.out = dx; g.u = da ? static_cast<float*>(workspace) : nullptr; g.offsets = offsets;
            g.adapter = adapter; g.scale = scale; g.ldi = lddy; g.ldb = ldb; g.ldo = lddx; g.rows = rows; g.R = R; g.L = L; g.r = r; g.len = N; g.cols = K;
            rc = adapter_rows<T, true>(g, st);
        }
        adapters::Grads ga{}, gb{};
        ga.offsets = offsets; ga.adapter = adapter; ga.rows = rows; ga.R = R; ga.L = L; ga.r = r; ga.wide_out = grad_dtype == 0;
        gb = ga;
        ga.in = x; ga.c = static_cast<const float*>(workspace); ga.out = da; ga.ldi = ldx; ga.cols = K;
        gb.in = dy; gb.c = u; gb.out = db; gb.db = true; gb.scale = scale; gb.ldi = lddy; gb.cols = N;
        if (rc == cudaSuccess) rc = adapter_grads<T>(ga, gb, st);
        return finish(call, rc);
    });
}

}  // extern "C"
