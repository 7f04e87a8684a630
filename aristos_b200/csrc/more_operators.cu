// C ABI of further operators around the experts: the activation between an expert's two products with its gradient, a whole
// layer for the few tokens of a decode step, and low-rank adapters of many requests with their gradients.  No counterpart in the
// reference.  None of them needs kleos_initialize, allocates, synchronises or keeps anything between calls.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "activation.cuh"
#include "adapters.cuh"
#include "adapters_mma.cuh"
#include "moe_stream.cuh"
#include "moe_tokens.cuh"

namespace kleos {
namespace {
using namespace ops;

constexpr int kMostColumns = 1 << 22;
constexpr char kNull[] = "null device pointer";
constexpr char kNoDevice[] = "no current CUDA device";
constexpr char kAct[] = "hidden_act must be 0 (ReLU), 1 (GELU) or 2 (SiLU)";

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

// ---------------------------------------------------------------- layer for a few tokens
long long moe_workspace(int T, int I, int K) { return (long long)T * K * 4 * ((I + 7) / 8 * 8); }

// Shared memory of a launch that takes `rows` of an expert at a time, and where what is in it lies.
template <typename T, int kMode, int kLines, int kSets, int kDepth>
int moe_smem(const tokens::Args& a, tokens::Cut& c, int rows) {
    using namespace tokens;
    c.rows = rows;
    c.slot = (kSets * kTileColumns + rows) * kLines * kLine;
    c.past = (padded_rows(rows) - rows) * kLines * kLine;
    const int teams = kStreamWarps / team_size(std::min(a.E, a.T * a.K));  // at most
    return groups_bytes(a.T * a.K, a.E) + kStreamWarps * kDepth * c.slot + c.past + 4 * (2 * meet_floats(kSets, rows) + (kMode == kDown ? teams * a.T * c.tile : 0));
}

// False where not even `least` rows of an expert fit at a time.
template <typename T, int kMode, int kLines, int kSets, int kUnit, int kDepth>
bool moe_stream_of(const tokens::Args& a, tokens::Cut c, int least, cudaStream_t st, cudaError_t* rc) {
    using namespace tokens;
    int rows = c.rows, smem;
    least = std::min(least, rows);
    while ((smem = moe_smem<T, kMode, kLines, kSets, kDepth>(a, c, rows)) > kMostSmem) {
        if (rows <= least) return false;
        rows = std::max(least, (rows - 1) / 8 * 8);
    }
    const int cols = kMode == kDown ? a.H : a.I;
    const auto kernel = stream_kernel<T, kMode, kLines, kSets, kUnit, kDepth>;
    static bool allowed[64];
    *rc = allow_smem(kernel, allowed, kMostSmem);
    if (*rc == cudaSuccess) *rc = launch(kernel, dim3((cols + c.share - 1) / c.share * c.spread), kStreamThreads, smem, kMode == kDown ? c.spread : 1, st, a, c);
    return true;
}

template <typename T, int kMode, int kUnit>
cudaError_t moe_stream(const tokens::Args& a, cudaStream_t st) {
    using namespace tokens;
    const int sms = sm_count(), cols = kMode == kDown ? a.H : a.I;
    cudaError_t rc = cudaErrorInvalidConfiguration;
    Cut c{};
    // Blocks that share columns: a step costs as much as some six rows of weights, and experts are dealt unevenly by about half a one.
    // (Clusters of four and more leave some multiprocessors of a group out.)
    const double used = a.E * (1 - std::pow(1 - std::min(1.0, (double)a.K / a.E), a.T));
    double best = 0;
    for (int spread = 1; spread <= 8 && spread <= std::min(a.E, a.T * a.K); spread *= 2) {
        const int over = (kMode == kDown && spread > 2 ? sms * 7 / 8 : sms) / spread;
        if (over < 1) break;
        const int share = (cols + over - 1) / over, most = kMode == kUpGated || (sizeof(T) == 4 && a.T > 8) ? kTileColumns : 2 * kTileColumns;
        const int tiles = (share + most - 1) / most, tile = (share + tiles - 1) / tiles, halves = kMode == kUpGated ? 2 : 1;
        const double even = a.T == 1 ? used / (spread * std::ceil(used / spread)) : used / (used + 0.5 * (spread - 1)), filled = (double)cols / ((cols + share - 1) / share) / share;
        const double good = even * filled * over * spread / sms * (halves * tile) / (halves * tile + 6.0);
        if (good > best * 1.02) best = good, c.spread = spread, c.share = share;
    }
    // rows of an expert at a time: as many as it has on average and some
    c.rows = std::min(a.T, a.T * a.K > 12 * a.E ? kMostRowsAtOnce : kMostRowsAtOnce / 2);
    if (sizeof(T) == 4) c.rows = std::min(c.rows, kMode == kUpGated ? 8 : 16);  // (registers)
    // two sets of 16 columns where that takes fewer tiles (a gated expert's are its halves)
    const bool two = kMode != kUpGated && (sizeof(T) == 2 || c.rows <= 8) && (c.share + 31) / 32 < (c.share + 15) / 16;
    auto cut = [&](int most) {
        const int tiles = (c.share + most - 1) / most;
        c.tile = (c.share + tiles - 1) / tiles;
    };
    cut(two ? 2 * kTileColumns : kTileColumns);
    // Three steps ahead where that leaves room for all but the fullest experts' rows (16 tokens of eight experts, four each on average: 453 us with
    // two steps, 427 with three).
    const int enough = std::min(c.rows, a.T * a.K <= 4 * a.E ? 8 : 16);
    if constexpr (kMode == kUpGated) {
        if constexpr (kUnit == 16)
            if (moe_stream_of<T, kMode, 1, 2, kUnit, 4>(a, c, enough, st, &rc)) return rc;
        if (moe_stream_of<T, kMode, 1, 2, kUnit, 3>(a, c, 8, st, &rc)) return rc;
    } else {
        if constexpr (kUnit == 16)
            if (two && moe_stream_of<T, kMode, 1, 2, kUnit, 4>(a, c, enough, st, &rc)) return rc;
        if (two && moe_stream_of<T, kMode, 1, 2, kUnit, 3>(a, c, 8, st, &rc)) return rc;
        cut(kTileColumns);
        if (moe_stream_of<T, kMode, 2, 1, kUnit, 3>(a, c, 8, st, &rc) || moe_stream_of<T, kMode, 1, 1, kUnit, 3>(a, c, 8, st, &rc)) return rc;
    }
    return rc;
}

template <typename T>
cudaError_t moe_layer(tokens::Args a, bool gated, bool route, cudaStream_t st) {
    using namespace tokens;
    constexpr int W = 16 / sizeof(T);
    const int sms = sm_count();
    cudaError_t rc = cudaSuccess;
    if (route) {
        a.group = std::min(kGateTokens, (a.T * kGateBlocks + 2 * sms - 1) / (2 * sms));  // clusters that run at once: two blocks a multiprocessor
        const bool wide = by_16(sizeof(T), {a.x, a.gate}, {a.ldx, a.H});
        const auto kernel = wide ? gate_kernel<T, W> : gate_kernel<T, 1>;
        static bool allowed[64];
        if (wide) rc = allow_smem(gate_kernel<T, W>, allowed, kGateSmem);
        if (rc == cudaSuccess) rc = launch(kernel, dim3((a.T + a.group - 1) / a.group * kGateBlocks), 32 * kGateWarps, wide ? kGateSmem : 0, kGateBlocks, st, a);
    }
    if (rc != cudaSuccess) return rc;
    auto with_unit = [&](int bytes, auto f) {
        using std::integral_constant;
        if constexpr (sizeof(T) == 2)
            if (bytes < 4) return f(integral_constant<int, 2>());
        return bytes < 16 ? f(integral_constant<int, 4>()) : f(integral_constant<int, 16>());
    };
    auto unit_of = [](const void* x, const void* w, std::initializer_list<long long> elems) {
        return by(16, sizeof(T), {x, w}, elems) ? 16 : by(4, sizeof(T), {x, w}, elems) ? 4 : 2;
    };
    rc = with_unit(unit_of(a.x, a.w1, {a.ldx, a.H}), [&](auto u) {
        constexpr int kUnit = decltype(u)::value;
        return gated ? moe_stream<T, kUpGated, kUnit>(a, st) : moe_stream<T, kUp, kUnit>(a, st);
    });
    if (rc != cudaSuccess) return rc;
    return with_unit(unit_of(a.h, a.w2, {a.ldh, a.I}), [&](auto u) { return moe_stream<T, kDown, decltype(u)::value>(a, st); });
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
    return launch(kernel, dim3((unsigned)(tiles * cluster)), 256, 0, cluster, st, a);
}

template <typename T, bool kDb>
cudaError_t adapter_grads(const adapters::Grads& a, cudaStream_t st) {
    using namespace adapters;
    if constexpr (sizeof(T) == 2) {
        if (a.r % 2 == 0 && by_16(2, {a.in}, {a.ldi, a.cols}) && aligned(a.c, 8))
            return with_rank(std::min(a.r, 64), [&](auto rt) {
                constexpr int RT = decltype(rt)::value, kBytes = GradShape<T, RT>::kBytes;
                const auto kernel = grads_mma_kernel<T, kDb, RT>;
                const long long strips = (a.cols + kGradColumns - 1) / kGradColumns, groups = strips * a.L * ((a.r + RT - 1) / RT);
                int cluster = 1;
                while (cluster < 8 && 2 * groups * cluster <= 2LL * sm_count() && a.rows > cluster * kGradRows * 4LL) cluster *= 2;
                static bool allowed[64];
                cudaError_t rc = allow_smem(kernel, allowed, kBytes);
                if (rc == cudaSuccess) rc = launch(kernel, dim3((unsigned)(strips * cluster), a.L, (a.r + RT - 1) / RT), 256, kBytes, cluster, st, a);
                return rc;
            });
    }
    const long long strips = (a.cols + 31) / 32, groups = strips * a.L * ((a.r + 15) / 16);
    int cluster = 1;
    while (cluster < 8 && 2 * groups * cluster <= 6LL * sm_count() && a.rows > cluster * 256) cluster *= 2;
    return launch(grads_kernel<T, kDb>, dim3((unsigned)(strips * cluster), a.L, (a.r + 15) / 16), 256, 0, cluster, st, a);
}

}  // namespace
}  // namespace kleos

using namespace kleos;

extern "C" {

int kleos_activation(const void* z, long long ldz, long long rows, int I, int hidden_act, int gated, int torch_dtype, void* h, long long ldh,
                     void* stream) {
    const char* call = "kleos_activation";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (hidden_act < 0 || hidden_act >= act::kKinds) return refuse(call, KLEOS_E_ARG, kAct);
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
    if (hidden_act < 0 || hidden_act >= act::kKinds) return refuse(call, KLEOS_E_ARG, kAct);
    if (const char* bad = bad_activation(rows, I, gated, std::min(ldz, lddz), lddh)) return refuse(call, KLEOS_E_ARG, bad);
    if (rows == 0) return KLEOS_OK;
    if (!dh || !z || !dz) return refuse(call, KLEOS_E_ARG, kNull);
    if (!whole(bytes_of(torch_dtype), {dh, z, dz})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, kNoDevice);
    act::Args a{};
    a.z = z; a.dh = dh; a.out = dz; a.ldz = ldz; a.ldh = lddh; a.ldo = lddz; a.rows = rows; a.I = I;
    return activation<true>(call, a, hidden_act, gated != 0, torch_dtype, stream_of(stream));
}

long long kleos_moe_tokens_workspace(int T, int I, int K) {
    return T < 0 || T > tokens::kMostTokens || I < 1 || I > kMostColumns || K < 1 || K > kMaxTopK ? KLEOS_E_ARG : moe_workspace(T, I, K);
}

int kleos_moe_tokens(const void* x, long long ldx, const void* gate, const float* gate_bias, const void* w1, const void* b1, const void* w2,
                     const void* b2, int T, int H, int I, int E, int K, int hidden_act, int gated, int torch_dtype, void* out,
                     long long ldo, int32_t* topk, float* weights, void* workspace, long long workspace_bytes, void* stream) {
    const char* call = "kleos_moe_tokens";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (hidden_act < 0 || hidden_act >= act::kKinds) return refuse(call, KLEOS_E_ARG, kAct);
    if (T < 0 || T > tokens::kMostTokens || K < 1 || K > kMaxTopK || E < 1 || E > kMaxExperts || (gate && K > E))
        return refuse(call, KLEOS_E_ARG, "T must be from 0 to 128, K from 1 to 8, E from 1 (with a gate K) to 1024");
    if (H < 1 || I < 1 || H > kMostColumns || I > kMostColumns || ldx < H || ldo < H)
        return refuse(call, KLEOS_E_ARG, "H and I must be from 1 to 2^22, and no row longer than its stride");
    if (T == 0) return KLEOS_OK;
    if (!x || !w1 || !w2 || !out || !topk || !weights || (gate_bias && !gate)) return refuse(call, KLEOS_E_ARG, kNull);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < moe_workspace(T, I, K))
        return refuse(call, KLEOS_E_ARG, "a 16-byte aligned workspace of kleos_moe_tokens_workspace(T, I, K) bytes is needed");
    if (!whole(bytes_of(torch_dtype), {x, gate, w1, b1, w2, b2, out}) || !whole(4, {gate_bias, topk, weights})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, kNoDevice);
    tokens::Args a{};
    a.x = x; a.gate = gate; a.w1 = w1; a.w2 = w2; a.b1 = b1; a.b2 = b2; a.gate_bias = gate_bias; a.out = out; a.topk = topk;
    a.weights = weights; a.h = workspace; a.ldx = ldx; a.ldo = ldo; a.ldh = (I + 7) / 8 * 8;
    a.T = T; a.H = H; a.I = I; a.E = E; a.K = K; a.act = hidden_act;
    return with_type(call, torch_dtype, [&](auto* null) {
        return finish(call, moe_layer<std::remove_pointer_t<decltype(null)>>(a, gated != 0, gate != nullptr, stream_of(stream)));
    });
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
        adapters::Grads g{};
        g.offsets = offsets; g.adapter = adapter; g.rows = rows; g.R = R; g.L = L; g.r = r; g.wide_out = grad_dtype == 0;
        if (rc == cudaSuccess && da) {
            g.in = x; g.c = static_cast<const float*>(workspace); g.out = da; g.ldi = ldx; g.cols = K;
            rc = adapter_grads<T, false>(g, st);
        }
        if (rc == cudaSuccess && db) {
            g.in = dy; g.c = u; g.out = db; g.scale = scale; g.ldi = lddy; g.cols = N;
            rc = adapter_grads<T, true>(g, st);
        }
        return finish(call, rc);
    });
}

}  // extern "C"
