// C ABI of the operators around the experts: layer norm, the sort of tokens by expert with the rows there and back, and
// the experts' products over the sorted rows, each with its gradients.  No counterpart in the reference, whose layer is
// one fused forward.  None of them needs kleos_initialize, allocates, synchronises or keeps anything between calls.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "expert_f32.cuh"
#include "expert_rows.cuh"
#include "expert_simt.cuh"
#include "expert_split.cuh"
#include "expert_tc.cuh"
#include "layer_norm.cuh"
#include "sort_tokens.cuh"

namespace kleos {
namespace {
using namespace ops;

size_t bytes_of(int torch_dtype) { return torch_dtype == 0 ? 4 : 2; }
bool known_type(int torch_dtype) { return torch_dtype == 0 || torch_dtype == 2 || torch_dtype == 3; }
constexpr int kMostColumns = 1 << 28;
constexpr int kMostRows = 0x7fff0000;  // launches count rows in ints, and round them up to whole blocks
constexpr char kNormSizes[] = "rows must be from 0 to 2^31 - 2^16, H from 1 to 2^28, and no row longer than its stride";
constexpr char kTypes[] = "torch_dtype must be 0 (float), 2 (bf16) or 3 (fp16)";

// Whether every pointer (null ones too) is where an element of so many bytes may be.
bool whole(size_t bytes, std::initializer_list<const void*> ptrs) {
    for (const void* p : ptrs)
        if (!aligned(p, bytes)) return false;
    return true;
}
constexpr char kWhole[] = "a device pointer is no multiple of its element's size";

// Whether all of it can be moved 16 bytes at a time.
bool by(int bytes, size_t elem, std::initializer_list<const void*> ptrs, std::initializer_list<long long> elems) {
    for (const void* p : ptrs)
        if (!aligned(p, bytes)) return false;
    for (const long long n : elems)
        if (n * (long long)elem % bytes) return false;
    return true;
}
bool by_16(size_t elem, std::initializer_list<const void*> ptrs, std::initializer_list<long long> elems) { return by(16, elem, ptrs, elems); }

constexpr long long kWaitCycles = 20000000000LL;  // about ten seconds: nothing but a copy or an MMA is waited for

// ---------------------------------------------------------------- layer norm
// Stages of a ring, `bytes` each, for `most` bytes on their way: one at least.
constexpr int kRingMost = 224 * 1024;
int ring_depth(size_t bytes, int most) { return std::max(1, std::min(norm::kMostDepth, (int)(most / bytes))); }

template <typename T>
cudaError_t norm_forward(norm::Args a, cudaStream_t st) {
    const int sms = sm_count();
    constexpr int W = 16 / sizeof(T);
    cudaError_t rc = cudaSuccess;
    bool done;
    if (by_16(sizeof(T), {a.x, a.y}, {a.ldx, a.ldy, a.H})) {
        done = norm::with_shape<W, false>(a.H, [&](auto g, auto n) {
            constexpr int G = decltype(g)::value, P = norm::kForwardGroups<G>, kThreads = G * P;
            const auto kernel = norm::forward_kernel<T, W, G, decltype(n)::value>;
            const size_t stage = (size_t)P * a.H * sizeof(T);
            static bool allowed[64];
            rc = allow_smem(kernel, allowed, kRingMost);
            a.depth = ring_depth(stage, G > 256 ? 98304 : 49152);
            const int blocks = a.rows <= sms ? a.rows : std::min((a.rows + P - 1) / P, std::max(1, resident_blocks(kernel, kThreads, a.depth * stage)));
            a.depth = std::min(a.depth, (a.rows + blocks * P - 1) / (blocks * P));
            if (rc == cudaSuccess) rc = launch(kernel, dim3(blocks), kThreads, a.depth * stage, 1, st, a);
        });
    } else {
        done = norm::with_odd_shape(a.H, [&](auto g, auto n) {
            constexpr int G = decltype(g)::value, P = norm::kForwardGroups<G>, kThreads = G * P;
            const auto kernel = norm::forward_odd_kernel<T, G, decltype(n)::value>;
            const int blocks = a.rows <= sms ? a.rows : std::min((a.rows + P - 1) / P, std::max(1, resident_blocks(kernel, kThreads, 0)));
            rc = launch(kernel, dim3(blocks), kThreads, 0, 1, st, a);
        });
    }
    if (!done) rc = launch(norm::forward_long_kernel<T>, dim3(std::min(a.rows, sms * 2)), 1024, 0, 1, st, a);
    return rc;
}

template <typename T>
cudaError_t norm_backward(norm::Args a, cudaStream_t st) {
    const int sms = sm_count();
    constexpr int W = 16 / sizeof(T);
    cudaError_t rc = cudaSuccess;
    int partials = 0;
    if (a.rows > 0) {
        bool done;
        if (by_16(sizeof(T), {a.x, a.dy, a.dx}, {a.ldx, a.lddy, a.lddx, a.H})) {
            done = norm::with_shape<W, true>(a.H, [&](auto g, auto n) {
                constexpr int G = decltype(g)::value, N = decltype(n)::value, P = norm::kGroups<G>;
                const auto kernel = norm::backward_kernel<T, W, G, N>;
                const size_t stage = 2 * (size_t)P * a.H * sizeof(T), least = P > 1 && a.partial ? 8 * (size_t)a.H * P : 0;
                partials = std::min(a.rows, std::min(sms, norm::kMaxPartials));
                const size_t weights = (size_t)(a.H * 4 + 127) / 128 * 128;
                a.depth = std::min(ring_depth(stage, kRingMost - (int)weights), (a.rows + partials * P - 1) / (partials * P));
                static bool allowed[64];
                rc = allow_smem(kernel, allowed, kRingMost);
                if (rc == cudaSuccess) rc = launch(kernel, dim3(partials), G * P, weights + std::max(a.depth * stage, least), 1, st, a);
            });
        } else {
            done = norm::with_odd_shape(a.H, [&](auto g, auto n) {
                constexpr int G = decltype(g)::value, P = norm::kGroups<G>, kThreads = G * P;
                const auto kernel = norm::backward_odd_kernel<T, G, decltype(n)::value>;
                const size_t smem = P > 1 && a.partial ? 8 * (size_t)a.H * P : 0;
                partials = a.rows <= sms ? a.rows : std::min({(a.rows + P - 1) / P, norm::kMaxPartials, std::max(1, resident_blocks(kernel, kThreads, smem))});
                rc = launch(kernel, dim3(partials), kThreads, smem, 1, st, a);
            });
        }
        if (!done) {
            rc = launch(norm::backward_long_kernel<T>, dim3(std::min(a.rows, sms * 2)), 1024, 0, 1, st, a);
            partials = std::min(a.rows, norm::kMaxPartials);
            if (rc == cudaSuccess && a.partial)
                rc = launch(norm::column_kernel<T>, dim3((a.H + 255) / 256, partials), 256, 0, 1, st, a);
        }
    }
    if (rc == cudaSuccess && a.partial) rc = launch(norm::finish_kernel<T>, dim3((2 * a.H + 31) / 32), 1024, 0, 1, st, a, partials);
    return rc;
}

// ---------------------------------------------------------------- sort, gather, combine
template <template <typename, int, int> class Kernel>
int move_rows(const char* call, sorting::Move m, int torch_dtype, std::initializer_list<const void*> ptrs, cudaStream_t st) {
    return with_type(call, torch_dtype, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        constexpr int W = 16 / sizeof(T);
        const int V = by_16(sizeof(T), ptrs, {m.ld, m.H}) ? W : by(2 * sizeof(T), sizeof(T), ptrs, {m.ld, m.H}) ? 2 : 1;
        // four vectors a thread, or one where there are few tokens; a token a block, or eight where a warp is enough for one
        const bool many = m.T >= 4 * sm_count();
        const int vectors = (m.H + V - 1) / V, per = many ? 4 : 1;
        m.lanes = std::min(256, std::max(32, (vectors + 32 * per - 1) / (32 * per) * 32));
        const int groups = many && m.lanes == 32 ? 8 : 1;
        auto run = [&](auto v, auto kt) {
            constexpr int kV = decltype(v)::value, KT = decltype(kt)::value, U = Kernel<T, kV, KT>::kAhead;
            const int parts = U == 0 || many ? 1 : std::min(65535, (vectors + m.lanes * U - 1) / (m.lanes * U));
            m.span = parts * m.lanes * U * V;
            return finish(call, launch(Kernel<T, kV, KT>::get(), dim3((m.T + groups - 1) / groups, parts), groups * m.lanes, 0, 1, st, m));
        };
        auto with_k = [&](auto kt) {
            using std::integral_constant;
            return V == W ? run(integral_constant<int, W>(), kt) : V == 2 ? run(integral_constant<int, 2>(), kt) : run(integral_constant<int, 1>(), kt);
        };
        using std::integral_constant;
        if (m.K == 1) return with_k(integral_constant<int, 1>());
        if (m.K == 2) return with_k(integral_constant<int, 2>());
        if (m.K <= 4) return with_k(integral_constant<int, 4>());
        return with_k(integral_constant<int, kMaxTopK>());
    });
}
// kAhead: vectors of a row that a thread takes at a time; 0: a token's sums take all of a row.
template <typename T, int V, int KT>
struct Gather {
    static constexpr int kAhead = sorting::kAhead<V, 1>;
    static auto get() { return sorting::gather_kernel<T, V, KT>; }
};
template <typename T, int V, int KT>
struct Combine {
    static constexpr int kAhead = sorting::kAhead<V, KT>;
    static auto get() { return sorting::combine_kernel<T, V, KT>; }
};
template <typename T, int V, int KT>
struct CombineBack {
    static constexpr int kAhead = 0;
    static auto get() { return sorting::combine_back_kernel<T, V, KT>; }
};

const char* bad_places(int T, int K, int H, long long ld) {
    if (T < 0 || K < 1 || K > kMaxTopK || (long long)T * K > 0x7fffff00LL) return "T must be 0 or more, K from 1 to 8, T * K below 2^31";
    if (H < 1 || H > kMostColumns || ld < H) return "H must be from 1 to 2^28, and no row longer than its stride";
    return nullptr;
}

// ---------------------------------------------------------------- products
template <int kMode>
int products_simt(const char* call, const experts::Args& a, int torch_dtype, cudaStream_t st) {
    return with_type(call, torch_dtype, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        const int tile = experts::kTile, cols = kMode == experts::kForward ? a.N : a.K;
        const dim3 grid = kMode == experts::kDw ? dim3((a.N + tile - 1) / tile, (cols + tile - 1) / tile, a.E)
                                                : dim3(a.rows / tile + a.E + 1, (cols + tile - 1) / tile);
        const bool wide = by_16(sizeof(T), {a.x, a.dy, a.w, a.out}, {a.ldx, a.ldy, a.ldo, a.N, a.K});
        if (wide) return finish(call, launch(experts::product_kernel<T, kMode, 4>, grid, 256, 0, 1, st, a));
        return finish(call, launch(experts::product_kernel<T, kMode, 1>, grid, 256, 0, 1, st, a));
    });
}

// Tensor of up to three dimensions (sizes and strides from the innermost, which is contiguous), copied in boxes of 128
// bytes by `lines` lines, 128-byte swizzle.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
bool encode(CUtensorMap* map, int torch_dtype, const void* base, int dims, const cuuint64_t* sizes, const long long* strides, int lines) {
    static const EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeTiledFn>(f);
    }();
    if (!fn) return false;
    const size_t elem = bytes_of(torch_dtype);
    const CUtensorMapDataType type = torch_dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : torch_dtype == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t pitch[2] = {(cuuint64_t)strides[0] * elem, dims > 2 ? (cuuint64_t)strides[1] * elem : 0};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / elem), (cuuint32_t)lines, 1}, one[3] = {1, 1, 1};
    return fn(map, type, (cuuint32_t)dims, const_cast<void*>(base), sizes, pitch, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode_rows(CUtensorMap* map, int torch_dtype, const void* base, int rows, int cols, long long ld, int lines) {
    const cuuint64_t sizes[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    return encode(map, torch_dtype, base, 2, sizes, &ld, lines);
}
bool encode_weights(CUtensorMap* map, int torch_dtype, const void* base, int E, int N, int K, int lines) {
    const cuuint64_t sizes[3] = {(cuuint64_t)K, (cuuint64_t)N, (cuuint64_t)E};
    const long long strides[2] = {K, (long long)N * K};
    return encode(map, torch_dtype, base, 3, sizes, strides, lines);
}

constexpr int kLeastSteps = 4;  // of 64 elements that a part of a split sum has

// Pairs of blocks for so many tiles at most.
int pair_grid(long long tiles) { return 2 * (int)std::max<long long>(1, std::min<long long>(sm_count() / 2, tiles)); }

// Clusters of a kernel that the device holds at once.
template <typename... P>
int resident_clusters(void (*kernel)(P...), int cluster, int threads, size_t smem) {
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3((unsigned)cluster);
    lc.blockDim = dim3((unsigned)threads);
    lc.dynamicSmemBytes = smem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    lc.attrs = &at;
    lc.numAttrs = 1;
    int n = 0;
    return cudaOccupancyMaxActiveClusters(&n, kernel, &lc) == cudaSuccess ? n : 0;
}

// Whether the call's tiles, `tiles` at most, are so few that a cluster of kParts pairs of blocks can take each and run at once;
// the call is launched then and its result is in *code.
template <typename TE, bool kDx, int kParts>
bool products_split(const char* call, const experts::Args& a, const experts::tcp::TcArgs& g, long long tiles, int torch_dtype, cudaStream_t st, int* code) {
    using namespace experts;
    if ((g.len + tcp::BK - 1) / tcp::BK < kLeastSteps * kParts) return false;
    const auto kernel = tcs::split_tc_kernel<TE, kDx, kParts>;
    static bool done[64];
    static int known[64];
    int dev = -1, most = 0;
    cudaError_t rc = cudaGetDevice(&dev);
    if (rc == cudaSuccess) rc = allow_smem(kernel, done, tcs::SMEM_BYTES);
    if (rc == cudaSuccess && dev < 64) most = known[dev];
    if (rc == cudaSuccess && !most) {
        most = resident_clusters(kernel, 2 * kParts, tcp::kThreads, tcs::SMEM_BYTES);
        if (dev < 64) known[dev] = most;
    }
    if (rc == cudaSuccess && tiles > most) return false;
    tcs::HalfMaps rows;
    CUtensorMap w;
    bool ok = rc == cudaSuccess && encode_weights(&w, torch_dtype, a.w, a.E, a.N, a.K, kDx ? 64 : 128);
    for (int i = 0; i < 2; ++i) ok = ok && encode_rows(&rows.box[i], torch_dtype, kDx ? a.dy : a.x, a.rows, g.len, kDx ? a.ldy : a.ldx, 16 << i);
    if (rc == cudaSuccess && !ok) {
        *code = refuse(call, KLEOS_E_CUDA, "cuTensorMapEncodeTiled failed");
        return true;
    }
    if (rc == cudaSuccess) rc = launch(kernel, dim3(2 * kParts * (int)tiles), tcp::kThreads, tcs::SMEM_BYTES, 2 * kParts, st, rows, w, g);
    *code = finish(call, rc);
    return true;
}

template <typename TE, bool kDx>
int products_tc(const char* call, const experts::Args& a, int torch_dtype, cudaStream_t st) {
    using namespace experts::tcp;
    TcArgs g{};
    g.offsets = a.offsets; g.bias = a.bias; g.out = a.out; g.ldo = a.ldo; g.rows = a.rows; g.E = a.E; g.wait_cycles = kWaitCycles;
    g.M = kDx ? a.K : a.N;
    g.len = kDx ? a.N : a.K;
    const long long pairs = (g.M + 2 * BM - 1) / (2 * BM), at_most = pairs * (a.rows / experts::tcs::kRows + std::min(a.E, a.rows));
    int code;
    if (products_split<TE, kDx, 4>(call, a, g, at_most, torch_dtype, st, &code) || products_split<TE, kDx, 2>(call, a, g, at_most, torch_dtype, st, &code)) return code;
    // tiles of fewer rows where there would be fewer tiles than pairs of blocks (one expert's 1000 rows, N = K = 1024: 12.3 -> 9.4 us)
    g.units = (int)std::min(9LL, std::max(2LL, (pairs * (a.rows / 32 + std::min(a.E, a.rows)) * 2 + sm_count() - 1) / sm_count()));
    RowMaps rows;
    CUtensorMap w;
    bool ok = encode_weights(&w, torch_dtype, a.w, a.E, a.N, a.K, kDx ? 64 : 128);
    for (int i = 0; i < kBoxes; ++i) ok = ok && encode_rows(&rows.box[i], torch_dtype, kDx ? a.dy : a.x, a.rows, g.len, kDx ? a.ldy : a.ldx, box_rows(i));
    if (!ok) return refuse(call, KLEOS_E_CUDA, "cuTensorMapEncodeTiled failed");
    static bool done[64];
    cudaError_t rc = allow_smem(product_tc_kernel<TE, kDx>, done, SMEM_BYTES);
    const long long tiles = pairs * (a.rows / (g.units < 9 ? 32 * g.units : 256) + std::min(a.E, a.rows));  // at most
    if (rc == cudaSuccess) rc = launch(product_tc_kernel<TE, kDx>, dim3(pair_grid(tiles)), kThreads, SMEM_BYTES, 1, st, rows, w, g);
    return finish(call, rc);
}

template <typename TE, bool kWideOut>
int weights_tc(const char* call, const experts::Args& a, int torch_dtype, cudaStream_t st) {
    using namespace experts::tcp;
    TcArgs g{};
    g.offsets = a.offsets; g.out = a.out; g.rows = a.rows; g.E = a.E; g.M = a.N; g.len = a.K; g.wait_cycles = kWaitCycles;
    CUtensorMap dy, x, dw;
    const bool ok = encode_rows(&dy, torch_dtype, a.dy, a.rows, a.N, a.ldy, BK) && encode_rows(&x, torch_dtype, a.x, a.rows, a.K, a.ldx, BK) &&
                    encode_weights(&dw, kWideOut ? 0 : torch_dtype, a.out, a.E, a.N, a.K, 32);
    if (!ok) return refuse(call, KLEOS_E_CUDA, "cuTensorMapEncodeTiled failed");
    static bool done[64];
    cudaError_t rc = allow_smem(weight_tc_kernel<TE, kWideOut>, done, wg::SMEM_BYTES);
    const long long tiles = (long long)a.E * ((a.N + 255) / 256) * ((a.K + 255) / 256);
    if (rc == cudaSuccess) rc = launch(weight_tc_kernel<TE, kWideOut>, dim3(pair_grid(tiles)), kThreads, wg::SMEM_BYTES, 1, st, dy, x, dw, g);
    return finish(call, rc);
}

template <int kMode>
int products_f32(const char* call, const experts::Args& a, cudaStream_t st) {
    using namespace experts;
    tcp::TcArgs g{};
    g.offsets = a.offsets; g.bias = a.bias; g.out = a.out; g.rows = a.rows; g.E = a.E; g.wait_cycles = kWaitCycles;
    g.M = kMode == kForward ? a.N : a.K;
    g.len = kMode == kForward ? a.K : a.N;
    g.ldo = kMode == kDw ? a.K : a.ldo;
    CUtensorMap m, n;
    bool ok;
    long long tiles = (g.M + 2 * tcp::BM - 1) / (2 * tcp::BM);  // at most
    if constexpr (kMode == kDw) {
        ok = encode_rows(&m, 0, a.x, a.rows, a.K, a.ldx, f32::BK) && encode_rows(&n, 0, a.dy, a.rows, a.N, a.ldy, f32::BK);
        tiles *= (long long)a.E * ((a.N + f32::BN - 1) / f32::BN);
    } else {
        ok = encode_weights(&m, 0, a.w, a.E, a.N, a.K, kMode == kForward ? tcp::BM : f32::BK) &&
             encode_rows(&n, 0, kMode == kForward ? a.x : a.dy, a.rows, g.len, kMode == kForward ? a.ldx : a.ldy, f32::kHalf);
        tiles *= a.rows / f32::BN + std::min(a.E, a.rows);
    }
    if (!ok) return refuse(call, KLEOS_E_CUDA, "cuTensorMapEncodeTiled failed");
    static bool done[64];
    cudaError_t rc = allow_smem(f32::product_f32_kernel<kMode>, done, f32::SMEM_BYTES);
    if (rc == cudaSuccess) rc = launch(f32::product_f32_kernel<kMode>, dim3(pair_grid(tiles)), f32::kThreads, f32::SMEM_BYTES, 1, st, m, n, g);
    return finish(call, rc);
}

// A few rows: the weights are streamed from all multiprocessors.
template <int kMode>
int products_few(const char* call, const experts::Args& a, int torch_dtype, cudaStream_t st) {
    using namespace experts::few;
    return with_type(call, torch_dtype, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        if constexpr (kMode == experts::kForward) {
            constexpr int W = 16 / sizeof(T);
            const bool wide = by_16(sizeof(T), {a.x, a.w}, {a.ldx, a.K});
            // one or two rows: twice the blocks, for which two columns a warp are enough
            const int columns = a.rows <= 2 ? 16 : 32;
            auto of = [&](auto v) {
                constexpr int V = decltype(v)::value;
                return a.rows <= 2 ? forward_rows_kernel<T, V, 2, 2> : a.rows <= 2 * a.E ? forward_rows_kernel<T, V, 2, 4> : forward_rows_kernel<T, V, 4, 4>;
            };
            const auto kernel = wide ? of(std::integral_constant<int, W>()) : of(std::integral_constant<int, 1>());
            return finish(call, launch(kernel, dim3((a.N + columns - 1) / columns, a.rows), 256, 0, 1, st, a));
        } else {
            const int V = by_16(sizeof(T), {a.w}, {a.K}) ? 4 : 1, tiles = (a.K + 32 * V - 1) / (32 * V);
            // a cluster shares the weights' rows, 512 a block in turn, where the blocks would leave multiprocessors idle
            const int parts = std::max(1, std::min({8, (a.N + 32 * kDxWarps - 1) / (32 * kDxWarps), (int)(sm_count() / ((long long)tiles * std::max(std::min(a.rows, a.E), a.rows / 4)))}));
            const auto kernel = V == 4 ? dx_rows_kernel<T, 4> : dx_rows_kernel<T, 1>;
            return finish(call, launch(kernel, dim3(tiles * parts, a.rows), 32 * kDxWarps, kDxWarps * (32 * V + 1) * sizeof(float), parts, st, a));
        }
    });
}

// The tensor cores' kernels load by TMA, whose rows begin and end on 16-byte boundaries; everything else goes to the FP32
// pipes: up to so many rows with the weights streamed, more in tiles.
constexpr int kFewRows = 32;

// Whether float products are sooner done by streaming the weights once for every four rows, at 6.2 TB/s (c chunks of rows, every
// second expert's last one shorter), than by tiles of 128 rows, a microsecond for every 64 of the sums in as many rounds as
// there are tiles for a pair of blocks.  33 and 64 rows, N = K = 2048, forward: one expert 24 and 42 us (tiles 37 and 37), 16 experts
// 55 and 76 (67 and 68); 64 experts, N = K = 1024 24 and 36 (40 and 56); one expert, N = 512, K = 8192 32 and 34 (123 and 124), its
// dx 43 and 80 (16 and 16).
bool few_floats(const experts::Args& a, int M, int len) {
    if (a.rows > 256) return false;
    const double c = a.rows / 4.0 + std::min(a.rows, a.E) / 2.0, pairs = std::max(1, sm_count() / 2);
    const double tiles = (double)((M + 255) / 256) * (a.rows / 128 + std::min(a.rows, a.E));
    return 4 + c * a.N * a.K * 4 / 6.2e6 < 7 + std::ceil(tiles / pairs) * len / 64.0;
}

template <int kMode>
int products(const char* call, const experts::Args& a, int torch_dtype, cudaStream_t st) {
    const bool tensor = a.rows > 0 && by_16(bytes_of(torch_dtype), {a.x, a.dy, a.w, a.out}, {a.ldx, a.ldy, a.ldo, a.N, a.K});
    if constexpr (kMode != experts::kDw) {
        const bool forward = kMode == experts::kForward;
        if (!tensor ? a.rows <= kFewRows : torch_dtype == 0 && few_floats(a, forward ? a.N : a.K, forward ? a.K : a.N))
            return products_few<kMode>(call, a, torch_dtype, st);
        // (64 experts, N = K = 2048, a row: 5.6 us and 8.9 on the tensor cores; 2 rows of 8 experts, N = K = 4096: 23.9 and 16.5;
        // 1 row, N = 256, K = 8192: 13.8 and 11.7)
        if (kMode == experts::kForward && a.rows <= 2 && a.K <= 4096 && (long long)((a.N + 255) / 256) * a.rows * a.K <= 65536)
            return products_few<kMode>(call, a, torch_dtype, st);
    }
    if (!tensor) return products_simt<kMode>(call, a, torch_dtype, st);
    // Weight gradients of few rows an expert are little but stores, and a tile of floats on the tensor cores has a long way
    // through its roles (128 experts, N = 4424, K = 384: 1 row 199 us on the FP32 pipes and 646, 32 355 and 648, 48 482 and 648;
    // the host knows the average only: 4096 rows on four of the 128 experts 371).
    if (kMode == experts::kDw && torch_dtype == 0 && a.rows <= 48LL * a.E) return products_simt<kMode>(call, a, torch_dtype, st);
    if (torch_dtype == 0) return products_f32<kMode>(call, a, st);
    if constexpr (kMode != experts::kDw) {
        return torch_dtype == 2 ? products_tc<__nv_bfloat16, kMode == experts::kDx>(call, a, torch_dtype, st)
                                : products_tc<__half, kMode == experts::kDx>(call, a, torch_dtype, st);
    } else if (a.wide_out) {
        return torch_dtype == 2 ? weights_tc<__nv_bfloat16, true>(call, a, torch_dtype, st) : weights_tc<__half, true>(call, a, torch_dtype, st);
    } else {
        return torch_dtype == 2 ? weights_tc<__nv_bfloat16, false>(call, a, torch_dtype, st) : weights_tc<__half, false>(call, a, torch_dtype, st);
    }
}

const char* bad_products(int rows, int E, int N, int K, long long ld_n, long long ld_k) {
    if (rows < 0 || rows > kMostRows || E < 1 || E > kMaxExperts) return "rows must be from 0 to 2^31 - 2^16, E from 1 to 1024";
    if (N < 1 || K < 1 || N > 1 << 22 || K > 1 << 22) return "N and K must be from 1 to 2^22";
    // tiles are counted in ints: of rows by columns, and of the weights
    const long long n = (N + 127) / 128, k = (K + 127) / 128;
    if ((rows / 32 + (long long)E + 1) * std::max(n, k) > 0x7fffffff || E * n * k > 0x7fffffff) return "too many experts, rows and columns at once";
    if (ld_n < N || ld_k < K) return "no row may be longer than its stride";
    return nullptr;
}

}  // namespace
}  // namespace kleos

using namespace kleos;

extern "C" {

long long kleos_layer_norm_workspace(int H) { return H < 1 || H > kMostColumns ? KLEOS_E_ARG : (long long)norm::kMaxPartials * 2 * H * (long long)sizeof(float); }

int kleos_layer_norm(const void* x, long long ldx, const void* weight, const void* bias, int rows, int H, float eps,
                     int torch_dtype, int param_dtype, void* y, long long ldy, float* mean, float* rstd, void* stream) {
    const char* call = "kleos_layer_norm";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (param_dtype != 0 && param_dtype != torch_dtype) return refuse(call, KLEOS_E_UNSUPPORTED, "param_dtype must be 0 (float) or the element type");
    if (rows < 0 || rows > kMostRows || H < 1 || H > kMostColumns || ldx < H || ldy < H) return refuse(call, KLEOS_E_ARG, kNormSizes);
    if (!(eps >= 0.f)) return refuse(call, KLEOS_E_ARG, "eps must not be negative");
    if (rows == 0) return KLEOS_OK;
    if (!x || !y) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {x, y}) || !whole(bytes_of(param_dtype), {weight, bias}) || !whole(4, {mean, rstd})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    norm::Args a{};
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    a.ldx = ldx; a.ldy = ldy; a.rows = rows; a.H = H; a.wide = param_dtype == 0; a.eps = eps; a.wait_cycles = kWaitCycles;
    a.param_vec = whole(16, {weight, bias});
    return with_type(call, torch_dtype, [&](auto* null) { return finish(call, norm_forward<std::remove_pointer_t<decltype(null)>>(a, stream_of(stream))); });
}

int kleos_layer_norm_backward(const void* dy, long long lddy, const void* x, long long ldx, const void* weight, const float* mean,
                              const float* rstd, int rows, int H, int torch_dtype, int param_dtype, void* dx, long long lddx,
                              void* dweight, void* dbias, void* workspace, long long workspace_bytes, void* stream) {
    const char* call = "kleos_layer_norm_backward";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (param_dtype != 0 && param_dtype != torch_dtype) return refuse(call, KLEOS_E_UNSUPPORTED, "param_dtype must be 0 (float) or the element type");
    if (rows < 0 || rows > kMostRows || H < 1 || H > kMostColumns || ldx < H || lddy < H || lddx < H) return refuse(call, KLEOS_E_ARG, kNormSizes);
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return refuse(call, KLEOS_E_ARG, "null device pointer");
    const bool sums = dweight || dbias;
    if (sums && (!workspace || !aligned(workspace, 16) || workspace_bytes < kleos_layer_norm_workspace(H)))
        return refuse(call, KLEOS_E_ARG, "dweight and dbias need a 16-byte aligned workspace of kleos_layer_norm_workspace(H) bytes");
    if (!whole(bytes_of(torch_dtype), {dy, x, dx}) || !whole(bytes_of(param_dtype), {weight, dweight, dbias}) || !whole(4, {mean, rstd})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    norm::Args a{};
    a.x = x; a.dy = dy; a.weight = weight; a.dx = dx; a.dweight = dweight; a.dbias = dbias;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    a.ldx = ldx; a.lddy = lddy; a.lddx = lddx; a.rows = rows; a.H = H; a.wide = param_dtype == 0; a.wait_cycles = kWaitCycles;
    a.param_vec = whole(16, {weight});
    return with_type(call, torch_dtype, [&](auto* null) { return finish(call, norm_backward<std::remove_pointer_t<decltype(null)>>(a, stream_of(stream))); });
}

int kleos_sort_tokens(const int32_t* topk, int T, int K, int E, int32_t* offsets, int32_t* row_of, int32_t* source, void* stream) {
    const char* call = "kleos_sort_tokens";
    if (const char* bad = bad_places(T, K, 1, 1)) return refuse(call, KLEOS_E_ARG, bad);
    if (E < 1 || E > kMaxExperts) return refuse(call, KLEOS_E_ARG, "E must be from 1 to 1024");
    if (!offsets || (T > 0 && (!topk || !row_of))) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(4, {topk, offsets, row_of, source})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    // one block up to 4096 places, where meeting the others costs more than they take off it
    const int cluster = (long long)T * K <= 4096 ? 1 : sorting::kCluster;
    const bool kept = (long long)T * K <= 32LL * sorting::kKeep * sorting::kWarps * cluster;
    const bool wide = E > 255;  // the number of bits that an id, E among them, takes: 8, or 11
    const auto kernel = wide ? kept ? sorting::sort_kernel<true, 11> : sorting::sort_kernel<false, 11>
                             : kept ? sorting::sort_kernel<true, 8> : sorting::sort_kernel<false, 8>;
    const size_t smem = sizeof(int) * sorting::kWarps * E;
    static bool allowed[4][64];
    cudaError_t rc = allow_smem(kernel, allowed[2 * wide + kept], (int)sizeof(int) * sorting::kWarps * kMaxExperts);
    if (rc == cudaSuccess) rc = launch(kernel, dim3(cluster), sorting::kThreads, smem, cluster, stream_of(stream), topk, T * K, E, offsets, row_of, source);
    return finish(call, rc);
}

int kleos_gather_tokens(const void* x, long long ldx, const int32_t* row_of, const int32_t* offsets, int T, int K, int E, int H,
                        int torch_dtype, void* rows, void* stream) {
    const char* call = "kleos_gather_tokens";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (const char* bad = bad_places(T, K, H, ldx)) return refuse(call, KLEOS_E_ARG, bad);
    if (E < 1 || E > kMaxExperts) return refuse(call, KLEOS_E_ARG, "E must be from 1 to 1024");
    if (T == 0) return KLEOS_OK;
    if (!x || !row_of || !offsets || !rows) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {x, rows}) || !whole(4, {row_of, offsets})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    sorting::Move m{};
    m.from = x; m.to = rows; m.row_of = row_of; m.offsets = offsets; m.ld = ldx; m.T = T; m.K = K; m.E = E; m.H = H; m.n = T * K;
    return move_rows<Gather>(call, m, torch_dtype, {x, rows}, stream_of(stream));
}

int kleos_combine_tokens(const void* rows, const int32_t* row_of, const float* weights, int T, int K, int H, int torch_dtype,
                         void* out, long long ldo, void* stream) {
    const char* call = "kleos_combine_tokens";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (const char* bad = bad_places(T, K, H, ldo)) return refuse(call, KLEOS_E_ARG, bad);
    if (T == 0) return KLEOS_OK;
    if (!rows || !row_of || !out) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {rows, out}) || !whole(4, {row_of, weights})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    sorting::Move m{};
    m.from = rows; m.to = out; m.row_of = row_of; m.weights = weights; m.ld = ldo; m.T = T; m.K = K; m.H = H; m.n = T * K;
    return move_rows<Combine>(call, m, torch_dtype, {rows, out}, stream_of(stream));
}

int kleos_combine_tokens_backward(const void* dout, long long ldd, const void* rows, const int32_t* row_of, const float* weights,
                                  const int32_t* offsets, int T, int K, int E, int H, int torch_dtype, void* drows,
                                  float* dweights, void* stream) {
    const char* call = "kleos_combine_tokens_backward";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (const char* bad = bad_places(T, K, H, ldd)) return refuse(call, KLEOS_E_ARG, bad);
    if (E < 1 || E > kMaxExperts) return refuse(call, KLEOS_E_ARG, "E must be from 1 to 1024");
    if (T == 0) return KLEOS_OK;
    if (!dout || !rows || !row_of || !offsets || !drows) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {dout, rows, drows}) || !whole(4, {row_of, weights, offsets, dweights})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    sorting::Move m{};
    m.from = dout; m.other = rows; m.to = drows; m.row_of = row_of; m.offsets = offsets; m.weights = weights; m.dweights = dweights;
    m.ld = ldd; m.T = T; m.K = K; m.E = E; m.H = H; m.n = T * K;
    return move_rows<CombineBack>(call, m, torch_dtype, {dout, rows, drows}, stream_of(stream));
}

int kleos_expert_products(const void* x, long long ldx, const int32_t* offsets, const void* w, const void* bias, int rows, int E,
                          int N, int K, int torch_dtype, void* y, long long ldy, void* stream) {
    const char* call = "kleos_expert_products";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (const char* bad = bad_products(rows, E, N, K, ldy, ldx)) return refuse(call, KLEOS_E_ARG, bad);
    if (rows == 0) return KLEOS_OK;
    if (!x || !offsets || !w || !y) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {x, w, bias, y}) || !whole(4, {offsets})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    experts::Args a{};
    a.x = x; a.w = w; a.bias = bias; a.out = y; a.offsets = offsets; a.ldx = ldx; a.ldo = ldy; a.rows = rows; a.E = E; a.N = N; a.K = K;
    return products<experts::kForward>(call, a, torch_dtype, stream_of(stream));
}

int kleos_expert_products_dx(const void* dy, long long lddy, const int32_t* offsets, const void* w, int rows, int E, int N, int K,
                             int torch_dtype, void* dx, long long lddx, void* stream) {
    const char* call = "kleos_expert_products_dx";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (const char* bad = bad_products(rows, E, N, K, lddy, lddx)) return refuse(call, KLEOS_E_ARG, bad);
    if (rows == 0) return KLEOS_OK;
    if (!dy || !offsets || !w || !dx) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {dy, w, dx}) || !whole(4, {offsets})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    experts::Args a{};
    a.dy = dy; a.w = w; a.out = dx; a.offsets = offsets; a.ldy = lddy; a.ldo = lddx; a.rows = rows; a.E = E; a.N = N; a.K = K;
    return products<experts::kDx>(call, a, torch_dtype, stream_of(stream));
}

int kleos_expert_products_dw(const void* dy, long long lddy, const void* x, long long ldx, const int32_t* offsets, int rows, int E,
                             int N, int K, int torch_dtype, int grad_dtype, void* dw, void* dbias, void* stream) {
    const char* call = "kleos_expert_products_dw";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (grad_dtype != 0 && grad_dtype != torch_dtype) return refuse(call, KLEOS_E_UNSUPPORTED, "grad_dtype must be 0 (float) or the element type");
    if (const char* bad = bad_products(rows, E, N, K, lddy, ldx)) return refuse(call, KLEOS_E_ARG, bad);
    if (!offsets || !dw || (rows > 0 && (!x || !dy))) return refuse(call, KLEOS_E_ARG, "null device pointer");
    if (!whole(bytes_of(torch_dtype), {dy, x}) || !whole(bytes_of(grad_dtype), {dw, dbias}) || !whole(4, {offsets})) return refuse(call, KLEOS_E_ARG, kWhole);
    if (!sm_count()) return refuse(call, KLEOS_E_CUDA, "no current CUDA device");
    experts::Args a{};
    a.dy = dy; a.x = x; a.out = dw; a.offsets = offsets; a.ldy = lddy; a.ldx = ldx; a.rows = rows; a.E = E; a.N = N; a.K = K;
    a.wide_out = grad_dtype == 0;
    const cudaStream_t st = stream_of(stream);
    if (const int rc = products<experts::kDw>(call, a, torch_dtype, st)) return rc;
    if (!dbias) return KLEOS_OK;
    a.out = dbias;
    return with_type(call, torch_dtype, [&](auto* null) {
        using T = std::remove_pointer_t<decltype(null)>;
        constexpr int W = 16 / sizeof(T);
        const bool wide = by_16(sizeof(T), {dy}, {lddy, N});
        const int columns = experts::kBiasLanes * (wide ? W : 1), tiles = (N + columns - 1) / columns;
        // two blocks a multiprocessor; blocks that share an expert's rows have 128 of them each (on average, which is what the host
        // knows: N = 2048, bf16, 16384 rows of 64 experts 24 us, by Zipf 56, all of one expert 170)
        const int parts = (int)std::max(1LL, std::min({8LL, 2LL * sm_count() / ((long long)tiles * E), (long long)rows / E / 128}));
        const auto kernel = wide ? experts::bias_kernel<T, W> : experts::bias_kernel<T, 1>;
        return finish(call, launch(kernel, dim3(tiles * parts, E), 1024, 0, parts, st, a));
    });
}

}  // extern "C"
