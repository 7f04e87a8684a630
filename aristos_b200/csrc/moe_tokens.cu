// C ABI of a whole MoE layer for the few tokens of a decode step.  No counterpart in the reference.  It needs no kleos_initialize, allocates
// nothing, does not synchronise and keeps nothing between calls.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "moe_stream.cuh"

namespace kleos {
namespace {
using namespace ops;

constexpr int kMostSize = 1 << 22;  // H and I

// h: floats, or 16-bit values and (fp16) as many second parts (PastRange).  One size for all types.
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
template <typename T, int kMode, int kLines, int kSets, int kUnit, int kDepth, bool kLong = false>
bool moe_stream_of(const tokens::Args& a, tokens::Cut c, int least, cudaStream_t st, cudaError_t* rc) {
    using namespace tokens;
    int rows = c.rows, smem;
    least = std::min(least, rows);
    while ((smem = moe_smem<T, kMode, kLines, kSets, kDepth>(a, c, rows)) > kMostSmem) {
        if (rows <= least) return false;
        rows = std::max(least, (rows - 1) / 8 * 8);
    }
    const int cols = kMode == kDown ? a.H : a.I;
    const auto kernel = stream_kernel<T, kMode, kLines, kSets, kUnit, kDepth, kLong>;
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
    if (sizeof(T) == 4) c.rows = std::min(c.rows, kMode == kUpGated ? 8 : 16);  // (registers, here and next)
    if (kUnit == 2) c.rows = std::min(c.rows, 16);
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
    if constexpr (sizeof(T) == 2)
        if (longer_sums((kMode == kDown ? a.I : a.H) * (int)sizeof(T), std::min(a.E, a.T * a.K) / c.spread)) {
            if (kMode != kUpGated) cut(kTileColumns);
            moe_stream_of<T, kMode, kMode == kUpGated ? 1 : 2, kMode == kUpGated ? 2 : 1, kUnit, 3, true>(a, c, 8, st, &rc);
            return rc;
        }
    if constexpr (kMode == kUpGated) {
        if constexpr (kUnit == 16)
            if (moe_stream_of<T, kMode, 1, 2, kUnit, 4>(a, c, enough, st, &rc)) return rc;
        moe_stream_of<T, kMode, 1, 2, kUnit, 3>(a, c, 8, st, &rc);
    } else {
        if constexpr (kUnit == 16)
            if (two && moe_stream_of<T, kMode, 1, 2, kUnit, 4>(a, c, enough, st, &rc)) return rc;
        if (two && moe_stream_of<T, kMode, 1, 2, kUnit, 3>(a, c, 8, st, &rc)) return rc;
        cut(kTileColumns);
        moe_stream_of<T, kMode, 2, 1, kUnit, 3>(a, c, 8, st, &rc);  // (eight rows fit with every T, K and E)
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

}  // namespace
}  // namespace kleos

using namespace kleos;

extern "C" {

long long kleos_moe_tokens_workspace(int T, int I, int K) {
    return T < 0 || T > tokens::kMostTokens || I < 1 || I > kMostSize || K < 1 || K > kMaxTopK ? KLEOS_E_ARG : moe_workspace(T, I, K);
}

int kleos_moe_tokens(const void* x, long long ldx, const void* gate, const float* gate_bias, const void* w1, const void* b1, const void* w2,
                     const void* b2, int T, int H, int I, int E, int K, int hidden_act, int gated, int torch_dtype, void* out,
                     long long ldo, int32_t* topk, float* weights, void* workspace, long long workspace_bytes, void* stream) {
    const char* call = "kleos_moe_tokens";
    if (!known_type(torch_dtype)) return refuse(call, KLEOS_E_UNSUPPORTED, kTypes);
    if (hidden_act < 0 || hidden_act >= act::kKinds) return refuse(call, KLEOS_E_ARG, act::kWhich);
    if (T < 0 || T > tokens::kMostTokens || K < 1 || K > kMaxTopK || E < 1 || E > kMaxExperts || (gate && K > E))
        return refuse(call, KLEOS_E_ARG, "T must be from 0 to 128, K from 1 to 8, E from 1 (with a gate K) to 1024");
    if (H < 1 || I < 1 || H > kMostSize || I > kMostSize || ldx < H || ldo < H)
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

}  // extern "C"
