// The experts of a few tokens (moe_tokens.cuh): the chosen experts' weights are streamed once.
//
//   stream_kernel<kUp>    h of every place, the second factor of a gated expert in the same pass
//   stream_kernel<kDown>  out, all experts' shares of a column added up by the block that owns it
//
// One block a multiprocessor owns a share of the columns of EVERY expert, so the work is even however the tokens were sent and each sum is
// finished where it began.  Where that would be too few columns at once, two to eight blocks share columns and deal the experts among them (kDown:
// a cluster, which adds its results up; 23 tokens, 8 of 128 experts, H = 1280, I = 256, floats: 291 -> 139 us).  A block's eight warps are teams
// that take the experts in turn; each warp of a team goes through its own 128 or 256 bytes of the weights' rows, and of the rows they are
// multiplied with, by 16-byte copies to shared memory that are two or three steps ahead, across experts.  A step is multiplied on the tensor cores
// (warp_mma.cuh), weights on the instruction's 16 rows, up to 32 rows of an expert on its columns; floats by 32-bit multiply-adds, which up to 16
// rows an expert are fewer than the splitting that the tensor cores would want.  A team's partial sums meet in shared memory once an
// expert and tile of columns.  (Copies of whole rows by the bulk engine took 90 cycles each of the warp that issued them: 1480 us for 128
// tokens instead of 383 at that stage.)
//
// h goes from one kernel to the other rounded to the element type, as in the library's other layer: a second value for what that leaves would
// halve the rounding error of a result (2-norm 0.0024 to 0.0017, bf16) and read h twice.  A value past fp16's range is kept all the same
// (PastRange): sums that it made no number are added up anew, by a warp each from memory (16 tokens of the large FFN 436 us; with a token that is no
// number 492; with all of h past the range 11 ms).
//
// The second kernel's first weights are on their way before the first kernel has ended: which experts those are was written by the kernel
// before both, and no kernel lets its successor begin before it has waited for its predecessor (common.cuh).
//
// Bound by HBM where rows are long and experts many: alone, kUp of 128 tokens (64 gated experts, H = I = 2048, bf16, 1.07 GB) 167 us = 6.4 TB/s,
// 16 tokens of the large FFN (2.8 GB, both kernels) 427 us = 6.5 TB/s; by issue and latency where a block's share of an expert is small: kDown of
// those 128 tokens (0.54 GB, 28 rows of 4 KB at a time) 105 us, 37 tokens with H = 1088, I = 2880 (135 MB each) 57 and 65.  One token: 23 us for all
// three launches, of which the weights take 8 and an empty layer 12.
#pragma once

#include <cuda.h>

#include "moe_tokens.cuh"
#include "tc_common.cuh"
#include "warp_mma.cuh"

namespace kleos {
namespace tokens {

constexpr int kUp = 0, kUpGated = 1, kDown = 2;
constexpr int kStreamWarps = 8, kStreamThreads = 32 * kStreamWarps;
constexpr int kMostSmem = 226 * 1024;
constexpr int kMostRowsAtOnce = 32, kTileColumns = 16;
constexpr int kTeam2 = 16, kTeam4 = 8;               // experts from which teams are of two warps, of four
constexpr int kLine = 128;                           // bytes of a row that a warp takes at a time

// How a launch cuts the work up; the same for all its blocks.
struct Cut {
    int spread;  // blocks that share the same columns, each with every so-manyth expert (kDown: a cluster, whose results are added up)
    int share;   // columns of a block
    int tile;    // columns of those at a time
    int rows;    // rows of an expert at a time
    int slot;    // bytes of a warp's step
    int past;    // bytes behind the last slot that are read for rows that it does not have, whose products nobody takes
};
// Rows of a slot: 16 of the weights (32 of a gated expert, or of more columns), then those that they are multiplied with.
__host__ __device__ constexpr int padded_rows(int rows) { return (rows + 7) / 8 * 8; }
__host__ __device__ constexpr int even_rows(int rows) { return (rows + 1) / 2 * 2; }
// Floats that the warps need beside their slots: two buffers to meet in, and (kDown) a tile's results by team.
__host__ __device__ constexpr int meet_floats(int sets, int rows) { return kStreamWarps * 16 * sets * even_rows(rows); }

// Places by expert, within an expert in their own order; those without an expert are left out.
struct Groups {
    float* weight;         // of the places in order (kDown)
    short *of, *token;     // the places in order, and whose they are
    short *expert;         // those that have a place, ascending
    short *begin;          // where their places begin
    int n;                 // experts
};
// Shared memory for them, as little as the call needs: where it is little, the down kernel's blocks are there before the up kernel's have ended.
__host__ __device__ __forceinline__ int groups_bytes(int places, int experts) { return (places * 8 + (experts < places ? experts : places) * 4 + 2 + 127) / 128 * 128; }
struct Counts {
    short of[kMaxExperts];
};

// All threads of the block call it; one warp goes through the places, 32 at a time.  `counts` is only used where there are more than 32.
__device__ __forceinline__ Groups group_places(const Args& a, char* memory, Counts& counts) {
    __shared__ int experts;
    const int lane = threadIdx.x & 31, n = a.T * a.K;
    Groups g;
    g.weight = reinterpret_cast<float*>(memory);
    g.of = reinterpret_cast<short*>(g.weight + n);
    g.token = g.of + n;
    g.expert = g.token + n;
    g.begin = g.expert + min(a.E, n);
    if (n > 32) {
        for (int e = threadIdx.x; e < a.E; e += blockDim.x) counts.of[e] = 0;
        __syncthreads();
    }
    auto expert_of = [&](int i) {
        const int e = i < n ? __ldcg(a.topk + i) : -1;
        return e >= 0 && e < a.E ? e : -1;
    };
    auto put = [&](int to, int i) {
        g.of[to] = (short)i;
        g.token[to] = (short)(i / a.K);
    };
    const unsigned below_me = (1u << lane) - 1;
    if (threadIdx.x < 32 && n <= 32) {
        const int e = expert_of(lane);
        const unsigned same = __match_any_sync(0xffffffffu, e), firsts = __ballot_sync(0xffffffffu, e >= 0 && (same & below_me) == 0);
        int rank = __popc(same & below_me), used = 0;
        for (unsigned m = firsts; m; m &= m - 1) {  // experts before this one
            const int from = __ffs(m) - 1, other = __shfl_sync(0xffffffffu, e, from), places = __popc(__shfl_sync(0xffffffffu, same, from));
            if (other < e) rank += places, ++used;
        }
        if (e >= 0) {
            put(rank, lane);
            if ((same & below_me) == 0) g.expert[used] = (short)e, g.begin[used] = (short)rank;
        }
        const int places = __popc(__ballot_sync(0xffffffffu, e >= 0));
        if (lane == 0) experts = __popc(firsts), g.begin[__popc(firsts)] = (short)places;
    } else if (threadIdx.x < 32) {
        constexpr int kSteps = kMostPlaces / 32;
        short at[kSteps], expert[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) expert[s] = s * 32 < n ? (short)expert_of(s * 32 + lane) : (short)-1;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (s * 32 >= n) break;
            const unsigned same = __match_any_sync(0xffffffffu, expert[s]);
            const int below = __popc(same & below_me);
            if (expert[s] >= 0) at[s] = (short)(counts.of[expert[s]] + below);
            __syncwarp();
            if (expert[s] >= 0 && below == 0) counts.of[expert[s]] += (short)__popc(same);
            __syncwarp();
        }
        int begin = 0, used = 0;
        for (int e0 = 0; e0 < a.E; e0 += 32) {
            const int e = e0 + lane, c = e < a.E ? counts.of[e] : 0;
            int up = c;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, up, o);
                if (lane >= o) up += v;
            }
            const unsigned any = __ballot_sync(0xffffffffu, c > 0);
            if (e < a.E) counts.of[e] = (short)(begin + up - c);
            if (c > 0) {
                const int u = used + __popc(any & below_me);
                g.expert[u] = (short)e;
                g.begin[u] = (short)(begin + up - c);
            }
            begin += __shfl_sync(0xffffffffu, up, 31);
            used += __popc(any);
        }
        if (lane == 0) experts = used, g.begin[used] = (short)begin;
        __syncwarp();
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (s * 32 >= n) break;
            if (expert[s] >= 0) put(counts.of[expert[s]] + at[s], s * 32 + lane);
        }
    }
    __syncthreads();
    g.n = experts;
    return g;
}

// With experts enough for every team to have several, a warp goes through more of a sum before it meets others (128 tokens of 63 experts:
// teams of eight 383 us, of four 355, of two 346; 37 tokens of 22: 186, 163, 158).
__host__ __device__ __forceinline__ int team_size(int experts) { return experts >= kTeam2 ? 2 : experts >= kTeam4 ? 4 : 8; }

// An fp16 value of h past the type's range.  In its place stands a number that is none, with the sign and ten bits of the value behind them; sixteen more are
// as far behind the place as the workspace's first half is long: a float but for its last five bits.
struct PastRange {
    uint16_t first, second;
    static __device__ __forceinline__ bool is(uint16_t v) { return (v & 0x7c00) == 0x7c00; }
    __device__ __forceinline__ explicit PastRange(float h) {
        const uint32_t v = ((h != h ? 0x7fc00000u : __float_as_uint(h)) + 16) >> 5;
        first = (uint16_t)(v >> 26 << 15 | 0x7c00 | (v >> 16 & 0x3ff));
        second = (uint16_t)v;
    }
    static __device__ __forceinline__ float value(uint16_t first, uint16_t second) {
        return __uint_as_float((uint32_t)(first & 0x8000) << 16 | (uint32_t)(first & 0x3ff) << 21 | (uint32_t)second << 5);
    }
};

__device__ __forceinline__ void copy_4(uint32_t to, const void* from, bool there) {  // (zeros, and nothing is read, where it is not there)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void zero_16(uint32_t to) { asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory"); }

// The matrix unit cuts its running sums off instead of rounding them: by half a unit in 2^23 a step of 16 terms, about 2^-16 of 8192 terms of one sign.
// That is a sixteenth and less of a 16-bit result's own rounding; a warp with more of a sum than that adds it up in the place where the team's sums meet, every kWhole
// bytes.  (In all calls: one token 22.6 -> 24.8 us, 37 tokens with H = 1088, I = 2880 111 -> 117; every 256 terms, to registers, 128 tokens 279 -> 377.)
constexpr int kWhole = 8192, kWholeAtMost = 16384;
__host__ __device__ __forceinline__ bool longer_sums(int row_bytes, int experts) { return row_bytes > kWholeAtMost * team_size(experts); }

// Where a warp's copies are in a launch's work: columns c0 .. c0 + w - 1 of expert e (number u of those that have a place), its places
// p0 .. p0 + n - 1, step along the sum.
struct At {
    int c0, w, u, e, p0, n, end, step;
};

// kLines: lines of a row in a warp's step.  kSets: sets of 16 rows of the weights (of a gated expert one a half).  kUnit: bytes that all rows
// may be copied in: 16 or 4, by the asynchronous copies, or 2.  kDepth: steps of a warp in shared memory.  kLong: sums leave the matrix unit
// (longer_sums()).
template <typename T, int kMode, int kLines, int kSets, int kUnit, int kDepth, bool kLong>
__global__ void __launch_bounds__(kStreamThreads) stream_kernel(Args a, Cut c) {
    constexpr bool kGated = kMode == kUpGated, kIsDown = kMode == kDown, kMma = sizeof(T) == 2, kHalf = std::is_same<T, __half>::value;
    static_assert(!kGated || kSets == 2, "a set for each half");
    constexpr int kHalves = kGated ? 2 : 1;              // row sets of W1
    constexpr int kNTiles = kMostRowsAtOnce / 8;
    constexpr int kFloatRows = kSets == 2 ? 8 : 16;      // floats: rows at a time
    constexpr int kRowBytes = kLines * kLine;            // of a slot's row
    extern __shared__ __align__(128) char memory[];
    char* const ring = memory + groups_bytes(a.T * a.K, a.E);

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, t = lane & 3;
    const int cols = kIsDown ? a.H : a.I, row_bytes = (kIsDown ? a.I : a.H) * (int)sizeof(T);
    const int rank = blockIdx.x % c.spread, first = blockIdx.x / c.spread * c.share, last = min(cols, first + c.share);
    const int pitch = even_rows(c.rows);  // of the sums that meet
    char* mine = ring + warp * kDepth * c.slot;
    float* const behind = reinterpret_cast<float*>(ring + kStreamWarps * kDepth * c.slot + c.past);

    // the down kernel waits for the kernel before it only where it needs h: the choice of experts was there before that began
    if (!kIsDown) pdl_wait();
    const Groups g = group_places(a, memory, *reinterpret_cast<Counts*>(ring));
    if (kIsDown)
        for (int i = threadIdx.x; i < g.begin[g.n]; i += kStreamThreads) g.weight[i] = __ldcg(a.weights + g.of[i]);
    __syncthreads();
    if (!kIsDown) pdl_trigger();

    // Warps that share a sum, and teams of so many that take every other expert.
    const int size = team_size(g.n / c.spread), teams = kStreamWarps / size, team = warp / size, part = warp % size;
    const int u_first = team * c.spread + rank, u_next = teams * c.spread;
    const int stride = size * kRowBytes, steps = (row_bytes + stride - 1) / stride;
    float* const results = behind + 2 * meet_floats(kSets, c.rows);
    float* const sums = results + team * a.T * c.tile;
    auto team_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * size) : "memory"); };
    auto team_any = [&](bool mine) {  // meets as well
        int any;
        asm volatile("{.reg .pred p, q; setp.ne.s32 p, %3, 0; bar.red.or.pred q, %1, %2, p; selp.s32 %0, 1, 0, q;}" : "=r"(any) : "r"(1 + team), "r"(32 * size), "r"((int)mine) : "memory");
        return any != 0;
    };
    const size_t past = (size_t)a.T * a.K * a.ldh;  // elements to the second parts of h

    // Copies: 8 lanes a line, 16 bytes each.  In odd rows the halves of a line change places: eight rows of 64 bytes are read without two of
    // them on one bank.
    const int line = kUnit == 16 ? lane >> 3 : 0, sub = lane & 7, my_byte = part * kRowBytes + (kUnit == 16 ? sub * 16 : lane * 4);
    const size_t next_set = (size_t)(kGated ? a.I : kTileColumns) * row_bytes;
    const uint32_t to_lane = tc::smem_u32(mine) + line * kRowBytes + ((sub ^ (line & 1) * 4) * 16);
    const char* const w_all = static_cast<const char*>(kIsDown ? a.w2 : a.w1);
    const char* const x_all = static_cast<const char*>(kIsDown ? a.h : a.x);
    const size_t x_row = (kIsDown ? a.ldh : a.ldx) * sizeof(T);
    const short* const x_of = kIsDown ? g.of : g.token;
    const char *weights = nullptr, *row0 = nullptr;  // of this lane's first rows, at the step where the copies are
    const size_t next_rows = (size_t)4 * row_bytes;
    int byte = 0;                                    // of the row, there
    At ahead{};
    auto enter = [&] {
        ahead.e = g.expert[ahead.u];
        ahead.p0 = g.begin[ahead.u];
        ahead.end = g.begin[ahead.u + 1];
    };
    auto find = [&] {
        ahead.n = min(c.rows, ahead.end - ahead.p0);
        const size_t row = kIsDown ? (size_t)ahead.e * a.H + ahead.c0 : (size_t)ahead.e * kHalves * a.I + ahead.c0;
        weights = w_all + (row + line) * row_bytes + my_byte;
        if (line < ahead.n) row0 = x_all + x_of[ahead.p0 + line] * x_row + my_byte;
        byte = my_byte;
    };
    auto begin = [&] {
        ahead.u = u_first;
        ahead.c0 = u_first < g.n ? first : last;
        ahead.w = min(c.tile, last - first);
        ahead.step = 0;
        if (u_first < g.n) enter(), find();
    };
    auto go_on = [&] {
        weights += stride;
        row0 += stride;
        byte += stride;
        if (++ahead.step < steps) return;
        ahead.step = 0;
        ahead.p0 += c.rows;
        if (ahead.p0 >= ahead.end) {
            ahead.u += u_next;
            if (ahead.u >= g.n) {
                ahead.u = u_first;
                ahead.c0 += c.tile;
                ahead.w = min(c.tile, last - ahead.c0);
            }
            enter();
        }
        find();
    };
    // Rows that do not begin on 16 bytes: a line at a time, each lane 4 bytes of it.  Where they do not begin on 4 either, by way of registers: a
    // step's elements are loaded before the step at hand is multiplied and stored after it.
    const uint32_t mine_at = tc::smem_u32(mine);
    auto place_of = [&](int row, int l) { return mine_at + row * kRowBytes + l * kLine + (lane * 4 ^ (row & 1) * 64); };
    auto copy_words = [&](int slot, bool take_weights, bool take_rows) {
        const uint32_t at = slot * c.slot;
#pragma unroll 1
        for (int l = 0; l < kLines; ++l) {
            const bool there = byte + l * kLine < row_bytes;
            auto lines = [&](int row0, int rows, auto from_of) {
                for (int r = 0; r < rows; ++r) copy_4(at + place_of(row0 + r, l), there ? from_of(r) + l * kLine : w_all, there);
            };
            if (take_weights)
                for (int m = 0; m < kSets; ++m)
                    lines(m * kTileColumns, min(kTileColumns, kGated ? ahead.w : ahead.w - m * kTileColumns), [&](int r) { return weights + (m ? next_set : 0) + (size_t)r * row_bytes; });
            if (take_rows) lines(kSets * kTileColumns, ahead.n, [&](int r) { return x_all + x_of[ahead.p0 + r] * x_row + byte; });
        }
    };
    constexpr int kHeldRows = (kSets + 1) * kTileColumns;
    uint16_t held[kUnit == 2 ? kLines * kHeldRows : 1][2];
    int held_slot = -1, held_w = 0, held_n = 0;
    bool held_weights = false, held_rows = false;
    auto row_is_held = [&](int i) {  // row i of a slot
        if (i >= kSets * kTileColumns) return held_rows && i - kSets * kTileColumns < held_n;
        return held_weights && (kGated ? i % kTileColumns : i) < held_w;
    };
    auto fetch = [&](int slot, bool take_weights, bool take_rows) {
        held_slot = slot, held_w = ahead.w, held_n = ahead.n, held_weights = take_weights, held_rows = take_rows;
#pragma unroll
        for (int l = 0; l < kLines; ++l)
#pragma unroll
            for (int i = 0; i < kHeldRows; ++i) {
                const int here = byte + l * kLine, m = i / kTileColumns, r = i % kTileColumns;
                const char* from = w_all;
                if (row_is_held(i)) from = (m < kSets ? weights + (m ? next_set : 0) + (size_t)r * row_bytes : x_all + x_of[ahead.p0 + r] * x_row + byte) + l * kLine;
#pragma unroll
                for (int k = 0; k < 2; ++k) held[l * kHeldRows + i][k] = row_is_held(i) && here + 2 * k < row_bytes ? reinterpret_cast<const uint16_t*>(from)[k] : (uint16_t)0;
            }
    };
    auto stash = [&] {
        if (held_slot < 0) return;
#pragma unroll
        for (int l = 0; l < kLines; ++l)
#pragma unroll
            for (int i = 0; i < kHeldRows; ++i)
                if (row_is_held(i))
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(held_slot * c.slot + place_of(i, l)), "r"((uint32_t)held[l * kHeldRows + i][0] | (uint32_t)held[l * kHeldRows + i][1] << 16) : "memory");
        held_slot = -1;
    };
    // (a row may end inside a step: there the copies are of zeros.  A line ends in one too, or is whole: 128 bytes are eight lanes' 16.)
    auto copy = [&](int slot, bool take_weights, bool take_rows) {
        if constexpr (kUnit == 4) return copy_words(slot, take_weights, take_rows);
        if constexpr (kUnit == 2) {
            stash();
            fetch(slot, take_weights, take_rows);
            return;
        }
        const uint32_t to = to_lane + slot * c.slot;
#pragma unroll
        for (int l = 0; l < kLines; ++l) {
            const bool there = byte + l * kLine < row_bytes;
            if (take_weights) {
                const char* p = weights + l * kLine;
#pragma unroll
                for (int m = 0; m < kSets; ++m) {
                    const int rows = (kGated ? ahead.w : ahead.w - m * kTileColumns) - line;
                    const char* q = p + (m ? next_set : 0);
#pragma unroll
                    for (int i = 0; i < kTileColumns / 4; ++i, q += next_rows) {
                        const uint32_t at = to + (m * kTileColumns + 4 * i) * kRowBytes + l * kLine;
                        if (there && 4 * i < rows) copy_16(at, q);
                    }
                }
            }
            if (take_rows) {
                const uint32_t to_row = to + kSets * kTileColumns * kRowBytes + l * kLine;
                if (there && line < ahead.n) copy_16(to_row, row0 + l * kLine);
                if (ahead.n > 4)
                    for (int r = line + 4; r < ahead.n; r += 4) {
                        const char* q = x_all + x_of[ahead.p0 + r] * x_row + byte + l * kLine;
                        if (!there) break;
                        copy_16(to_row + (r - line) * kRowBytes, q);
                    }
            }
            if (!there) {  // zeros for all the slot's rows: what is multiplied with zeros has to be a number
                if (take_weights)
                    for (int r = 0; r < kSets * kTileColumns; r += 4) zero_16(to + r * kRowBytes + l * kLine);
                if (take_rows) {
                    const uint32_t to_row = to + kSets * kTileColumns * kRowBytes + l * kLine;
                    for (int r = line; r < ahead.n; r += 4) zero_16(to_row + (r - line) * kRowBytes);
                }
            }
        }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

    begin();
    if constexpr (kIsDown) {
        for (int i = 0; i < kDepth - 1 && ahead.c0 < last; ++i) {
            copy(i, true, false);
            go_on();
        }
        pdl_wait();  // (who reads what is in out, or wrote what h is made of, is done)
        pdl_trigger();
        begin();
    }
    for (int i = 0; i < kDepth - 1; ++i) {
        if (ahead.c0 < last) {
            copy(i, !kIsDown, true);
            go_on();
        }
        commit();
    }
    if (kUnit == 2) stash();

    int slot = 0, turn = 0;
    const int lane_in_team = part * 32 + lane;
    const char* in_lane = mine + quad * kRowBytes;
    const int chunk[2] = {(t ^ (quad & 1) * 4) * 16, ((4 + t) ^ (quad & 1) * 4) * 16};  // this lane's 16 bytes of either half of a line
    auto next_slot = [&] {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
        __syncwarp();
        if (ahead.c0 < last) {  // into the slot that the step before has left
            copy(slot == 0 ? kDepth - 1 : slot - 1, true, true);
            go_on();
        }
        commit();
        const char* in = in_lane + slot * c.slot;
        if (++slot == kDepth) slot = 0;
        return in;
    };
    for (int c0 = first; c0 < last; c0 += c.tile) {
        const int w = min(c.tile, last - c0);
        if (kIsDown)
            for (int i = lane_in_team; i < a.T * w; i += 32 * size) sums[i] = 0.f;
        for (int u = u_first; u < g.n; u += u_next) {
            const int e = g.expert[u], end = g.begin[u + 1];
            for (int p0 = g.begin[u]; p0 < end; p0 += c.rows) {
                const int n = min(c.rows, end - p0);
                // what a finished sum becomes: of a gated expert, z and what it is multiplied with
                auto finish_up = [&](int column, int row, float z, float z2) {
                    const T* b1 = static_cast<const T*>(a.b1) + (size_t)e * kHalves * a.I + c0 + column;
                    if (a.b1) z += Elem<T>::to_f(*b1);
                    float h = a.act == 0 ? act::value<0, kMma>(z) : a.act == 1 ? act::value<1, kMma>(z) : act::value<2, kMma>(z);
                    if constexpr (kGated) h *= a.b1 ? z2 + Elem<T>::to_f(b1[a.I]) : z2;
                    T* out = static_cast<T*>(a.h) + (size_t)g.of[p0 + row] * a.ldh + c0 + column;
                    *out = Elem<T>::from_f(h);
                    if constexpr (kHalf) {
                        uint16_t* bits = reinterpret_cast<uint16_t*>(out);
                        if (PastRange::is(__half_as_ushort(Elem<T>::from_f(h)))) {
                            const PastRange p(h);
                            bits[0] = p.first, bits[past] = p.second;
                        }
                    }
                };
                // two buffers in turn, so that a team meets once a sum
                bool odd = false;  // whether a sum of this lane is no number
                float* meet = behind + (turn ? meet_floats(kSets, c.rows) : 0) + team * size * 16 * kSets * pitch;
                turn ^= 1;
                if constexpr (kMma) {
                    const int tiles = (n + 7) / 8;
                    float s[kSets][kNTiles][4];
#pragma unroll
                    for (int m = 0; m < kSets; ++m)
#pragma unroll
                        for (int j = 0; j < kNTiles; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[m][j][i] = 0.f;
                    auto place = [&](int m, int j, int h) { return reinterpret_cast<float2*>(meet + ((part * kSets + m) * 16 + quad + h * 8) * pitch + j * 8 + t * 2); };
                    // the sums so far to their places, or all of them back
                    auto keep = [&](bool first, bool back) {
#pragma unroll
                        for (int m = 0; m < kSets; ++m)
#pragma unroll
                            for (int j = 0; j < kNTiles; ++j)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    if (j >= tiles || j * 8 + t * 2 >= pitch) continue;
                                    float2 v = make_float2(s[m][j][2 * h], s[m][j][2 * h + 1]);
                                    if (!first) v.x += place(m, j, h)->x, v.y += place(m, j, h)->y;
                                    if (!back) *place(m, j, h) = v;
                                    s[m][j][2 * h] = back ? v.x : 0.f, s[m][j][2 * h + 1] = back ? v.y : 0.f;
                                }
                    };
                    constexpr int kEvery = kWhole / kRowBytes;
                    for (int step = 0; step < steps; ++step) {
                        if (kLong && step > 0 && step % kEvery == 0) keep(step == kEvery, false);
                        const char* in = next_slot();
#pragma unroll
                        for (int b = 0; b < 2 * kLines; ++b) {
                            const char* at_block = in + b / 2 * kLine + chunk[b & 1];
                            wm::Rows16<T> q[kSets];
#pragma unroll
                            for (int m = 0; m < kSets; ++m)
                                q[m].set(*reinterpret_cast<const uint4*>(at_block + 16 * m * kRowBytes), *reinterpret_cast<const uint4*>(at_block + (16 * m + 8) * kRowBytes));
                            at_block += kSets * kTileColumns * kRowBytes;
#pragma unroll
                            for (int j = 0; j < kNTiles; ++j) {
                                if (j >= tiles) break;
                                wm::Rows8<T> x;
                                x.set(*reinterpret_cast<const uint4*>(at_block + j * 8 * kRowBytes));
#pragma unroll
                                for (int m = 0; m < kSets; ++m) wm::multiply<T>(s[m][j], q[m], x);
                            }
                        }
                        if (kUnit == 2) stash();
                        __syncwarp();
                    }
                    if (kLong && steps > kEvery) keep(false, true);
#pragma unroll
                    for (int m = 0; m < kSets; ++m)
#pragma unroll
                        for (int j = 0; j < kNTiles; ++j) {
                            if (j >= tiles) break;
                            if (j * 8 + t * 2 >= pitch) break;
                            *place(m, j, 0) = make_float2(s[m][j][0], s[m][j][1]);
                            *place(m, j, 1) = make_float2(s[m][j][2], s[m][j][3]);
                            if constexpr (kIsDown && kHalf) {
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (m * 16 + quad + i / 2 * 8 < w && j * 8 + t * 2 + i % 2 < n) odd |= !isfinite(s[m][j][i]);
                            }
                        }
                } else {
                    // floats: a lane multiplies its 16 bytes of two rows of each set with the same bytes of every row
                    F2 s[2 * kSets][kFloatRows];
#pragma unroll
                    for (int m = 0; m < 2 * kSets; ++m)
#pragma unroll
                        for (int j = 0; j < kFloatRows; ++j) s[m][j] = both(0.f);
                    for (int step = 0; step < steps; ++step) {
                        const char* in = next_slot();
#pragma unroll
                        for (int b = 0; b < 2 * kLines; ++b) {
                            F2 q[2 * kSets][2];
#pragma unroll
                            for (int m = 0; m < 2 * kSets; ++m)
                                to_pairs<float, 4>(load_vec<float, 4>(reinterpret_cast<const float*>(in + 8 * m * kRowBytes + b / 2 * kLine + chunk[b & 1])), q[m]);
                            const char* x0 = in - quad * kRowBytes + kSets * kTileColumns * kRowBytes + b / 2 * kLine;
#pragma unroll
                            for (int j = 0; j < kFloatRows; ++j) {
                                if (j >= n) break;
                                F2 x[2];
                                to_pairs<float, 4>(load_vec<float, 4>(reinterpret_cast<const float*>(x0 + j * kRowBytes + ((((b & 1) * 4 + t) ^ (j & 1) * 4) * 16))), x);
#pragma unroll
                                for (int m = 0; m < 2 * kSets; ++m) s[m][j] = fma2(q[m][1], x[1], fma2(q[m][0], x[0], s[m][j]));
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < kFloatRows; ++j) {
                        if (j >= n) break;
#pragma unroll
                        for (int m = 0; m < 2 * kSets; ++m) {
                            float v = sum2(s[m][j]);
                            v += __shfl_xor_sync(0xffffffffu, v, 1);
                            v += __shfl_xor_sync(0xffffffffu, v, 2);
                            if (t == 0) meet[(part * 16 * kSets + 8 * m + quad) * pitch + j] = v;
                        }
                    }
                }
                if constexpr (kIsDown && kHalf) odd = team_any(odd);
                else team_sync();
                auto sum_of = [&](int column, int row) {
                    const float* from = meet + column * pitch + row;
                    float v = *from;
                    for (int k = 1; k < size; ++k) v += *(from += 16 * kSets * pitch);
                    return v;
                };
                if constexpr (kIsDown && kHalf) {
                    if (odd) {  // a warp a sum
                        for (int i = part; i < w * n; i += size) {
                            const int row = i / w, column = i - row * w;
                            float v = sum_of(column, row);
                            if (isfinite(v)) continue;
                            const uint16_t* h = static_cast<const uint16_t*>(a.h) + (size_t)g.of[p0 + row] * a.ldh;
                            const T* w2 = static_cast<const T*>(a.w2) + ((size_t)e * a.H + c0 + column) * a.I;
                            v = 0.f;
                            for (int k0 = 0; k0 < a.I && !__any_sync(0xffffffffu, v != v); k0 += 128)  // (a token that is no number is soon done)
#pragma unroll
                                for (int k = k0 + lane; k < min(a.I, k0 + 128); k += 32) {
                                    const uint16_t bits = h[k];
                                    v = fmaf(Elem<T>::to_f(w2[k]), PastRange::is(bits) ? PastRange::value(bits, h[past + k]) : __half2float(__ushort_as_half(bits)), v);
                                }
                            v = ops::warp_sum(v);
                            if (lane < size) meet[(lane * 16 * kSets + column) * pitch + row] = lane == 0 ? v : 0.f;
                        }
                        team_sync();
                    }
                }
                for (int i = lane_in_team; i < w * n; i += 32 * size) {
                    const int row = i / w, column = i - row * w;
                    if constexpr (!kIsDown) {
                        finish_up(column, row, sum_of(column, row), kGated ? sum_of(kTileColumns + column, row) : 0.f);
                    } else {  // one thread a column and token: a choice may name an expert twice
                        const int token = g.token[p0 + row];
                        if (row > 0 && g.token[p0 + row - 1] == token) continue;
                        const float b2 = a.b2 ? Elem<T>::to_f(static_cast<const T*>(a.b2)[(size_t)e * a.H + c0 + column]) : 0.f;
                        float v = sums[token * w + column];
                        for (int r = row; r < n && g.token[p0 + r] == token; ++r) v += g.weight[p0 + r] * (sum_of(column, r) + b2);
                        sums[token * w + column] = v;
                    }
                }
            }
        }
        if constexpr (kIsDown) {
            namespace cg = cooperative_groups;
            cg::cluster_group cluster = cg::this_cluster();
            __syncthreads();
            for (int i = threadIdx.x; i < a.T * w; i += kStreamThreads) {
                float v = results[i];
                for (int k = 1; k < teams; ++k) v += results[k * a.T * c.tile + i];
                if (c.spread > 1) results[i] = v;
                else static_cast<T*>(a.out)[i / w * a.ldo + c0 + i % w] = Elem<T>::from_f(v);
            }
            if (c.spread == 1) {
                __syncthreads();
                continue;
            }
            cluster.sync();
            for (int i = rank * kStreamThreads + threadIdx.x; i < a.T * w; i += c.spread * kStreamThreads) {
                float v = 0.f;
                for (int k = 0; k < c.spread; ++k) v += *cluster.map_shared_rank(results + i, k);
                static_cast<T*>(a.out)[i / w * a.ldo + c0 + i % w] = Elem<T>::from_f(v);
            }
            cluster.sync();
        }
    }
}

}  // namespace tokens
}  // namespace kleos
