// The experts' products of floats on the tensor cores (tcgen05, paired blocks), over operands that are split into three
// bf16 parts each, as in the float layers' GEMM (gemm_f32.cuh says where the splitting and the short sums come from).
//
//   x = h + m + l, the leading, middle and trailing eight significand bits; of the nine products of two operands six are
//   computed: h h, h m, m h, m m, h l, l h.  The others are below 2^-23 of the product together, half a unit of the last
//   place of an fp32 product each, which is what an fp32 multiply-add rounds away.
//
// The matrix unit does not round its running sums to nearest, so none stays there for long: the h h sums are read back
// every 128 steps, the five small products' sums (below 2^-6 of them) every 512, and both are added up in registers.  2-norm
// error of 2048 terms, N(0,1) and all positive: 1.9e-7 and 2.8e-7 (every 64 and 128: 1.7e-7 twice; 256 and 512: 2.9e-7 and
// 4.8e-7; fp32 multiply-adds 8.1e-7 and 7.0e-7).
// 512 to 8192 terms: 1.8e-7 to 2.4e-7 and 2.6e-7 to 3.0e-7.
// An infinity or NaN makes the h h sums what fp32 multiply-adds give; the small sums beside it are limited to finite values
// and leave it as it is.  A part has bf16's exponents: of an operand below 2^-110 what is below 2^-133 is lost, which fp32
// multiply-adds keep.
//
//   kForward  y[r]  = x[r] W[e]^T + b[e]       M: columns of y    N: rows of e    sum over K
//   kDx       dx[r] = dy[r] W[e]               M: columns of dx   N: rows of e    sum over N of W
//   kDw       dW[e] = sum over r dy[r]^T x[r]  M: columns of dW   N: rows of dW   sum over the rows of e
//
// M is always the direction in which the result is contiguous: a read-back lane is a column, and a store instruction
// writes 128 bytes of a row as it is.  256 columns a pair of blocks by up to 128 rows, which are 32 to 128 of an expert's as
// its number needs.  Per block, 576 threads: warps 0..7 read back and add up, 8..11 split the M operand into tensor
// memory (a lane a column), 12..15 the N operand into shared memory, 16 issues the MMAs (leader) and owns
// tensor memory, 17 loads by TMA, two slices of 32 steps at a time.  What is contiguous along the sums is loaded and split line by
// line; what is contiguous across them comes in tiles of 32 x 32 that are read down a column (M operand) or split into
// N-major parts (N operand).  Rows that are not the expert's are cleared when they are split.
//
// What bounds it: the roles' own time, about 1900 to 2200 cycles for a step of 64, for the split of either operand as for
// the read-back, where its MMAs take 1536 (without them a launch took as long); 2048 columns, 256 rows an expert: 4.3 tiles a
// pair of blocks in five rounds.  4096 rows, 16 experts, N = K = 2048: 222, 217 and 249 us (34.4 GFLOP each: 155, 158 and 138
// TFLOP/s; the FP32 pipes 1014, 965 and 734).  Steps, from 287, 289 and 288: a step a barrier instead of a slice, four
// warps for the N operand instead of two 252, 251, 288; sums read back half and a quarter as often.  Eight warps for the M operand,
// whose registers the others then lack, 282, 270 and 332 instead of 252, 251 and 288; six for the N operand 219, 221 and 256.
#pragma once

#include <cfloat>

#include "expert_tc.cuh"

namespace kleos {
namespace experts {
namespace f32 {
using namespace tcp;

constexpr int BK = 32, ROW = BK * 2;           // steps of a slice; bytes of a part's row of them
constexpr int kDrain = 8, kSplitA = 4, kSplitB = 4, kSplit = kSplitA + kSplitB;  // warps
constexpr int kMmaWarp = kDrain + kSplit, kTmaWarp = kMmaWarp + 1;
constexpr int kThreads = (kTmaWarp + 1) * 32;  // 96 registers a thread; forward and dx spill 16 bytes
constexpr int kStep = 2;   // slices that are loaded, split and multiplied at a time
constexpr int kHigh = 2;   // steps whose h h products share a read-back
constexpr int kGroup = 8;  // steps whose small products share one
constexpr int kStages = 2, kRing = 3;  // of a step each
constexpr int kHalf = 64;  // rows of N per block
constexpr int BN = 2 * kHalf;
constexpr int PLANE = kHalf * ROW, PARTS_BYTES = 3 * PLANE;                        // of a slice
constexpr int A_BYTES = BM * BK * 4, SLICE_BYTES = A_BYTES + kHalf * BK * 4;  // as loaded
constexpr int STAGE_BYTES = kStep * PARTS_BYTES, SLOT_BYTES = kStep * SLICE_BYTES;
constexpr int A_COLS = 3 * BK / 2, A_COL0 = 2 * BN;  // tensor memory: h h sums, small sums, then the M operand's parts
static_assert(A_COL0 + kStages * kStep * A_COLS <= TMEM_COLS, "tensor memory has 512 columns");

struct Control {
    unsigned long long ring_full[kRing];   // TMA bytes of the slot have landed
    unsigned long long ring_empty[kRing];  // the split warps have read the slot
    unsigned long long full[kStages];      // used on the leader: the step's parts are in place, split warps of both blocks
    unsigned long long done[kStages];      // one per block: the MMAs of the step have completed
    unsigned long long sum_full[2];        // one per block: [0] h h sums of a step, [1] small sums of a group are complete
    unsigned long long sum_empty[2];       // used on the leader: ... and have been read, drain warps of both blocks
    uint32_t tmem_base;
    int abort;
    int first[kMaxExperts + 1];
};
constexpr int SMEM_BYTES = kStages * STAGE_BYTES + kRing * SLOT_BYTES + 1024 + (int)sizeof(Control);
static_assert(SMEM_BYTES <= 232448, "227 KiB of shared memory per block");

// Descriptors of a part of the N operand: rows of 64 bytes with the swizzle of that span, groups of 8 rows 512 bytes
// apart; or N-major, 64 elements (128 bytes) a step, groups of 8 steps 1024 bytes apart.
template <bool kAcross>
__device__ __forceinline__ uint64_t part_desc(uint32_t addr) {
    if constexpr (kAcross) return make_major_desc(addr);
    return (make_smem_desc(addr) & ~((7ull << 61) | (0x3fffull << 32))) | (4ull << 61) | (static_cast<uint64_t>(512 >> 4) << 32);
}
// 256 x N accumulator += A (tensor memory of each block of the pair, 128 lanes) x B (shared memory)
__device__ __forceinline__ void umma_ta(uint32_t issue, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
// 16 registers per thread -> 32 lanes x 16 columns of tensor memory
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// Four fp32 values -> their leading, middle and trailing eight bits as bf16 (the conversion keeps every NaN a NaN).
__device__ __forceinline__ void split4(const float (&v)[4], uint2* h, uint2* m, uint2* l) {
    uint32_t top[2], mid[4], low[4];
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(top[k / 2]) : "f"(v[k + 1]), "f"(v[k]));
        const float r[2] = {v[k] - __uint_as_float(top[k / 2] << 16), v[k + 1] - __uint_as_float(top[k / 2] & 0xffff0000u)};  // exact
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mid[k + i] = __float_as_uint(r[i]);
            low[k + i] = __float_as_uint(r[i] - __uint_as_float(mid[k + i] & 0xffff0000u));
        }
    }
    *h = make_uint2(top[0], top[1]);
    *m = make_uint2(__byte_perm(mid[0], mid[1], 0x7632), __byte_perm(mid[2], mid[3], 0x7632));
    *l = make_uint2(__byte_perm(low[0], low[1], 0x7632), __byte_perm(low[2], low[3], 0x7632));
}
// Bounded wait without a pause between the polls: the waits hand a slice of under a thousand cycles from role to role.
__device__ __forceinline__ bool spin(unsigned long long* bar, uint32_t parity, long long budget, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity))
        if (*abort || clock64() - t0 > budget) {
            *abort = 1;
            return false;
        }
    return true;
}
struct Turn {  // position in a ring of n buffers and the parity of the current round
    int n, at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ explicit Turn(int n_) : n(n_) {}
    __device__ __forceinline__ void next() {
        if (++at == n) at = 0, parity ^= 1;
    }
};

struct Tile {
    int e, col;          // expert, first column of the pair
    int row, n, half;    // first row of the result, how many, rows per block in the MMA
    int k0, len;         // first row (weight gradients: the sums' first step) and length of the sums
    __device__ __forceinline__ int steps() const { return (len + kStep * BK - 1) / (kStep * BK); }
};
// Tiles in order of expert, columns, rows.  Products: an expert's rows split evenly in units of 32 into as few tiles of up to
// 128 as hold them.  `at`: the caller's place in the list.
template <int kMode>
__device__ __forceinline__ Tile tile_at(int t, const int* first, const TcArgs& g, int per, int RT, int* at) {
    Tile x;
    if constexpr (kMode == kDw) {
        const int e = t / per, r = t - e * per, mt = r / RT;
        const Group rows = group_rows(g.offsets, e, g.rows);
        x.e = e;
        x.col = mt * 2 * BM;
        x.row = (r - mt * RT) * BN;
        x.n = min(BN, g.len - x.row);
        x.half = kHalf;
        x.k0 = rows.begin;
        x.len = rows.end - rows.begin;
    } else {
        int e = *at;
        while (first[e + 1] <= t) ++e;
        *at = e;
        const Group rows = group_rows(g.offsets, e, g.rows);
        const int n = rows.end - rows.begin, splits = (n + BN - 1) / BN, r = t - first[e], mt = r / splits, j = r - mt * splits;
        const int units = (n + 31) >> 5, share = units / splits, more = units - share * splits;
        const int u0 = j * share + min(j, more), u = share + (j < more ? 1 : 0);
        x.e = e;
        x.col = mt * 2 * BM;
        x.row = rows.begin + 32 * u0;
        x.half = 16 * u;
        x.n = min(32 * u, n - 32 * u0);
        x.k0 = 0;
        x.len = g.len;
    }
    return x;
}

// g.M: columns of the result; g.len: length of the sums (products), rows of dW[e] (weight gradients).
template <int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
product_f32_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, TcArgs g) {
    constexpr bool kAcrossA = kMode != kForward, kAcrossB = kMode == kDw;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* ring = stages + kStages * STAGE_BYTES;
    Control* ctl = reinterpret_cast<Control*>(ring + kRing * SLOT_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)cluster_ctarank();
    volatile int* abort_flag = &ctl->abort;
    if (tid == 0) {
        for (int s = 0; s < kRing; ++s) {
            mbar_init(&ctl->ring_full[s], 1);
            mbar_init(&ctl->ring_empty[s], kSplit);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&ctl->full[s], 2 * kSplit);
            mbar_init(&ctl->done[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->sum_full[b], 1);
            mbar_init(&ctl->sum_empty[b], 2 * kDrain);
        }
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    const int MT = (g.M + 2 * BM - 1) / (2 * BM), RT = kMode == kDw ? (g.len + BN - 1) / BN : 0, per = MT * RT;
    if constexpr (kMode != kDw) count_tiles(ctl->first, g, [&](int n) { return (n + BN - 1) / BN * MT; });
    __syncthreads();
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem_base = ctl->tmem_base;
    const int total = kMode == kDw ? g.E * per : ctl->first[g.E], t0 = blockIdx.x >> 1, dt = gridDim.x >> 1;
    int at = 0;

    if (warp == kTmaWarp) {
        // ------------------------------------------------------------ TMA (both blocks)
        if (lane == 0) {
            Turn slot(kRing);
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt) {
                const Tile x = tile_at<kMode>(t, ctl->first, g, per, RT, &at);
                const int steps = x.steps(), col = x.col + rank * BM;
                for (int i = 0; i < steps; ++i) {
                    if (!(ok = spin(&ctl->ring_empty[slot.at], slot.parity ^ 1, g.wait_cycles, abort_flag))) break;
                    unsigned long long* bar = &ctl->ring_full[slot.at];
                    const uint32_t own = map_to_cta(smem_u32(bar), rank);
                    mbar_expect_tx(bar, SLOT_BYTES);
#pragma unroll
                    for (int h = 0; h < kStep; ++h) {
                        uint8_t *a = ring + slot.at * SLOT_BYTES + h * SLICE_BYTES, *b = a + A_BYTES;
                        const int k = (i * kStep + h) * BK;
                        if constexpr (kMode == kForward) tma_load_3d_pair(a, &map_a, k, col, x.e, own);
#pragma unroll
                        for (int j = 0; j < BM / 32; ++j) {
                            if constexpr (kMode == kDx) tma_load_3d_pair(a + j * 4096, &map_a, col + 32 * j, k, x.e, own);
                            if constexpr (kMode == kDw) tma_load_2d(a + j * 4096, &map_a, col + 32 * j, x.k0 + k, bar);
                        }
                        if constexpr (kAcrossB) {
                            tma_load_2d(b, &map_b, x.row + rank * kHalf, x.k0 + k, bar);
                            tma_load_2d(b + 4096, &map_b, x.row + rank * kHalf + 32, x.k0 + k, bar);
                        } else {
                            tma_load_2d(b, &map_b, k, x.row + rank * x.half, bar);
                        }
                    }
                    slot.next();
                }
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ MMA issuer (leader only)
        if (rank == 0) {
            // parts of the operands whose products are summed apart from h h, smallest first
            constexpr int kPartA[5] = {2, 0, 1, 1, 0}, kPartB[5] = {0, 2, 1, 0, 1};
            const uint32_t elected = elect_one(), tmem = (uint32_t)uniform((int)tmem_base);
            const uint32_t bars = smem_u32(ctl), parts = smem_u32(stages);
            auto wait = [&](unsigned long long* bar, uint32_t parity) {
                const bool ok = __all_sync(0xffffffffu, spin(bar, parity, g.wait_cycles, abort_flag));
                tc_fence_after();
                return ok;
            };
            int s = 0;                        // stage
            uint32_t sp = 0, hp = 0, lp = 0;  // parities: stages, h h sums, small sums
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt) {
                const Tile x = tile_at<kMode>(t, ctl->first, g, per, RT, &at);
                const int steps = uniform(x.steps());
                const uint32_t idesc = make_instr_desc_bf16(2 * BM, uniform(2 * x.half)) | (kAcrossB ? kBMajor : 0u);
                auto multiply = [&](int slice, int pa, int pb, uint32_t d, bool more) {  // slice: of all stages
                    const uint32_t ta = tmem + A_COL0 + slice * A_COLS + pa * (BK / 2);
                    const uint64_t db = part_desc<kAcrossB>(parts + slice * PARTS_BYTES + pb * PLANE);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)
                        umma_ta(elected, d, ta + k * 8, db + (kAcrossB ? kMajorStep / 16 : 2u) * k, idesc, (more || k > 0) ? 1u : 0u);
                };
                for (int kd = 0; kd < steps; ++kd) {
                    const bool fresh = kd % kHigh == 0;
                    if (fresh) {
                        if (!(ok = wait(&ctl->sum_empty[0], hp ^ 1))) break;
                        hp ^= 1;
                    }
                    if (!(ok = wait(&ctl->full[s], sp))) break;
#pragma unroll
                    for (int j = 0; j < kStep; ++j) multiply(s * kStep + j, 0, 0, tmem, !fresh || j > 0);
                    if (kd + 1 == steps || kd % kHigh == kHigh - 1) umma_commit_both_if(elected, bars + (uint32_t)offsetof(Control, sum_full));
                    const bool first = kd % kGroup == 0;
                    if (first) {
                        if (!(ok = wait(&ctl->sum_empty[1], lp ^ 1))) break;
                        lp ^= 1;
                    }
#pragma unroll
                    for (int j = 0; j < kStep; ++j)
#pragma unroll
                        for (int p = 0; p < 5; ++p) multiply(s * kStep + j, kPartA[p], kPartB[p], tmem + BN, !first || (j | p) != 0);
                    umma_commit_both_if(elected, bars + (uint32_t)offsetof(Control, done) + 8 * s);
                    if (kd + 1 == steps || kd % kGroup == kGroup - 1) umma_commit_both_if(elected, bars + (uint32_t)offsetof(Control, sum_full) + 8);
                    if (++s == kStages) s = 0, sp ^= 1;
                }
            }
        }
        __syncwarp();
    } else if (warp >= kDrain) {
        // ------------------------------------------------------------ split (both blocks)
        const bool m_side = warp < kDrain + kSplitA;
        const int q = warp & 3, line = q * 32 + lane, tb = tid - (kDrain + kSplitA) * 32;
        Turn stage(kStages), slot(kRing);
        bool ok = true;
        for (int t = t0; ok && t < total; t += dt) {
            const Tile x = tile_at<kMode>(t, ctl->first, g, per, RT, &at);
            const int steps = x.steps();
            for (int i = 0; i < steps; ++i) {
                // the stage is free once the MMAs of the step before in it have completed
                ok = spin(&ctl->done[stage.at], stage.parity ^ 1, g.wait_cycles, abort_flag) &&
                     spin(&ctl->ring_full[slot.at], slot.parity, g.wait_cycles, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int half = 0; half < kStep; ++half) {
                    const uint8_t* src = ring + slot.at * SLOT_BYTES + half * SLICE_BYTES;
                    const int valid = kMode == kDw ? x.len - (i * kStep + half) * BK : BK;  // steps of the slice that are the expert's rows
                    if (m_side) {
                        uint32_t h[16], m[16], l[16];
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            float v[4];
                            if constexpr (kAcrossA) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const int k = 4 * c + j;
                                    v[j] = *reinterpret_cast<const float*>(src + q * 4096 + k * 128 + (((lane >> 2) ^ (k & 7)) << 4) + (lane & 3) * 4);
                                    if (kMode == kDw && k >= valid) v[j] = 0.f;
                                }
                            } else {
                                const float4 f = *reinterpret_cast<const float4*>(src + line * 128 + ((c ^ (line & 7)) << 4));
                                v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
                            }
                            split4(v, reinterpret_cast<uint2*>(h + 2 * c), reinterpret_cast<uint2*>(m + 2 * c), reinterpret_cast<uint2*>(l + 2 * c));
                        }
                        const uint32_t ta = tmem_base + A_COL0 + (stage.at * kStep + half) * A_COLS + (static_cast<uint32_t>(q * 32) << 16);
                        tmem_st_32x16(ta, h);
                        tmem_st_32x16(ta + BK / 2, m);
                        tmem_st_32x16(ta + BK, l);
                    } else {
                        src += A_BYTES;
                        uint8_t* dst = stages + stage.at * STAGE_BYTES + half * PARTS_BYTES;
#pragma unroll
                        for (int j = 0; j < 16 / kSplitB; ++j) {
                            uint32_t from, to;
                            bool in = true;
                            if constexpr (kAcrossB) {  // four columns of step k
                                const int k = (tb >> 4) + 2 * kSplitB * j, c = tb & 15;
                                from = (uint32_t)((c >> 3) * 4096 + k * 128 + (((c & 7) ^ (k & 7)) << 4));
                                to = (uint32_t)(k * 128 + (((c >> 1) ^ (k & 7)) << 4) + ((c & 1) << 3));
                                in = k < valid;
                            } else {  // four steps of row r
                                const int r = (tb >> 3) + 4 * kSplitB * j, c = tb & 7;
                                if (r >= x.half) break;
                                from = (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
                                to = (uint32_t)(r * ROW + (((c >> 1) ^ ((r >> 1) & 3)) << 4) + ((c & 1) << 3));
                            }
                            const float4 f = *reinterpret_cast<const float4*>(src + from);
                            const float v[4] = {in ? f.x : 0.f, in ? f.y : 0.f, in ? f.z : 0.f, in ? f.w : 0.f};
                            uint2 h, m, l;
                            split4(v, &h, &m, &l);
                            *reinterpret_cast<uint2*>(dst + to) = h;
                            *reinterpret_cast<uint2*>(dst + to + PLANE) = m;
                            *reinterpret_cast<uint2*>(dst + to + 2 * PLANE) = l;
                        }
                    }
                }
                if (m_side) {
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                } else {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_pair(map_to_cta(smem_u32(&ctl->full[stage.at]), 0));
                    mbar_arrive(&ctl->ring_empty[slot.at]);
                }
                stage.next();
                slot.next();
            }
        }
    } else {
        // ------------------------------------------------------------ drain (both blocks)
        // Tensor-memory lane = column of the result; warps 0..3 have the rows of block 0, warps 4..7 those of block 1.
        const int q = warp & 3, part = warp >> 2;
        float* out = static_cast<float*>(g.out);
        uint32_t hp = 0, lp = 0;
        bool dead = false;
        for (int t = t0; t < total; t += dt) {
            const Tile x = tile_at<kMode>(t, ctl->first, g, per, RT, &at);
            const int steps = x.steps();
            float acc[kHalf];
#pragma unroll
            for (int j = 0; j < kHalf; ++j) acc[j] = 0.f;
            // Adds an accumulator to the registers and hands it back to the MMA issuer.
            auto add = [&](int which, uint32_t parity, auto small) {
                if (dead) return;
                dead = !__all_sync(0xffffffffu, spin(&ctl->sum_full[which], parity, g.wait_cycles, abort_flag));
                if (dead) return;
                tc_fence_after();
                const uint32_t taddr = tmem_base + which * BN + part * x.half + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll
                for (int c = 0; c < kHalf / 16; ++c) {
                    if (c * 16 >= x.half) break;
                    uint32_t v[16];
                    tmem_ld_32x16(taddr + c * 16, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float f = __uint_as_float(v[j]);
                        if (decltype(small)::value) f = fmaxf(fminf(f, FLT_MAX), -FLT_MAX);
                        acc[c * 16 + j] += f;
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(map_to_cta(smem_u32(&ctl->sum_empty[which]), 0));
            };
            for (int kd = 0; kd < steps; ++kd) {
                if (kd + 1 == steps || kd % kHigh == kHigh - 1) {
                    add(0, hp, std::false_type());
                    hp ^= 1;
                }
                if (kd + 1 == steps || kd % kGroup == kGroup - 1) {
                    add(1, lp, std::true_type());
                    lp ^= 1;
                }
            }
            const int col = x.col + rank * BM + q * 32 + lane, rows = min(x.half, x.n - part * x.half);
            if (col < g.M) {
                const float b = kMode == kForward && g.bias ? static_cast<const float*>(g.bias)[(size_t)x.e * g.M + col] : 0.f;
                float* o = out + (kMode == kDw ? (size_t)x.e * g.len * g.M : 0) + (long long)(x.row + part * x.half) * g.ldo + col;
#pragma unroll
                for (int j = 0; j < kHalf; ++j)
                    if (j < rows) o[(long long)j * g.ldo] = dead ? __uint_as_float(0x7fffffffu) : acc[j] + b;
            }
            __syncwarp();
        }
        if constexpr (kMode != kDw) {
            // rows of nobody
            const int end = min(max(g.offsets[g.E], 0), g.rows);
            for (long long r = end + (int)blockIdx.x; r < g.rows; r += gridDim.x)
                for (int c = tid; c < g.M; c += kDrain * 32) out[r * g.ldo + c] = 0.f;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) settle_after_abort();
    cluster_sync_all();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace f32
}  // namespace experts
}  // namespace kleos
