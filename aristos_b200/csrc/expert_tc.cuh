// The experts' products on the tensor cores (bf16, fp16): tcgen05 with paired blocks, operands staged by TMA.
//
//   product_tc_kernel<TE, false>  y[r]  = x[r] W[e]^T + b[e]
//   product_tc_kernel<TE, true>   dx[r] = dy[r] W[e]
//   weight_tc_kernel              dW[e] = sum over the rows r of e of dy[r]^T x[r]
//
// Products: result columns (of W) on the MMA's M side, 256 a pair of blocks, the rows of an expert on its N side, 32 to
// 288 of them: an expert may have any number of rows, and the weights are what a small batch has to stream.  For dx the
// weights' other direction is summed over, so W is read in M-major tiles (64 columns of 64 rows, 128-byte swizzle)
// instead of K-major ones; nothing is transposed in memory.
// Weight gradients: both operands lie with the summed direction (the rows) outermost, so both are M-major / N-major
// tiles of 64 rows.  An expert's last 64 rows may reach into the next expert's: only the steps of 16 rows that it has
// are multiplied, and in the last of those a warp of each block clears the rows that are not its own before the MMA
// reads them (a factor of zero would not do: the other expert's row may be infinite).
// Sums are fp32 in tensor memory: sixteen slots of 32 columns of which a tile of products takes as many as its rows need,
// two accumulators of 256 columns for the weight gradients (see kRead for those in floats), so that the read-back of a tile runs
// beside the next one's main loop.  No load is multicast; every wait is bounded, and a block that gives up stores NaN for what it owes.
//
// What bounds them, measured alone: few rows an expert the weight stream (256 rows of 64 experts, N = K = 2048: 82 us for
// 529 MB = 6.5 TB/s); 256 rows an expert HBM, and the tensor pipe at the clock the power limit leaves (16384 rows: 127 us forward,
// 125 dx, 152 dW for 671 MB each; without their MMAs 112, 108 and 129, dW without its stores 111); thousands of rows the
// tensor pipe (one expert of 16384 rows: 99, 100 and 96 us, 1.37 to 1.43 PFLOP/s; 8192 rows of 8 experts, N = 14336, K =
// 4096: 690 to 820 us, 1.2 to 1.4 PFLOP/s, the operand traffic alone 1.8).  An expert's dW is written once, 256 x 256 at a
// time, through shared memory twice the size of what is on its way; with one such buffer and a list of tiles in shared
// memory 160 us instead of 161: the stores themselves, not the wait for them, are what is left.
#pragma once

#include <cuda.h>

#include "expert_simt.cuh"
#include "tc_common.cuh"

namespace kleos {
namespace experts {
namespace tcp {
using namespace tc;

constexpr int BM = 128, BK = 64;          // per block: M, elements of a slice of the sums
constexpr int kMaxHalf = 144;             // rows of a tile of products, per block
constexpr int HALF_BYTES = 128 * 128;     // 128 lines' slice of an operand
constexpr int kBackWarps = 8, kThreads = (4 + kBackWarps) * 32;
constexpr int TMEM_COLS = 512, ACC_COLS = 256;
constexpr int kSlotCols = 32, kSlots = TMEM_COLS / kSlotCols;
constexpr int kBoxes = 6;

struct RowMaps {
    CUtensorMap box[kBoxes];
};
__host__ __device__ constexpr int box_rows(int i) { return i == 0 ? 16 : i == 1 ? 32 : i == 2 ? 64 : i == 3 ? 96 : i == 4 ? 128 : kMaxHalf; }
__device__ __forceinline__ int box_of(int rows) {
    int i = 0;
    while (box_rows(i) < rows) ++i;
    return i;
}

struct TcArgs {
    const int* offsets;
    const void* bias;
    void* out;
    long long ldo;
    int rows, E;
    int M;            // columns of the result (kernels of products), rows of dW[e] (weight gradients)
    int len;          // length of the sums (products), columns of dW[e]
    int units;        // products: units of 32 rows that a tile has at most, nine
    long long wait_cycles;
};

// Operand tiles of 64 contiguous elements (128 bytes, swizzled) by any number of steps, 64 x 64 blocks 8 KiB apart.
__device__ __forceinline__ uint64_t make_major_desc(uint32_t smem_addr) {
    return (static_cast<uint64_t>(8192 >> 4) << 16) | make_smem_desc(smem_addr) & ~(static_cast<uint64_t>(0x3fff) << 16);
}
constexpr uint32_t kAMajor = 1u << 15, kBMajor = 1u << 16;  // of the instruction descriptor: operand is M- (N-) major
constexpr uint32_t kMajorStep = 16 * 128;                   // bytes of sixteen steps

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar_cluster) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar_cluster)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair_hint(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar_cluster, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %4}], [%5], %6;"
        ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar_cluster), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t smem_src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// 16 lanes x 16 columns as two 16 x 8 fragments: register 4 x + 2 h + i of thread t is lane t / 4 + 8 h, column
// 8 x + 2 (t % 4) + i
__device__ __forceinline__ void tmem_ld_16x256_x2(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
// Four 8 x 8 blocks of 16-bit elements, transposed: thread 8 i + j gives the address of column j of block i.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, const uint32_t* r) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// An arrival that announces nothing in memory: the tensor-memory reads before it have completed.
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool all_of_group(bool yes, int barrier) {  // whether all 128 threads at the barrier say yes
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)yes), "r"(barrier)
        : "memory");
    return all != 0;
}

// kAccs accumulators are announced in turn, kFree parts of tensor memory given back.
template <int kSlices, int kAccs, int kFree>
struct Barriers {
    unsigned long long full[kSlices];   // used on the leader
    unsigned long long empty[kSlices];  // one per block
    unsigned long long tail[kSlices];   // one per block: a slice whose rows are not all the expert's (weight gradients)
    unsigned long long acc_full[kAccs];   // one per block
    unsigned long long acc_empty[kFree];  // used on the leader: the read-back warps of both blocks
    uint32_t tmem_base;
    int abort;
};
// Barriers, tensor memory and the start of the block's life, the same in all kernels here.
template <int kSlices, int kAccs, int kFree>
__device__ __forceinline__ void set_up(Barriers<kSlices, kAccs, kFree>* b, int full_count) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlices; ++i) {
            mbar_init(&b->full[i], full_count);
            mbar_init(&b->empty[i], 1);
            mbar_init(&b->tail[i], 1);
        }
        for (int i = 0; i < kAccs; ++i) mbar_init(&b->acc_full[i], 1);
        for (int i = 0; i < kFree; ++i) mbar_init(&b->acc_empty[i], 2 * kBackWarps);
        b->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x >> 5 == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b->tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
// Neither block may leave while its partner can still touch its shared memory, barriers or tensor memory.
template <int kSlices, int kAccs, int kFree>
__device__ __forceinline__ void tear_down(Barriers<kSlices, kAccs, kFree>* b) {
    tc_fence_before();
    __syncthreads();
    if (*(volatile int*)&b->abort) settle_after_abort();
    cluster_sync_all();
    if (threadIdx.x >> 5 == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(b->tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------- products
constexpr int kSlices = 6;
constexpr int SLICE_BYTES = HALF_BYTES + kMaxHalf * 128;
constexpr int STG_ROW = BM * 2 + 16;  // bytes of a staged row: padded, so that eight rows meet no bank conflict
using ProductBarriers = Barriers<kSlices, kSlots, kSlots>;
struct Control {
    ProductBarriers b;
    int first[kMaxExperts + 1];  // tiles before every expert
    __align__(16) unsigned char stage[2][2][16 * STG_ROW];  // per read-back group, two turns: 16 rows x 256 bytes
};
constexpr int SMEM_BYTES = kSlices * SLICE_BYTES + 1024 + (int)sizeof(Control);
static_assert(SMEM_BYTES <= 232448, "227 KiB of shared memory per block");
static_assert(SLICE_BYTES % 1024 == 0, "the swizzle repeats every 1024 bytes");

// Tiles along the rows of an expert.  A K slice of a tile of n rows takes the larger of 2 n cycles of the tensor pipe and
// n + 256 of shared memory; one of 288 rows is two instructions a step, which read the weights twice, 672 cycles.  Of the
// two counts that come into question, fewest tiles of up to 288 rows or of up to 256, the cheaper one.
__device__ __forceinline__ int split_cost(int units, int s) {  // units of 32 rows, shared out evenly
    const int low = units / s, more = units - low * s;
    auto cost = [](int u) { return u > 8 ? 672 : u > 7 ? 512 : 32 * u + 256; };
    return more * cost(low + 1) + (s - more) * cost(low);
}
__device__ __forceinline__ int row_splits(int n, int most) {
    const int units = (n + 31) >> 5, a = (units + 8) / 9, b = (units + 7) >> 3;
    if (most < 9) return (units + most - 1) / most;
    return a == b || split_cost(units, a) <= split_cost(units, b) ? a : b;
}

// The slots of a tile that starts at ring position `at`: as one run, or as two when they wrap around or are more than the
// 256 columns of an instruction.
struct Runs {
    int n0, n1, slot0, slot1;
    __device__ __forceinline__ Runs(uint32_t at, int half) {
        const int n = half >> 4, room = kSlots - (int)(at % kSlots);
        slot0 = (int)(at % kSlots);
        n0 = n > room ? room : n > 8 ? (n + 1) >> 1 : n;
        n1 = n - n0;
        slot1 = (slot0 + n0) % kSlots;
    }
};

struct Tile {
    int e, col, row, n, half;  // expert, first column of the pair, first row, rows, rows per block in the MMA
    bool once;                 // no other tile reads these weights
};
// Tiles in order of expert, columns, rows: those that run together read the same weights.  An expert's rows are split
// evenly in units of 32 into row_splits() tiles.  `at`: the caller's place in the list.
__device__ __forceinline__ Tile tile_at(int t, const int* first, const TcArgs& g, int* at) {
    int e = *at;
    while (first[e + 1] <= t) ++e;
    *at = e;
    const Group rows = group_rows(g.offsets, e, g.rows);
    const int n = rows.end - rows.begin, splits = row_splits(n, g.units), r = t - first[e];
    Tile x;
    x.e = e;
    const int mt = r / splits, j = r - mt * splits;
    const int units = (n + 31) >> 5, share = units / splits, more = units - share * splits;
    const int u0 = j * share + min(j, more), u = share + (j < more ? 1 : 0);
    x.col = mt * 2 * BM;
    x.row = rows.begin + 32 * u0;
    x.half = 16 * u;
    x.n = min(32 * u, n - 32 * u0);
    x.once = splits == 1;
    return x;
}

// first[e] = sum over the experts before e of tiles(rows of it); warp 0 computes it
template <typename F>
__device__ __forceinline__ void count_tiles(int* first, const TcArgs& g, F tiles) {
    if (threadIdx.x < 32) {
        int at = 0;
        for (int e0 = 0; e0 < g.E; e0 += 32) {
            const int e = e0 + (int)threadIdx.x;
            int n = 0;
            if (e < g.E) {
                const Group r = group_rows(g.offsets, e, g.rows);
                n = tiles(r.end - r.begin);
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if ((int)threadIdx.x >= o) upto += v;
            }
            if (e < g.E) first[e] = at + upto - n;
            at += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (threadIdx.x == 0) first[g.E] = at;
    }
}

template <typename TE, bool kDx>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
product_tc_kernel(const __grid_constant__ RowMaps map_x, const __grid_constant__ CUtensorMap map_w, TcArgs g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    Control* ctl = reinterpret_cast<Control*>(tiles + kSlices * SLICE_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    volatile int* abort_flag = &ctl->b.abort;
    set_up(&ctl->b, 1);
    pdl_wait();
    const int MT = (g.M + 2 * BM - 1) / (2 * BM);
    count_tiles(ctl->first, g, [&](int n) { return row_splits(n, g.units) * MT; });
    __syncthreads();
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem_base = ctl->b.tmem_base;
    const int KS = (g.len + BK - 1) / BK, total = ctl->first[g.E];
    const int t0 = blockIdx.x >> 1, dt = gridDim.x >> 1;

    if (warp == 0 || warp == 3) {
        // ------------------------------------------------------------ TMA: rows (warp 0) and weights (warp 3)
        // The leader announces the bytes of both blocks on its own barrier; a slice that lands before the
        // announcement only makes the barrier's byte count negative for a moment.
        if (lane == 0) {
            // weights that one tile reads leave L2 first, those that others read too stay
            uint64_t stream, keep;
            asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(stream));
            asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(keep));
            uint32_t it = 0;
            int at = 0;
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt) {
                const Tile x = tile_at(t, ctl->first, g, &at);
                const int box = box_of(x.half);
                const uint32_t bytes = 2u * (HALF_BYTES + box_rows(box) * 128);
                for (int kb = 0; kb < KS; ++kb, ++it) {
                    const int s = it % kSlices;
                    if (!mbar_wait(&ctl->b.empty[s], ((it / kSlices) & 1) ^ 1, g.wait_cycles, abort_flag)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    const uint32_t full = map_to_cta(smem_u32(&ctl->b.full[s]), 0);
                    uint8_t* dst = tiles + s * SLICE_BYTES;
                    if (warp == 0) {
                        if (leader) mbar_expect_tx(&ctl->b.full[s], bytes);
                        tma_load_2d_pair(dst + HALF_BYTES, &map_x.box[box], kb * BK, x.row + (int)rank * x.half, full);
                    } else if constexpr (kDx) {
                        const int col = x.col + (int)rank * BM;
                        tma_load_3d_pair_hint(dst, &map_w, col, kb * BK, x.e, full, x.once ? stream : keep);
                        tma_load_3d_pair_hint(dst + 8192, &map_w, col + 64, kb * BK, x.e, full, x.once ? stream : keep);
                    } else {
                        tma_load_3d_pair_hint(dst, &map_w, kb * BK, x.col + (int)rank * BM, x.e, full, x.once ? stream : keep);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader; see tc::elect_one)
        if (leader) {
            const uint32_t elected = elect_one();
            const uint32_t slices = smem_u32(tiles), bars = smem_u32(&ctl->b), tmem = (uint32_t)uniform((int)tmem_base);
            uint32_t s = 0, ph = 0, i = 0, slots = 0;
            int at = 0;
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt, ++i) {
                const int half = uniform(tile_at(t, ctl->first, g, &at).half);
                const Runs runs(slots, half);
                {
                    const uint32_t slot = slots + (uint32_t)lane;  // a lane per slot
                    if (lane < runs.n0 + runs.n1) ok = mbar_wait(&ctl->b.acc_empty[slot % kSlots], ((slot / kSlots) & 1) ^ 1, g.wait_cycles, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                }
                slots += runs.n0 + runs.n1;
                tc_fence_after();
                // N of a run: 32 columns a slot, 16 rows of each block
                const uint32_t idesc = make_instr_desc_16b(2 * BM, 0, Pack2<TE>::kMmaFormat) | (kDx ? kAMajor : 0u);
                const uint32_t idesc0 = idesc | ((uint32_t)runs.n0 << 19), idesc1 = idesc | ((uint32_t)runs.n1 << 19);
                const uint32_t d0 = tmem + runs.slot0 * kSlotCols, d1 = tmem + runs.slot1 * kSlotCols;
                for (int kb = 0; ok && kb < KS; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&ctl->b.full[s], ph, g.wait_cycles, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = slices + s * SLICE_BYTES;
                    const uint64_t da = kDx ? make_major_desc(sa) : make_smem_desc(sa), db = make_smem_desc(sa + HALF_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)
                        umma_bf16_pair_if(elected, d0, da + (kDx ? kMajorStep / 16 : 2u) * k, db + 2 * k, idesc0, k != 0 ? 1u : (uint32_t)(kb != 0));
                    if (runs.n1 > 0) {
                        const uint64_t db1 = make_smem_desc(sa + HALF_BYTES + (uint32_t)runs.n0 * 2048);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            umma_bf16_pair_if(elected, d1, da + (kDx ? kMajorStep / 16 : 2u) * k, db1 + 2 * k, idesc1, k != 0 ? 1u : (uint32_t)(kb != 0));
                    }
                    umma_commit_both_if(elected, bars + (uint32_t)offsetof(ProductBarriers, empty) + 8 * s);
                    if (++s == kSlices) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) *abort_flag = 1;
                else umma_commit_both_if(elected, bars + (uint32_t)offsetof(ProductBarriers, acc_full) + 8 * (i % kSlots));
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------ read-back (both blocks)
        // Tensor-memory lane = result column, column = row.  Group 0 takes the first 16 columns of every slot, group 1 the
        // others; a warp reads the 32 lanes of its quadrant.
        const int q = warp & 3, grp = (warp - 4) >> 2, tg = tid - 128 - grp * 128;
        TE* out = static_cast<TE*>(g.out);
        uint32_t i = 0, slots = 0, turn = 0;
        int at = 0;
        bool dead = false;
        for (int t = t0; t < total; t += dt, ++i) {
            const Tile x = tile_at(t, ctl->first, g, &at);
            const Runs runs(slots, x.half);
            const int n0 = x.col + (int)rank * BM;  // this block's first column
            float bv[4] = {};
            if (!kDx && g.bias) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int n = n0 + q * 32 + 8 * k + (lane >> 2);
                    if (n < g.M) bv[k] = Elem<TE>::to_f(static_cast<const TE*>(g.bias)[(size_t)x.e * g.M + n]);
                }
            }
            if (!dead) {
                const bool ok = mbar_wait(&ctl->b.acc_full[i % kSlots], (i / kSlots) & 1, g.wait_cycles, abort_flag);
                if (!ok) *abort_flag = 1;
                dead = !all_of_group(ok, 1 + grp);
                tc_fence_after();
            }
            // A turn is 16 columns: 16 rows of one block's share.  Two turns' loads are in flight together.
            auto fetch = [&](uint32_t slot, uint32_t* r) {
                if (dead) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) r[k] = 0x7fffffffu;  // NaN
                    return;
                }
                const uint32_t taddr = tmem_base + (slot % kSlots) * kSlotCols + grp * 16 + (static_cast<uint32_t>(q * 32) << 16);
                tmem_ld_16x256_x2(taddr, r);
                tmem_ld_16x256_x2(taddr + (16u << 16), r + 8);
            };
            auto store = [&](int k, const uint32_t* r) {
                // columns of a run: its rows of block 0, then those of block 1
                const bool run1 = k >= runs.n0;
                const int len = (run1 ? runs.n1 : runs.n0) * 16, off = run1 ? runs.n0 * 16 : 0;
                const int c = (k - (run1 ? runs.n0 : 0)) * kSlotCols + grp * 16;
                const int r0 = c >= len ? x.half + off + c - len : off + c;  // row of the tile
                const int valid = min(16, x.n - r0);
                if (valid <= 0) return;  // (the same for all warps of the group)
                // transposed through shared memory: the group's four warps put the block's 128 columns of 16 rows
                // there, and every store instruction writes 256 bytes of two rows
                const uint32_t stg = smem_u32(ctl->stage[grp][turn & 1]);
                ++turn;
#pragma unroll
                for (int x8 = 0; x8 < 2; ++x8) {
                    uint32_t m[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) {  // columns 8 b .. 8 b + 7 of the warp's 32
                        const uint32_t* f = r + (b >> 1) * 8 + x8 * 4 + (b & 1) * 2;
                        const auto p = Pack2<TE>::from_f2(__uint_as_float(f[0]) + bv[b], __uint_as_float(f[1]) + bv[b]);
                        m[b] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    stmatrix_x4_trans(stg + (uint32_t)((8 * x8 + (lane & 7)) * STG_ROW + q * 64 + (lane >> 3) * 16), m);
                }
                // (before the turn after next is staged here, all threads have met for the next one)
                asm volatile("bar.sync %0, 128;" ::"r"(1 + grp) : "memory");
                const int col = (tg & 15) * 8;
                TE* o = out + (long long)(x.row + r0) * g.ldo + n0 + col;
#pragma unroll
                for (int j = tg >> 4; j < 16; j += 8)
                    if (j < valid && n0 + col < g.M) {
                        uint4 v;
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                     : "r"(stg + (uint32_t)(j * STG_ROW + col * 2)));
                        *reinterpret_cast<uint4*>(o + j * g.ldo) = v;
                    }
            };
            const int n_slots = runs.n0 + runs.n1;
#pragma unroll 1
            for (int k = 0; k < n_slots; k += 2) {
                uint32_t r0[16], r1[16];
                const bool two = k + 1 < n_slots;
                fetch(slots + k, r0);
                if (two) fetch(slots + k + 1, r1);
                tmem_ld_wait();
                // this warp's part of the slots is in registers: back to the MMA issuer
                tc_fence_before();
                __syncwarp();
                if (lane < (two ? 2 : 1)) arrive_relaxed(map_to_cta(smem_u32(&ctl->b.acc_empty[(slots + k + lane) % kSlots]), 0));
                store(k, r0);
                if (two) store(k + 1, r1);
            }
            slots += n_slots;
        }
        // rows of nobody
        const int chunks = g.M / 8, end = min(max(g.offsets[g.E], 0), g.rows);
        for (long long r = end + (int)blockIdx.x; r < g.rows; r += gridDim.x)
            for (int c = tid - 128; c < chunks; c += kBackWarps * 32) *reinterpret_cast<uint4*>(out + r * g.ldo + c * 8) = make_uint4(0, 0, 0, 0);
    }
    tear_down(&ctl->b);
}

// ---------------------------------------------------------------- weight gradients
namespace wg {
constexpr int kSlices = 5;
constexpr int SLICE_BYTES = 2 * HALF_BYTES;
constexpr int STG_BYTES = 32 * 128;  // a warp's 32 rows of 128 bytes, twice
// The matrix unit cuts its running sums off instead of rounding them: about 2^-27 of the sum of magnitudes a term, of one sign.  16-bit
// results' own rounding covers that (16384 rows 1.1e-4, where rounding to fp16 takes up to 4.9e-4); that of floats does not: their sums
// are read back every kRead slices, 256 rows, and added up in registers (128 a thread; 60 bytes of them spill).  2-norm error of 16384
// rows, N(0,1) and of one sign: bf16 2.7e-7 and 4.0e-7, fp16 3.7e-7 and 1.2e-6 (all of the sum in the unit 1.9e-5 both, 8.3e-5 and
// 1.1e-4).  One expert of 16384 rows, N = K = 2048: 112 us instead of 96; 8192 rows of 8, N = 14336, K = 4096 876 instead of 815;
// 16384 of 64, N = K = 2048 232 instead of 227.  Tiles of 128 columns, whose sums are 64 registers, 198, 1186 and 249.
constexpr int kRead = 4;
using WeightBarriers = Barriers<kSlices, 2, 2>;
struct Control {
    WeightBarriers b;
};
constexpr int SMEM_BYTES = kSlices * SLICE_BYTES + 2 * kBackWarps * STG_BYTES + 1024 + (int)sizeof(Control);
static_assert(SMEM_BYTES <= 232448, "227 KiB of shared memory per block");

struct Tile {
    int e, row, n, m, c;  // expert, first row and how many, first row and column of dW[e]
};
// Tiles in order of expert, rows, columns of dW: `per` of each expert, `CT` of each row.
__device__ __forceinline__ Tile tile_at(int t, const TcArgs& g, int per, int CT) {
    const int e = t / per, r = t - e * per, mt = r / CT;
    const Group rows = group_rows(g.offsets, e, g.rows);
    return Tile{e, rows.begin, rows.end - rows.begin, mt * 2 * BM, (r - mt * CT) * 256};
}
}  // namespace wg

template <typename TE, bool kWideOut>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
weight_tc_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dw,
                 TcArgs g) {
    constexpr int kSlices = wg::kSlices, SLICE_BYTES = wg::SLICE_BYTES;
    using WeightBarriers = wg::WeightBarriers;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* stage = tiles + kSlices * SLICE_BYTES;
    wg::Control* ctl = reinterpret_cast<wg::Control*>(stage + 2 * kBackWarps * wg::STG_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    volatile int* abort_flag = &ctl->b.abort;
    set_up(&ctl->b, 2);  // a slice of the expert's own rows: the leader twice; another: a warp of each block
    pdl_wait();
    const int MT = (g.M + 2 * BM - 1) / (2 * BM), CT = (g.len + 255) / 256;
    __syncthreads();
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem_base = ctl->b.tmem_base;
    const int per = MT * CT, total = g.E * per;
    const int t0 = blockIdx.x >> 1, dt = gridDim.x >> 1;
    // the last slice of an expert's rows ends inside a step of sixteen: rows of others must not reach the MMA
    auto ragged = [](int n, int kb) { return kb == (n - 1) / BK && (n & 15) != 0; };

    if (warp == 0 || warp == 3) {
        // ------------------------------------------------------------ TMA: x (warp 0) and dy (warp 3)
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt) {
                const wg::Tile x = wg::tile_at(t, g, per, CT);
                for (int kb = 0; kb * BK < x.n; ++kb, ++it) {
                    const int s = it % kSlices;
                    if (!mbar_wait(&ctl->b.empty[s], ((it / kSlices) & 1) ^ 1, g.wait_cycles, abort_flag)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    uint8_t* dst = tiles + s * SLICE_BYTES + (warp == 0 ? HALF_BYTES : 0);
                    const CUtensorMap* map = warp == 0 ? &map_x : &map_dy;
                    const int c = (warp == 0 ? x.c : x.m) + (int)rank * 128, row = x.row + kb * BK;
                    if (ragged(x.n, kb)) {
                        if (warp == 0) mbar_expect_tx(&ctl->b.tail[s], SLICE_BYTES);
                        tma_load_2d(dst, map, c, row, &ctl->b.tail[s]);
                        tma_load_2d(dst + 8192, map, c + 64, row, &ctl->b.tail[s]);
                    } else {
                        const uint32_t full = map_to_cta(smem_u32(&ctl->b.full[s]), 0);
                        if (warp == 0 && leader) {
                            mbar_expect_tx(&ctl->b.full[s], 2 * SLICE_BYTES);
                            mbar_arrive(&ctl->b.full[s]);
                        }
                        tma_load_2d_pair(dst, map, c, row, full);
                        tma_load_2d_pair(dst + 8192, map, c + 64, row, full);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------------------ rows of others in a last slice (both blocks)
        uint32_t it = 0, phases = 0;
        bool ok = true;
        for (int t = t0; ok && t < total; t += dt) {
            const wg::Tile x = wg::tile_at(t, g, per, CT);
            if (x.n == 0) continue;
            const int slices = (x.n + BK - 1) / BK;
            it += slices;
            if (!ragged(x.n, slices - 1)) continue;
            const int s = (it - 1) % kSlices;
            ok = __all_sync(0xffffffffu, mbar_wait(&ctl->b.tail[s], (phases >> s) & 1, g.wait_cycles, abort_flag));
            if (!ok) {
                *abort_flag = 1;
                break;
            }
            phases ^= 1u << s;
            // rows [own, next step of sixteen) of the four 64 x 64 blocks: 128 bytes each
            const int own = x.n - (slices - 1) * BK, others = 16 - (own & 15);
            const uint32_t base = smem_u32(tiles + s * SLICE_BYTES) + own * 128;
            for (int j = lane; j < others * 32; j += 32) {
                const int block = j / (others * 8), k = j - block * (others * 8);
                st_shared_v4(base + block * 8192 + k * 16, make_uint4(0, 0, 0, 0));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_pair(map_to_cta(smem_u32(&ctl->b.full[s]), 0));
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader; see tc::elect_one)
        if (leader) {
            const uint32_t elected = elect_one();
            const uint32_t slices = smem_u32(tiles), bars = smem_u32(&ctl->b), tmem = (uint32_t)uniform((int)tmem_base);
            constexpr uint32_t idesc = make_instr_desc_16b(2 * BM, 256, Pack2<TE>::kMmaFormat) | kAMajor | kBMajor;
            uint32_t s = 0, ph = 0, i = 0;
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt) {
                const int n = uniform(wg::tile_at(t, g, per, CT).n);
                // (a sum is all of an expert's rows, or, of floats, the part that is read back at once)
                for (int k0 = 0; ok && k0 * BK < n; k0 += wg::kRead) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&ctl->b.acc_empty[i & 1], ((i >> 1) & 1) ^ 1, g.wait_cycles, abort_flag));
                    tc_fence_after();
                    const uint32_t d = tmem + (i & 1) * ACC_COLS;
                    const int end = kWideOut ? min(n, (k0 + wg::kRead) * BK) : n;
                    for (int kb = k0; ok && kb * BK < end; ++kb) {
                        ok = __all_sync(0xffffffffu, mbar_wait(&ctl->b.full[s], ph, g.wait_cycles, abort_flag));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t sa = slices + s * SLICE_BYTES;
                        const uint64_t da = make_major_desc(sa), db = make_major_desc(sa + HALF_BYTES);
                        const int steps = min(BK / 16, (end - kb * BK + 15) >> 4);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            if (k < steps) umma_bf16_pair_if(elected, d, da + kMajorStep / 16 * k, db + kMajorStep / 16 * k, idesc, k != 0 ? 1u : (uint32_t)(kb != k0));
                        umma_commit_both_if(elected, bars + (uint32_t)offsetof(WeightBarriers, empty) + 8 * s);
                        if (++s == kSlices) {
                            s = 0;
                            ph ^= 1;
                        }
                    }
                    if (!ok) *abort_flag = 1;
                    else umma_commit_both_if(elected, bars + (uint32_t)offsetof(WeightBarriers, acc_full) + 8 * (i & 1));
                    ++i;
                    if (!kWideOut) break;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------ read-back (both blocks)
        // Tensor-memory lane = row of dW[e], column = its column.  A warp takes the 32 rows of its quadrant, 128 bytes of
        // each at a time: through shared memory, swizzled, and from there by TMA, which leaves out what is past the edges.
        constexpr int kCols = kWideOut ? 32 : 64, kMine = 128;  // columns of a turn, of a group
        const int q = warp & 3, grp = (warp - 4) >> 2;
        const uint32_t stg = smem_u32(stage + 2 * (warp - 4) * wg::STG_BYTES);
        uint32_t i = 0, turn = 0;
        bool dead = false;
        for (int t = t0; t < total; t += dt) {
            const wg::Tile x = wg::tile_at(t, g, per, CT);
            const int m = x.m + (int)rank * BM + q * 32;
            auto await = [&] {  // the next accumulator
                if (dead) return;
                const bool ok = mbar_wait(&ctl->b.acc_full[i & 1], (i >> 1) & 1, g.wait_cycles, abort_flag);
                if (!ok) *abort_flag = 1;
                dead = !__all_sync(0xffffffffu, ok);
                tc_fence_after();
            };
            auto acc = [&] { return tmem_base + (i & 1) * ACC_COLS + (static_cast<uint32_t>(q * 32) << 16) + grp * kMine; };
            auto give_back = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_relaxed(map_to_cta(smem_u32(&ctl->b.acc_empty[i & 1]), 0));
                ++i;
            };
            auto store = [&](int c, const uint32_t* r) {  // columns grp * kMine + c ..
                const int col = x.c + grp * kMine + c;
                if (m >= g.M || col >= g.len) return;  // (the same for the whole warp)
                // the rows of the turn before the last have left shared memory
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                __syncwarp();
                const uint32_t half = stg + (turn++ & 1) * wg::STG_BYTES, line = half + lane * 128;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint4 v;
                    if constexpr (kWideOut) {
                        v = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                    } else {
                        uint32_t p[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const auto two = Pack2<TE>::from_f2(__uint_as_float(r[8 * j + 2 * k]), __uint_as_float(r[8 * j + 2 * k + 1]));
                            p[k] = *reinterpret_cast<const uint32_t*>(&two);
                        }
                        v = make_uint4(p[0], p[1], p[2], p[3]);
                    }
                    st_shared_v4(line + ((j ^ (lane & 7)) << 4), v);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tma_store_3d(&map_dw, half, col, m, x.e);
            };
            if constexpr (kWideOut) {
                uint32_t sum[kMine] = {};
                for (int left = x.n; left > 0; left -= wg::kRead * BK) {
                    await();
                    if (!dead) {
#pragma unroll
                        for (int c = 0; c < kMine; c += 16) {
                            uint32_t r[16];
                            tmem_ld_32x16(acc() + c, r);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) sum[c + k] = __float_as_uint(__uint_as_float(sum[c + k]) + __uint_as_float(r[k]));
                        }
                    }
                    give_back();
                }
                if (x.n > 0 && dead) {
#pragma unroll
                    for (int k = 0; k < kMine; ++k) sum[k] = 0x7fffffffu;  // NaN
                }
#pragma unroll
                for (int c = 0; c < kMine; c += kCols) store(c, sum + c);
            } else {
                if (x.n > 0) await();
#pragma unroll 1
                for (int c = 0; c < kMine; c += kCols) {
                    uint32_t r[kCols];
                    if (x.n == 0 || dead) {
#pragma unroll
                        for (int k = 0; k < kCols; ++k) r[k] = x.n == 0 ? 0u : 0x7fffffffu;
                    } else {
                        tmem_ld_32x32(acc() + c, r);
                        tmem_ld_32x32(acc() + c + 32, r + 32);
                        tmem_ld_wait();
                    }
                    if (c + kCols == kMine && x.n > 0) {
                        // (store() is behind: the accumulator is in registers)
                        give_back();
                    }
                    store(c, r);
                }
            }
        }
        if (lane == 0) bulk_store_wait_all();
    }
    tear_down(&ctl->b);
}

}  // namespace tcp
}  // namespace experts
}  // namespace kleos
