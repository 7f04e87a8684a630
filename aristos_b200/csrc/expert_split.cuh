// The experts' products on the tensor cores where tiles are few: the sums of a tile are split over the pairs of blocks of a
// cluster and joined through their shared memory.
//
//   y[r] = x[r] W[e]^T + b[e]   or   dx[r] = dy[r] W[e]   = sum over the parts p of the elements that part p sums
//
// A pair of blocks streams 256 weights' columns by 64 of the sums at about 70 GB/s a block, which is what bounds a call whose
// tiles leave most multiprocessors idle.  Here kParts pairs, one cluster, take a tile of up to 64 rows: part p sums the p-th
// share of the 64-element steps as product_tc_kernel does, every block puts its 128 columns of fp32 sums into shared memory
// and tells the other parts' blocks of the same columns; then each part adds up its share of the rows, in order of the
// parts, and stores them.  Every call gives the same bits; every wait is bounded, and a block that gives up stores NaN.
//
// Four parts where all tiles' clusters of eight blocks run at once, else two where those of four do; each has 256 elements of the
// sums at least.  What bounds it is still the stream of a block, then the launch and a cluster's two meetings (about 7 us
// together).  bf16, split and not: 3 rows of 12 experts, dx of N = 8920, K = 256 14.0 and 37.5 us; 7 rows, N = 576, K = 6016 10.7 and
// 23.0; 538 rows, N = 728, K = 5888 16.9 and 37.2; dx of 33 rows, N = 14336, K = 4096 (117 MB) 33 and 58; 8 rows of 8 experts, N = K =
// 1024 7.7 and 8.6.
#pragma once

#include "expert_tc.cuh"

namespace kleos {
namespace experts {
namespace tcs {
using namespace tcp;

constexpr int kRows = 64, kHalf = kRows / 2;  // rows of a tile; of the MMA's N side per block
constexpr int kStages = 8, STAGE_BYTES = HALF_BYTES + kHalf * 128;
constexpr int SUM_BYTES = kRows * BM * 4, kCols = 128;  // fp32 sums of a tile; tensor memory: two accumulators
static_assert(STAGE_BYTES % 1024 == 0, "the swizzle repeats every 1024 bytes");

struct HalfMaps {
    CUtensorMap box[2];  // 16 and 32 rows
};
struct Control {
    unsigned long long full[kStages];   // used on a pair's first block
    unsigned long long empty[kStages];  // one per block
    unsigned long long acc_full[2];     // one per block
    unsigned long long acc_empty[2];    // used on a pair's first block: the read-back warps of both blocks
    unsigned long long sum_full;        // one per block: the read-back warps of the blocks with the same columns
    unsigned long long sum_empty;       // ... have read this block's sums
    uint32_t tmem_base;
    int abort;
    int first[kMaxExperts + 1];  // tiles before every expert
};
constexpr int SMEM_BYTES = kStages * STAGE_BYTES + SUM_BYTES + 1024 + (int)sizeof(Control);
static_assert(SMEM_BYTES <= 232448, "227 KiB of shared memory per block");

__host__ __device__ constexpr int row_splits(int n) { return (n + kRows - 1) / kRows; }

struct Tile {
    int e, col, row, n, half;
    bool once;
};
// As tcp::tile_at, in tiles of up to 64 rows.
__device__ __forceinline__ Tile rows_tile_at(int t, const int* first, const TcArgs& g, int* at) {
    int e = *at;
    while (first[e + 1] <= t) ++e;
    *at = e;
    const Group rows = group_rows(g.offsets, e, g.rows);
    const int n = rows.end - rows.begin, splits = row_splits(n), r = t - first[e], mt = r / splits, j = r - mt * splits;
    Tile x;
    x.e = e;
    x.col = mt * 2 * BM;
    x.row = rows.begin + j * kRows;
    x.n = min(kRows, n - j * kRows);
    x.half = x.n > kRows / 2 ? kHalf : kHalf / 2;
    x.once = splits == 1;
    return x;
}

// A wait for what another block of the cluster has written.
__device__ __forceinline__ bool try_wait_cluster(unsigned long long* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_cluster(unsigned long long* bar, uint32_t parity, long long budget, volatile int* abort) {
    if (try_wait_cluster(bar, parity)) return true;
    const long long t0 = clock64();
    uint32_t polls = 0;
    while (!try_wait_cluster(bar, parity))
        if ((++polls & 31u) == 0 && (*abort || clock64() - t0 > budget)) return false;
    return true;
}
__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void commit_pair_if(uint32_t issue, uint32_t bar, uint32_t pair) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "cvt.u16.u32 m, %2;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
        ::"r"(bar), "r"(issue), "r"(3u << pair)
        : "memory");
}

template <typename TE, bool kDx, int kParts>
__global__ void __launch_bounds__(kThreads, 1)
split_tc_kernel(const __grid_constant__ HalfMaps map_x, const __grid_constant__ CUtensorMap map_w, TcArgs g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* sums = reinterpret_cast<float*>(stages + kStages * STAGE_BYTES);  // [row of the tile][column of the block]
    Control* ctl = reinterpret_cast<Control*>(stages + kStages * STAGE_BYTES + SUM_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank(), side = rank & 1, pair = rank & ~1u;
    const int part = (int)(rank >> 1);
    volatile int* abort_flag = &ctl->abort;
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&ctl->full[i], 1);
            mbar_init(&ctl->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl->acc_full[i], 1);
            mbar_init(&ctl->acc_empty[i], 2 * kBackWarps);
        }
        mbar_init(&ctl->sum_full, kParts * kBackWarps);
        mbar_init(&ctl->sum_empty, kParts * kBackWarps);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(kCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    const int MT = (g.M + 2 * BM - 1) / (2 * BM);
    count_tiles(ctl->first, g, [&](int n) { return row_splits(n) * MT; });
    __syncthreads();
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem_base = ctl->tmem_base;
    const int KS = (g.len + BK - 1) / BK, k0 = (int)((long long)KS * part / kParts), k1 = (int)((long long)KS * (part + 1) / kParts);
    const int total = ctl->first[g.E], t0 = blockIdx.x / (2 * kParts), dt = gridDim.x / (2 * kParts);

    if (warp == 0 || warp == 3) {
        // ------------------------------------------------------------ TMA: rows (warp 0) and weights (warp 3)
        if (lane == 0) {
            uint64_t stream, keep;
            asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(stream));
            asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(keep));
            uint32_t it = 0;
            int at = 0;
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt) {
                const Tile x = rows_tile_at(t, ctl->first, g, &at);
                const uint32_t bytes = 2u * (HALF_BYTES + x.half * 128);
                for (int kb = k0; kb < k1; ++kb, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait(&ctl->empty[s], ((it / kStages) & 1) ^ 1, g.wait_cycles, abort_flag)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    const uint32_t full = map_to_cta(smem_u32(&ctl->full[s]), pair);
                    uint8_t* dst = stages + s * STAGE_BYTES;
                    if (warp == 0) {
                        if (side == 0) mbar_expect_tx(&ctl->full[s], bytes);
                        tma_load_2d_pair(dst + HALF_BYTES, &map_x.box[x.half == kHalf], kb * BK, x.row + (int)side * x.half, full);
                    } else if constexpr (kDx) {
                        const int col = x.col + (int)side * BM;
                        tma_load_3d_pair_hint(dst, &map_w, col, kb * BK, x.e, full, x.once ? stream : keep);
                        tma_load_3d_pair_hint(dst + 8192, &map_w, col + 64, kb * BK, x.e, full, x.once ? stream : keep);
                    } else {
                        tma_load_3d_pair_hint(dst, &map_w, kb * BK, x.col + (int)side * BM, x.e, full, x.once ? stream : keep);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (a pair's first block)
        if (side == 0) {
            const uint32_t elected = elect_one();
            const uint32_t slices = smem_u32(stages), bars = smem_u32(ctl), tmem = (uint32_t)uniform((int)tmem_base);
            uint32_t s = 0, ph = 0, i = 0;
            int at = 0;
            bool ok = true;
            for (int t = t0; ok && t < total; t += dt, ++i) {
                const int half = uniform(rows_tile_at(t, ctl->first, g, &at).half);
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl->acc_empty[i & 1], ((i >> 1) & 1) ^ 1, g.wait_cycles, abort_flag));
                tc_fence_after();
                const uint32_t idesc = make_instr_desc_16b(2 * BM, 0, Pack2<TE>::kMmaFormat) | (kDx ? kAMajor : 0u) | ((uint32_t)(2 * half / 8) << 17);
                const uint32_t d = tmem + (i & 1) * kRows;
                for (int kb = k0; ok && kb < k1; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&ctl->full[s], ph, g.wait_cycles, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = slices + s * STAGE_BYTES;
                    const uint64_t da = kDx ? make_major_desc(sa) : make_smem_desc(sa), db = make_smem_desc(sa + HALF_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k)
                        umma_bf16_pair_if(elected, d, da + (kDx ? kMajorStep / 16 : 2u) * k, db + 2 * k, idesc, k != 0 ? 1u : (uint32_t)(kb != k0));
                    commit_pair_if(elected, bars + (uint32_t)offsetof(Control, empty) + 8 * s, pair);
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) *abort_flag = 1;
                else commit_pair_if(elected, bars + (uint32_t)offsetof(Control, acc_full) + 8 * (i & 1), pair);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------ read-back, exchange, store
        // Tensor-memory lane = column of the block, column = row of the tile.  Group 0 takes every other sixteen rows.
        const int q = warp & 3, grp = (warp - 4) >> 2;
        TE* out = static_cast<TE*>(g.out);
        uint32_t i = 0;
        int at = 0;
        bool dead = false;
        auto decide = [&](bool ok) {  // the 256 threads go on or give up together
            if (!ok) *abort_flag = 1;
            uint32_t all;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.ne.b32 p, %1, 0;\n\t"
                "bar.red.and.pred q, 1, 256, p;\n\t"
                "selp.u32 %0, 1, 0, q;\n\t}"
                : "=r"(all)
                : "r"((uint32_t)ok)
                : "memory");
            dead = all == 0;
        };
        auto tell = [&](unsigned long long* bar) {  // the blocks of all parts with these columns
            __syncwarp();
            if (lane < kParts) mbar_arrive_cluster(map_to_cta(smem_u32(bar), 2 * lane + side));
        };
        for (int t = t0; t < total; t += dt, ++i) {
            const Tile x = rows_tile_at(t, ctl->first, g, &at);
            const int col = x.col + (int)side * BM + 4 * lane;  // of the row that this warp stores
            if (!dead) {
                // the sums of the tile before have been read by all parts; this one's are complete
                decide(wait_cluster(&ctl->sum_empty, (i & 1) ^ 1, g.wait_cycles, abort_flag) &&
                       mbar_wait(&ctl->acc_full[i & 1], (i >> 1) & 1, g.wait_cycles, abort_flag));
                tc_fence_after();
            }
            if (!dead) {
                const uint32_t acc = tmem_base + (i & 1) * kRows + (static_cast<uint32_t>(q * 32) << 16);
                for (int c = grp * 16; c < 2 * x.half; c += 32) {
                    uint32_t r[16];
                    tmem_ld_32x16(acc + c, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int k = 0; k < 16; ++k) sums[(c + k) * BM + q * 32 + lane] = __uint_as_float(r[k]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_relaxed(map_to_cta(smem_u32(&ctl->acc_empty[i & 1]), pair));
                tell(&ctl->sum_full);
                decide(wait_cluster(&ctl->sum_full, i & 1, g.wait_cycles, abort_flag));
            }
            float bv[4] = {};
            if (!kDx && g.bias && col < g.M) {
#pragma unroll
                for (int k = 0; k < 4; ++k) bv[k] = Elem<TE>::to_f(static_cast<const TE*>(g.bias)[(size_t)x.e * g.M + col + k]);
            }
            const int r1 = x.n * (part + 1) / kParts;
            for (int r = x.n * part / kParts + warp - 4; r < r1; r += kBackWarps) {
                float v[4];
                if (dead) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(0x7fffffffu);
                } else {
                    float4 f[kParts];
#pragma unroll
                    for (int p = 0; p < kParts; ++p) f[p] = load_cluster(map_to_cta(smem_u32(sums + r * BM + 4 * lane), 2 * p + side));
                    v[0] = f[0].x, v[1] = f[0].y, v[2] = f[0].z, v[3] = f[0].w;
#pragma unroll
                    for (int p = 1; p < kParts; ++p) v[0] += f[p].x, v[1] += f[p].y, v[2] += f[p].z, v[3] += f[p].w;
                }
                if (col < g.M) {  // M is a multiple of eight
                    Vec<TE, 4> o;
#pragma unroll
                    for (int k = 0; k < 4; ++k) o.v[k] = Elem<TE>::from_f(v[k] + bv[k]);
                    store_vec<TE, 4>(out + (long long)(x.row + r) * g.ldo + col, o);
                }
            }
            if (!dead) tell(&ctl->sum_empty);
        }
        // rows of nobody
        const int chunks = g.M / 8, end = min(max(g.offsets[g.E], 0), g.rows);
        for (long long r = end + (int)blockIdx.x; r < g.rows; r += gridDim.x)
            for (int c = tid - 128; c < chunks; c += kBackWarps * 32) *reinterpret_cast<uint4*>(out + r * g.ldo + c * 8) = make_uint4(0, 0, 0, 0);
    }
    // No block may leave while another can still touch its shared memory, barriers or tensor memory.
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) settle_after_abort();
    cluster_sync_all();
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kCols) : "memory");
    }
}

}  // namespace tcs
}  // namespace experts
}  // namespace kleos
