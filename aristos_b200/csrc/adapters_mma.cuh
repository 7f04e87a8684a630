// The adapters' products (adapters.cuh) where 16-bit rows begin on 16-byte boundaries and the rank is a multiple of 8 (up to 16, of 4; for the
// gradients, of 2): on the tensor cores, straight from memory (warp_mma.cuh).
//
//   rows_mma_kernel   u and y, or v and dx: a cluster of blocks takes up to TR rows of a request
//   grads_mma_kernel  dA or dB: a cluster takes 256 columns of one adapter and goes through the rows of its requests
//
// A block has eight warps.  First product: RG groups of warps have 16 MT rows each, the KS warps of a group (times the blocks of the cluster)
// take 128 bytes of those rows in turn; the partial sums meet in shared memory, across the cluster where few rows make few blocks.
// Second product: the same groups, the warps take 32 columns in turn; columns are dealt to the instruction's so that a lane ends
// with eight neighbours, which it adds to base and stores in one piece.
// Where the summed direction is not the contiguous one (both products of the backward pass, the gradients' rows), 8 x 8 blocks change rows
// and columns between lanes on their way (movmatrix); nothing is transposed in memory.
//
// What bounds them, alone: few rows latency (one row, N = K = 2048, rank 16: 5 us; 128 requests of a row each 11); prompts latency of loads
// (7919 rows, N = 2880, K = 1088, rank 32, fp16: 44 us, 104 MB of HBM); many rows of a large rank shared memory, which the tensor cores' operands
// cross four times (16384 rows, N = K = 4096, rank 64: 120 us forward and for dx, 402 MB each), and instructions beside it (both gradients 148 us for
// 278 MB: the adapter with the most rows sets the time).
//
// u and v are factors of the second products as values of the element type: rounded once, as a projection's own input would be (both parts of
// them would double those products' time on the tensor cores and halve the rounding error of a result).  Gradients in floats, which would show
// that, are made of both parts.  fp16 has too little range for either:
// a row is divided by a power of two first (in the gradients: every rank by itself, all its rows by that of the largest so far).
#pragma once

#include "adapters.cuh"
#include "warp_mma.cuh"

namespace kleos {
namespace adapters {

constexpr int kWarps = 8;

__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// The power of two that brings a largest value m to [2^14, 2^15), which leaves fp16 as much as it has below: values down to 2^-28 of the largest keep all their
// bits, those down to 2^-38 some.  2^126 at most, which zero has too.
__device__ __forceinline__ float top_of(float m) { return __uint_as_float(min(268u - (__float_as_uint(m) >> 23), 253u) << 23); }
// What a rounding left of a value; nothing of one that is no number or became an infinity.
__device__ __forceinline__ float rest_of(float v, float rounded) { return fabsf(rounded) < INFINITY ? v - rounded : 0.f; }
__device__ __forceinline__ float finite_size(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.f; }

template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const typename Pack2<T>::type p = Pack2<T>::from_f2(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}

template <int RT, int TR>
struct Shape {
    static constexpr int MT = TR == 16 || RT == 128 ? 1 : 2;  // of 16 rows, a warp's
    static constexpr int RG = TR / (16 * MT), KS = kWarps / RG;
    static constexpr int NT = RT / 8;                         // columns of u, by eight
    static constexpr int kPitch = RT + 4;                     // floats of a row of partial sums
    static constexpr int kBytes = KS * TR * kPitch * 4;
};

template <typename T, bool kBack, int RT, int TR>
__global__ void __launch_bounds__(256, RT == 64 && TR == 64 ? 1 : 2) rows_mma_kernel(Args a) {
    namespace cg = cooperative_groups;
    using S = Shape<RT, TR>;
    constexpr int MT = S::MT, RG = S::RG, KS = S::KS, NT = S::NT;
    constexpr int kQ = RT == 16 ? 2 : 4;   // n-tiles of a vector of P, backward
    constexpr bool kShrink = std::is_same<T, __half>::value;
    extern __shared__ __align__(128) char memory[];
    float* const part = reinterpret_cast<float*>(memory);  // [KS][TR][pitch]
    __shared__ __align__(16) T ub[TR][RT + 8];
    __shared__ float grow[TR];                          // what a row's second product is multiplied with
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, t = lane & 3;
    const int rg = warp % RG, ks = warp / RG;
    pdl_wait();
    pdl_trigger();
    Tile tile;
    if (!find_tile<TR>(a, blockIdx.x / blocks, &tile)) return;  // (all blocks of the cluster)
    const int n = tile.end - tile.begin;
    if (tile.adapter < 0) {
        const int share = ((a.cols + blocks - 1) / blocks + 7) / 8 * 8, c0 = min(a.cols, block * share);
        copy_base<T, 8>(a, tile, c0, min(a.cols, c0 + share));
        if (a.u && block == 0)
            for (int i = threadIdx.x; i < n * a.r; i += 256) a.u[(long long)tile.begin * a.r + i] = 0.f;
        return;
    }
    const float scale = a.scale ? a.scale[tile.adapter] : 1.f;
    const T* P = static_cast<const T*>(a.p) + (size_t)tile.adapter * a.r * a.len;
    const T* Q = static_cast<const T*>(a.q) + (size_t)tile.adapter * a.r * a.cols;

    // ------------------------------------------------ first product
    const T* in[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)  // rows past the last are the last; nobody takes their sums
            in[m][h] = static_cast<const T*>(a.in) + (long long)(tile.begin + min((rg * MT + m) * 16 + h * 8 + quad, n - 1)) * a.ldi + t * 8;
    float d[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[m][j][i] = 0.f;
    // The matrix unit cuts its running sums off instead of rounding them, and u is a 32-bit result: every kWhole steps of 64 elements a warp's sums are
    // added to those that it has in shared memory (columns of tile j in their own order; backward: as they were dealt).
    constexpr int kWhole = 4;
    bool begun = false;
    auto put = [&] {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int col = !kBack ? j * 8 + t * 2 : RT == 16 ? t * 4 + j * 2 : j / 4 * 32 + t * 8 + j % 4 * 2;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float2* to = reinterpret_cast<float2*>(part + (ks * TR + (rg * MT + m) * 16 + h * 8 + quad) * S::kPitch + col);
                    const float2 before = begun ? *to : make_float2(0.f, 0.f);
                    *to = make_float2(before.x + d[m][j][2 * h], before.y + d[m][j][2 * h + 1]);
                    d[m][j][2 * h] = d[m][j][2 * h + 1] = 0.f;
                }
            }
        begun = true;
    };
    // 32 elements at a time, two of those next to each other
    const int pieces = (a.len + 31) / 32, next = 2 * KS * blocks;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto load_in = [&](int piece, uint4 (&x)[MT][2]) {
        const bool there = piece < pieces && piece * 32 + t * 8 < a.len;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[m][h] = there ? *reinterpret_cast<const uint4*>(in[m][h] + piece * 32) : zero;
    };
    const bool rows_here = rg * MT * 16 < n;
    if (rows_here) {
        const int first = 2 * (block * KS + ks);
        uint4 x[2][MT][2];
        load_in(first, x[0]);
        load_in(first + 1, x[1]);
        int taken = 0;
        for (int p0 = first; p0 < pieces; p0 += next) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int k0 = (p0 + half) * 32;
                wm::Rows16<T> q[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) q[m].set(x[half][m][0], x[half][m][1]);
                if (k0 < a.len) {
                    if constexpr (!kBack) {
                        const T* p = P + (size_t)quad * a.len + k0 + t * 8;
                        const bool there = k0 + t * 8 < a.len;
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            wm::Rows8<T> w;
                            w.set(there && j * 8 + quad < a.r ? *reinterpret_cast<const uint4*>(p + (size_t)j * 8 * a.len) : zero);
#pragma unroll
                            for (int m = 0; m < MT; ++m) wm::multiply<T>(d[m][j], q[m], w);
                        }
                    } else {
                        // rows k0 + 8 (i / 8) + (i / 4) % 2 + 2 g of P: transposed, the pairs of k that a lane of `in` has in its words
                        const int row = k0 + 8 * (quad >> 1) + (quad & 1);
                        const bool there = row < a.len;
#pragma unroll
                        for (int v = 0; v < NT / kQ; ++v) {
                            uint32_t w[4][kQ];
#pragma unroll
                            for (int g = 0; g < 4; ++g) {
                                const int at = RT == 16 ? t * 4 : v * 32 + t * 8;
                                const T* p = P + (size_t)(row + 2 * g) * a.r + at;
                                if constexpr (kQ == 2) {
                                    const uint2 l = there && at < a.r ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
                                    w[g][0] = l.x, w[g][1] = l.y;
                                } else {
                                    const uint4 l = there && at < a.r ? *reinterpret_cast<const uint4*>(p) : zero;
                                    w[g][0] = l.x, w[g][1] = l.y, w[g][2] = l.z, w[g][3] = l.w;
                                }
                            }
#pragma unroll
                            for (int k = 0; k < kQ; ++k) {
                                const uint32_t b0 = transposed(w[0][k]), b1 = transposed(w[1][k]), b2 = transposed(w[2][k]), b3 = transposed(w[3][k]);
#pragma unroll
                                for (int m = 0; m < MT; ++m) {
                                    wm::mma16<T>(d[m][v * kQ + k], q[m].u.x, q[m].v.x, q[m].u.y, q[m].v.y, b0, b1);
                                    wm::mma16<T>(d[m][v * kQ + k], q[m].u.z, q[m].v.z, q[m].u.w, q[m].v.w, b2, b3);
                                }
                            }
                        }
                    }
                }
                load_in(p0 + next + half, x[half]);
            }
            if (++taken % kWhole == 0) put();
        }
    }
    put();  // the warps' sums meet
    __syncthreads();
    for (int i = threadIdx.x; i < n * RT; i += 256) {
        float* at = part + i / RT * S::kPitch + i % RT;
        float v = *at;
#pragma unroll
        for (int k = 1; k < KS; ++k) v += at[k * TR * S::kPitch];
        *at = kBack ? v * scale : v;
    }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    // a warp takes a row: its sum over the cluster, and what of it the second product takes
    for (int row = warp; row < n; row += kWarps) {
        constexpr int V = RT >= 32 ? RT / 32 : 1;
        float v[V], most = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = i * 32 + lane;
            v[i] = 0.f;
            if (j < RT) {
                float* at = part + row * S::kPitch + j;
                if (blocks == 1) v[i] = *at;
                else
                    for (int k = 0; k < blocks; ++k) v[i] += *cluster.map_shared_rank(at, k);
                if (a.u && block == 0 && j < a.r) a.u[(long long)(tile.begin + row) * a.r + j] = v[i];
            }
            most = fmaxf(most, finite_size(v[i]));
        }
        float shrink = 1.f;
        if constexpr (kShrink) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            shrink = top_of(most);
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * 32 + lane < RT) ub[row][i * 32 + lane] = Elem<T>::from_f(v[i] * shrink);
        if (lane == 0) grow[row] = (kBack ? 1.f : scale) / shrink;
    }
    if (blocks > 1) cluster.sync();  // (no block leaves while its sums may still be read)
    else __syncthreads();
    if (!rows_here) return;

    // ------------------------------------------------ second product
    constexpr int KB = RT / 16;  // steps of 16 along the rank
    uint32_t f[MT][KB][4];
    float up[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = (rg * MT + m) * 16 + h * 8 + quad;
            up[m][h] = row < n ? grow[row] : 0.f;
#pragma unroll
            for (int s = 0; s < KB; ++s) {
                // the elements that a lane has of Q in the same words
                const int c0 = kBack ? s * 16 + t * 2 : RT == 16 ? t * 4 : s / 2 * 32 + t * 8 + s % 2 * 4, c1 = kBack ? c0 + 8 : c0 + 2;
                f[m][s][h] = row < n ? *reinterpret_cast<const uint32_t*>(&ub[row][c0]) : 0u;
                f[m][s][2 + h] = row < n ? *reinterpret_cast<const uint32_t*>(&ub[row][c1]) : 0u;
            }
        }
    const T* base = static_cast<const T*>(a.base);
    T* out = static_cast<T*>(a.out);
    for (int c0 = (block * KS + ks) * 32; c0 < a.cols; c0 += KS * blocks * 32) {
        const int mine = c0 + t * 8;  // this lane's columns of the result
        const bool there = mine < a.cols;
        uint4 before[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = (rg * MT + m) * 16 + h * 8 + quad;
                before[m][h] = base && there && row < n ? *reinterpret_cast<const uint4*>(base + (long long)(tile.begin + row) * a.ldb + mine) : zero;
            }
        float s[MT][4][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][j][i] = 0.f;
        if constexpr (!kBack) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int col = c0 + 8 * (quad >> 1) + 2 * j + (quad & 1);
                const T* q = Q + (size_t)col * a.r;
#pragma unroll
                for (int b = 0; b < (RT + 31) / 32; ++b) {
                    uint32_t w[4];
                    if constexpr (RT == 16) {
                        const uint2 l = col < a.cols && t * 4 < a.r ? *reinterpret_cast<const uint2*>(q + t * 4) : make_uint2(0, 0);
                        w[0] = l.x, w[1] = l.y;
                    } else {
                        const uint4 l = col < a.cols && b * 32 + t * 8 < a.r ? *reinterpret_cast<const uint4*>(q + b * 32 + t * 8) : zero;
                        w[0] = l.x, w[1] = l.y, w[2] = l.z, w[3] = l.w;
                    }
#pragma unroll
                    for (int i = 0; i < (RT == 16 ? 1 : 2); ++i)
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            const uint32_t* g = f[m][RT == 16 ? 0 : 2 * b + i];
                            wm::mma16<T>(s[m][j], g[0], g[1], g[2], g[3], w[2 * i], w[2 * i + 1]);
                        }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                uint4 l[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = k * 16 + h * 8 + quad;
                    l[h] = there && row < a.r ? *reinterpret_cast<const uint4*>(Q + (size_t)row * a.cols + mine) : zero;
                }
                const uint32_t w[2][4] = {{l[0].x, l[0].y, l[0].z, l[0].w}, {l[1].x, l[1].y, l[1].z, l[1].w}};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t b0 = transposed(w[0][j]), b1 = transposed(w[1][j]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) wm::mma16<T>(s[m][j], f[m][k][0], f[m][k][1], f[m][k][2], f[m][k][3], b0, b1);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = (rg * MT + m) * 16 + h * 8 + quad;
                if (!there || row >= n) continue;
                const uint32_t o[4] = {before[m][h].x, before[m][h].y, before[m][h].z, before[m][h].w};
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 b = Pack2<T>::to_f2(*reinterpret_cast<const typename Pack2<T>::type*>(&o[j]));
                    r[j] = pack<T>(fmaf(up[m][h], s[m][j][2 * h], b.x), fmaf(up[m][h], s[m][j][2 * h + 1], b.y));
                }
                *reinterpret_cast<uint4*>(out + (long long)(tile.begin + row) * a.ldo + mine) = make_uint4(r[0], r[1], r[2], r[3]);
            }
    }
}

// ---------------------------------------------------------------- many rows
// The same for tiles enough to fill the GPU: a block takes 64 rows alone.  What it multiplies comes through a ring of kStages
// steps of 64 elements in shared memory, 16-byte copies that run ahead from the first product into the second, and reaches the tensor cores by
// ldmatrix (transposed where the summed direction is not the contiguous one).  Rows of 128, 64 or 32 bytes with their 16-byte pieces
// exchanged, so that eight of them meet no bank twice.
constexpr int kPipeRows = 64, kPipeStep = 64, kPipeThreads = 256, kStages = 4;

template <int kRowBytes>
__device__ __forceinline__ int piece_at(int row, int piece) {
    if constexpr (kRowBytes == 128) return row * 128 + (piece ^ (row & 7)) * 16;
    if constexpr (kRowBytes == 64) return row * 64 + (piece ^ (row >> 1 & 3)) * 16;
    return row * 32 + (piece ^ (row >> 2 & 1)) * 16;
}
__device__ __forceinline__ void copy_or_zero(uint32_t to, const void* from, bool there) {  // (nothing is read where it is not there)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
template <bool kTrans>
__device__ __forceinline__ void load_blocks(uint32_t (&f)[4], uint32_t at) {  // four 8 x 8 blocks, a row's address a lane
    if constexpr (kTrans)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(at) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(at) : "memory");
}

template <int RT>
struct PipeShape {
    static constexpr int kRowTile = kPipeRows * kPipeStep * 2, kOther = RT * kPipeStep * 2, kStage = kRowTile + kOther;
    static constexpr int kSumPitch = RT + 4, kFactorPitch = RT + 8;
    static constexpr int kFactors = kStages * kStage, kSums = kFactors + kPipeRows * kFactorPitch * 2;
    static constexpr int kBytes = kSums + kPipeRows * kSumPitch * 4;
};

template <typename T, bool kBack, int RT>
__global__ void __launch_bounds__(kPipeThreads, 2) rows_pipe_kernel(Args a) {
    using S = PipeShape<RT>;
    constexpr int MT = RT == 64 ? 2 : 1, RG = 4 / MT;        // of 16 rows: a warp's, and groups of warps
    constexpr int NT1 = RT / 8 / MT, KB = RT / 16;           // first product: the ranks of a warp by eight; two warps share the elements of a step
    constexpr int CG = kWarps / RG, NT2 = 8 / CG;            // second: the warps of a group share the columns
    constexpr bool kShrink = std::is_same<T, __half>::value;
    extern __shared__ __align__(128) char memory[];
    __shared__ float grow[kPipeRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, t = lane & 3, rg = warp % RG, group = warp / RG;
    const int half = group % MT, kpart = group / MT;
    pdl_wait();
    pdl_trigger();
    Tile tile;
    if (!find_tile<kPipeRows>(a, blockIdx.x, &tile)) return;
    const int n = tile.end - tile.begin;
    if (tile.adapter < 0) {
        copy_base<T, 8>(a, tile, 0, a.cols);
        if (a.u)
            for (int i = threadIdx.x; i < n * a.r; i += kPipeThreads) a.u[(long long)tile.begin * a.r + i] = 0.f;
        return;
    }
    const float scale = a.scale ? a.scale[tile.adapter] : 1.f;
    const T* P = static_cast<const T*>(a.p) + (size_t)tile.adapter * a.r * a.len;
    const T* Q = static_cast<const T*>(a.q) + (size_t)tile.adapter * a.r * a.cols;
    const T* in = static_cast<const T*>(a.in) + (long long)tile.begin * a.ldi;
    const T* base = a.base ? static_cast<const T*>(a.base) + (long long)tile.begin * a.ldb : nullptr;
    T* out = static_cast<T*>(a.out) + (long long)tile.begin * a.ldo;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(memory));
    const int steps1 = (a.len + kPipeStep - 1) / kPipeStep, steps = steps1 + (a.cols + kPipeStep - 1) / kPipeStep;

    // A thread's copies: a piece of 16 bytes of every so many rows, at addresses that only move on from step to step.
    struct Lane {
        const T* from;    // of the first of its rows
        long long rows;   // elements from one of its rows to the next
        uint32_t to;      // in the stage
        int first;        // row
    };
    constexpr int kRows = kPipeThreads / 8;                      // of 128 bytes at a time
    const int row8 = threadIdx.x / 8, piece = threadIdx.x % 8;
    constexpr int kTallPieces = RT / 8, kTallRows = kPipeThreads / kTallPieces;
    const int tall_row = threadIdx.x / kTallPieces, tall_piece = threadIdx.x % kTallPieces;
    auto lane_of = [&](const T* m, long long ld) { return Lane{m + row8 * ld + piece * 8, kRows * ld, (uint32_t)piece_at<128>(row8, piece), row8}; };
    // rows: of a tile, or [RT] rows of 64 elements of a matrix [r][width].  What is not there is zeros; rows that are not are left out
    // where nobody takes their sums (kZeros false).
    auto copy_rows = [&](uint32_t to, Lane& l, int rows, int width, int k0, auto all, auto zeros) {
        constexpr int kAll = decltype(all)::value;
        const bool whole = k0 + kPipeStep <= width;
        const T* from = l.from;
#pragma unroll
        for (int i = 0; i < kAll; i += kRows, from += l.rows) {
            const bool there = l.first + i < rows;
            if (whole && there) copy_16(to + l.to + i * 128, from);
            else if (there || (decltype(zeros)::value && l.first + i < kAll)) {
                const bool in_row = there && k0 + piece * 8 < width;
                copy_or_zero(to + l.to + i * 128, in_row ? from : static_cast<const T*>(a.p), in_row);
            }
        }
        l.from += kPipeStep;
    };
    // 64 rows of a matrix [width][r]
    auto tall_of = [&](const T* m) { return Lane{m + (long long)tall_row * a.r + tall_piece * 8, (long long)kTallRows * a.r, (uint32_t)piece_at<RT * 2>(tall_row, tall_piece), tall_row}; };
    auto copy_tall = [&](uint32_t to, Lane& l, int width, int k0) {
        const T* from = l.from;
#pragma unroll
        for (int i = 0; i < kPipeStep; i += kTallRows, from += l.rows) {
            const bool there = tall_piece * 8 < a.r && k0 + l.first + i < width;
            if (l.first + i < kPipeStep) copy_or_zero(to + l.to + i * RT * 2, there ? from : static_cast<const T*>(a.p), there);
        }
        l.from += (long long)kPipeStep * a.r;
    };
    using std::integral_constant;
    Lane rows_at = lane_of(in, a.ldi), other = kBack ? tall_of(P) : lane_of(P, a.len);
    uint32_t fill = ring, take = ring;  // stages that are copied to and read next
    int copied = 0;
    auto copy = [&] {
        if (copied < steps) {
            if (copied == steps1) {
                if (base) rows_at = lane_of(base, a.ldb);
                other = kBack ? lane_of(Q, a.cols) : tall_of(Q);
            }
            const bool second = copied >= steps1;
            const int width = second ? a.cols : a.len, k0 = (copied - (second ? steps1 : 0)) * kPipeStep;
            if (!second || base) copy_rows(fill, rows_at, n, width, k0, integral_constant<int, kPipeRows>(), std::false_type());
            if (kBack != second) copy_tall(fill + S::kRowTile, other, width, k0);
            else copy_rows(fill + S::kRowTile, other, a.r, width, k0, integral_constant<int, RT>(), std::true_type());
            ++copied;
            fill = fill == ring + (kStages - 1) * S::kStage ? ring : fill + S::kStage;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto next = [&] {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();
        copy();
        const uint32_t from = take;
        take = take == ring + (kStages - 1) * S::kStage ? ring : take + S::kStage;
        return from;
    };
    for (int i = 0; i < kStages - 1; ++i) copy();

    // ------------------------------------------------ first product
    const int low = lane & 7, mid = lane >> 3 & 1, high = lane >> 4;  // which row of which 8 x 8 block this lane's address is of
    float d[MT][NT1][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT1; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[m][j][i] = 0.f;
    float whole[MT][NT1][4] = {};  // as above: what the accumulators have had for kWhole steps is added up in registers
    constexpr int kWhole = 4;
    auto add_up = [&] {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT1; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) whole[m][j][i] += d[m][j][i], d[m][j][i] = 0.f;
    };
    for (int step = 0; step < steps1; ++step) {
        if (step % kWhole == 0) add_up();
        const uint32_t from = next();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = 2 * kpart + i;
            uint32_t f[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) load_blocks<false>(f[m], from + piece_at<128>((rg * MT + m) * 16 + low + mid * 8, 2 * k + high));
#pragma unroll
            for (int j = 0; j < NT1; j += 2) {
                uint32_t b[4];
                const int j0 = half * NT1 + j;
                if constexpr (kBack) load_blocks<true>(b, from + S::kRowTile + piece_at<RT * 2>(16 * k + low + mid * 8, j0 + high));
                else load_blocks<false>(b, from + S::kRowTile + piece_at<128>(j0 * 8 + low + high * 8, 2 * k + mid));
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    wm::mma16<T>(d[m][j], f[m][0], f[m][1], f[m][2], f[m][3], b[0], b[1]);
                    wm::mma16<T>(d[m][j + 1], f[m][0], f[m][1], f[m][2], f[m][3], b[2], b[3]);
                }
            }
        }
    }
    add_up();
    float* sums = reinterpret_cast<float*>(memory + S::kSums);
    T* factors = reinterpret_cast<T*>(memory + S::kFactors);
    for (int part = 0; part < 2; ++part) {  // one half of the sums, and the other onto it
        if (kpart == part)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NT1; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float2* to = reinterpret_cast<float2*>(sums + ((rg * MT + m) * 16 + h * 8 + quad) * S::kSumPitch + (half * NT1 + j) * 8 + t * 2);
                        const float2 before = part ? *to : make_float2(0.f, 0.f);
                        *to = make_float2(before.x + whole[m][j][2 * h], before.y + whole[m][j][2 * h + 1]);
                    }
        __syncthreads();
    }
    // a warp takes a row: u, and what of it the second product takes
    for (int row = warp; row < kPipeRows; row += kPipeThreads / 32) {
        constexpr int V = RT >= 32 ? RT / 32 : 1;
        float v[V], most = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = i * 32 + lane;
            v[i] = j < RT && row < n ? sums[row * S::kSumPitch + j] * (kBack ? scale : 1.f) : 0.f;
            if (a.u && row < n && j < a.r) a.u[(long long)(tile.begin + row) * a.r + j] = v[i];
            most = fmaxf(most, finite_size(v[i]));
        }
        float shrink = 1.f;
        if constexpr (kShrink) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            shrink = top_of(most);
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * 32 + lane < RT) factors[row * S::kFactorPitch + i * 32 + lane] = Elem<T>::from_f(v[i] * shrink);
        if (lane == 0) grow[row] = (kBack ? 1.f : scale) / shrink;
    }
    __syncthreads();

    // ------------------------------------------------ second product
    uint32_t f[MT][KB][4];
    float up[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = (rg * MT + m) * 16;
        up[m][0] = grow[row + quad], up[m][1] = grow[row + 8 + quad];
#pragma unroll
        for (int k = 0; k < KB; ++k)
            load_blocks<false>(f[m][k], ring + S::kFactors + ((row + low + mid * 8) * S::kFactorPitch + k * 16 + high * 8) * 2);
    }
    for (int step = steps1; step < steps; ++step) {
        const uint32_t from = next();
        const int c0 = (step - steps1) * kPipeStep;
        float s[MT][NT2][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][j][i] = 0.f;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int j = 0; j < NT2; j += 2) {
                uint32_t b[4];
                const int j0 = group * NT2 + j;
                if constexpr (kBack) load_blocks<true>(b, from + S::kRowTile + piece_at<128>(16 * k + low + mid * 8, j0 + high));
                else load_blocks<false>(b, from + S::kRowTile + piece_at<RT * 2>(j0 * 8 + low + high * 8, 2 * k + mid));
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    wm::mma16<T>(s[m][j], f[m][k][0], f[m][k][1], f[m][k][2], f[m][k][3], b[0], b[1]);
                    wm::mma16<T>(s[m][j + 1], f[m][k][0], f[m][k][1], f[m][k][2], f[m][k][3], b[2], b[3]);
                }
            }
        // onto base, in its place in the ring, whence the warp stores its rows 16 bytes at a time
        char* tile_at = memory + (from - ring);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t* at = reinterpret_cast<uint32_t*>(tile_at + piece_at<128>((rg * MT + m) * 16 + h * 8 + quad, group * NT2 + j) + t * 4);
                    const float2 b = base ? Pack2<T>::to_f2(*reinterpret_cast<const typename Pack2<T>::type*>(at)) : make_float2(0.f, 0.f);
                    *at = pack<T>(fmaf(up[m][h], s[m][j][2 * h], b.x), fmaf(up[m][h], s[m][j][2 * h + 1], b.y));
                }
        __syncwarp();
#pragma unroll
        for (int i = lane; i < 16 * MT * NT2; i += 32) {
            const int row = rg * MT * 16 + i / NT2, piece = group * NT2 + i % NT2;
            if (row < n && c0 + piece * 8 < a.cols)
                *reinterpret_cast<uint4*>(out + row * a.ldo + c0 + piece * 8) = *reinterpret_cast<const uint4*>(tile_at + piece_at<128>(row, piece));
        }
    }
}

// ---------------------------------------------------------------- gradients of the adapters
// Up to so many rows results in 16 bits are made of both parts of u and v as well: a rank of a few rows is a few values, whose rounding shows in a whole row of
// dA (column of dB) and is not evened out (four rows of one adapter, rank 32: 2-norm 0.0025 of dB, now 0.0017).  N = K = 4096, rank 64: 256 rows 25.9 us instead
// of 24.9, 512 rows 35.8 instead of 33.5, 2048 rows 53 instead of 47.
constexpr int kBothParts = 512;
constexpr int kGradRows = 32, kGradColumns = 256, kGradStages = 4;

template <typename T, int RT>
struct GradShape {
    static constexpr int kRowPitch = kGradColumns * 2 + 16;        // bytes of a row of the other factor
    static constexpr int kPitch = RT * 4 + 16;                     // bytes of a row of c: values, then both parts of every eight in their 32 bytes
    static constexpr int kRows = kGradRows * kRowPitch, kStage = kRows + kGradRows * kPitch;
    static constexpr int kSums = RT * (kGradColumns + 1) * 4, kRing = kGradStages * kStage;
    static constexpr int kBytes = kSums > kRing ? kSums : kRing;
};

// RT: columns of c (u or v) from blockIdx.z * RT on.  The cluster's blocks take kGradRows rows of a request in turn; both factors come through a
// ring in shared memory, c a step before it is needed, when it is rounded to a factor of the products.
//
// The matrix unit cuts its running sums off instead of rounding them (expert_tc.cuh), and u and v have 32 bits: 16-bit results' own rounding covers what is
// lost of either from some rows on (kParts, kBothParts).  Where results are floats (kWide), every 16 rows are a sum of their own, which is added up in registers (there is no room for a second
// set of sums that would be read back less often), of both parts of c.  16384 rows, N = K = 4096, rank 64, bf16: 200 us instead of 149; the sums alone 166, and
// 16-bit results of both parts 197.
template <typename T, int RT, bool kWide, int kParts>
__global__ void __launch_bounds__(256, 2) grads_mma_kernel(Grads first_of_two, Grads second_of_two) {
    namespace cg = cooperative_groups;
    using S = GradShape<T, RT>;
    constexpr int MT = RT / 16;
    constexpr bool kShrink = std::is_same<T, __half>::value;
    extern __shared__ __align__(128) char memory[];
    constexpr int kRanks = kShrink ? RT : 2;
    constexpr float kNoneYet = 0x1p127f;
    __shared__ __align__(16) float largest[kWarps][kRanks], shrink[kRanks], change[kRanks];
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, t = lane & 3;
    const int strip = blockIdx.x / blocks;
    const bool second = strip >= first_of_two.strips;
    const Grads a = second ? second_of_two : first_of_two;
    const int l = blockIdx.y, j0 = blockIdx.z * RT, c0 = (strip - (second ? first_of_two.strips : 0)) * kGradColumns;
    pdl_wait();
    pdl_trigger();
    float s[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][j][i] = 0.f;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(memory));

    // This block's share of the adapter's rows, kGradRows of a request at a time.
    struct {
        int i0, row, end, count;
        unsigned of;
    } walk{-32, 0, 0, 0, 0};
    auto advance = [&](int* row0) {  // rows of the next step, 0 at the end; uniform over the block
        for (;;) {
            while (walk.row < walk.end) {
                const int row = walk.row, n = min(kGradRows, walk.end - row);
                walk.row += kGradRows;
                if (walk.count++ % blocks != block) continue;
                *row0 = row;
                return n;
            }
            while (!walk.of) {
                walk.i0 += 32;
                if (walk.i0 >= a.R) {
                    walk.i0 = a.R;  // (stays at the end)
                    return 0;
                }
                const int i = walk.i0 + lane;
                walk.of = __ballot_sync(0xffffffffu, i < a.R && a.adapter[i] == l);
            }
            const Group g = group_rows(a.offsets, walk.i0 + __ffs(walk.of) - 1, a.rows);
            walk.of &= walk.of - 1;
            walk.row = g.begin;
            walk.end = g.end;
        }
    };
    // a thread's copies: 16 bytes of every eighth row
    const int my_row = threadIdx.x / 32, my_col = threadIdx.x % 32 * 8;
    const bool my_column = c0 + my_col < a.cols;
    const T* const in = static_cast<const T*>(a.in) + my_row * a.ldi + c0 + my_col;
    const uint32_t ring_end = ring + kGradStages * S::kStage;
    uint32_t fill = ring + my_row * S::kRowPitch + my_col * 2, take = ring;
    // 8 bytes of c, of every so-manyth row
    constexpr int kMine = kGradRows * RT / 256 / 2, kEvery = 512 / RT;
    const int c_row = (int)threadIdx.x * 2 / RT, c_col = (int)threadIdx.x * 2 % RT;
    const bool c_column = j0 + c_col < a.r;
    const float* const c_in = a.c + (long long)c_row * a.r + j0 + c_col;
    const int c_at = S::kRows + c_row * S::kPitch + c_col * 4;
    uint32_t fill_c = ring + c_at;
    auto copy = [&](int row0, int n) {
        const T* from = in + row0 * a.ldi;
#pragma unroll
        for (int i = 0; i < kGradRows; i += 8, from += 8 * a.ldi) {
            const bool there = my_column && my_row + i < n;  // (rows of others are zeros here, not multiplied by zero)
            copy_or_zero(fill + i * S::kRowPitch, there ? from : static_cast<const T*>(a.in), there);
        }
        const float* c_from = c_in + (long long)row0 * a.r;
#pragma unroll
        for (int k = 0; k < kMine; ++k, c_from += (long long)kEvery * a.r) {
            const bool there = c_column && c_row + k * kEvery < n;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(fill_c + k * kEvery * S::kPitch), "l"(there ? c_from : a.c), "r"(there ? 8 : 0) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        fill += S::kStage;
        fill_c += S::kStage;
        if (fill >= ring_end) fill -= kGradStages * S::kStage, fill_c -= kGradStages * S::kStage;
    };
    // shrink: what a rank's values of c are multiplied with (a power of two; its sums then have it too).  It goes by the rank's finite values alone: what
    // is not a number stays so, in that rank's sums, and another rank's size costs this one no bits.
    if (kShrink && threadIdx.x < RT) shrink[threadIdx.x] = kNoneYet;
    // The factors of a step whose copies are there, in the values' place: both parts of each.
    auto round = [&](char* stage) {
        if constexpr (kShrink) {
            float2 v[kMine], most = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kMine; ++k) {
                v[k] = *reinterpret_cast<const float2*>(stage + c_at + k * kEvery * S::kPitch);
                most = make_float2(fmaxf(most.x, finite_size(v[k].x)), fmaxf(most.y, finite_size(v[k].y)));
            }
#pragma unroll
            for (int o = RT / 2; o < 32; o *= 2)  // lanes with the same columns
                most = make_float2(fmaxf(most.x, __shfl_xor_sync(0xffffffffu, most.x, o)), fmaxf(most.y, __shfl_xor_sync(0xffffffffu, most.y, o)));
            if (lane < RT / 2) *reinterpret_cast<float2*>(&largest[warp][c_col]) = most;
            __syncthreads();
            bool larger = false;
            if (threadIdx.x < RT) {
                float m = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, largest[w][threadIdx.x]);
                const float want = top_of(m), now = shrink[threadIdx.x];
                larger = m > 0.f && want < now;
                // (not zero: an infinity that is there already stays one)
                change[threadIdx.x] = larger ? fmaxf(want / now, 0x1p-126f) : 1.f;
                if (larger) shrink[threadIdx.x] = want;
            }
            if (__syncthreads_or(larger)) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float f = change[m * 16 + q / 2 * 8 + quad];
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[m][j][q] *= f;
                    }
            }
            if constexpr (kParts == 1) {  // (all have read theirs)
                const float2 by = *reinterpret_cast<const float2*>(shrink + c_col);
                char* const to = stage + S::kRows + c_row * S::kPitch + c_col / 8 * 32 + c_col % 8 * 2;
#pragma unroll
                for (int k = 0; k < kMine; ++k) *reinterpret_cast<uint32_t*>(to + k * kEvery * S::kPitch) = pack<T>(v[k].x * by.x, v[k].y * by.y);
                return;
            }
        }
        if (threadIdx.x < 4 * RT) {  // eight values a thread
            const int row = (int)threadIdx.x / (RT / 8), eight = (int)threadIdx.x % (RT / 8);
            char* const c = stage + S::kRows + row * S::kPitch + eight * 32;
            float v[8], by[8];
            uint32_t part[2][4];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(c + i * 4);
                if constexpr (kShrink) *reinterpret_cast<float4*>(by + i) = *reinterpret_cast<const float4*>(shrink + eight * 8 + i);
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float x = kShrink ? v[i] * by[i] : v[i], y = kShrink ? v[i + 1] * by[i + 1] : v[i + 1];
                part[0][i / 2] = pack<T>(x, y);
                if (kParts == 1) continue;
                const float2 first = Pack2<T>::to_f2(*reinterpret_cast<const typename Pack2<T>::type*>(&part[0][i / 2]));
                part[1][i / 2] = pack<T>(rest_of(x, first.x), rest_of(y, first.y));
            }
#pragma unroll
            for (int p = 0; p < kParts; ++p)
                *reinterpret_cast<uint4*>(c + p * 16) = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
        }
    };

    // rows of this step and of those that are on their way
    int n[kGradStages];
    auto one_more = [&](int i) {
        int row0 = 0;
        n[i] = advance(&row0);
        copy(row0, n[i]);
    };
#pragma unroll
    for (int i = 0; i < kGradStages - 1; ++i) one_more(i);
    asm volatile("cp.async.wait_group %0;" ::"n"(kGradStages - 2) : "memory");
    __syncthreads();
    if (n[0] > 0) round(memory);
    const int low = lane & 7, mid = lane >> 3 & 1, high = lane >> 4;
    while (n[0] > 0) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kGradStages - 3) : "memory");
        __syncthreads();
        one_more(kGradStages - 1);
        const uint32_t from = take;
        take = take + S::kStage == ring_end ? ring : take + S::kStage;
        // 8 x 8 blocks: of c rows lane % 8 (+ 8 for lanes 16 on) and columns + 8 for every second eight lanes; of the other the other way round
        auto columns = [&](int k, uint32_t (&b)[2][4]) {
#pragma unroll
            for (int j = 0; j < 2; ++j) load_blocks<true>(b[j], from + (k * 16 + low + mid * 8) * S::kRowPitch + (warp * 32 + j * 16 + high * 8) * 2);
        };
        auto multiply = [&](int k, int m, const uint32_t (&b)[2][4], float (&d)[4][4]) {
#pragma unroll
            for (int p = kParts - 1; p >= 0; --p) {
                uint32_t f[4];
                load_blocks<true>(f, from + S::kRows + (k * 16 + low + high * 8) * S::kPitch + ((m * 2 + mid) * 2 + p) * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) wm::mma16<T>(d[j], f[0], f[1], f[2], f[3], b[j / 2][j % 2 * 2], b[j / 2][j % 2 * 2 + 1]);
            }
        };
        if constexpr (kWide) {
#pragma unroll
            for (int k = 0; k < kGradRows / 16; ++k) {
                if (k * 16 >= n[0]) break;
                uint32_t b[2][4];
                columns(k, b);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float d[4][4] = {};
                    multiply(k, m, b, d);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int q = 0; q < 4; q += 2) {
                            const float2 v = split(add2(pair(s[m][j][q], s[m][j][q + 1]), pair(d[j][q], d[j][q + 1])));
                            s[m][j][q] = v.x, s[m][j][q + 1] = v.y;
                        }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < kGradRows / 16; ++k) {
                if (k * 16 >= n[0]) break;
                uint32_t b[2][4];
                columns(k, b);
#pragma unroll
                for (int m = 0; m < MT; ++m) multiply(k, m, b, s[m]);
            }
        }
#pragma unroll
        for (int i = 0; i < kGradStages - 1; ++i) n[i] = n[i + 1];
        if (n[0] > 0) round(memory + (take - ring));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // the cluster's sums meet; the blocks share what is then to be stored
    float* sums = reinterpret_cast<float*>(memory);  // [RT][columns + 1]
    constexpr int kPitch = kGradColumns + 1;
    const float scale = a.scale ? a.scale[l] : 1.f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int rank = m * 16 + h * 8 + quad;
            const float grow = kShrink ? 1.f / shrink[rank] : 1.f;  // (exact; scale may not be)
            float* to = sums + rank * kPitch + warp * 32 + t * 2;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[8 * j] = s[m][j][2 * h] * grow * scale, to[8 * j + 1] = s[m][j][2 * h + 1] * grow * scale;
        }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    // (neighbours in a row of the sums are read together from the other blocks; dB's results change places in this block's own memory)
    const int width = min(RT, a.r - j0), share = kGradColumns / blocks, first = block * share, columns = min(share, a.cols - c0 - first);
    T* const out = static_cast<T*>(a.out);
    float* const wide_out = static_cast<float*>(a.out);
    auto store = [&](int j, int col, float v) {
        const size_t to = a.db ? ((size_t)l * a.cols + c0 + first + col) * a.r + j0 + j : ((size_t)l * a.r + j0 + j) * a.cols + c0 + first + col;
        if constexpr (kWide) wide_out[to] = v;
        else out[to] = Elem<T>::from_f(v);
    };
    for (int i = threadIdx.x; i < width * share; i += 256) {
        const int j = i / share, col = i % share;
        float* at = sums + j * kPitch + first + col;
        float v = 0.f;
        if (blocks == 1) v = *at;
        else
            for (int k = 0; k < blocks; ++k) v += *cluster.map_shared_rank(at, k);
        if (a.db) *at = v;  // (nobody else reads this block's share of its own sums but itself)
        else if (col < columns) store(j, col, v);
    }
    if (a.db) {
        __syncthreads();
        for (int i = threadIdx.x; i < width * columns; i += 256) store(i % width, i / width, sums[i % width * kPitch + first + i / width]);
    }
    if (blocks > 1) cluster.sync();
}

}  // namespace adapters
}  // namespace kleos
