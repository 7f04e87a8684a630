// The adapters' products (adapters.cuh) where 16-bit rows begin on 16-byte boundaries and the rank is a multiple of 8: on the tensor
// cores, straight from memory (warp_mma.cuh).
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
// u and v are factors of the second products as values of the element type: rounded once, as a projection's own input would be (both parts of
// them would double those products' time on the tensor cores and halve the rounding error of a result).  fp16 has too little range for that:
// a row is divided by a power of two first (in the gradients: all rows, by the largest so far).
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

// The power of two that brings a largest value m to [1, 2); 1 for zero, infinities and NaN.
__device__ __forceinline__ float shrink_of(float m) {
    const uint32_t e = __float_as_uint(m) >> 23 & 255;
    return e == 0 || e >= 254 ? 1.f : __uint_as_float((254 - e) << 23);
}

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
    extern __shared__ __align__(16) float part[];       // [KS][TR][pitch]
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
        const int share = (a.cols + blocks - 1) / blocks, c0 = min(a.cols, block * share);
        copy_base<T>(a, tile, c0, min(a.cols, c0 + share));
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
        }
    }
    // the warps' sums meet: columns of tile j in their own order (backward: as they were dealt)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int col = !kBack ? j * 8 + t * 2 : RT == 16 ? t * 4 + j * 2 : j / 4 * 32 + t * 8 + j % 4 * 2;
            float* to = part + (ks * TR + (rg * MT + m) * 16 + quad) * S::kPitch + col;
            *reinterpret_cast<float2*>(to) = make_float2(d[m][j][0], d[m][j][1]);
            *reinterpret_cast<float2*>(to + 8 * S::kPitch) = make_float2(d[m][j][2], d[m][j][3]);
        }
    __syncthreads();
    if (KS > 1 || kBack) {
        for (int i = threadIdx.x; i < n * RT; i += 256) {
            float* at = part + i / RT * S::kPitch + i % RT;
            float v = *at;
#pragma unroll
            for (int k = 1; k < KS; ++k) v += at[k * TR * S::kPitch];
            *at = kBack ? v * scale : v;
        }
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
            most = fmaxf(most, fabsf(v[i]));
        }
        float shrink = 1.f;
        if constexpr (kShrink) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            shrink = shrink_of(most);
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

// ---------------------------------------------------------------- gradients of the adapters
constexpr int kGradRows = 64, kGradColumns = 256;

template <typename T, int RT>
struct GradShape {
    static constexpr int kPitch = RT + 8;                          // elements of a row of c
    static constexpr int kSums = RT * (kGradColumns + 4) * 4;
    static constexpr int kBytes = kSums > 2 * kGradRows * kPitch * 2 ? kSums : 2 * kGradRows * kPitch * 2;
};

// RT: columns of c (u or v) from blockIdx.z * RT on.  The cluster's blocks take 64 rows of a request in turn.
template <typename T, bool kDb, int RT>
__global__ void __launch_bounds__(256, RT == 64 ? 1 : 2) grads_mma_kernel(Grads a) {
    namespace cg = cooperative_groups;
    using S = GradShape<T, RT>;
    constexpr int MT = RT / 16;
    constexpr bool kShrink = std::is_same<T, __half>::value;
    extern __shared__ __align__(16) char memory[];
    __shared__ float largest[kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, t = lane & 3;
    const int l = blockIdx.y, j0 = blockIdx.z * RT, c0 = (int)(blockIdx.x / blocks) * kGradColumns, mine = c0 + warp * 32 + t * 8;
    pdl_wait();
    pdl_trigger();
    float s[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[m][j][i] = 0.f;
    T* c = reinterpret_cast<T*>(memory);
    float shrink = 1.f;  // what the values of c are multiplied with (a power of two; the sums then have it too)
    bool any = false;    // whether one of them was not zero
    int turn = 0, count = 0;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int i0 = 0; i0 < a.R; i0 += 32) {
        const int i = i0 + lane;
        unsigned of = __ballot_sync(0xffffffffu, i < a.R && a.adapter[i] == l);
        for (; of; of &= of - 1) {
            const Group g = group_rows(a.offsets, i0 + __ffs(of) - 1, a.rows);
            for (int row0 = g.begin; row0 < g.end; row0 += kGradRows) {
                if (count++ % blocks != block) continue;
                const int n = min(kGradRows, g.end - row0);
                // this step's rows of the other factor are on their way while c is made
                const T* in = static_cast<const T*>(a.in) + (long long)(row0 + quad) * a.ldi + mine;
                auto load = [&](int k, uint4 (&x)[2]) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        x[h] = mine < a.cols && k * 16 + h * 8 + quad < n ? *reinterpret_cast<const uint4*>(in + (long long)(k * 16 + h * 8) * a.ldi) : zero;
                };
                uint4 x[kGradRows / 16][2];
#pragma unroll
                for (int k = 0; k < kGradRows / 16; ++k) load(k, x[k]);
                constexpr int kMine = kGradRows * RT / 256 / 2;  // pairs of c of a thread
                float2 v[kMine];
                float most = 0.f;
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    const int at = (k * 256 + (int)threadIdx.x) * 2, row = at / RT, j = at % RT;
                    v[k] = row < n && j0 + j < a.r ? *reinterpret_cast<const float2*>(a.c + (long long)(row0 + row) * a.r + j0 + j) : make_float2(0.f, 0.f);
                    most = fmaxf(most, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));
                }
                if constexpr (kShrink) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    if (lane == 0) largest[warp] = most;
                    __syncthreads();
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, largest[w]);
                    const float want = shrink_of(most);
                    if (most > 0.f && (!any || want < shrink)) {  // (the first, or larger ones than before)
                        any = true;
                        const float by = want / shrink;
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
#pragma unroll
                                for (int q = 0; q < 4; ++q) s[m][j][q] *= by;
                        shrink = want;
                    }
                }
                T* to = c + turn * kGradRows * S::kPitch;
                turn ^= 1;
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    const int at = (k * 256 + (int)threadIdx.x) * 2;
                    *reinterpret_cast<uint32_t*>(to + at / RT * S::kPitch + at % RT) = pack<T>(v[k].x * shrink, v[k].y * shrink);
                }
                __syncthreads();  // (two buffers in turn)
#pragma unroll
                for (int k = 0; k < kGradRows / 16; ++k) {
                    if (k * 16 >= n) break;
                    const uint32_t w[2][4] = {{x[k][0].x, x[k][0].y, x[k][0].z, x[k][0].w}, {x[k][1].x, x[k][1].y, x[k][1].z, x[k][1].w}};
                    uint32_t b[4][2];
#pragma unroll
                    for (int j = 0; j < 4; ++j) b[j][0] = transposed(w[0][j]), b[j][1] = transposed(w[1][j]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        uint32_t f[4];
                        // four 8 x 8 blocks of c: rows (k) lane % 8 (+ 8 for lanes 16 on), columns (m) + 8 for every second eight lanes
                        const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to + (k * 16 + (lane & 7) + (lane >> 4) * 8) * S::kPitch + m * 16 + (lane >> 3 & 1) * 8));
                        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "r"(at) : "memory");
#pragma unroll
                        for (int j = 0; j < 4; ++j) wm::mma16<T>(s[m][j], f[0], f[1], f[2], f[3], b[j][0], b[j][1]);
                    }
                }
            }
        }
    }
    __syncthreads();
    // the cluster's sums meet; the blocks share what is then to be stored
    float* sums = reinterpret_cast<float*>(memory);  // [RT][columns + 4]
    constexpr int kPitch = kGradColumns + 4;
    const float scale = a.scale ? a.scale[l] : 1.f, grow = scale / shrink;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* to = sums + (m * 16 + h * 8 + quad) * kPitch + warp * 32 + t * 8;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[2 * j] = s[m][j][2 * h] * grow, to[2 * j + 1] = s[m][j][2 * h + 1] * grow;
        }
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    const int width = min(RT, a.r - j0), columns = min(kGradColumns, a.cols - c0);
    for (int i = block * 256 + threadIdx.x; i < width * columns; i += blocks * 256) {
        const int j = kDb ? i % width : i / columns, col = kDb ? i / width : i % columns;
        float* at = sums + j * kPitch + col;
        float v = 0.f;
        if (blocks == 1) v = *at;
        else
            for (int k = 0; k < blocks; ++k) v += *cluster.map_shared_rank(at, k);
        const size_t to = kDb ? ((size_t)l * a.cols + c0 + col) * a.r + j0 + j : ((size_t)l * a.r + j0 + j) * a.cols + c0 + col;
        if (a.wide_out) static_cast<float*>(a.out)[to] = v;
        else static_cast<T*>(a.out)[to] = Elem<T>::from_f(v);
    }
    if (blocks > 1) cluster.sync();
}

}  // namespace adapters
}  // namespace kleos
