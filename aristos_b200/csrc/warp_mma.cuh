// Products of a warp on the tensor cores straight from rows of memory (mma.sync, 16-bit elements), for operators that few rows or a short
// sum keep bound by memory: 16 rows of one operand by 8 of the other, summed over 64 bytes of each row.
//
// A lane holds, of row lane / 4 (and lane / 4 + 8), the 16 bytes that begin at 16 (lane % 4): one vector load.  Which elements
// those are does not matter to the sum as long as both operands take the same, so nothing is rearranged: the halves of the
// 16 bytes are the k pairs that the instruction wants, and 64 bytes are two instructions.
#pragma once

#include "ops_common.cuh"

namespace kleos {
namespace wm {
using namespace ops;

// acc[0..1]: row lane / 4 of a, columns (rows of b) 2 (lane % 4) and the next; acc[2..3]: row lane / 4 + 8.
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One operand's 64 bytes of rows, as the instruction takes them.
template <typename T>
struct Rows16 {  // 16 rows
    uint4 u, v;  // rows lane / 4 and lane / 4 + 8
    __device__ __forceinline__ void set(const uint4& first, const uint4& second) { u = first, v = second; }
};
template <typename T>
struct Rows8 {
    uint4 u;
    __device__ __forceinline__ void set(const uint4& q) { u = q; }
};
template <typename T>
__device__ __forceinline__ void multiply(float (&d)[4], const Rows16<T>& a, const Rows8<T>& b) {
    mma16<T>(d, a.u.x, a.v.x, a.u.y, a.v.y, b.u.x, b.u.y);
    mma16<T>(d, a.u.z, a.v.z, a.u.w, a.v.w, b.u.z, b.u.w);
}

}  // namespace wm
}  // namespace kleos
