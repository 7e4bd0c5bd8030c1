// What the kernels of attention over a paged cache share (attention_paged.hip:
// few rows of a sequence; many: attention_paged_many.hip over f16 rows,
// attention_paged_f32.hip over f32 ones).
//
// Row r of a sequence and kv head (new token r / G at position p, query head r % G):
//   s_j = (q . K[j]) / sqrt(HD)   for j <= p and, with a window, j > p - window or j < first tokens, j's page there
//   out = sum_j exp(s_j - max) V[j] / sum_j exp(s_j - max), zero where no j is left
// S^T = K Q^T and O^T += V^T P^T on the matrix cores, so that a query is a lane's
// column throughout: its maximum, sum and rescaling need no exchange but the one
// over the lane groups, and P^T is already PV's operand.
//
// Numerics over an f16 cache (f32 results of f32 queries).  K and V are exact f16
// operands.  A query row times scale log2(e) is multiplied by a power of two so
// that its largest element is in [2^14, 2^15) and split into hi + 2^-11 lo, two
// f16 values whose products have sums of their own: an element is off by 2^-23
// of itself down to 2^-29 of the row's largest, by 2^-52 of the largest below that.
// A weight exp2(s - max + 15), at most 2^15, is split into two f16 values likewise
// but joined in one sum: the split is off by 2^-22 of it (many rows, which cut the first part: 2^-21) down to 2^-17 of the
// row's largest weight, by 2^-40 of the largest below that; an exponent of 8 to 16 is rounded by 2^-21, which is
// 2^-21.5 of the weight, and exp2 by 2^-23: 2^-20 in all.  That is half of the matrix rate for results
// that one f16 value a weight would have at 2^-12.  The MFMA's f32 sums are not rounded to
// nearest, so each step's start from zero and join O in one fma.
// Over an f32 cache few rows take the f32 MFMA (they are bound by the reading all the
// same), many rows six products of bf16 parts: within 2^-23 of |x y| for values from 2^-110 on (those from
// 3.3961e38 on read as NaN where they are seen, for bf16 rounds them to infinity).  Weights are at most 1 / kv_len there
// (paged_weight_unit).
//
// V in unseen places: a weight of zero keeps finite values out, not NaN.  Steps
// that some row does not see all of replace what is not finite (or has bf16 parts that
// are not) by zero, and put NaN where a row does see one.
#pragma once
#include "common.hpp"
#include "f16_split.hpp"
#include "launch.hpp"
#include "mfma_common.hpp"
#include "paged.hpp"

namespace barq {

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// What the weights over an f32 cache of n positions (1 or more) are multiplied by: below 1 / n, a power of two.  Their sum is then below
// 1, so that no sum of weights times V, of a step, an item or a merge, is larger than the largest |V| (the division by the weights' sum
// takes it out again, exactly); products below 2^-126 lose bits, of V below 2^-126 n.
__device__ __forceinline__ float paged_weight_unit(int n) { return __builtin_bit_cast(float, (uint32_t)(95 + __builtin_clz(n)) << 23); }

__device__ __forceinline__ float paged_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// An item, in scalar registers.
__device__ __forceinline__ PagedItem paged_item(const PagedItem* p) {
    PagedItem it;
    const int* from = reinterpret_cast<const int*>(p);
    int* to = reinterpret_cast<int*>(&it);
    #pragma unroll
    for (int i = 0; i < 12; i++) to[i] = __builtin_amdgcn_readfirstlane(from[i]);
    return it;
}

// What a row sees.
struct PagedSight {
    int window, n_sink;
    // bit x, below 64: the row at row_pos sees position base + x (windows are at most 2^31 - 4096)
    __device__ __forceinline__ uint64_t mask(int row_pos, int base) const {
        const auto below = [](int n) { return n > 0 ? ~0ull >> (64 - min(n, 64)) : 0ull; };
        uint64_t m = below(row_pos - base + 1);
        if (window) m &= ~below(row_pos - base - window + 1) | below(n_sink - base);
        return m;
    }
    // all positions base .. base + n - 1 by all rows at positions first .. last
    __device__ __forceinline__ bool all(int base, int n, int first, int last) const {
        return base + n - 1 <= first && (!window || base > last - window || base + n <= n_sink);
    }
};

// Scale of a query row (a power of two) whose largest |element| is m; 1 / it.
__device__ __forceinline__ float paged_row_scale(float m, float& back) {
    // at least 2^-100 and below infinity, so that both are normal f32 values
    uint32_t e = __builtin_bit_cast(uint32_t, m) >> 23;
    e = e < 27u ? 27u : e > 254u ? 254u : e;
    back = __builtin_bit_cast(float, (e - 14u) << 23);
    return __builtin_bit_cast(float, (254u + 14u - e) << 23);
}

// x -> f16 hi and f16 of (x - hi) 2^11
__device__ __forceinline__ void paged_split(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const h2v h = {(_Float16)x0, (_Float16)x1};
    const h2v l = {(_Float16)((x0 - (float)h[0]) * 2048.0f), (_Float16)((x1 - (float)h[1]) * 2048.0f)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// x where `keep` is all ones, -infinity where it is zero
__device__ __forceinline__ float seen_or_none(float x, int keep) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(int, x) & keep) | (0xFF800000 & ~keep));
}
__device__ __forceinline__ int bit_as_mask(uint32_t bits, int i) { return (int)(bits << (31 - i)) >> 31; }

// Bit 15 of an f16 half that is not finite, bit 31 of the other or of an f32; other bits say nothing.
__device__ __forceinline__ uint32_t f16_bad_mark(uint32_t x) { return (x & 0x7C007C00u) + 0x04000400u; }
__device__ __forceinline__ uint32_t f32_bad_mark(uint32_t x) { return (x & 0x7F800000u) + 0x00800000u; }
// The f16 halves of a dword that are not finite, as 0xFFFF each.
__device__ __forceinline__ uint32_t f16_bad(uint32_t x) {
    return ((((x & 0x7C007C00u) + 0x04000400u) >> 15) & 0x00010001u) * 0xFFFFu;
}
__device__ __forceinline__ uint32_t f32_bad(uint32_t x) { return (x & 0x7F800000u) == 0x7F800000u ? 0xFFFFFFFFu : 0u; }

}  // namespace barq
