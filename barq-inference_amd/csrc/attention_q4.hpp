// What the kernels of attention over a 4-bit KV cache share (attention_q4.hip:
// few query rows, attention_q4_prompt.hip: many): 16 query rows of one kv head
// against 32 positions by one wave.
//
// The query rows that share a kv head are flattened as query * G + head.
//   S^T[pos, row] = sum over blocks b of dk[pos, b] * ((codes_K[pos, b, :] - 8) . Q[row, b, :])
//                                      16x16x32 MFMAs, A = K rows, B = Q^T
//   P = exp2(S - max), online per row
//   O^T[dim, row] += V^T[dim, pos] P^T[pos, row]     A = V^T, B = P^T
// Row i of S's tile t (of two) stands for position 8 (i / 4) + 4 t + i % 4, so
// that lane group g ends with the weights of positions 8 g .. 8 g + 7: P^T is
// already PV's B operand, the 8 positions are one tile of V, and K's and V's
// scales of them are 16 bytes a block.
//
// Numerics (f32 results from f32 queries).  A K code minus 8 is exact in f16.
// A query row is scaled by a power of two so that its largest element is in
// [2^14, 2^15) and split into two f16 values, off by at most 2^-23 of an element
// down to 2^-17 of the largest and by 2^-40 of the largest below that.  (A normal
// query has such an element in one row of 300.)  What that can do to a score is
// bounded by the keys' scales; where the bound passes 2^-20 in log2 units the wave
// forms the step's scores from three bf16 values instead, which hold any f32
// exactly.  With the largest key there may be (65504) and 128 dims that is from one such
// element on beside a largest one of 64 or more; with keys up to 64 beside one of 2^16.
// The products are exact, the sums f32, the block's scale joins in
// f32 and the row's in the exponent's fma.
// A V element (code - 8) * d has 15 bits and is exactly hi + lo in f16: all
// its parts are multiples of 2^-24, the least f16 step, and the quantizer keeps it
// within +-65504.  A weight is scaled by the step's largest to at most 2^15 and
// split into two f16 values: off by at most 2^-23 of itself down to 2^-16 of the
// step's largest weight, by 2^-40 of the largest below that.  Weights under
// 2^-20 of the largest (14 nats; beside a position that takes nearly all the
// weight) are therefore left to another pass over the step's V with a scale of
// their own, and so on down to f32's least; lo lo products (2^-22 of theirs at
// most) are left out.  The MFMA does not round its f32 sums to nearest, so each
// step's products start from zero and join O in one fma.  Nor does it keep
// everything of products of f16 values below 2^-14, to which zero belongs: a sum
// is cut at about 2^-24.  Three sums a step with a largest weight of 2^14 or more: an output may
// be off by 2^-36 of 1 besides (seen: V values of 2^-24 by 6e-5 of themselves).
#pragma once
#include "common.hpp"
#include "f16_split.hpp"
#include "kv_q4.hpp"
#include "mfma_common.hpp"

namespace barq {

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int Q4A_ROWS = 16;    // query rows of a tile
constexpr int Q4A_STEP = 32;    // positions of a step
constexpr int Q4A_NW = 4;       // waves of a workgroup
constexpr int Q4A_WINDOW = 20;  // log2 of the spread that a step's weights may have

struct Q4Args {
    const float* q;        // [n_head, q_len, HD]
    Q4View kv;
    int n_head, n_head_kv, G, groups, q_len, kv_len;   // groups of G query heads that share a kv head
    int q_rows;            // rows of q per head (the call's are the first q_len)
    long long start_pos;
    int chunk, n_split;    // positions of a split, splits
    int tiles;             // workgroups' row tiles
    float scale;           // log2(e) / sqrt(HD)
    float* part;           // [q_len][n_head][splits][HD + 2] (SC, or more than one split)
    float* out;            // [q_len, n_head, HD]
    float* scores;         // SC: [q_len * n_head][score_stride], log2 units
    size_t score_stride;
};

// Constants in registers that the compiler knows nothing of, so that a mask
// and an or stay one instruction (two scalar operands would not fit it) and
// split_f16's fma stays one.
struct Q4Const {
    uint32_t lo = 0x64006400u, hi = 0x54005400u;   // f16 pairs of 1024 and of 64
    float minus_one = f16_minus_one();
    __device__ __forceinline__ Q4Const() {
        asm("" : "+v"(lo));
        asm("" : "+v"(hi));
    }
};

// Eight codes -> code - 8 in f16 pairs.  With n in the mantissa's lowest four bits
// 0x6400 | n is 1024 + n, in the next four 0x5400 | 16 n is 64 + n.
__device__ __forceinline__ void q4_codes(uint32_t w, const Q4Const& kc, h2v (&n)[4]) {
    const uint32_t w8 = w >> 8;
    const uint32_t u[4] = {(w & 0x000F000Fu) | kc.lo, (w & 0x00F000F0u) | kc.hi, (w8 & 0x000F000Fu) | kc.lo, (w8 & 0x00F000F0u) | kc.hi};
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        const _Float16 off = j & 1 ? (_Float16)-72.0f : (_Float16)-1032.0f;
        n[j] = __builtin_bit_cast(h2v, u[j]) + h2v{off, off};
    }
}
__device__ __forceinline__ h8v q4_k_frag(uint32_t w, const Q4Const& kc) {
    h2v n[4];
    q4_codes(w, kc, n);
    u32x4v v;
    #pragma unroll
    for (int j = 0; j < 4; j++) v[j] = __builtin_bit_cast(uint32_t, n[j]);
    return __builtin_bit_cast(h8v, v);
}
// Eight positions of a V dim, times their scales -> f16 hi + lo, exactly.
__device__ __forceinline__ void q4_v_frag(uint32_t w, u32x4v sc, const Q4Const& kc, h8v& hi, h8v& lo) {
    h2v n[4], d[4], a[4];
    q4_codes(w, kc, n);
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t pair = sc[j];   // (a bit cast of the vector's element itself would take element 0)
        d[j] = __builtin_bit_cast(h2v, pair);
        a[j] = n[j] * d[j];
    }
    u32x4v h, l;
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        h[j] = __builtin_bit_cast(uint32_t, a[j]);
        l[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n[j], d[j], -a[j]));
    }
    hi = __builtin_bit_cast(h8v, h);
    lo = __builtin_bit_cast(h8v, l);
}

// Maximum / sum over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float groups_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, (int)a[0]), __builtin_bit_cast(float, (int)a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (int)b[0]), __builtin_bit_cast(float, (int)b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
    v = swap16_add(v, v);
    return swap32_add(v, v);
}

// A value that all lanes hold, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// The lane's part of a query row: hi + lo.
template <int HD>
struct Q4Query {
    h8v hi[HD / 32], lo[HD / 32];
    const float* at;     // its dims 0 .. 7 of block 0
    float scale, back;   // what the row is multiplied by; scores times back are in log2 units
    // Returns what the split may cost a score (log2 units), in steps of 2^-22 times the
    // keys' largest scale: each element below 2^-2 is off by 2^-25 at most, its key is
    // at most 8 scales.
    __device__ __forceinline__ float load(const float* row, float score_scale, int g, const Q4Const& kc) {
        at = row + 8 * g;
        float4 y[HD / 16];
        float m = 0.0f;
        #pragma unroll
        for (int b = 0; b < HD / 32; b++)
            #pragma unroll
            for (int u = 0; u < 2; u++) {
                const float4 v = y[2 * b + u] = *reinterpret_cast<const float4*>(at + 32 * b + 4 * u);
                m = fmaxf(fmaxf(fmaxf(m, __builtin_fabsf(v.x)), fmaxf(__builtin_fabsf(v.y), __builtin_fabsf(v.z))), __builtin_fabsf(v.w));
            }
        m = groups_max(m);
        // 2^14 over the largest element's power of two, which is at least 2^-112 so that the scales are normal f32 values
        uint32_t e = __builtin_bit_cast(uint32_t, m) >> 23;
        e = e > 15u ? e : 15u;
        scale = __builtin_bit_cast(float, (254u + 14u - e) << 23);
        back = __builtin_bit_cast(float, (e - 14u) << 23) * score_scale;
        float small = 0.0f;
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            u32x4v h, l;
            #pragma unroll
            for (int u = 0; u < 4; u++) {
                const float4 v = y[2 * b + u / 2];
                const float x0 = (u & 1 ? v.z : v.x) * scale, x1 = (u & 1 ? v.w : v.y) * scale;
                uint32_t hh, ll;
                split_f16(x0, x1, kc.minus_one, hh, ll);
                h[u] = hh;
                l[u] = ll;
                small += __builtin_fabsf(x0) < 0.25f && x0 != 0.0f ? 1.0f : 0.0f;
                small += __builtin_fabsf(x1) < 0.25f && x1 != 0.0f ? 1.0f : 0.0f;
            }
            hi[b] = __builtin_bit_cast(h8v, h);
            lo[b] = __builtin_bit_cast(h8v, l);
        }
        return groups_sum(small) * back;
    }
    // block b in three bf16 values, which hold any f32 exactly
    __device__ __forceinline__ void exact(int b, bf8v (&p)[3]) const {
        const float* x = at + 32 * b;
        asm volatile("" : "+v"(x));   // (loaded where it is used: ahead of the loop it would take its registers)
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            float y = x[e] * scale;
            #pragma unroll
            for (int i = 0; i < 3; i++) {
                p[i][e] = (__bf16)y;
                y -= (float)p[i][e];
            }
        }
    }
};

// A lane's running state of a row: its reference maximum, the sum over its
// group's positions, O's dims 16 c + 4 g + r.
template <int HD>
struct Q4State {
    float m, l;
    f32x4 o[HD / 16];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
        #pragma unroll
        for (int c = 0; c < HD / 16; c++) o[c] = f32x4{};
    }
    __device__ __forceinline__ bool not_finite() const {
        float z = 0.0f;
        #pragma unroll
        for (int c = 0; c < HD / 16; c++)
            #pragma unroll
            for (int e = 0; e < 4; e++) z = __builtin_fmaf(o[c][e], 0.0f, z);
        return z != 0.0f;
    }
    // NaN in the dims of the blocks whose first NaN position is below end
    __device__ __forceinline__ void put_nan(const int* nan_at, int end) {
        #pragma unroll
        for (int b = 0; b < HD / 32; b++)
            if (nan_at[b] < end) o[2 * b] = o[2 * b + 1] = f32x4{NAN, NAN, NAN, NAN};
    }
};

// What a lane's row sees of the positions at hand.
struct Q4Seen {
    int end;   // the row's positions end here
    int all;   // every row of its tile sees the positions up to here
};

// The scores of the tile's rows (times their scale).  lost: the largest of what the
// rows' load returned, in a scalar register.  kfrag(t, b, fresh): K
// codes minus 8 of S tile t, block b, as f16 (fresh: not values it gave before,
// which would stay in registers between the calls); kscale(b): the group's 8
// positions' scales.
template <int HD, class K, class S>
__device__ __forceinline__ void q4_scores(float (&x)[8], const Q4Query<HD>& q, float lost, K kfrag, S kscale) {
    #pragma unroll
    for (int e = 0; e < 8; e++) x[e] = 0.0f;
    bool exact = false;
    if (lost * Q4_D_MAX > 4.0f) {   // 2^(-20 + 22)
        h2v m = {};
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            const u32x4v d = kscale(b);
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t pair = d[j] & 0x7FFF7FFFu;
                m = __builtin_elementwise_max(m, __builtin_bit_cast(h2v, pair));   // (a NaN is passed over: its scores are NaN either way)
            }
        }
        exact = __any(fmaxf((float)m[0], (float)m[1]) * lost > 4.0f);
    }
    if (exact) {
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            bf8v p[3];
            q.exact(b, p);
            const h8v d = __builtin_bit_cast(h8v, kscale(b));
            #pragma unroll
            for (int t = 0; t < 2; t++) {
                const h8v n = kfrag(t, b, true);
                bf8v k;
                #pragma unroll
                for (int e = 0; e < 8; e++) k[e] = (__bf16)(float)n[e];
                f32x4 c = {};
                #pragma unroll
                for (int i = 2; i >= 0; i--) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, p[i], c, 0, 0, 0);
                #pragma unroll
                for (int e = 0; e < 4; e++) x[4 * t + e] = __builtin_fmaf(c[e], (float)d[4 * t + e], x[4 * t + e]);
            }
            __builtin_amdgcn_sched_barrier(0);   // (one block's values at a time)
        }
    } else {
        // a block's products run while the next one's codes are fetched (or formed), and the one before is scaled
        h8v k[2][2];
        u32x4v d[2];
        f32x4 c[2][2];
        #pragma unroll
        for (int t = 0; t < 2; t++) k[0][t] = kfrag(t, 0, false);
        d[0] = kscale(0);
        #pragma unroll
        for (int b = 0; b <= HD / 32; b++) {
            const int cur = b & 1, old = cur ^ 1;
            if (b < HD / 32) {
                #pragma unroll
                for (int t = 0; t < 2; t++)
                    c[cur][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[cur][t], q.lo[b], f32x4{}, 0, 0, 0);
                #pragma unroll
                for (int t = 0; t < 2; t++)
                    c[cur][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[cur][t], q.hi[b], c[cur][t], 0, 0, 0);
            }
            if (b) {
                const h8v s = __builtin_bit_cast(h8v, d[old]);
                #pragma unroll
                for (int t = 0; t < 2; t++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) x[4 * t + e] = __builtin_fmaf(c[old][t][e], (float)s[4 * t + e], x[4 * t + e]);
            }
            if (b + 1 < HD / 32) {
                #pragma unroll
                for (int t = 0; t < 2; t++) k[old][t] = kfrag(t, b + 1, false);
                d[old] = kscale(b + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// O += V times the weights y (at most 2^15, times inv).  vfrag(c, hi, lo): dims 16 c + lane % 16
// at the group's 8 positions.
template <int HD, class V>
__device__ __forceinline__ void q4_pv(const float (&y)[8], float inv, const Q4Const& kc, Q4State<HD>& st, V vfrag) {
    h8v bh, bl;
    u32x4v ph, pl;
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t h, l;
        split_f16(y[2 * j], y[2 * j + 1], kc.minus_one, h, l);
        ph[j] = h;
        pl[j] = l;
    }
    bh = __builtin_bit_cast(h8v, ph);
    bl = __builtin_bit_cast(h8v, pl);
    // two dims' products run while the next two's values are fetched (or formed), and the two before join O
    h8v v[2][2][2];
    f32x4 d[2][2];
    #pragma unroll
    for (int i = 0; i < 2; i++) vfrag(i, v[0][i][0], v[0][i][1]);
    #pragma unroll
    for (int u = 0; u <= HD / 32; u++) {
        const int cur = u & 1, old = cur ^ 1;
        if (u < HD / 32) {
            #pragma unroll
            for (int i = 0; i < 2; i++)
                d[cur][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[cur][i][1], bh, f32x4{}, 0, 0, 0);
            #pragma unroll
            for (int i = 0; i < 2; i++)
                d[cur][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[cur][i][0], bl, d[cur][i], 0, 0, 0);
            #pragma unroll
            for (int i = 0; i < 2; i++)
                d[cur][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[cur][i][0], bh, d[cur][i], 0, 0, 0);
        }
        if (u)
            #pragma unroll
            for (int i = 0; i < 2; i++)
                #pragma unroll
                for (int e = 0; e < 4; e++) st.o[2 * u - 2 + i][e] = __builtin_fmaf(d[old][i][e], inv, st.o[2 * u - 2 + i][e]);
        if (u + 1 < HD / 32)
            #pragma unroll
            for (int i = 0; i < 2; i++) vfrag(2 * u + 2 + i, v[old][i][0], v[old][i][1]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Moves the weights below 2^-20 of 2^15 to `later`, times 2^20; whether there are any.
__device__ __forceinline__ bool q4_window(float (&x)[8], float (&later)[8]) {
    bool any = false;
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        const bool small = x[e] < 0x1p15f / (float)(1 << Q4A_WINDOW);   // (false for NaN)
        later[e] = small ? x[e] * (float)(1 << Q4A_WINDOW) : 0.0f;
        x[e] = small ? 0.0f : x[e];
        any |= later[e] > 0.0f;
    }
    return __any(any);
}

// Scores to weights to O, for the positions from base (at: this group's first).
template <int HD, bool SC, class V>
__device__ __forceinline__ void q4_attend(float (&x)[8], int base, int at, const Q4Seen& seen, const Q4Query<HD>& q,
                                          const Q4Const& kc, Q4State<HD>& st, float* score_row, V vfrag) {
    float bm = -INFINITY, least = INFINITY;
    if (base + Q4A_STEP <= seen.all) {
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            bm = fmaxf(bm, x[e]);
            least = fminf(least, x[e]);
        }
    } else {
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool in = at + e < seen.end;
            least = fminf(least, in ? x[e] : INFINITY);
            x[e] = in ? x[e] : -INFINITY;
            bm = fmaxf(bm, x[e]);
        }
    }
    float back = q.back;
    if constexpr (SC) {   // (the weights from the scores as they are kept: the sums match)
        #pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= back;
        bm *= back;
        least *= back;
        back = 1.0f;
        if (score_row) {   // (a row's stride is whole steps)
            *reinterpret_cast<f32x4*>(score_row + at) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(score_row + at + 4) = f32x4{x[4], x[5], x[6], x[7]};
        }
    }
    bm = groups_max(bm) * back;
    // O and l are relative to m, a multiple of 2^-14 (which every f32 value from 2^9
    // on is); it moves when the maximum has grown by 2^32.  The step's weights are
    // relative to ref, m plus a whole number as f32 rounds it, and at most 2^15.5.
    if (__any(bm > st.m + 32.0f)) {
        const float mn = fmaxf(st.m, __builtin_fabsf(bm) < 0x1p9f ? __builtin_ceilf(bm * 0x1p14f) * 0x1p-14f : bm);
        const float corr = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - mn);
        st.m = mn;
        st.l *= corr;
        #pragma unroll
        for (int c = 0; c < HD / 16; c++) st.o[c] *= corr;
    }
    const bool none = bm == -INFINITY;   // a row that sees no position of the step
    float ref = none ? 0.0f : st.m + (__builtin_ceilf(bm - st.m) - 15.0f);
    // From scores of 2^21 on their rounding (bm's against the product below, ref's) would let
    // weights pass 65504: there the scores are rounded first, and ref is bm itself where it came out lower.
    if (__any(__builtin_fabsf(ref) >= 0x1p21f || bm - ref > 15.5f)) {
        #pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= back;
        least *= back;
        back = 1.0f;
        ref = bm - ref > 15.5f ? bm : ref;
    }
    float w = none ? 0.0f : __builtin_amdgcn_exp2f(ref - st.m);
    #pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], back, -ref));
    st.l = __builtin_fmaf(((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])), w, st.l);
    const bool spread = least * back < ref + (15.0f - Q4A_WINDOW);
    // weights that span more than f16 pairs hold are taken in windows of
    // 2^20, each scaled by itself
    float later[8];
    bool more = __any(spread);
    if (more) more = q4_window(x, later);
    for (;;) {
        q4_pv<HD>(x, w, kc, st, vfrag);
        if (!more) break;
        w *= 1.0f / (float)(1 << Q4A_WINDOW);
        #pragma unroll
        for (int e = 0; e < 8; e++) x[e] = later[e];
        more = q4_window(x, later);
    }
}

// The lane's row of a row tile (the last row again where there are no more).
struct Q4Row {
    int i, h;     // query, query head
    bool ok;
    int vis;      // positions it sees
};
__device__ __forceinline__ Q4Row q4_row(const Q4Args& a, int grp, int row) {
    const int n = a.q_len * a.G;
    Q4Row r;
    r.ok = row < n;
    row = r.ok ? row : n - 1;
    r.i = row / a.G;
    r.h = grp * a.G + (row - r.i * a.G);
    const long long v = a.start_pos + r.i + 1;
    r.vis = (int)(v < a.kv_len ? v : a.kv_len);
    return r;
}
// positions that row `row` (or the last one) sees
__device__ __forceinline__ int q4_vis(const Q4Args& a, int row) {
    const int n = a.q_len * a.G;
    const long long v = a.start_pos + (row < n ? row : n - 1) / a.G + 1;
    return (int)(v < a.kv_len ? v : a.kv_len);
}

// The row's state (its sum complete) as results, or as partial state `split`.
template <int HD, bool PART>
__device__ __forceinline__ void q4_store(const Q4Args& a, const Q4Row& row, int split, int g, const Q4State<HD>& st, float lsum) {
    const size_t at = (size_t)row.i * a.n_head + row.h;
    if constexpr (!PART) {
        typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
        #pragma unroll
        for (int u = 0; u < HD / 16; u++) {
            const f32x4 o = st.o[u];
            *reinterpret_cast<f32x4u*>(a.out + at * HD + 16 * u + 4 * g) = f32x4u{o[0] / lsum, o[1] / lsum, o[2] / lsum, o[3] / lsum};
        }
    } else {
        float* pp = a.part + (at * a.n_split + split) * (HD + 2);   // 8-byte aligned
        #pragma unroll
        for (int u = 0; u < HD / 16; u++) {
            const f32x4 o = st.o[u];
            *reinterpret_cast<float2*>(pp + 2 + 16 * u + 4 * g) = make_float2(o[0], o[1]);
            *reinterpret_cast<float2*>(pp + 4 + 16 * u + 4 * g) = make_float2(o[2], o[3]);
        }
        if (g == 0) *reinterpret_cast<float2*>(pp) = make_float2(st.m, lsum);
    }
}

// attention_q4_prompt.hip (64 and 128 dims)
hipError_t attn_q4_prompt_launch(const Q4Args& a, size_t head_dim, hipStream_t s);

}  // namespace barq
