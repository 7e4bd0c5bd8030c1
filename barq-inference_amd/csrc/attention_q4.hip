// Attention over a KV cache held in 4 bits (kv_q4.hpp), for any number of
// query rows: the decode kernel of such a cache.  See attention.hip for the
// reference's functions and the layouts of q and the output.
//
// The query rows that share a kv head are flattened as query * G + head and
// taken 16 at a time (one decoded token: its G heads); the positions are
// split over workgroups and, in steps of 32, over the four waves of one.  A
// step of a wave:
//   S^T[pos, row] = sum over blocks b of dk[pos, b] * (codes_K[pos, b, :] . Q[row, b, :])
//                                      16x16x32 MFMAs, A = K rows, B = Q^T
//   P = exp2(S - max), online per row
//   O^T[dim, row] += V^T[dim, pos] P^T[pos, row]     A = V^T, B = P^T
// Row i of S's tile t stands for position 8 (i / 4) + 4 t + i % 4 of the step, so
// that lane group g ends with the weights of positions 8 g .. 8 g + 7: P^T is
// already PV's B operand, the 8 positions are one tile of V, and K's and V's
// scales of them are 16 bytes a block.  Nothing passes through LDS but the
// merge of the four waves.
//
// Numerics (f32 results from f32 queries): a K code is an integer, exact in
// bf16; a query element times 16 log2(e) / sqrt(HD) is rounded once and split
// into three bf16 values that add up to it exactly, over all of f32's range.
// The products are exact, the sums f32, the block's scale joins in f32.
// A V element (code - 8) * d has 15 bits and is exactly hi + lo in f16: all
// its parts are multiples of 2^-24, the least f16 step, and the quantizer keeps it
// within +-65504.  A weight is scaled by the step's largest to at most 2^15 and
// split into two f16 values: off by at most 2^-23 of itself down to 2^-16 of the
// step's largest weight, by 2^-40 of the largest below that.  Weights under
// 2^-20 of the largest (14 nats; beside a position that takes nearly all the
// weight) are therefore left to another pass over the step's V with a scale of
// their own, and so on down to f32's least; lo lo products (2^-22 of theirs at
// most) are left out.  The MFMA does not round its
// f32 sums to nearest, so each step's products start from zero and join O in
// one fma.
#include "common.hpp"
#include "kv_q4.hpp"
#include "launch.hpp"
#include "mfma_common.hpp"

#include <cmath>

namespace barq {

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int Q4A_ROWS = 16;    // query rows of a workgroup
constexpr int Q4A_STEP = 32;    // positions of a wave's step
constexpr int Q4A_NW = 4;
constexpr float Q4A_WINDOW = 0x1p-20f;

struct Q4Args {
    const float* q;        // [n_head, q_len, HD]
    Q4View kv;
    int n_head, n_head_kv, G, q_len, kv_len;
    int q_rows;            // rows of q per head (the call's are the first q_len)
    long long start_pos;
    int chunk, n_split;    // positions of a split, splits
    float scale;           // 16 log2(e) / sqrt(HD)
    float* part;           // [q_len][n_head][splits][HD + 2] (SC, or more than one split)
    float* out;            // [q_len, n_head, HD]
    float* scores;         // SC: [q_len * n_head][score_stride], log2 units
    size_t score_stride;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t q4_rsrc(const uint8_t* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), (short)0, (int)bytes, 0x00020000);
}

// N dwords at off (N = 2, or a multiple of 4); past the descriptor's limit zeros.
template <int N>
__device__ __forceinline__ void q4_ld(uint32_t (&d)[N], __amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (N == 2) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
        d[0] = (uint32_t)v[0];
        d[1] = (uint32_t)v[1];
    } else {
        #pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, 0, 0);
            #pragma unroll
            for (int j = 0; j < 4; j++) d[4 * i + j] = (uint32_t)v[j];
        }
    }
}

// Eight K codes -> (code - 8) / 16 in bf16 (four bits: the upper halves of the f32 values hold them).
__device__ __forceinline__ bf8v q4_k_frag(uint32_t w) {
    uint32_t p[4];
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        const float a = __builtin_amdgcn_cvt_off_f32_i4((int)(w >> (8 * j)));
        const float b = __builtin_amdgcn_cvt_off_f32_i4((int)(w >> (8 * j + 4)));
        p[j] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
    }
    return __builtin_bit_cast(bf8v, u32x4v{p[0], p[1], p[2], p[3]});
}

// Eight positions of a V dim, times their scales -> f16 hi + lo, exactly.
__device__ __forceinline__ void q4_v_frag(uint32_t w, const uint32_t* sc, h8v& hi, h8v& lo) {
    u32x4v h, l;
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        // 0x6400 | n is the f16 1024 + n
        const h2v n = __builtin_bit_cast(h2v, ((w >> (4 * j)) & 0x000F000Fu) | 0x64006400u) + h2v{(_Float16)-1032.0f, (_Float16)-1032.0f};
        const h2v d = __builtin_bit_cast(h2v, sc[j]);
        const h2v a = n * d;
        h[j] = __builtin_bit_cast(uint32_t, a);
        l[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, d, -a));
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

template <int HD>
struct Q4Step {   // a step's packed rows
    uint32_t k[2][HD / 32];     // S tile t: this lane's quarter of its row
    uint32_t v[HD / 16];        // this lane's dims 16 c + l % 16 of its group's tile
    uint32_t ks[HD / 32][4];    // its group's tile: 8 f16 a block
    uint32_t vs[HD / 32][4];
};

template <int HD>
struct Q4Rows {
    __amdgpu_buffer_rsrc_t kc, vc, ks, vs;   // from the split's first position (a multiple of 8)
    uint32_t ko[2], vo, so;                  // this lane's offsets in a step
    // rows j0 .. j1 of a kv head
    __device__ __forceinline__ void init(const Q4View& kv, int hk, int j0, int j1, int l) {
        const size_t co = (size_t)hk * kv.code_head + (size_t)j0 * (HD / 2), cs = (size_t)hk * kv.scale_head + (size_t)j0 * (HD / 16);
        const uint32_t n = (uint32_t)(j1 - j0 + KV_TILE - 1) / KV_TILE * KV_TILE;   // whole tiles
        kc = q4_rsrc(kv.kc + co, n * (HD / 2));
        vc = q4_rsrc(kv.vc + co, n * (HD / 2));
        ks = q4_rsrc(kv.ks + cs, n * (HD / 16));
        vs = q4_rsrc(kv.vs + cs, n * (HD / 16));
        const uint32_t c = l & 15, g = l >> 4;
        #pragma unroll
        for (int t = 0; t < 2; t++) ko[t] = (8 * (c / 4) + 4 * t + c % 4) * (HD / 2) + g * (HD / 8);
        vo = g * (KV_TILE * HD / 2) + c * (HD / 4);
        so = g * (KV_TILE * HD / 16);
    }
    __device__ __forceinline__ void load(Q4Step<HD>& s, uint32_t at) const {   // at: positions from j0
        #pragma unroll
        for (int t = 0; t < 2; t++) q4_ld(s.k[t], kc, at * (HD / 2) + ko[t]);
        q4_ld(s.v, vc, at * (HD / 2) + vo);
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            q4_ld(s.ks[b], ks, at * (HD / 16) + so + 16 * b);
            q4_ld(s.vs[b], vs, at * (HD / 16) + so + 16 * b);
        }
    }
};

// The lane's part of its query row, split in three: registers, or with 256
// dims (whose 96 registers the kernel does not have) LDS, which the four
// waves share since their rows are the same.
template <int HD>
struct Q4Query {
    static constexpr bool IN_LDS = HD == 256;
    static constexpr int LDS = IN_LDS ? 3 * (HD / 32) * 64 : 1;   // fragments
    bf8v reg[IN_LDS ? 1 : 3][IN_LDS ? 1 : HD / 32];
    const bf8v* lds;   // this lane's: [piece][block] 64 apart
    __device__ __forceinline__ bf8v get(int piece, int b) const {
        if constexpr (IN_LDS) return lds[(piece * (HD / 32) + b) * 64];
        else return reg[piece][b];
    }
    __device__ __forceinline__ void load(const float* row, float scale, int g, int l, int wave, bf8v* store) {
        lds = store + l;
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            if (IN_LDS && b % Q4A_NW != wave) continue;   // each wave its share
            const float4 u = *reinterpret_cast<const float4*>(row + 32 * b + 8 * g), w = *reinterpret_cast<const float4*>(row + 32 * b + 8 * g + 4);
            const float y[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
            bf8v p[3];
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = y[e] * scale;
                p[0][e] = (__bf16)x;
                const float x1 = x - (float)p[0][e];
                p[1][e] = (__bf16)x1;
                p[2][e] = (__bf16)(x1 - (float)p[1][e]);
            }
            #pragma unroll
            for (int i = 0; i < 3; i++) {
                if constexpr (IN_LDS) store[(i * (HD / 32) + b) * 64 + l] = p[i];
                else reg[i][b] = p[i];
            }
        }
        if constexpr (IN_LDS) __syncthreads();
    }
};

// A lane's running state: its row's reference maximum, the sum over its
// group's positions, O's dims 16 c + 4 g + r of the row.
template <int HD>
struct Q4State {
    float m, l;
    f32x4 o[HD / 16];
};

// One step: positions base .. base + 31 (of the cache), seen up to `end` by this lane's row.
// FIX: V scales that are NaN count as zero and leave their position in
// nan_at[block] instead (the rows that see it get NaN at the end): 0 * NaN
// would reach rows that do not.
template <int HD, bool SC, bool FIX>
__device__ __forceinline__ void q4_step(Q4Step<HD>& s, int base, int j1, int end, const Q4Query<HD>& q, int g,
                                        Q4State<HD>& st, float* score_row, int (&nan_at)[HD / 32]) {
    f32x4 sc[2] = {};
    #pragma unroll
    for (int t = 0; t < 2; t++)
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            const bf8v k = q4_k_frag(s.k[t][b]);
            f32x4 c = {};
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q.get(2, b), c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q.get(1, b), c, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q.get(0, b), c, 0, 0, 0);
            const h8v d = __builtin_bit_cast(h8v, u32x4v{s.ks[b][0], s.ks[b][1], s.ks[b][2], s.ks[b][3]});
            #pragma unroll
            for (int r = 0; r < 4; r++) sc[t][r] = __builtin_fmaf(c[r], (float)d[4 * t + r], sc[t][r]);
        }
    const int at = base + 8 * g;
    float x[8];
    float bm = -INFINITY;
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = at + e < end ? sc[e >> 2][e & 3] : -INFINITY;
        bm = fmaxf(bm, x[e]);
    }
    if constexpr (SC) {
        if (score_row) {   // (a row's stride is whole steps)
            *reinterpret_cast<f32x4*>(score_row + at) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(score_row + at + 4) = f32x4{x[4], x[5], x[6], x[7]};
        }
    }
    bm = groups_max(bm);
    // O and l are relative to m, a multiple of 2^-14; it moves when the
    // maximum has grown by 2^32.  The step's weights are relative to m plus a
    // whole number k, at most 1.
    if (__any(bm > st.m + 32.0f)) {
        const float mn = fmaxf(st.m, __builtin_ceilf(bm * 0x1p14f) * 0x1p-14f);
        const float corr = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - mn);
        st.m = mn;
        st.l *= corr;
        #pragma unroll
        for (int c = 0; c < HD / 16; c++) st.o[c] *= corr;
    }
    const bool none = bm == -INFINITY;   // a row that sees no position of the step
    const float k = none ? 0.0f : __builtin_ceilf(bm - st.m);
    const float ref = none ? 0.0f : st.m + k, w = none ? 0.0f : __builtin_amdgcn_exp2f(k);
    float p[8], sum = 0.0f;
    #pragma unroll
    for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(x[e] - ref);
    sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    st.l = __builtin_fmaf(sum, w, st.l);
    if (base + Q4A_STEP > j1) {   // the range's last step: what lies behind it is not the cache's
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t m = (at + 2 * j < j1 ? 0xFFFFu : 0u) | (at + 2 * j + 1 < j1 ? 0xFFFF0000u : 0u);
            #pragma unroll
            for (int b = 0; b < HD / 32; b++) s.vs[b][j] &= m;
        }
    }
    if constexpr (FIX) {
        #pragma unroll
        for (int b = 0; b < HD / 32; b++)
            #pragma unroll
            for (int j = 3; j >= 0; j--)
                #pragma unroll
                for (int u = 1; u >= 0; u--) {
                    const uint32_t m = 0x7C00u << (16 * u);
                    if ((s.vs[b][j] & m) == m) {
                        s.vs[b][j] &= u ? 0x0000FFFFu : 0xFFFF0000u;
                        nan_at[b] = min(nan_at[b], at + 2 * j + u);
                    }
                }
    }
    // The least weight that is not zero (bits - 1 orders zero last): where the
    // step's weights span more than f16 pairs hold, they are taken in windows
    // of 2^20, each scaled by itself.
    uint32_t least = 0xFFFFFFFFu;
    #pragma unroll
    for (int e = 0; e < 8; e++) least = min(least, __builtin_bit_cast(uint32_t, p[e]) - 1u);
    const bool spread = __any(least < __builtin_bit_cast(uint32_t, Q4A_WINDOW) - 1u);
    float inv = w * 0x1p-15f;
    bool more = false;
    do {
        float y[8];
        #pragma unroll
        for (int e = 0; e < 8; e++) y[e] = p[e] * 0x1p15f;
        if (spread) {
            bool left = false;
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool later = p[e] < Q4A_WINDOW;   // (false for NaN)
                y[e] = later ? 0.0f : y[e];
                p[e] = later ? p[e] * (1.0f / Q4A_WINDOW) : 0.0f;
                left |= p[e] > 0.0f;
            }
            more = __any(left);
        }
        u32x4v ph, pl;
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const h2v h = {(_Float16)y[2 * j], (_Float16)y[2 * j + 1]};
            const h2v r = {(_Float16)(y[2 * j] - (float)h[0]), (_Float16)(y[2 * j + 1] - (float)h[1])};
            ph[j] = __builtin_bit_cast(uint32_t, h);
            pl[j] = __builtin_bit_cast(uint32_t, r);
        }
        const h8v bh = __builtin_bit_cast(h8v, ph), bl = __builtin_bit_cast(h8v, pl);
        #pragma unroll
        for (int c = 0; c < HD / 16; c++) {
            h8v vh, vl;
            q4_v_frag(s.v[c], s.vs[c / 2], vh, vl);
            f32x4 d = {};
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, bh, d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, bl, d, 0, 0, 0);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, bh, d, 0, 0, 0);
            #pragma unroll
            for (int r = 0; r < 4; r++) st.o[c][r] = __builtin_fmaf(d[r], inv, st.o[c][r]);
        }
        inv *= Q4A_WINDOW;
    } while (more);
}

// A wave's steps of positions j0 .. j1.
template <int HD, bool SC, bool FIX>
__device__ __forceinline__ void q4_walk(const Q4Rows<HD>& rows, int j0, int j1, int end, int wave, const Q4Query<HD>& q,
                                        int g, Q4State<HD>& st, float* score_row, int (&nan_at)[HD / 32]) {
    st.m = -INFINITY;
    st.l = 0.0f;
    #pragma unroll
    for (int c = 0; c < HD / 16; c++) st.o[c] = f32x4{};
    constexpr int ALL = Q4A_NW * Q4A_STEP;
    int at = wave * Q4A_STEP;
    const int n = j1 - j0;
    if (at >= n) return;
    if constexpr (HD == 256) {   // no registers for a second set
        Q4Step<HD> a;
        for (; at < n; at += ALL) {
            rows.load(a, (uint32_t)at);
            q4_step<HD, SC, FIX>(a, j0 + at, j1, end, q, g, st, score_row, nan_at);
        }
        return;
    }
    Q4Step<HD> a, b;
    rows.load(a, (uint32_t)at);
    // two register sets in turn, each loaded one step ahead (past the range zeros, no memory access)
    for (; at < n; at += 2 * ALL) {
        rows.load(b, (uint32_t)(at + ALL));
        q4_step<HD, SC, FIX>(a, j0 + at, j1, end, q, g, st, score_row, nan_at);
        if (at + ALL >= n) break;
        rows.load(a, (uint32_t)(at + 2 * ALL));
        q4_step<HD, SC, FIX>(b, j0 + at + ALL, j1, end, q, g, st, score_row, nan_at);
    }
}

// Grid: x = tile of 16 rows * splits + split, y = group of G heads.
template <int HD, bool SC>
__global__ __launch_bounds__(64 * Q4A_NW, 2)
void attn_q4_kernel(Q4Args a) {
    constexpr int NB = HD / 32, ORS = HD + 4;   // LDS row: 16 rows on distinct banks
    constexpr int MERGE = Q4A_NW * Q4A_ROWS * ORS * 4, QUERY = Q4Query<HD>::LDS * 16;
    __shared__ __align__(16) uint8_t lds[MERGE > QUERY ? MERGE : QUERY];   // the queries, then the merge
    __shared__ float lml[Q4A_NW][Q4A_ROWS][2];
    float (*lo)[Q4A_ROWS][ORS] = reinterpret_cast<float (*)[Q4A_ROWS][ORS]>(lds);
    const int t = threadIdx.x, l = t & 63, c = l & 15, g = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int grp = blockIdx.y, rows_n = a.q_len * a.G, n_split = a.n_split;
    const int r0 = (int)(blockIdx.x / n_split) * Q4A_ROWS, split = (int)(blockIdx.x % n_split);
    const int hk = (int)((long long)(grp * a.G) * a.n_head_kv / a.n_head);
    const int row = r0 + c < rows_n ? r0 + c : rows_n - 1;
    const int i = row / a.G, h = grp * a.G + (row - i * a.G);
    const long long seen = a.start_pos + i + 1;
    const int vis = (int)(seen < a.kv_len ? seen : a.kv_len);
    // what the tile's last row sees bounds the positions
    const int i_last = (r0 + Q4A_ROWS < rows_n ? r0 + Q4A_ROWS - 1 : rows_n - 1) / a.G;
    const long long last = a.start_pos + i_last + 1;
    const int visible = (int)(last < a.kv_len ? last : a.kv_len);
    const int j0 = min(split * a.chunk, visible), j1 = min(visible, j0 + a.chunk), end = min(vis, j1);

    Q4Query<HD> q;
    q.load(a.q + ((size_t)h * a.q_rows + i) * HD, a.scale, g, l, wave, reinterpret_cast<bf8v*>(lds));
    float* score_row = nullptr;
    if (SC && r0 + c < rows_n) score_row = a.scores + ((size_t)i * a.n_head + h) * a.score_stride;
    Q4State<HD> st;
    int nan_at[NB];
    #pragma unroll
    for (int b = 0; b < NB; b++) nan_at[b] = 0x7FFFFFFF;
    Q4Rows<HD> rows;
    rows.init(a.kv, hk, split * a.chunk, max(j1, split * a.chunk), l);
    q4_walk<HD, SC, false>(rows, j0, j1, end, wave, q, g, st, score_row, nan_at);
    // NaN somewhere: again with V's NaN blocks kept out of the products
    float z = 0.0f;
    #pragma unroll
    for (int u = 0; u < HD / 16; u++)
        #pragma unroll
        for (int r = 0; r < 4; r++) z = __builtin_fmaf(st.o[u][r], 0.0f, z);
    if (__any(z != 0.0f)) {
        q4_walk<HD, false, true>(rows, j0, j1, end, wave, q, g, st, nullptr, nan_at);
        #pragma unroll
        for (int b = 0; b < NB; b++) {
            // the earliest of the four groups' positions
            int n = nan_at[b];
            n = min(n, __shfl_xor(n, 16));
            n = min(n, __shfl_xor(n, 32));
            if (n < end)
                #pragma unroll
                for (int u = 0; u < 2; u++) st.o[2 * b + u] = f32x4{NAN, NAN, NAN, NAN};
        }
    }

    // the four waves' states
    if constexpr (Q4Query<HD>::IN_LDS) __syncthreads();
    #pragma unroll
    for (int u = 0; u < HD / 16; u++) *reinterpret_cast<f32x4*>(&lo[wave][c][16 * u + 4 * g]) = st.o[u];
    const float lsum = groups_sum(st.l);
    if (g == 0) {
        lml[wave][c][0] = st.m;
        lml[wave][c][1] = lsum;
    }
    __syncthreads();
    const int live = min(Q4A_ROWS, rows_n - r0);
    for (int e = t; e < live * HD; e += 64 * Q4A_NW) {
        const int rr = e / HD, d = e % HD;
        float M = -INFINITY;
        #pragma unroll
        for (int w = 0; w < Q4A_NW; w++) M = fmaxf(M, lml[w][rr][0]);
        float L = 0.0f, O = 0.0f;
        #pragma unroll
        for (int w = 0; w < Q4A_NW; w++) {
            const float f = lml[w][rr][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lml[w][rr][0] - M);
            L = __builtin_fmaf(lml[w][rr][1], f, L);
            O = __builtin_fmaf(lo[w][rr][d], f, O);
        }
        const int ii = (r0 + rr) / a.G, hh = grp * a.G + (r0 + rr - ii * a.G);
        const size_t at = (size_t)ii * a.n_head + hh;
        if (n_split == 1 && !SC) {
            a.out[at * HD + d] = O / L;
        } else {
            float* pp = a.part + (at * n_split + split) * (HD + 2);
            pp[2 + d] = O;
            if (d == 0) {
                pp[0] = M;
                pp[1] = L;
            }
        }
    }
}

// ---- launch ------------------------------------------------------------------------

// Splits of the positions, of whole turns of a workgroup's four waves.
struct Q4Plan {
    int G, groups, tiles, n_split, chunk;
};

static Q4Plan q4_plan(size_t n_head, size_t n_head_kv, size_t q_len, size_t kv_len) {
    constexpr size_t TURN = Q4A_NW * Q4A_STEP;
    Q4Plan p;
    const bool even = n_head % n_head_kv == 0;
    p.G = even ? (int)(n_head / n_head_kv) : 1;
    p.groups = even ? (int)n_head_kv : (int)n_head;
    p.tiles = (int)((q_len * p.G + Q4A_ROWS - 1) / Q4A_ROWS);
    const size_t wg = (size_t)p.groups * p.tiles, target = (size_t)cu_count_attn() * 2;
    size_t ns = (target + wg - 1) / wg;
    const size_t most = (kv_len + TURN - 1) / TURN;
    if (ns > most) ns = most;
    if (ns > 1024) ns = 1024;   // the merge's limit
    // at most 2^20 positions a split (32-bit byte offsets)
    const size_t least = (kv_len + ((size_t)1 << 20) - 1) >> 20;
    if (ns < least) ns = least;
    size_t ch = (kv_len + ns - 1) / ns;
    ch = (ch + TURN - 1) / TURN * TURN;
    p.chunk = (int)ch;
    p.n_split = (int)((kv_len + ch - 1) / ch);
    return p;
}

size_t attention_q4_workspace(size_t n_head, size_t n_head_kv, size_t head_dim, size_t q_len, size_t kv_len) {
    const Q4Plan p = q4_plan(n_head, n_head_kv, q_len, kv_len);
    return p.n_split > 1 ? (size_t)p.n_split * n_head * q_len * (head_dim + 2) * sizeof(float) : 0;
}

bool attention_q4_q8_direct(const AttnArgs& a) {
    return (a.n_head * a.head_dim) % 256 == 0 && q4_plan(a.n_head, a.n_head_kv, a.q_len, a.kv_len).n_split > 1;
}

int attention_q4_scores_splits(size_t n_head, size_t n_head_kv, size_t q_len, size_t kv_len) {
    return q4_plan(n_head, n_head_kv, q_len, kv_len).n_split;
}

template <int HD>
static hipError_t attn_q4_launch_t(const AttnArgs& a, const AttnScores* sc, const Q4View& kv, hipStream_t s) {
    const Q4Plan p = q4_plan(a.n_head, a.n_head_kv, a.q_len, a.kv_len);
    Q4Args k{};
    k.q = a.q;
    k.kv = kv;
    k.n_head = (int)a.n_head;
    k.n_head_kv = (int)a.n_head_kv;
    k.G = p.G;
    k.q_len = (int)a.q_len;
    k.kv_len = (int)a.kv_len;
    k.q_rows = (int)(sc ? sc->q_rows : a.q_len);
    k.start_pos = (long long)a.start_pos;
    k.chunk = p.chunk;
    k.n_split = p.n_split;
    k.scale = 16.0f * 1.44269504088896340736f / sqrtf((float)HD);
    k.part = a.part;
    k.out = a.out;
    const dim3 grid((unsigned)p.n_split * (unsigned)p.tiles, p.groups), block(64 * Q4A_NW);
    if (sc) {
        k.scores = sc->scores;
        k.score_stride = sc->stride;
        hipLaunchKernelGGL((attn_q4_kernel<HD, true>), grid, block, 0, s, k);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((attn_q4_kernel<HD, false>), grid, block, 0, s, k);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.n_split == 1) return e;
    return attention_combine_launch(a, p.n_split, attention_q4_q8_direct(a) ? a.out_q8 : nullptr, s);
}

static hipError_t attn_q4_launch(const AttnArgs& a, const AttnScores* sc, const Q4View& kv, hipStream_t s) {
    switch (a.head_dim) {
    case 64: return attn_q4_launch_t<64>(a, sc, kv, s);
    case 128: return attn_q4_launch_t<128>(a, sc, kv, s);
    case 256: return attn_q4_launch_t<256>(a, sc, kv, s);
    default: return hipErrorInvalidValue;
    }
}

hipError_t attention_q4_launch(const AttnArgs& a, const Q4View& kv, hipStream_t s) {
    if (a.q_len == 0 || a.n_head == 0) return hipSuccess;
    return attn_q4_launch(a, nullptr, kv, s);
}

hipError_t attention_q4_scores_launch(const AttnArgs& a, const AttnScores& sc, const Q4View& kv, hipStream_t s) {
    return attn_q4_launch(a, &sc, kv, s);
}

}  // namespace barq
