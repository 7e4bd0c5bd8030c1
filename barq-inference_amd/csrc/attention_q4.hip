// Attention over a KV cache held in 4 bits for few query rows (a decoded
// token): see attention_q4.hpp for the products and attention.hip for the
// reference's functions and the layouts of q and the output.
//
// 16 rows a workgroup (one decoded token: its G heads); the positions are split
// over workgroups and, in steps of 32, over the four waves of one.
//
// What bounds it: vector issue.  A step of 128 dims takes about 380 vector
// instructions (K's codes to f16 72, V's codes and scales to hi and lo 136, the
// scores' scales and O's sums 64, the softmax and the weights' split the rest)
// beside 40 MFMAs of 16 cycles, for 4.5 KB of the cache, and a 16-column product
// serves the G rows alone.  One row of 32/8 heads of 128 dims against 65536
// positions (75.5 MB): 25.0 us and 3.8 for the merge, 3.0 TB/s (vector issue 59 % and
// the matrix unit 18 % busy, counted at 26.2); 4096 positions 6.5 + 3.8 (first bytes
// and launches); five rows of 16/16 heads of 256 against 3003 14.9 + 3.8 (one step a wave).
#include "attention_q4.hpp"
#include "attention_q4_plan.hpp"
#include "launch.hpp"

#include <cmath>

namespace barq {

// A wave's packed rows on their way through LDS: each lane copies what it (or
// for the scales, its group) will read, one step ahead, straight from memory
// (no registers, no barrier: the wave waits for its own copies).
template <int HD>
struct Q4Fifo {
    static constexpr int KB = 16 * HD, SB = HD < 128 ? 256 : 2 * HD;   // bytes of a step's codes and scales (each of K's and V's)
    static constexpr int STAGE = 2 * KB + 2 * SB, BYTES = 2 * STAGE;
    static constexpr int COPIES = 2 * (KB / 1024) + 2 * (SB / 256);
    i32x4v kc, vc, ks, vs;   // from the range's first position (a multiple of 8)
    uint32_t ko[2], vo, so;  // this lane's offsets in a step
    uint32_t lds;            // the wave's two stages

    // positions j0 .. j1 of kv head hk (reads behind the last one's tile give zeros)
    __device__ __forceinline__ void init(const Q4View& kv, int hk, int j0, int j1, int l, uint32_t at) {
        const size_t co = (size_t)hk * kv.code_head + (size_t)j0 * (HD / 2), cs = (size_t)hk * kv.scale_head + (size_t)j0 * (HD / 16);
        const uint32_t n = (uint32_t)(j1 - j0 + KV_TILE - 1) / KV_TILE * KV_TILE;   // whole tiles
        kc = make_rsrc4(kv.kc + co, n * (HD / 2));
        vc = make_rsrc4(kv.vc + co, n * (HD / 2));
        ks = make_rsrc4(kv.ks + cs, n * (HD / 16));
        vs = make_rsrc4(kv.vs + cs, n * (HD / 16));
        const uint32_t c = l & 15, g = l >> 4;
        #pragma unroll
        for (int t = 0; t < 2; t++) ko[t] = HD == 64 ? 16 * l : (8 * (c / 4) + 4 * t + c % 4) * (HD / 2) + g * (HD / 8);
        vo = g * (KV_TILE * HD / 2) + c * (HD / 4);
        so = 4 * l;
        lds = at;
    }
    __device__ __forceinline__ void issue(int stage, uint32_t at) const {   // at: positions from j0
        const uint32_t base = lds + stage * STAGE, ca = at * (HD / 2), sa = at * (HD / 16);
        wait_lgkmcnt0();   // (the stage's last readers)
        #pragma unroll
        for (int t = 0; t < (HD == 64 ? 1 : 2); t++)
            #pragma unroll
            for (int u = 0; u < (HD == 256 ? 2 : 1); u++)
                lds_load16_at(kc, base + 1024 * ((HD == 256 ? 2 * t : t) + u), ko[t] + 16 * u, ca);
        #pragma unroll
        for (int u = 0; u < HD / 64; u++) lds_load16_at(vc, base + KB + 1024 * u, vo + 16 * u, ca);
        #pragma unroll
        for (int u = 0; u < SB / 256; u++) {
            lds_load4_at(ks, base + 2 * KB + 256 * u, so + 256 * u, sa);
            lds_load4_at(vs, base + 2 * KB + SB + 256 * u, so + 256 * u, sa);
        }
    }
};

// A stage as this lane reads it.
template <int HD>
struct Q4Stage {
    uint8_t* p;
    int c, g;
    // K codes of S tile t: this lane's dwords of its row, one per block
    __device__ __forceinline__ void k_row(int t, uint32_t (&w)[HD / 32]) const {
        if constexpr (HD == 64) {
            const uint2 v = *reinterpret_cast<const uint2*>(p + (8 * (c / 4) + 4 * t + c % 4) * 32 + 8 * g);
            w[0] = v.x;
            w[1] = v.y;
        } else {
            #pragma unroll
            for (int u = 0; u < HD / 128; u++) {
                const uint4 v = *reinterpret_cast<const uint4*>(p + 1024 * (t * (HD / 128) + u) + 16 * (16 * g + c));
                w[4 * u] = v.x; w[4 * u + 1] = v.y; w[4 * u + 2] = v.z; w[4 * u + 3] = v.w;
            }
        }
    }
    // V codes of dims 16 (4 u + i) + c, i < 4, at the group's 8 positions
    __device__ __forceinline__ uint4 v_dims(int u) const {
        return *reinterpret_cast<const uint4*>(p + Q4Fifo<HD>::KB + 1024 * u + 16 * (16 * g + c));
    }
    __device__ __forceinline__ u32x4v* scale(int which, int b) const {   // the group's 8 positions, K's (0) or V's (1)
        return reinterpret_cast<u32x4v*>(p + 2 * Q4Fifo<HD>::KB + which * Q4Fifo<HD>::SB + 16 * (g * (HD / 32) + b));
    }
};

// One step: positions base .. base + 31 (of the cache) of a range up to j1.
// nan_at (LDS, unless null): V scales that are NaN count as zero, and the
// first position of one goes there, block by block; the rows that see it get
// NaN at the end.  (0 * NaN would reach rows that do not.)
template <int HD, bool SC>
__device__ __forceinline__ void q4_step(const Q4Stage<HD>& s, int base, int j1, const Q4Seen& seen, const Q4Query<HD>& q,
                                        float lost, const Q4Const& kc, Q4State<HD>& st, float* score_row,
                                        int* nan_at) {
    float x[8];
    uint32_t kw[2][HD / 32];
    #pragma unroll
    for (int t = 0; t < 2; t++) s.k_row(t, kw[t]);
    const auto kfrag = [&](int t, int b, bool fresh) {
        uint32_t w = kw[t][b];
        if (fresh) asm volatile("" : "+v"(w));
        return q4_k_frag(w, kc);
    };
    q4_scores<HD>(x, q, lost, kfrag, [&](int b) { return *s.scale(0, b); });
    const int at = base + 8 * s.g;
    if (base + Q4A_STEP > j1) {   // the range's last step: what lies behind it is not the cache's
        u32x4v m;
        #pragma unroll
        for (int j = 0; j < 4; j++) m[j] = (at + 2 * j < j1 ? 0xFFFFu : 0u) | (at + 2 * j + 1 < j1 ? 0xFFFF0000u : 0u);
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) *s.scale(1, b) &= m;   // (the group's 16 lanes write the same)
    }
    if (nan_at) {
        #pragma unroll
        for (int b = 0; b < HD / 32; b++) {
            u32x4v v = *s.scale(1, b);
            int n = 0x7FFFFFFF;
            #pragma unroll
            for (int j = 3; j >= 0; j--)
                #pragma unroll
                for (int u = 1; u >= 0; u--) {
                    const uint32_t m = 0x7C00u << (16 * u);
                    const bool bad = (v[j] & m) == m;
                    v[j] &= bad ? ~(0xFFFFu << (16 * u)) : 0xFFFFFFFFu;
                    n = bad ? at + 2 * j + u : n;
                }
            *s.scale(1, b) = v;
            if (s.c == 0 && n != 0x7FFFFFFF) atomicMin(&nan_at[b], n);
        }
    }
    uint4 vw;
    q4_attend<HD, SC>(x, base, at, seen, q, kc, st, score_row, [&](int c, h8v& hi, h8v& lo) {
        if (c % 4 == 0) vw = s.v_dims(c / 4);
        q4_v_frag(c % 4 == 0 ? vw.x : c % 4 == 1 ? vw.y : c % 4 == 2 ? vw.z : vw.w, *s.scale(1, c / 2), kc, hi, lo);
    });
}

// A wave's steps of positions j0 .. j1: every `turn` positions from the first.
template <int HD, bool SC>
__device__ __forceinline__ void q4_walk(const Q4Fifo<HD>& fifo, uint8_t* lds, int j0, int j1, int first, int turn, int l,
                                        const Q4Seen& seen, const Q4Query<HD>& q, float lost, const Q4Const& kc,
                                        Q4State<HD>& st, float* score_row, int* nan_at) {
    st.clear();
    const int n = j1 - j0;
    if (first >= n) return;
    fifo.issue(0, (uint32_t)first);
    int stage = 0;
    for (int at = first; at < n; at += turn, stage ^= 1) {
        fifo.issue(stage ^ 1, (uint32_t)q4_ahead(at, turn, n));   // (always as many copies: the wait counts them)
        wait_vmcnt<Q4Fifo<HD>::COPIES>();
        asm volatile("" ::: "memory");
        const Q4Stage<HD> s{lds + stage * Q4Fifo<HD>::STAGE, l & 15, l >> 4};
        q4_step<HD, SC>(s, j0 + at, j1, seen, q, lost, kc, st, score_row, nan_at);
    }
    wait_vmcnt<0>();   // nothing on its way to LDS any more
    asm volatile("" ::: "memory");
}

// Workgroup x: group of G heads x % groups, then split, then tile of 16 rows.
// The four waves share out the split's steps.
template <int HD, bool SC>
__global__ __launch_bounds__(64 * Q4A_NW, HD <= 128 ? 3 : 2)
void attn_q4_kernel(Q4Args a) {
    constexpr int NB = HD / 32, ORS = HD + 4;   // LDS row: 16 rows on distinct banks
    constexpr int MERGE = Q4A_NW * Q4A_ROWS * ORS * 4, FIFO = Q4A_NW * Q4Fifo<HD>::BYTES;
    __shared__ __align__(16) uint8_t lds[MERGE > FIFO ? MERGE : FIFO];   // the rows on their way, then the merge
    __shared__ float lml[Q4A_NW][Q4A_ROWS][2];
    __shared__ int nan_pos[Q4A_NW][NB];
    const int t = threadIdx.x, l = t & 63, c = l & 15, g = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int grp = (int)(blockIdx.x % a.groups), piece = (int)(blockIdx.x / a.groups), rows_n = a.q_len * a.G, n_split = a.n_split;
    const int r0 = piece / n_split * Q4A_ROWS, split = piece % n_split;
    const int hk = (int)((long long)(grp * a.G) * a.n_head_kv / a.n_head);
    // the tile's last row bounds the positions
    const int visible = q4_vis(a, r0 + Q4A_ROWS - 1);
    const int start = split * a.chunk, j0 = min(start, visible), j1 = q4_range_end(start, a.chunk, visible);

    Q4Fifo<HD> fifo;
    uint8_t* mine = lds + wave * Q4Fifo<HD>::BYTES;
    fifo.init(a.kv, hk, start, max(j1, start), l, lds_addr(mine));
    const Q4Const kc;
    const Q4Row row = q4_row(a, grp, r0 + c);
    const Q4Seen seen{min(row.vis, j1), min(q4_vis(a, r0), j1)};
    Q4Query<HD> q;
    const float lost = uniform(row16_max(q.load(a.q + ((size_t)row.h * a.q_rows + row.i) * HD, a.scale, g, kc)));
    float* const score_row = SC && row.ok ? a.scores + ((size_t)row.i * a.n_head + row.h) * a.score_stride : nullptr;
    Q4State<HD> st;
    int* nan_at = nullptr;
    for (;;) {
        q4_walk<HD, SC>(fifo, mine, j0, j1, wave * Q4A_STEP, Q4A_NW * Q4A_STEP, l, seen, q, lost, kc, st, score_row, nan_at);
        if (nan_at || !__any(st.not_finite())) break;
        // NaN somewhere: again with V's NaN blocks kept out of the products
        nan_at = nan_pos[wave];
        if (l < NB) nan_at[l] = 0x7FFFFFFF;
    }
    if (nan_at) {
        wait_lgkmcnt0();
        st.put_nan(nan_at, seen.end);
    }

    // the four waves' states
    float (*lo)[Q4A_ROWS][ORS] = reinterpret_cast<float (*)[Q4A_ROWS][ORS]>(lds);
    __syncthreads();
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

static Q4Plan q4_plan(size_t n_head, size_t n_head_kv, size_t hd, size_t q_len, size_t kv_len) {
    return q4_plan(n_head, n_head_kv, hd, q_len, kv_len, (size_t)cu_count_attn());
}

size_t attention_q4_workspace(size_t n_head, size_t n_head_kv, size_t head_dim, size_t q_len, size_t kv_len) {
    const Q4Plan p = q4_plan(n_head, n_head_kv, head_dim, q_len, kv_len);
    return p.n_split > 1 ? (size_t)p.n_split * n_head * q_len * (head_dim + 2) * sizeof(float) : 0;
}

bool attention_q4_fits(size_t n_head, size_t n_head_kv, size_t head_dim, size_t q_len, size_t kv_len) {
    return q4_fits(q4_plan(n_head, n_head_kv, head_dim, q_len, kv_len), n_head, head_dim, q_len);
}

bool attention_q4_q8_direct(const AttnArgs& a) {
    return (a.n_head * a.head_dim) % 256 == 0 && q4_plan(a.n_head, a.n_head_kv, a.head_dim, a.q_len, a.kv_len).n_split > 1;
}

int attention_q4_scores_splits(size_t n_head, size_t n_head_kv, size_t head_dim, size_t q_len, size_t kv_len) {
    return q4_plan(n_head, n_head_kv, head_dim, q_len, kv_len).n_split;
}

template <int HD>
static hipError_t attn_q4_launch_t(const AttnArgs& a, const AttnScores* sc, const Q4View& kv, hipStream_t s) {
    const Q4Plan p = q4_plan(a.n_head, a.n_head_kv, HD, a.q_len, a.kv_len);
    Q4Args k{};
    k.q = a.q;
    k.kv = kv;
    k.n_head = (int)a.n_head;
    k.n_head_kv = (int)a.n_head_kv;
    k.G = p.G;
    k.groups = p.groups;
    k.q_len = (int)a.q_len;
    k.kv_len = (int)a.kv_len;
    k.q_rows = (int)(sc ? sc->q_rows : a.q_len);
    k.start_pos = (long long)a.start_pos;
    k.chunk = p.chunk;
    k.n_split = p.n_split;
    k.tiles = p.tiles;
    k.scale = 1.44269504088896340736f / sqrtf((float)HD);
    k.part = a.part;
    k.out = a.out;
    if (sc) {
        k.scores = sc->scores;
        k.score_stride = sc->stride;
    }
    hipError_t e;
    if (p.prompt) {
        e = attn_q4_prompt_launch(k, HD, s);
    } else {
        const dim3 grid((unsigned)p.n_split * (unsigned)p.tiles * (unsigned)p.groups), block(64 * Q4A_NW);
        if (sc) hipLaunchKernelGGL((attn_q4_kernel<HD, true>), grid, block, 0, s, k);
        else hipLaunchKernelGGL((attn_q4_kernel<HD, false>), grid, block, 0, s, k);
        e = hipGetLastError();
    }
    if (e != hipSuccess || sc || p.n_split == 1) return e;
    return attention_combine_launch(a, p.n_split, attention_q4_q8_direct(a) ? a.out_q8 : nullptr, nullptr, s);
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
