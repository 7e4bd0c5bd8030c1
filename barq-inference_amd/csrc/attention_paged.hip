// Attention over a paged KV cache for sequences with few rows (new tokens x the
// query heads of a kv head): the next token, drafted tokens.  attention_paged.hpp
// has the formulas and numerics.
//
// Bound by the reading of K and V: 32 sequences of up to 8000 positions (8 kv heads of
// 128 dims, f16), 556 MB, in 96 us with the merge, 5.8 TB/s; loads alone, on the same pages and as many workgroups, have 6.5
// that pass the caches by and 5.9 otherwise.  A workgroup is four
// waves, each with key steps of its own (every fourth of the item's), so nothing is shared
// and nothing waits before the end: the pages' layout is the MFMA operands', 16 bytes a
// lane straight into registers.  A step is 32 positions in f16, 16 in f32: 16 KiB of K and V
// for 128 dims either way, and K's registers take the next step's keys as soon as the
// scores are there, V's after P V (with a second set of registers the compiler spilled, and the same
// read took 189 us).  One tile of 16 rows: two in one workgroup leave one workgroup a CU (eight
// sequences' 5 drafted tokens after 4000 positions: 43 us, tile by tile 29, the second reading from the caches).
// Short calls are bound by the launch and the chain of an item, its page ids, keys and values, the joining: one token
// against 4096 positions 6.3 us on the device, an empty launch 2.3.
#include "attention_paged.hpp"
#include "q8k_block.hpp"

namespace barq {

namespace {

constexpr int NW = 4;   // waves

// Over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48).
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

// A lane's part of one step: K of tile t (position 8 (i / 4) + 4 t + i % 4 of the
// step in f16, i in f32, for lane i of its group), dims E (4 c + g) .. ; V of dim
// 16 d + i, the group's E positions.
template <bool H, int HD>
struct Step {
    static constexpr int KT = H ? 2 : 1, NC = H ? HD / 32 : HD / 16, NV = HD / 16;
    u32x4v k[KT][NC], v[NV];
};

template <bool H, int HD>
struct Query {
    static constexpr int NC = H ? HD / 32 : HD / 16, E = H ? 8 : 4;
    u32x4v hi[NC], lo[H ? NC : 1];   // f32: the values in hi
    float back;
    // fetched first, split when the keys and values are on their way
    __device__ __forceinline__ static void fetch(const float* row, int g, float (&x)[NC][E]) {
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int u = 0; u < E / 4; u++) {
                const float4 y = *reinterpret_cast<const float4*>(row + E * (4 * c + g) + 4 * u);
                x[c][4 * u] = y.x, x[c][4 * u + 1] = y.y, x[c][4 * u + 2] = y.z, x[c][4 * u + 3] = y.w;
            }
    }
    __device__ __forceinline__ void split(float (&x)[NC][E], float scale) {
        float m = 0.0f;
        #pragma unroll
        for (int c = 0; c < NC; c++)
            #pragma unroll
            for (int e = 0; e < E; e++) {
                x[c][e] *= scale;
                m = fmaxf(m, __builtin_fabsf(x[c][e]));
            }
        back = 1.0f;
        if constexpr (H) {
            const float up = paged_row_scale(groups_max(m), back);
            #pragma unroll
            for (int c = 0; c < NC; c++)
                #pragma unroll
                for (int u = 0; u < 4; u++) {
                    uint32_t h, l;
                    paged_split(x[c][2 * u] * up, x[c][2 * u + 1] * up, h, l);
                    hi[c][u] = h;
                    lo[c][u] = l;
                }
        } else {
            #pragma unroll
            for (int c = 0; c < NC; c++)
                #pragma unroll
                for (int u = 0; u < 4; u++) hi[c][u] = __builtin_bit_cast(uint32_t, x[c][u]);
        }
    }
};

// The scores of the lane's positions (log2 units): index 4 t + r is position 8 g + 4 t + r (f16), 4 g + r (f32).
template <bool H, int HD>
__device__ __forceinline__ void scores(const Step<H, HD>& st, const Query<H, HD>& q, float (&s)[4 * Step<H, HD>::KT]) {
    constexpr int KT = Step<H, HD>::KT, NC = Step<H, HD>::NC;
    #pragma unroll
    for (int t = 0; t < KT; t++) {
        if constexpr (H) {
            f32x4 hi = {}, lo = {};
            #pragma unroll
            for (int c = 0; c < NC; c++) {
                const h8v k = __builtin_bit_cast(h8v, st.k[t][c]);
                lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, __builtin_bit_cast(h8v, q.lo[c]), lo, 0, 0, 0);
                hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, __builtin_bit_cast(h8v, q.hi[c]), hi, 0, 0, 0);
            }
            #pragma unroll
            for (int r = 0; r < 4; r++) s[4 * t + r] = __builtin_fmaf(lo[r], 1.0f / 2048, hi[r]) * q.back;
        } else {
            // four sums side by side: none waits for another, and each is cut a quarter as often
            f32x4 part[4] = {};
            #pragma unroll
            for (int c = 0; c < NC; c++) {
                const f32x4 k = __builtin_bit_cast(f32x4, st.k[t][c]), x = __builtin_bit_cast(f32x4, q.hi[c]);
                #pragma unroll
                for (int e = 0; e < 4; e++) part[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], x[e], part[e], 0, 0, 0);
            }
            #pragma unroll
            for (int r = 0; r < 4; r++) s[4 * t + r] = (part[0][r] + part[1][r]) + (part[2][r] + part[3][r]);
        }
    }
}

// V^T times the weights (or what stands for them) of the lane's positions, dims 16 d + 4 g + r of the lane's row.
template <bool H>
struct Weights {
    u32x4v hi, lo;
    float w[H ? 1 : 4];
    __device__ __forceinline__ void set(const float* p, float minus_one) {
        if constexpr (H) {
            #pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t h, l;
                split_f16(p[2 * j], p[2 * j + 1], minus_one, h, l);
                hi[j] = h;
                lo[j] = l;
            }
        } else {
            #pragma unroll
            for (int j = 0; j < 4; j++) w[j] = p[j];
        }
    }
    __device__ __forceinline__ f32x4 times(u32x4v v) const {
        f32x4 acc = {};
        if constexpr (H) {
            const h8v a = __builtin_bit_cast(h8v, v);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(h8v, lo), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(h8v, hi), acc, 0, 0, 0);
        } else {
            const f32x4 a = __builtin_bit_cast(f32x4, v);
            #pragma unroll
            for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], w[j], acc, 0, 0, 0);
        }
        return acc;
    }
};

// ONCE: keys and values that nothing reads again soon pass the caches by.
template <bool H, int HD, bool ONCE>
__global__ __launch_bounds__(64 * NW, HD == 256 ? 1 : 2)
void paged_few_kernel(PagedAttn a, int count) {
    constexpr int STEP = H ? 32 : 16, E = H ? 8 : 4, KT = H ? 2 : 1, NV = HD / 16, NP = 4 * KT;
    constexpr int ROW = HD + 4;   // floats of a row in LDS: 16-byte pieces, the four groups in other banks
    constexpr size_t BLOCK = (size_t)PAGE_BLOCK * HD * (H ? 2 : 4);
    __shared__ __align__(16) float o_s[NW][16][ROW];
    __shared__ float m_s[NW][16], l_s[NW][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    int n_tokens = a.n_tokens;
    if (n_tokens < 0) {
        n_tokens = a.counts->n_tokens;
        count = a.counts->few;
    }
    const float minus_one = f16_minus_one();
    const PagedSight sight = {a.window, a.n_sink};
    const size_t page_bytes = BLOCK << (a.log_page - 4);   // of one kv head
    for (int w = blockIdx.x, at = w / a.n_kv; w < count * a.n_kv;) {
        const int hk = w % a.n_kv;
        const PagedItem it = paged_item(&a.few[at]);
        const int p_first = it.past + it.row0 / a.G, p_last = it.past + (it.row0 + it.rows - 1) / a.G;
        float m = -INFINITY, l = 0.0f;
        f32x4 o[NV];
        #pragma unroll
        for (int d = 0; d < NV; d++) o[d] = f32x4{};
        const int32_t* table = a.table + it.table;
        const float unit = paged_weight_unit(it.kv_len);
        const int steps = (it.v1 - it.v0 - wave + NW - 1) / NW;   // this wave's (none: 0 or less)
        const auto base_of = [&](int j) {
            const int v = it.v0 + wave + NW * j;
            return (v < it.a ? v : v - it.a + it.b) * STEP;
        };
        // lane j holds the pages of the wave's step 64 n + j, of its first 16 positions and (f16) of the others
        int id0 = -1, id1 = -1;
        const auto fetch_ids = [&](int j0) {
            id0 = id1 = -1;
            const int j = j0 + lane;
            if (j < steps) {
                const int at = base_of(j);
                id0 = table[at >> a.log_page];
                if (H && at + 16 < it.kv_len) id1 = table[(at + 16) >> a.log_page];
            }
        };
        const auto block_at = [&](const uint8_t* pool, int id, int at) {   // (an absent page: the first one, unseen)
            return pool + ((size_t)max(id, 0) * a.n_kv + hk) * page_bytes + (size_t)((at & ((1 << a.log_page) - 1)) >> 4) * BLOCK;
        };
        // One set of registers: K's are free once the scores are there, V's after P V, and take the next step's at once.
        Step<H, HD> st;
        int k_pages = 0;   // bit 0, 1: the first 16 positions of the step in K's registers have a page, the others
        const auto fetch = [](const uint8_t* p) __attribute__((always_inline)) {
            return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const u32x4v*>(p)) : *reinterpret_cast<const u32x4v*>(p);
        };
        const auto load = [&](int j, bool keys) __attribute__((always_inline)) {
            if (j >= steps) return;
            const int at = base_of(j), p0 = __builtin_amdgcn_readlane(id0, j & 63), p1 = H ? __builtin_amdgcn_readlane(id1, j & 63) : -1;
            const uint8_t *pool = keys ? a.k : a.v, *b0 = block_at(pool, p0, at), *b1 = H ? block_at(pool, p1, at + 16) : b0;
            if (keys) {
                k_pages = (p0 >= 0 ? 1 : 0) | (p1 >= 0 ? 2 : 0);
                const uint8_t* b = H && i >= 8 ? b1 : b0;
                #pragma unroll
                for (int t = 0; t < KT; t++) {
                    const int slot = H ? (8 * (i >> 2) + 4 * t + (i & 3)) & 15 : i;
                    #pragma unroll
                    for (int c = 0; c < Step<H, HD>::NC; c++) st.k[t][c] = fetch(b + ((4 * c + g) * 16 + slot) * 16);
                }
            } else {
                const uint8_t* b = H && g >= 2 ? b1 : b0;
                #pragma unroll
                for (int d = 0; d < NV; d++) st.v[d] = fetch(b + ((H ? g & 1 : g) * HD + 16 * d + i) * 16);
            }
        };
        if (steps > 0) fetch_ids(0);
        Query<H, HD> q;
        float raw[Query<H, HD>::NC][E];
        const int mine = it.row0 + min(i, it.rows - 1), tok = mine / a.G, pos = it.past + tok;
        Query<H, HD>::fetch(a.q + ((size_t)(hk * a.G + mine % a.G) * n_tokens + it.q0 + tok) * HD, g, raw);
        load(0, true);
        load(0, false);
        q.split(raw, a.scale);
        for (int j = 0; j < steps; j++) {
            const int base = base_of(j), have = k_pages;
            const bool whole = have == (H ? 3 : 1) && sight.all(base, STEP, p_first, p_last);
            uint32_t seen = 0;   // bit e: the lane's row sees the lane's position e
            if (!whole) {
                const bool here = H && g >= 2 ? have & 2 : have & 1;   // (a group's positions lie in one block)
                seen = here ? (uint32_t)sight.mask(pos, base + E * g) : 0u;
                uint32_t any = 0;
                #pragma unroll
                for (int d = 0; d < NV; d++)
                    #pragma unroll
                    for (int u = 0; u < 4; u++) any |= H ? f16_bad_mark(st.v[d][u]) : f32_bad_mark(st.v[d][u]);
                if (__any((any & (H ? 0x80008000u : 0x80000000u)) != 0)) {   // NaN where a row sees what is not finite, and zero in its place
                    Weights<H> ones;
                    float z[NP];
                    #pragma unroll
                    for (int e = 0; e < NP; e++) z[e] = (seen >> e) & 1 ? 1.0f : 0.0f;
                    ones.set(z, minus_one);
                    #pragma unroll
                    for (int d = 0; d < NV; d++) {
                        u32x4v is;
                        #pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const uint32_t b = H ? f16_bad(st.v[d][u]) : f32_bad(st.v[d][u]);
                            is[u] = b & (H ? 0x3C003C00u : 0x3F800000u);
                            st.v[d][u] &= ~b;
                        }
                        const f32x4 nan = ones.times(is);
                        #pragma unroll
                        for (int r = 0; r < 4; r++) o[d][r] = nan[r] > 0.0f ? NAN : o[d][r];
                    }
                }
            }
            float s[NP];
            scores<H, HD>(st, q, s);
            if (((j + 1) & 63) == 0) fetch_ids(j + 1);
            load(j + 1, true);
            if (!whole) {
                #pragma unroll
                for (int e = 0; e < NP; e++) s[e] = seen_or_none(s[e], bit_as_mask(seen, e));
            }
            float top = s[0];
            #pragma unroll
            for (int e = 1; e < NP; e++) top = fmaxf(top, s[e]);
            top = fmaxf(m, groups_max(top));
            const float ref = top == -INFINITY ? 0.0f : top, alpha = paged_exp2(m - ref);
            m = top;
            float sum = 0.0f;
            #pragma unroll
            for (int e = 0; e < NP; e++) {
                s[e] = H ? paged_exp2((s[e] - ref) + 15.0f) : paged_exp2(s[e] - ref) * unit;   // (in this order: at most 15 whatever the scores)
                sum += s[e];
            }
            l = __builtin_fmaf(l, alpha, sum);
            Weights<H> p;
            p.set(s, minus_one);
            #pragma unroll
            for (int d = 0; d < NV; d++) {
                const f32x4 y = p.times(st.v[d]);
                #pragma unroll
                for (int r = 0; r < 4; r++) o[d][r] = __builtin_fmaf(o[d][r], alpha, y[r]);
            }
            load(j + 1, false);
        }
        // the four waves' states, joined
        l = groups_sum(l);
        if (g == 0) {
            m_s[wave][i] = m;
            l_s[wave][i] = l;
        }
        __syncthreads();
        {
            float top = m_s[0][i];
            #pragma unroll
            for (int u = 1; u < NW; u++) top = fmaxf(top, m_s[u][i]);
            const float f = m == -INFINITY ? 1.0f : paged_exp2(m - top);   // (1: o is zero, or NaN and stays it)
            #pragma unroll
            for (int d = 0; d < NV; d++) {
                f32x4 y;
                #pragma unroll
                for (int r = 0; r < 4; r++) y[r] = o[d][r] * f;
                *reinterpret_cast<f32x4*>(&o_s[wave][i][16 * d + 4 * g]) = y;
            }
        }
        __syncthreads();
        for (int u = threadIdx.x; u < it.rows * (HD / 4); u += 64 * NW) {
            const int r = u / (HD / 4), d = 4 * (u % (HD / 4));
            float top = m_s[0][r];
            #pragma unroll
            for (int x = 1; x < NW; x++) top = fmaxf(top, m_s[x][r]);
            float sum = 0.0f;
            #pragma unroll
            for (int x = 0; x < NW; x++) sum = __builtin_fmaf(l_s[x][r], m_s[x][r] == -INFINITY ? 1.0f : paged_exp2(m_s[x][r] - top), sum);
            f32x4 y = *reinterpret_cast<const f32x4*>(&o_s[0][r][d]);
            #pragma unroll
            for (int x = 1; x < NW; x++) y += *reinterpret_cast<const f32x4*>(&o_s[x][r][d]);
            if (it.part < 0) {
                const int rr = it.row0 + r;
                float* out = a.out + ((size_t)(it.q0 + rr / a.G) * a.n_head + hk * a.G + rr % a.G) * HD + d;
                #pragma unroll
                for (int e = 0; e < 4; e++) out[e] = sum == 0.0f ? 0.0f : y[e] / sum;
            } else {
                const size_t at = (size_t)hk * a.part_rows + it.part + r;
                *reinterpret_cast<f32x4*>(a.part + at * HD + d) = y;
                if (d == 0) a.stat[at] = make_float2(top, sum);
            }
        }
        __syncthreads();   // (a next item's states go where this one's are read from)
        at = it.next;
        if (at < 0) {
            w += gridDim.x;
            at = w / a.n_kv;
        }
    }
}

// Joins the partial states of rows that several workgroups share.  Bound by its latencies: a wave's loads, eight
// states and the maxima and sums, are in flight together (3.6 us for 32 rows of 32 states, 11.0 one after
// another).  Up to 8 states a wave a row, beyond that the four waves of a workgroup share a row's.
template <int HD>
__global__ __launch_bounds__(64 * NW)
void paged_merge_kernel(PagedAttn a) {
    constexpr int PER = HD / 64, AHEAD = 8;
    __shared__ float part_s[NW][HD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int merges = a.n_tokens < 0 ? a.counts->merges : a.n_merges, hk = blockIdx.y, span = a.merge_span;
    for (int w = blockIdx.x; w < merges * span; w += gridDim.x) {
        const PagedMerge mg = a.merges[w / span];
        const bool shared = mg.n_split > PAGED_MERGE_WAVE;
        const int r = shared ? w % span : (w % span) * NW + wave;
        const int step = shared ? NW : 1, mine = shared ? (mg.n_split - wave + NW - 1) / NW : mg.n_split, s0 = shared ? wave : 0;
        if (shared ? r >= mg.rows : (w % span) * NW >= mg.rows) continue;
        const size_t at = (size_t)hk * a.part_rows + mg.part + min(r, mg.rows - 1);
        const auto states = [&](int k, float (&x)[AHEAD][PER]) __attribute__((always_inline)) {
            #pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const float* from = a.part + (at + (size_t)(s0 + step * max(min(k + u, mine - 1), 0)) * mg.rows) * HD + lane * PER;
                #pragma unroll
                for (int e = 0; e < PER; e++) x[u][e] = from[e];
            }
        };
        float x[AHEAD][PER], y[PER], top = -INFINITY, sum = 0.0f;
        states(0, x);
        float2 z = make_float2(-INFINITY, 0.0f);
        for (int s = lane; s < mg.n_split; s += 64) {
            const float2 t = a.stat[at + (size_t)s * mg.rows];
            if (s < 64) z = t;
            top = fmaxf(top, t.x);
        }
        top = wave_max_all(top);
        const auto factor = [&](float m) { return m == -INFINITY ? 1.0f : paged_exp2(m - top); };   // (1: zeros, or NaN)
        const float f = factor(z.x);
        sum = z.y * f;
        for (int s = lane + 64; s < mg.n_split; s += 64) {
            const float2 t = a.stat[at + (size_t)s * mg.rows];
            sum = __builtin_fmaf(t.y, factor(t.x), sum);
        }
        sum = wave_sum_all(sum);
        #pragma unroll
        for (int e = 0; e < PER; e++) y[e] = 0.0f;
        for (int k = 0; k < mine; k += AHEAD) {
            if (k) states(k, x);
            #pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const int s = s0 + step * (k + u);
                if (k + u < mine) {
                    const float g = s < 64 ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s & 63))
                                           : factor(a.stat[at + (size_t)s * mg.rows].x);
                    #pragma unroll
                    for (int e = 0; e < PER; e++) y[e] = __builtin_fmaf(x[u][e], g, y[e]);
                }
            }
        }
        if (shared) {
            __syncthreads();   // (an earlier row's sums have been read)
            #pragma unroll
            for (int e = 0; e < PER; e++) part_s[wave][lane * PER + e] = y[e];
            __syncthreads();
            #pragma unroll
            for (int e = 0; e < PER; e++) {
                y[e] = part_s[0][lane * PER + e];
                #pragma unroll
                for (int u = 1; u < NW; u++) y[e] += part_s[u][lane * PER + e];
            }
        }
        if (shared ? wave == 0 : r < mg.rows) {
            const int rr = mg.row0 + r, tok = mg.q0 + rr / a.G, head = hk * a.G + rr % a.G;
            float* out = a.out + ((size_t)tok * a.n_head + head) * HD + lane * PER;
            #pragma unroll
            for (int e = 0; e < PER; e++) out[e] = sum == 0.0f ? 0.0f : y[e] / sum;
        }
    }
}

// The output rows as Q8_K blocks: a wave a block.
__global__ __launch_bounds__(64 * NW)
void paged_q8k_kernel(const float* __restrict__ rows, uint8_t* __restrict__ out, int n_tokens, int blocks, const PagedCounts* counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t n = (size_t)(n_tokens < 0 ? counts->n_tokens : n_tokens) * blocks;
    for (size_t b = (size_t)blockIdx.x * NW + wave; b < n; b += (size_t)gridDim.x * NW) {
        const float4 v = reinterpret_cast<const float4*>(rows + b * 256)[lane];
        const float x[4] = {v.x, v.y, v.z, v.w};
        q8_k_block(x, lane, out + b * Q8_K_BYTES);
    }
}

}  // namespace

hipError_t paged_attention_launch(const PagedAttn& a, bool f16, int hd, hipStream_t s) {
    // A captured call replays with other counts: its grids are fixed, their workgroups go round the items.
    const bool captured = a.n_tokens < 0;
    const auto grid = [&](int n) { return dim3(captured ? 1024u : (unsigned)n * (unsigned)a.n_kv); };
    if (captured || a.n_few) {
        #define BARQ_FEW(H, D, O) \
            if (f16 == H && hd == D && a.once == O) \
                hipLaunchKernelGGL((paged_few_kernel<H, D, O>), grid(a.n_few), dim3(64 * NW), 0, s, a, a.n_few);
        BARQ_FEW(true, 64, false) BARQ_FEW(true, 128, false) BARQ_FEW(true, 256, false)
        BARQ_FEW(false, 64, false) BARQ_FEW(false, 128, false) BARQ_FEW(false, 256, false)
        BARQ_FEW(true, 64, true) BARQ_FEW(true, 128, true) BARQ_FEW(true, 256, true)
        BARQ_FEW(false, 64, true) BARQ_FEW(false, 128, true) BARQ_FEW(false, 256, true)
        #undef BARQ_FEW
    }
    if (captured || a.n_many) {
        const hipError_t e = paged_many_launch(a, f16, hd, s);
        if (e != hipSuccess) return e;
    }
    if (captured || a.n_merges) {
        const dim3 g(captured ? 256u : (unsigned)a.n_merges * (unsigned)a.merge_span, (unsigned)a.n_kv);
        if (hd == 64) hipLaunchKernelGGL(paged_merge_kernel<64>, g, dim3(256), 0, s, a);
        if (hd == 128) hipLaunchKernelGGL(paged_merge_kernel<128>, g, dim3(256), 0, s, a);
        if (hd == 256) hipLaunchKernelGGL(paged_merge_kernel<256>, g, dim3(256), 0, s, a);
    }
    if (a.out_q8) {
        const size_t blocks = (size_t)a.n_head * hd / 256, n = (captured ? 256 : (size_t)a.n_tokens) * blocks;
        hipLaunchKernelGGL(paged_q8k_kernel, dim3((unsigned)((n + NW - 1) / NW < 8192 ? (n + NW - 1) / NW : 8192)), dim3(256), 0, s, a.out,
                           a.out_q8, a.n_tokens, (int)blocks, a.counts);
    }
    return hipGetLastError();
}

}  // namespace barq
