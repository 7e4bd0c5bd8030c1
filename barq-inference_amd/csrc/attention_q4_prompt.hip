// Attention over a KV cache held in 4 bits for many query rows (a prompt's
// chunk): see attention_q4.hpp for the products and their numerics.
//
// A workgroup of four waves takes 64 query rows of one kv head, 16 a wave,
// and walks the positions they see in blocks of 32.  The waves share the work
// that does not depend on the rows: each turns a fourth of a block's codes
// into f16 (K as they are, V times its scales as hi + lo) and leaves them in
// one of two LDS stages, lane by lane as the products will read them; one
// barrier per block.  Loads run one block ahead of that.  NaN scales of V are
// taken out here, so that they cannot reach rows that do not see them.
//
// What bounds it: the softmax and the products follow one another in a wave, and
// with three workgroups a CU three waves share a SIMD.  2048 tokens of 32/8 heads of
// 128 dims: 104 to 121 us, 34.4 GFLOP at 285 to 330 TFLOP/s of results, 2.5 f16
// products each (hi and lo of q, of V and of the weights): 0.7 to 0.8 PFLOP/s on the
// matrix unit, which a large f16 matrix product runs at 1.09.  With each wave
// converting for itself 207.  Scores kept, 512 rows after 1536: 81.8, 134 MB of
// them among that.  256 dims would take a CU's LDS for one workgroup and stay
// with attn_q4_kernel.
#include "attention_q4.hpp"
#include "attention_q4_plan.hpp"
#include "launch.hpp"

namespace barq {

template <int HD>
struct Q4Block {
    static constexpr int NB = HD / 32, CT = HD / 16;
    static constexpr int V = 2 * NB * 1024, KS = V + 2 * CT * 1024, STAGE = KS + 2 * HD;
    static constexpr int W = HD / 64;   // fragments of K, and of V, that a wave converts
    static_assert(2 * NB == W * Q4P_NW && CT == W * Q4P_NW, "whole fragments");

    __amdgpu_buffer_rsrc_t kc, vc, ks, vs;   // from the range's first position (a multiple of 8)
    uint32_t k[W], v[W], sc[4], kscale;      // raw codes, V's scales of this wave's block, K's scales
    int c, g, wave;

    __device__ __forceinline__ void init(const Q4View& kv, int hk, int j0, int j1, int l, int w) {
        const size_t co = (size_t)hk * kv.code_head + (size_t)j0 * (HD / 2), cs = (size_t)hk * kv.scale_head + (size_t)j0 * (HD / 16);
        const uint32_t n = (uint32_t)(j1 - j0 + KV_TILE - 1) / KV_TILE * KV_TILE;   // whole tiles: behind them zeros
        const auto rsrc = [](uint8_t* p, uint32_t bytes) { return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, (int)bytes, 0x00020000); };
        kc = rsrc(kv.kc + co, n * (HD / 2));
        vc = rsrc(kv.vc + co, n * (HD / 2));
        ks = rsrc(kv.ks + cs, n * (HD / 16));
        vs = rsrc(kv.vs + cs, n * (HD / 16));
        c = l & 15;
        g = l >> 4;
        wave = w;
    }
    __device__ __forceinline__ bool has_kscale() const { return 256 * wave + 4 * (16 * g + c) < 2 * HD; }
    // K of S tile wave % 2, blocks W * (wave / 2) ..; V of dims 16 (W * wave + i) + c
    __device__ __forceinline__ void load(int at) {   // at: positions from j0
        const uint32_t ca = at * (HD / 2), sa = at * (HD / 16);
        const uint32_t ko = (8 * (c / 4) + 4 * (wave & 1) + c % 4) * (HD / 2) + g * (HD / 8) + 4 * W * (wave >> 1);
        const uint32_t vo = g * (KV_TILE * HD / 2) + c * (HD / 4) + 4 * W * wave;
        if constexpr (W == 2) {
            const auto a = __builtin_amdgcn_raw_buffer_load_b64(kc, ko, ca, 0), b = __builtin_amdgcn_raw_buffer_load_b64(vc, vo, ca, 0);
            k[0] = (uint32_t)a[0]; k[1] = (uint32_t)a[1];
            v[0] = (uint32_t)b[0]; v[1] = (uint32_t)b[1];
        } else {
            k[0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(kc, ko, ca, 0);
            v[0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(vc, vo, ca, 0);
        }
        const auto s = __builtin_amdgcn_raw_buffer_load_b128(vs, g * (KV_TILE * HD / 16) + 16 * (W * wave / 2), sa, 0);
        #pragma unroll
        for (int j = 0; j < 4; j++) sc[j] = (uint32_t)s[j];
        if (has_kscale()) kscale = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(ks, 256 * wave + 4 * (16 * g + c), sa, 0);
    }
    // base: the block's first position of the cache
    __device__ __forceinline__ void convert(uint8_t* st, int base, int j1, const Q4Const& kx, int* nan_at) {
        const int l = 16 * g + c;
        #pragma unroll
        for (int i = 0; i < W; i++)
            *reinterpret_cast<h8v*>(st + 1024 * ((wave & 1) * NB + W * (wave >> 1) + i) + 16 * l) = q4_k_frag(k[i], kx);
        if (has_kscale()) *reinterpret_cast<uint32_t*>(st + KS + 256 * wave + 4 * l) = kscale;
        const int at = base + 8 * g;
        u32x4v s{sc[0], sc[1], sc[2], sc[3]};
        if (base + Q4A_STEP > j1)   // what lies behind the range is not the cache's
            #pragma unroll
            for (int j = 0; j < 4; j++) s[j] &= (at + 2 * j < j1 ? 0xFFFFu : 0u) | (at + 2 * j + 1 < j1 ? 0xFFFF0000u : 0u);
        // scales are finite or NaN: an exponent of ones (adding one to it carries out)
        uint32_t top = 0;
        #pragma unroll
        for (int j = 0; j < 4; j++) top |= (((s[j] & 0x7C007C00u) >> 1) + 0x02000200u) & 0x40004000u;
        if (__any(top)) {
            int first = 0x7FFFFFFF;
            #pragma unroll
            for (int j = 3; j >= 0; j--) {
                const uint32_t w = s[j];
                const bool hi = (w & 0x7C000000u) == 0x7C000000u, lo = (w & 0x7C00u) == 0x7C00u;
                first = hi ? at + 2 * j + 1 : first;
                first = lo ? at + 2 * j : first;
                s[j] = w & (hi ? 0x0000FFFFu : 0xFFFFFFFFu) & (lo ? 0xFFFF0000u : 0xFFFFFFFFu);
            }
            if (c == 0 && first != 0x7FFFFFFF) atomicMin(&nan_at[W * wave / 2], first);
        }
        #pragma unroll
        for (int i = 0; i < W; i++) {
            h8v hi, lo;
            q4_v_frag(v[i], s, kx, hi, lo);
            *reinterpret_cast<h8v*>(st + V + 2048 * (W * wave + i) + 16 * l) = hi;
            *reinterpret_cast<h8v*>(st + V + 2048 * (W * wave + i) + 1024 + 16 * l) = lo;
        }
    }
};

// Workgroup x: group of G heads x % groups, then split, then row tile from the
// last one down.  The longest tiles of all heads start first (2048 tokens when this was
// chosen: 128 us, and 170 with one head's tiles before the next head's), and
// with eight kv heads an XCD keeps to one of them.
template <int HD, bool PART, bool SC>
__global__ __launch_bounds__(64 * Q4P_NW, 3)
void attn_q4_prompt_kernel(Q4Args a) {
    using B = Q4Block<HD>;
    __shared__ __align__(16) uint8_t lds[2 * B::STAGE];
    __shared__ int nan_at[B::NB];
    const int t = threadIdx.x, l = t & 63, c = l & 15, g = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int grp = (int)(blockIdx.x % a.groups), part = (int)(blockIdx.x / a.groups), rows_n = a.q_len * a.G;
    const int tile = a.tiles - 1 - part / a.n_split, split = part % a.n_split;
    const int hk = (int)((long long)(grp * a.G) * a.n_head_kv / a.n_head);
    const int visible = q4_vis(a, tile * Q4P_ROWS + Q4P_ROWS - 1);
    const int start = split * a.chunk, j0 = min(start, visible), j1 = q4_range_end(start, a.chunk, visible);
    const int r0 = tile * Q4P_ROWS + wave * Q4A_ROWS;
    const int mine = r0 < rows_n ? min(j1, q4_vis(a, r0 + Q4A_ROWS - 1)) : 0;   // the wave's rows see no more

    B blk;
    blk.init(a.kv, hk, start, max(j1, start), l, wave);
    const int n = (j1 - j0 + Q4A_STEP - 1) / Q4A_STEP;
    if (n > 0) blk.load(0);
    if (t < B::NB) nan_at[t] = 0x7FFFFFFF;
    const Q4Const kx;
    const Q4Row row = q4_row(a, grp, r0 + c);
    const Q4Seen seen{min(row.vis, j1), min(q4_vis(a, r0), j1)};
    Q4Query<HD> q;
    const float lost = uniform(row16_max(q.load(a.q + ((size_t)row.h * a.q_rows + row.i) * HD, a.scale, g, kx)));
    float* const score_row = SC && row.ok ? a.scores + ((size_t)row.i * a.n_head + row.h) * a.score_stride : nullptr;
    Q4State<HD> st;
    st.clear();
    __syncthreads();   // nan_at
    if (n > 0) blk.convert(lds, j0, j1, kx, nan_at);
    if (n > 1) blk.load(Q4A_STEP);
    for (int b = 0; b < n; b++) {
        __syncthreads();   // block b is in its stage, and every wave is done with the other one
        if (b + 1 < n) blk.convert(lds + ((b + 1) & 1) * B::STAGE, j0 + (b + 1) * Q4A_STEP, j1, kx, nan_at);
        if (b + 2 < n) blk.load((b + 2) * Q4A_STEP);
        const int base = j0 + b * Q4A_STEP;
        if (base >= mine) continue;
        const uint8_t* s = lds + (b & 1) * B::STAGE;
        float x[8];
        q4_scores<HD>(x, q, lost,
                      [&](int t, int b, bool) { return *reinterpret_cast<const h8v*>(s + 1024 * (t * B::NB + b) + 16 * l); },
                      [&](int b) { return *reinterpret_cast<const u32x4v*>(s + B::KS + 16 * (g * B::NB + b)); });
        q4_attend<HD, SC>(x, base, base + 8 * g, seen, q, kx, st, score_row, [&](int c, h8v& hi, h8v& lo) {
            hi = *reinterpret_cast<const h8v*>(s + B::V + 2048 * c + 16 * l);
            lo = *reinterpret_cast<const h8v*>(s + B::V + 2048 * c + 1024 + 16 * l);
        });
    }
    __syncthreads();   // nan_at
    st.put_nan(nan_at, seen.end);
    const float lsum = groups_sum(st.l);
    if (row.ok) q4_store<HD, PART>(a, row, split, g, st, lsum);
}

template <int HD>
static hipError_t prompt_launch_t(const Q4Args& a, hipStream_t s) {
    const dim3 grid((unsigned)a.tiles * (unsigned)a.n_split * (unsigned)a.groups), block(64 * Q4P_NW);
    if (a.scores) hipLaunchKernelGGL((attn_q4_prompt_kernel<HD, true, true>), grid, block, 0, s, a);
    else if (a.n_split > 1) hipLaunchKernelGGL((attn_q4_prompt_kernel<HD, true, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attn_q4_prompt_kernel<HD, false, false>), grid, block, 0, s, a);
    return hipGetLastError();
}

hipError_t attn_q4_prompt_launch(const Q4Args& a, size_t head_dim, hipStream_t s) {
    return head_dim == 64 ? prompt_launch_t<64>(a, s) : prompt_launch_t<128>(a, s);
}

}  // namespace barq
