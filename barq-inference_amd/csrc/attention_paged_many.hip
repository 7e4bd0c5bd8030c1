// Attention over a paged KV cache of f16 rows for sequences with many rows (new tokens
// x the query heads of a kv head): prompts and their chunks.  attention_paged.hpp has
// the formulas and numerics, attention_paged_f32.hip the kernel for f32 rows.
//
// Bound by the matrix products: two of f16 for each of an f32 result's.  A workgroup
// is four waves of 32 rows each, the queries in registers; a step's K and V (64
// positions) come by direct loads into one of two LDS buffers while the other is
// computed on.  The pages' blocks are the MFMA operands' layout already, so they
// are copied as they lie and read without bank conflicts: wave w fetches block w.
// 2048 tokens of 32 heads of 128 dims after 6000 positions: 442 to 472 us by card, 533 to 500 TFLOP/s counted once, twice
// that of f16 products.  The card's power holds that down, not a wait: a loop of nothing but these products reaches 2570
// TFLOP/s on equal operands, 1670 on random ones, 1190 with 8 fmas beside each (a step has 320 vector instructions
// for 64 products); an 8192^3 f16 product has 1158.  So what counts is instructions left out: O in scalars (as
// vectors they are copied once a step), what a row sees as bits (a step at a window's edge takes a third fewer): together
// 464 -> 454 here, 102 -> 96 for 4000 tokens of 64 dims that see 1024 back (half the products for the same softmax), 96 -> 91
// for attention_mixed's 256 dims (446 registers, one wave a SIMD).
#include "attention_paged.hpp"

namespace barq {

namespace {

constexpr int NW = 4;   // waves, of which each fetches a block of a step's four

// sched_barrier: vector and scalar arithmetic may move across, loads and matrix products stay where they are
#define BARQ_ONLY_ALU_CROSSES 0x0006

__device__ __forceinline__ float halves_max(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (int)b[0]), __builtin_bit_cast(float, (int)b[1]));
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Register r of a lane of half h is position 16 (r / 8) + 8 h + r % 8 of a tile of 32: row i of the MFMA stands for
// position 16 (i / 16) + 8 (i / 4 % 2) + 4 (i / 8 % 2) + i % 4, so that a half's eight positions of a block are one piece of V.

// Two weights as f16 hi (cut, one instruction for both) + lo (of what that leaves, to the nearest).
__device__ __forceinline__ void split_weights(float x0, float x1, float minus_one, uint32_t& hi, uint32_t& lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    asm("" : "+v"(hi));
    const h2v h = __builtin_bit_cast(h2v, hi);
    const float r0 = __builtin_fmaf((float)h[0], minus_one, x0), r1 = __builtin_fmaf((float)h[1], minus_one, x1);
    const h2v r = {(_Float16)r0, (_Float16)r1};
    lo = __builtin_bit_cast(uint32_t, r);
}

__device__ __forceinline__ u32x4v finite(u32x4v v) {
    #pragma unroll
    for (int e = 0; e < 4; e++) v[e] &= ~f16_bad(v[e]);
    return v;
}

template <int HD>
__global__ __launch_bounds__(64 * NW, HD == 256 ? 1 : 2)
void paged_many_kernel(PagedAttn a, int count) {
    constexpr int STEP = 64, T = STEP / 32, NB = STEP / PAGE_BLOCK, NC = HD / 16, ND = HD / 32;
    constexpr int BLOCK = PAGE_BLOCK * HD * 2;   // bytes
    extern __shared__ __align__(16) uint8_t lds[];         // [2][K, V][NB][BLOCK]
    __shared__ int bad_s[2][NW];                           // whether a step's block of V has what is not finite
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    int n_tokens = a.n_tokens;
    if (n_tokens < 0) {
        n_tokens = a.counts->n_tokens;
        count = a.counts->many;
    }
    const float minus_one = f16_minus_one();
    const PagedSight sight = {a.window, a.n_sink};
    const size_t page_bytes = (size_t)BLOCK << (a.log_page - 4);   // of one kv head
    const uint32_t lds0 = lds_addr(lds);
    for (int w = blockIdx.x; w < count * a.n_kv; w += gridDim.x) {
        const int hk = w % a.n_kv;
        const PagedItem it = paged_item(&a.many[w / a.n_kv]);
        const int32_t* table = a.table + it.table;
        const int steps = it.v1 - it.v0;
        const auto base_of = [&](int j) {
            const int v = it.v0 + j;
            return (v < it.a ? v : v - it.a + it.b) * STEP;
        };
        // lane j: of step 64 n + j the page of the block that this wave fetches, and which blocks have one
        int id = -1, has = 0;
        const auto fetch_ids = [&](int j0) {
            id = -1, has = 0;
            if (j0 + lane < steps) {
                const int at = base_of(j0 + lane);
                #pragma unroll
                for (int b = 0; b < NB; b++) {
                    const int p = at + 16 * b < it.kv_len ? table[(at + 16 * b) >> a.log_page] : -1;
                    has |= p >= 0 ? 1 << b : 0;
                    if (b == wave) id = p;
                }
            }
        };
        const auto fetch = [&](int j, int has_all) {
            const int p = __builtin_amdgcn_readlane(id, j & 63), at = base_of(j) + 16 * wave;
            const size_t off = ((size_t)max(p, 0) * a.n_kv + hk) * page_bytes + (size_t)((at & ((1 << a.log_page) - 1)) >> 4) * BLOCK;
            #pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                i32x4v r = make_rsrc4((kv ? a.v : a.k) + off, (has_all >> wave) & 1 ? BLOCK : 0);   // (no page: zeros)
                #pragma unroll
                for (int e = 0; e < 4; e++) r[e] = __builtin_amdgcn_readfirstlane(r[e]);
                const uint32_t to = lds0 + (((j & 1) * 2 + kv) * NB + wave) * BLOCK;
                #pragma unroll
                for (int u = 0; u < BLOCK / 1024; u++) lds_load16_at(r, to + 1024 * u, lane * 16, 1024 * u);
            }
        };
        fetch_ids(0);
        int has_now = __builtin_amdgcn_readlane(has, 0), has_next = 0;
        fetch(0, has_now);
        // the wave's rows
        const int row0 = it.row0 + 32 * wave, end = it.row0 + it.rows, mine = min(row0 + i, end - 1), tok = mine / a.G;
        const int pos = it.past + tok, p_first = it.past + min(row0, end - 1) / a.G, p_last = it.past + min(row0 + 31, end - 1) / a.G;
        const int all_first = it.past + it.row0 / a.G, all_last = it.past + (end - 1) / a.G;
        u32x4v qh[NC], ql[NC];
        float back = 1.0f;
        {
            const float* row = a.q + ((size_t)(hk * a.G + mine % a.G) * n_tokens + it.q0 + tok) * HD;
            float m = 0.0f;
            #pragma unroll
            for (int c = 0; c < 2 * NC; c++) {
                const float4 y = *reinterpret_cast<const float4*>(row + 16 * (c / 2) + 8 * h + 4 * (c & 1));
                m = fmaxf(fmaxf(fmaxf(m, __builtin_fabsf(y.x * a.scale)), fmaxf(__builtin_fabsf(y.y * a.scale), __builtin_fabsf(y.z * a.scale))),
                          __builtin_fabsf(y.w * a.scale));
            }
            const float up = paged_row_scale(halves_max(m), back);
            #pragma unroll
            for (int c = 0; c < NC; c++)
                #pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float4 y = *reinterpret_cast<const float4*>(row + 16 * c + 8 * h + 4 * u);
                    uint32_t x0, y0, x1, y1;
                    paged_split(y.x * a.scale * up, y.y * a.scale * up, x0, y0);
                    paged_split(y.z * a.scale * up, y.w * a.scale * up, x1, y1);
                    qh[c][2 * u] = x0, qh[c][2 * u + 1] = x1;
                    ql[c][2 * u] = y0, ql[c][2 * u + 1] = y1;
                }
        }
        if constexpr (HD == 256) {
            // (256 registers of a wave take only products' operands and results: the queries)
            #pragma unroll
            for (int c = 0; c < NC; c++) {
                asm("" : "+a"(qh[c]));
                asm("" : "+a"(ql[c]));
            }
        }
        float m = -INFINITY, l = 0.0f;
        float o[ND][16];
        #pragma unroll
        for (int d = 0; d < ND; d++)
            #pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
        for (int j = 0; j < steps; j++) {
            const int base = base_of(j), have = has_now;
            uint8_t *kt = lds + (size_t)(j & 1) * 2 * NB * BLOCK, *vt = kt + NB * BLOCK;
            const bool edge = have != (1 << NB) - 1 || !sight.all(base, STEP, all_first, all_last);
            wait_vmcnt<0>();
            asm volatile("" ::: "memory");
            if (edge) {   // (each wave looks through the block that it fetched)
                uint32_t any = 0;
                #pragma unroll
                for (int u = 0; u < BLOCK / 1024; u++) {
                    const u32x4v x = reinterpret_cast<const u32x4v*>(vt + wave * BLOCK)[64 * u + lane];
                    #pragma unroll
                    for (int e = 0; e < 4; e++) any |= f16_bad_mark(x[e]);
                }
                const bool found = __any((any & 0x80008000u) != 0);
                if (lane == 0) bad_s[j & 1][wave] = found;
            }
            __syncthreads();   // the step is there for all waves, and none still reads the other buffer
            if (j + 1 < steps) {
                if (((j + 1) & 63) == 0) fetch_ids(j + 1);
                has_next = __builtin_amdgcn_readlane(has, (j + 1) & 63);
                fetch(j + 1, has_next);
            }
            has_now = has_next;
            // bit 16 (r / 8) + r % 8 of word t: the lane's row sees its register r of tile t
            const bool whole = have == (1 << NB) - 1 && sight.all(base, STEP, p_first, p_last);
            uint32_t seen[T];
            if (!whole) {
                uint64_t m = sight.mask(pos, base);
                #pragma unroll
                for (int b = 0; b < NB; b++) m &= (have >> b) & 1 ? ~0ull : ~(0xFFFFull << (16 * b));
                m >>= 8 * h;
                seen[0] = (uint32_t)m;
                seen[1] = (uint32_t)(m >> 32);
            }
            if (edge) {
                // some row of the workgroup does not see all of the step: what is not finite in V becomes zero, after it
                // has been put as NaN into the dims of the rows that see it (all waves find the same)
                if (bad_s[j & 1][0] | bad_s[j & 1][1] | bad_s[j & 1][2] | bad_s[j & 1][3]) {
                    if (whole) seen[0] = seen[1] = ~0u;
                    #pragma unroll
                    for (int d = 0; d < ND; d++) {
                        f32x16 n = {};   // such places that a row sees
                        #pragma unroll
                        for (int t = 0; t < T; t++) {
                            #pragma unroll
                            for (int u = 0; u < 2; u++) {
                                u32x4v v = *reinterpret_cast<const u32x4v*>(vt + (2 * t + u) * BLOCK + (h * HD + 32 * d + i) * 16), one;
                                #pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const uint32_t two = seen[t] >> (16 * u + 2 * e);
                                    v[e] = f16_bad(v[e]) & 0x3C003C00u;
                                    one[e] = (two & 1 ? 0x3C00u : 0u) | (two & 2 ? 0x3C000000u : 0u);
                                }
                                n = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, v), __builtin_bit_cast(h8v, one), n, 0, 0, 0);
                            }
                        }
                        #pragma unroll
                        for (int r = 0; r < 16; r++) o[d][r] = n[r] > 0.0f ? NAN : o[d][r];
                    }
                    __syncthreads();
                    for (int u = threadIdx.x; u < NB * BLOCK / 16; u += 64 * NW) {
                        u32x4v* x = reinterpret_cast<u32x4v*>(vt) + u;
                        *x = finite(*x);
                    }
                    __syncthreads();
                }
            }
            // scores: the next pieces of K are fetched while the products of these run
            constexpr int KG = 4, GC = NC / KG;
            float s[T][16];
            u32x4v kf[2][KG];
            const auto keys = [&](int n, u32x4v (&k)[KG]) __attribute__((always_inline)) {
                const int t = n / GC, slot = 8 * ((i >> 2) & 1) + 4 * ((i >> 3) & 1) + (i & 3);
                const uint8_t* kb = kt + (2 * t + (i >> 4)) * BLOCK + slot * 16 + h * 256;
                #pragma unroll
                for (int u = 0; u < KG; u++) k[u] = *reinterpret_cast<const u32x4v*>(kb + (n % GC * KG + u) * 512);
            };
            keys(0, kf[0]);
            f32x16 hi, lo;
            #pragma unroll
            for (int n = 0; n < T * GC; n++) {
                if (n + 1 < T * GC) keys(n + 1, kf[(n + 1) & 1]);
                __builtin_amdgcn_sched_barrier(BARQ_ONLY_ALU_CROSSES);
                if (n % GC == 0) hi = lo = f32x16{};
                #pragma unroll
                for (int u = 0; u < KG; u++) {
                    const int c = n % GC * KG + u;
                    const h8v k = __builtin_bit_cast(h8v, kf[n & 1][u]);
                    lo = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, __builtin_bit_cast(h8v, ql[c]), lo, 0, 0, 0);
                    hi = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, __builtin_bit_cast(h8v, qh[c]), hi, 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(BARQ_ONLY_ALU_CROSSES);
                if (n % GC == GC - 1) {
                    #pragma unroll
                    for (int r = 0; r < 16; r++) s[n / GC][r] = __builtin_fmaf(lo[r], 1.0f / 2048, hi[r]);
                }
            }
            if (!whole) {
                #pragma unroll
                for (int t = 0; t < T; t++)
                    #pragma unroll
                    for (int r = 0; r < 16; r++) s[t][r] = seen_or_none(s[t][r], bit_as_mask(seen[t], 16 * (r / 8) + r % 8));
            }
            float top = s[0][0];
            #pragma unroll
            for (int t = 0; t < T; t++)
                #pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, s[t][r]);
            top = fmaxf(m, halves_max(top) * back);
            const float ref = top == -INFINITY ? 0.0f : top, alpha = paged_exp2(m - ref);
            m = top;
            // exponents s * back - ref + 15 in one fma, unless 15 - ref would round by more than 2^-4
            float mul = back, shift = 15.0f - ref;
            if (__any(__builtin_fabsf(ref) > 1048576.0f)) {
                #pragma unroll
                for (int t = 0; t < T; t++)
                    #pragma unroll
                    for (int r = 0; r < 16; r++) s[t][r] = s[t][r] * back - ref;
                mul = 1.0f, shift = 15.0f;
            }
            float sum = 0.0f;
            u32x4v ph[T][2], pl[T][2];
            #pragma unroll
            for (int t = 0; t < T; t++) {
                #pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[t][r] = paged_exp2(__builtin_fmaf(s[t][r], mul, shift));
                    sum += s[t][r];
                }
                #pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    uint32_t x, y;
                    split_weights(s[t][r], s[t][r + 1], minus_one, x, y);
                    ph[t][r / 8][r % 8 / 2] = x;
                    pl[t][r / 8][r % 8 / 2] = y;
                }
            }
            l = __builtin_fmaf(l, alpha, sum);
            // O: the next 32 dims' pieces of V likewise; the weights' small parts first, so that fewer sums are cut at y's size
            constexpr int PIECES = 2 * T;
            u32x4v vf[2][PIECES];
            const auto values = [&](int d, u32x4v (&v)[PIECES]) __attribute__((always_inline)) {
                #pragma unroll
                for (int u = 0; u < PIECES; u++)
                    v[u] = *reinterpret_cast<const u32x4v*>(vt + u * BLOCK + (h * HD + 32 * d + i) * 16);
            };
            values(0, vf[0]);
            f32x16 y[2];
            const auto join = [&](int d, int r) __attribute__((always_inline)) { o[d][r] = __builtin_fmaf(o[d][r], alpha, y[d & 1][r]); };
            #pragma unroll
            for (int d = 0; d < ND; d++) {
                if (d + 1 < ND) values(d + 1, vf[(d + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
                #pragma unroll
                for (int u = 0; u < 2 * PIECES; u++) {
                    const int at = u % PIECES;
                    const u32x4v w = u < PIECES ? pl[at / 2][at & 1] : ph[at / 2][at & 1];
                    y[d & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, vf[d & 1][at]), __builtin_bit_cast(h8v, w), u ? y[d & 1] : f32x16{}, 0, 0, 0);
                    // (the dims before these join in the products' shadow)
                    if (d) {
                        #pragma unroll
                        for (int r = u * 16 / (2 * PIECES); r < (u + 1) * 16 / (2 * PIECES); r++) join(d - 1, r);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            #pragma unroll
            for (int r = 0; r < 16; r++) join(ND - 1, r);
        }
        const float sum = swap32_add(l, l);
        if (row0 + i < end) {
            if (it.part < 0) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                float* out = a.out + ((size_t)(it.q0 + tok) * a.n_head + hk * a.G + mine % a.G) * HD;
                #pragma unroll
                for (int d = 0; d < ND; d++)
                    #pragma unroll
                    for (int r = 0; r < 16; r++) out[32 * d + 8 * (r / 4) + 4 * h + r % 4] = o[d][r] * inv;
            } else {
                const size_t at = (size_t)hk * a.part_rows + it.part + (mine - it.row0);
                float* out = a.part + at * HD;
                #pragma unroll
                for (int d = 0; d < ND; d++)
                    #pragma unroll
                    for (int r = 0; r < 16; r++) out[32 * d + 8 * (r / 4) + 4 * h + r % 4] = o[d][r];
                if (h == 0) a.stat[at] = make_float2(m, sum);
            }
        }
        __syncthreads();   // (a next item's first loads go where this one's last step may be read from)
    }
}

template <int HD>
hipError_t launch(const PagedAttn& a, hipStream_t s) {
    constexpr unsigned bytes = 2 * 2 * 64 * HD * 2;
    if (bytes > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_many_kernel<HD>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return e;
    }
    const dim3 g(a.n_tokens < 0 ? 1024u : (unsigned)a.n_many * (unsigned)a.n_kv);
    hipLaunchKernelGGL(paged_many_kernel<HD>, g, dim3(64 * NW), bytes, s, a, a.n_many);
    return hipGetLastError();
}

}  // namespace

hipError_t paged_many_launch(const PagedAttn& a, bool f16, int hd, hipStream_t s) {
    if (!f16) return paged_many_f32_launch(a, hd, s);
    return hd == 64 ? launch<64>(a, s) : hd == 128 ? launch<128>(a, s) : launch<256>(a, s);
}

}  // namespace barq
