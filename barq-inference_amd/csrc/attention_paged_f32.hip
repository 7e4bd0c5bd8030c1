// Attention over a paged KV cache of f32 rows for sequences with many rows: prompts
// and their chunks.  attention_paged.hpp has the formulas and numerics.
//
// Bound by the matrix products: six of bf16 for each f32 product.  An f32 value is
// exactly the sum of three bf16 values (8 bits each, f32's exponents: below 2^-110 the last has fewer bits), so that the three
// largest products of two values' parts and the three next are within 2^-23 of |x y|;
// the sums of the five smaller ones are kept apart from the largest's, so that the MFMA's cuts count
// a few times only.  That is 2.7 times the rate of the f32 MFMA.  A workgroup is four waves of 32 rows,
// the queries' parts in registers; a step's 32 positions come by direct loads into LDS as they lie, the waves share
// their conversion into the operands' layout there, and the next step is fetched while this one is computed on.
// A 2048-token prompt of 32 heads on 8, 128 dims: 259 to 273 us by card, 130 TFLOP/s counted once (on the f32 MFMA 397, which
// reaches 154 in an 8192^3 product).
#include "attention_paged.hpp"

namespace barq {

namespace {

constexpr int NW = 4, STEP = 32, NB = 2, PARTS = 3;   // waves, positions and blocks of a step, bf16 values of an f32 one

typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float halves_max(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (int)b[0]), __builtin_bit_cast(float, (int)b[1]));
}

// Two values -> three pairs of bf16.
__device__ __forceinline__ void split3(float x0, float x1, uint32_t (&p)[PARTS]) {
    #pragma unroll
    for (int k = 0; k < PARTS; k++) {
        const b2v h = {(__bf16)x0, (__bf16)x1};
        p[k] = __builtin_bit_cast(uint32_t, h);
        x0 -= __builtin_bit_cast(float, p[k] << 16);
        x1 -= __builtin_bit_cast(float, p[k] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void split3(const float (&x)[8], u32x4v (&p)[PARTS]) {
    #pragma unroll
    for (int u = 0; u < 4; u++) {
        uint32_t w[PARTS];
        split3(x[2 * u], x[2 * u + 1], w);
        #pragma unroll
        for (int k = 0; k < PARTS; k++) p[k][u] = w[k];
    }
}
// What split3 makes infinite or NaN: NaN, infinities, and finite values that round to bf16's infinity.  As a mark in bit 31
// (other bits say nothing), as a mask.
__device__ __forceinline__ uint32_t wild_mark(uint32_t x) { return (x & 0x7FFFFFFFu) + 0x00808000u; }
__device__ __forceinline__ uint32_t wild(uint32_t x) { return (x & 0x7FFFFFFFu) >= 0x7F7F8000u ? 0xFFFFFFFFu : 0u; }
__device__ __forceinline__ f32x16 product(u32x4v a, u32x4v b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}

// LDS: raw K, V as in the pages, then their parts: K [part][HD / 8][32 positions][8 dims], V [part][4][HD][8 positions], of
// which chunk 2 u + h holds positions 16 u + 4 h + {0 .. 3, 8 .. 11}: register 8 u + e of a lane of half h of S^T is position
// 16 u + 4 h + 8 (e / 4) + e % 4.
template <int HD>
__global__ __launch_bounds__(64 * NW, HD == 256 ? 1 : 2)
void paged_many_f32_kernel(PagedAttn a, int count) {
    constexpr int BLOCK = PAGE_BLOCK * HD * 4, RAW = NB * BLOCK, PLANE = STEP * HD * 2, NC = HD / 16, ND = HD / 32;
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *const raw_k = lds, *const raw_v = lds + RAW, *const part_k = lds + 2 * RAW, *const part_v = part_k + PARTS * PLANE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    int n_tokens = a.n_tokens;
    if (n_tokens < 0) {
        n_tokens = a.counts->n_tokens;
        count = a.counts->many;
    }
    const PagedSight sight = {a.window, a.n_sink};
    const size_t page_bytes = (size_t)BLOCK << (a.log_page - 4);   // of one kv head
    const uint32_t lds0 = lds_addr(lds);
    for (int w = blockIdx.x; w < count * a.n_kv; w += gridDim.x) {
        const int hk = w % a.n_kv;
        const PagedItem it = paged_item(&a.many[w / a.n_kv]);
        const int32_t* table = a.table + it.table;
        const int steps = it.v1 - it.v0;
        const float unit = paged_weight_unit(it.kv_len);
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
                    if (b == (wave & 1)) id = p;
                }
            }
        };
        const auto fetch = [&](int j, int has_all) {   // K by waves 0 and 1, V by the others, a block each
            const int blk = wave & 1, kv = wave >> 1, p = __builtin_amdgcn_readlane(id, j & 63), at = base_of(j) + 16 * blk;
            const size_t off = ((size_t)max(p, 0) * a.n_kv + hk) * page_bytes + (size_t)((at & ((1 << a.log_page) - 1)) >> 4) * BLOCK;
            i32x4v r = make_rsrc4((kv ? a.v : a.k) + off, (has_all >> blk) & 1 ? BLOCK : 0);   // (no page: zeros)
            #pragma unroll
            for (int e = 0; e < 4; e++) r[e] = __builtin_amdgcn_readfirstlane(r[e]);
            const uint32_t to = lds0 + (kv * NB + blk) * BLOCK;
            #pragma unroll
            for (int u = 0; u < BLOCK / 1024; u++) lds_load16_at(r, to + 1024 * u, lane * 16, 1024 * u);
        };
        fetch_ids(0);
        int has_now = __builtin_amdgcn_readlane(has, 0), has_next = 0;
        fetch(0, has_now);
        // the wave's rows
        const int row0 = it.row0 + 32 * wave, end = it.row0 + it.rows, mine = min(row0 + i, end - 1), tok = mine / a.G;
        const int pos = it.past + tok, p_first = it.past + min(row0, end - 1) / a.G, p_last = it.past + min(row0 + 31, end - 1) / a.G;
        const int all_first = it.past + it.row0 / a.G, all_last = it.past + (end - 1) / a.G;
        u32x4v q[PARTS][NC];
        {
            const float* row = a.q + ((size_t)(hk * a.G + mine % a.G) * n_tokens + it.q0 + tok) * HD;
            #pragma unroll
            for (int c = 0; c < NC; c++) {
                float x[8];
                #pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float4 y = *reinterpret_cast<const float4*>(row + 16 * c + 8 * h + 4 * u);
                    x[4 * u] = y.x * a.scale, x[4 * u + 1] = y.y * a.scale, x[4 * u + 2] = y.z * a.scale, x[4 * u + 3] = y.w * a.scale;
                }
                u32x4v p[PARTS];
                split3(x, p);
                #pragma unroll
                for (int k = 0; k < PARTS; k++) {
                    q[k][c] = p[k];
                    if constexpr (HD == 256) asm("" : "+a"(q[k][c]));   // (as in attention_paged_many.hip)
                }
            }
        }
        float m = -INFINITY, l = 0.0f;
        f32x16 o[ND];
        #pragma unroll
        for (int d = 0; d < ND; d++) o[d] = f32x16{};
        for (int j = 0; j < steps; j++) {
            wait_vmcnt<0>();
            __syncthreads();   // the step is there for all waves, and none still reads the parts of the one before
            const int base = base_of(j), have = has_now;
            // bit 8 (r / 4) + r % 4: the lane's row sees its register r
            const auto seen_by = [&]() __attribute__((always_inline)) {
                uint32_t m = (uint32_t)sight.mask(pos, base);
                #pragma unroll
                for (int b = 0; b < NB; b++) m &= (have >> b) & 1 ? ~0u : ~(0xFFFFu << (16 * b));
                return m >> (4 * h);
            };
            // Where some row of the workgroup does not see all of the step: what has no finite parts in V becomes zero, after it
            // has been put as NaN into the dims of the rows that see it (a weight of zero times infinity is not zero).
            const bool edge = have != (1 << NB) - 1 || !sight.all(base, STEP, all_first, all_last);
            if (edge) {
                uint32_t any = 0;
                for (int u = lane; u < RAW / 16; u += 64) {
                    const u32x4v x = reinterpret_cast<const u32x4v*>(raw_v)[u];
                    #pragma unroll
                    for (int e = 0; e < 4; e++) any |= wild_mark(x[e]);
                }
                if (__any((any >> 31) != 0)) {
                    const uint32_t seen = seen_by();
                    #pragma unroll
                    for (int d = 0; d < ND; d++) {
                        f32x16 n = {};   // such places that a row sees
                        #pragma unroll
                        for (int g = 0; g < 4; g++) {
                            const u32x4v v = *reinterpret_cast<const u32x4v*>(raw_v + (g / 2) * BLOCK + ((2 * (g & 1) + h) * HD + 32 * d + i) * 16);
                            #pragma unroll
                            for (int e = 0; e < 4; e++)
                                n = __builtin_amdgcn_mfma_f32_32x32x2f32(wild(v[e]) ? 1.0f : 0.0f, (seen >> (8 * g + e)) & 1 ? 1.0f : 0.0f, n, 0, 0, 0);
                        }
                        #pragma unroll
                        for (int r = 0; r < 16; r++) o[d][r] = n[r] > 0.0f ? NAN : o[d][r];
                    }
                }
            }
            // the step's parts
            for (int u = threadIdx.x; u < STEP * HD / 8; u += 64 * NW) {
                const int x = u & 31, c = u >> 5;   // position, dims 8 c ..
                const uint8_t* from = raw_k + (x >> 4) * BLOCK + (2 * c * 16 + (x & 15)) * 16;
                const f32x4 y0 = *reinterpret_cast<const f32x4*>(from), y1 = *reinterpret_cast<const f32x4*>(from + 256);
                const float y[8] = {y0[0], y0[1], y0[2], y0[3], y1[0], y1[1], y1[2], y1[3]};
                u32x4v p[PARTS];
                split3(y, p);
                #pragma unroll
                for (int k = 0; k < PARTS; k++) *reinterpret_cast<u32x4v*>(part_k + k * PLANE + u * 16) = p[k];
            }
            for (int u = threadIdx.x; u < STEP * HD / 8; u += 64 * NW) {
                const int d = u % HD, c = u / HD;   // dim, chunk 2 u + h
                const uint8_t* from = raw_v + (c >> 1) * BLOCK + ((c & 1) * HD + d) * 16;
                u32x4v y0 = *reinterpret_cast<const u32x4v*>(from), y1 = *reinterpret_cast<const u32x4v*>(from + 2 * HD * 16);
                if (edge) {
                    #pragma unroll
                    for (int e = 0; e < 4; e++) y0[e] &= ~wild(y0[e]), y1[e] &= ~wild(y1[e]);
                }
                const f32x4 x0 = __builtin_bit_cast(f32x4, y0), x1 = __builtin_bit_cast(f32x4, y1);
                const float y[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
                u32x4v p[PARTS];
                split3(y, p);
                #pragma unroll
                for (int k = 0; k < PARTS; k++) *reinterpret_cast<u32x4v*>(part_v + k * PLANE + u * 16) = p[k];
            }
            __syncthreads();   // the parts are there, and nothing reads the raw step any more
            f32x16 big = {}, small = {};
            #pragma unroll
            for (int c = 0; c < NC; c++) {
                u32x4v k[PARTS];
                #pragma unroll
                for (int p = 0; p < PARTS; p++) k[p] = *reinterpret_cast<const u32x4v*>(part_k + p * PLANE + ((2 * c + h) * 32 + i) * 16);
                small = product(k[2], q[0][c], small);
                small = product(k[0], q[2][c], small);
                small = product(k[1], q[1][c], small);
                small = product(k[1], q[0][c], small);
                small = product(k[0], q[1][c], small);
                big = product(k[0], q[0][c], big);
            }
            float s[16];
            #pragma unroll
            for (int r = 0; r < 16; r++) s[r] = small[r] + big[r];
            // (the next step's loads after the scores: what the compiler reloads for those from scratch would wait for them)
            if (j + 1 < steps) {
                if (((j + 1) & 63) == 0) fetch_ids(j + 1);
                has_next = __builtin_amdgcn_readlane(has, (j + 1) & 63);
                fetch(j + 1, has_next);
            }
            has_now = has_next;
            if (have != (1 << NB) - 1 || !sight.all(base, STEP, p_first, p_last)) {
                const uint32_t seen = seen_by();
                #pragma unroll
                for (int r = 0; r < 16; r++) s[r] = seen_or_none(s[r], bit_as_mask(seen, 8 * (r / 4) + r % 4));
            }
            float top = s[0];
            #pragma unroll
            for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
            top = fmaxf(m, halves_max(top));
            const float ref = top == -INFINITY ? 0.0f : top, alpha = paged_exp2(m - ref);
            m = top;
            float sum = 0.0f;
            u32x4v pw[2][PARTS];
            #pragma unroll
            for (int u = 0; u < 2; u++) {
                float y[8];
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    y[e] = paged_exp2(s[8 * u + e] - ref) * unit;
                    sum += y[e];
                }
                split3(y, pw[u]);
            }
            l = __builtin_fmaf(l, alpha, sum);
            #pragma unroll
            for (int d = 0; d < ND; d++) {
                u32x4v v[2][PARTS];
                #pragma unroll
                for (int u = 0; u < 2; u++)
                    #pragma unroll
                    for (int p = 0; p < PARTS; p++) v[u][p] = *reinterpret_cast<const u32x4v*>(part_v + p * PLANE + ((2 * u + h) * HD + 32 * d + i) * 16);
                f32x16 y = {};
                #pragma unroll
                for (int u = 0; u < 2; u++) {
                    y = product(v[u][2], pw[u][0], y);
                    y = product(v[u][0], pw[u][2], y);
                    y = product(v[u][1], pw[u][1], y);
                    y = product(v[u][1], pw[u][0], y);
                    y = product(v[u][0], pw[u][1], y);
                }
                #pragma unroll
                for (int u = 0; u < 2; u++) y = product(v[u][0], pw[u][0], y);
                #pragma unroll
                for (int r = 0; r < 16; r++) o[d][r] = __builtin_fmaf(o[d][r], alpha, y[r]);
            }
        }
        const float sum = swap32_add(l, l);
        if (row0 + i < end) {
            const bool whole = it.part < 0;
            const size_t at = (size_t)hk * a.part_rows + it.part + (mine - it.row0);
            const float f = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
            float* out = whole ? a.out + ((size_t)(it.q0 + tok) * a.n_head + hk * a.G + mine % a.G) * HD : a.part + at * HD;
            #pragma unroll
            for (int d = 0; d < ND; d++)
                #pragma unroll
                for (int r = 0; r < 16; r++) out[32 * d + 8 * (r / 4) + 4 * h + r % 4] = o[d][r] * f;
            if (!whole && h == 0) a.stat[at] = make_float2(m, sum);
        }
        __syncthreads();   // (a next item's first step goes where this one's last may be read from)
    }
}

template <int HD>
hipError_t launch(const PagedAttn& a, hipStream_t s) {
    constexpr unsigned bytes = 2 * (STEP * HD * 4 + PARTS * STEP * HD * 2);
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_many_f32_kernel<HD>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
    const dim3 g(a.n_tokens < 0 ? 1024u : (unsigned)a.n_many * (unsigned)a.n_kv);
    hipLaunchKernelGGL(paged_many_f32_kernel<HD>, g, dim3(64 * NW), bytes, s, a, a.n_many);
    return hipGetLastError();
}

}  // namespace

hipError_t paged_many_f32_launch(const PagedAttn& a, int hd, hipStream_t s) {
    return hd == 64 ? launch<64>(a, s) : hd == 128 ? launch<128>(a, s) : launch<256>(a, s);
}

}  // namespace barq
