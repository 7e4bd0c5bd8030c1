// Eviction from the KV cache: which positions each kv head keeps, and moving
// their rows together.
//
//   kept(h) = the newest `recent` positions and, of the others, the keep -
//   recent with the largest mass (equal masses: the earlier position), in the order
//   of their positions
//
// Selection: a workgroup per kv head looks for the want-th largest key (the
// mass as an unsigned integer of the same order) 11 bits at a time from the
// top, each time with a histogram of the keys that share the bits found so
// far, until all keys that share them are wanted; then it numbers the kept
// positions by a running count.  The histogram has four columns, since masses
// share their leading bits and lanes adding to one counter take turns.  Up to
// 16384 masses stay in LDS (and their keys in registers) over the passes, and the kept
// positions go through a list there, so that they leave by whole lines; longer
// heads are read again by each pass (from the L2).  One workgroup's latencies bound
// it, 14.5 us for 16384 positions: the load takes 3500 cycles, a pass 4000 to
// 6000.  Stores from where a thread finds a position, without the list, took
// 14400, and the zeros behind the kept masses, one a thread at a time, 4800.
//
// The rows then move in one launch (more where a launch would pass 2^32 threads), bound by
// memory: f32 rows as they are (2048 of 8 heads of 128 dims 7.0 us, 33.6 MB at
// 4.8 TB/s); of a 4-bit cache, whose tiles hold 8 positions of V in one dword per
// dim, a thread builds the dwords of a tile's dims from those of its 8 sources,
// which reads V's codes up to eight times (4096 of 16384 positions 7.7 us, 9.4 MB and
// the rest of the tiles' lines).  In place they go by way of the workspace, since a row may
// move onto one that is still to be read, and back: the 2048 f32 rows 6.5 us, 4096
// 4-bit ones 4.6.  A budget's own step, 2112 positions to 2048, takes 7.1 + 4.8
// + 3.2 us in 4 bits and 7.1 + 7.2 + 6.5 in f32.
#include "common.hpp"
#include "kv_evict_plan.hpp"
#include "kv_q4.hpp"
#include "launch.hpp"

namespace barq {

constexpr int EV_NT = 1024;
constexpr int EV_DIGITS = 2 * EV_NT;
constexpr int EV_COLS = 4;
constexpr int EV_CHUNK = 4 * EV_NT;   // keys of a pass over the workgroup, four in a row per thread
constexpr int EV_KEEP = 4 * EV_CHUNK;   // masses that stay in LDS

struct EvictArgs {
    const float* mass_in;
    float* mass_out;     // may be mass_in or null
    size_t stride;
    int n, m, recent;    // positions, kept ones, the newest among them
    int32_t* kept;       // [heads][m]
};

// The order of f32 values as unsigned integers; NaN as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t ev_key(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x != x ? -INFINITY : x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of the lanes before this one, and of all (64 lanes): within rows of 16
// by shifts, then the rows' last lanes to the rows behind them.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t& total) {
    int s = (int)v;
    s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xF, 0xF, true);
    s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xA, 0xF, false);
    s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xC, 0xF, false);
    total = (uint32_t)__builtin_amdgcn_readlane(s, 63);
    return (uint32_t)s - v;
}

// Sum of part[0 .. w), and of all 16 (w: the same in every lane).
__device__ __forceinline__ uint32_t waves_before(const uint32_t* part, int w, uint32_t& total) {
    const int l = threadIdx.x & 63;
    const uint32_t before = wave_scan(l < EV_NT / 64 ? part[l] : 0u, total);
    return (uint32_t)__builtin_amdgcn_readlane((int)before, w);
}

// LDS: the masses stay there, and their keys in registers (n <= EV_KEEP).
template <bool LDS>
__global__ __launch_bounds__(EV_NT)
void evict_select_kernel(EvictArgs a) {
    static_assert(EV_NT == 1024 && EV_DIGITS == 2 * EV_NT, "16 waves, two digits a thread");
    __shared__ __align__(16) uint32_t hist[EV_COLS][EV_DIGITS + 8];   // (a digit's columns on distinct banks)
    __shared__ __align__(16) float4 kept_in[LDS ? EV_KEEP / 4 : 1];
    __shared__ uint32_t part[EV_NT / 64];
    __shared__ uint32_t found[3];   // the digit, what is left to find within it, its keys
    const int t = threadIdx.x, l = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6), h = blockIdx.x;
    const float* in = a.mass_in + (size_t)h * a.stride;
    float* out = a.mass_out ? a.mass_out + (size_t)h * a.stride : nullptr;
    int32_t* kept = a.kept + (size_t)h * a.m;
    const int old = a.n - a.recent, want = a.m - a.recent, chunks = (a.n + EV_CHUNK - 1) / EV_CHUNK;

    // masses 4 q .. 4 q + 3, 0 behind the last
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const auto load = [&](int q) {
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (4 * q + 4 <= a.n) {
            const f32x4u v = *reinterpret_cast<const f32x4u*>(in + 4 * q);
            x = make_float4(v.x, v.y, v.z, v.w);
        } else {
            if (4 * q < a.n) x.x = in[4 * q];
            if (4 * q + 1 < a.n) x.y = in[4 * q + 1];
            if (4 * q + 2 < a.n) x.z = in[4 * q + 2];
        }
        return x;
    };
    // their place in LDS: threads that read four such in a row each do so from distinct banks
    const auto place = [](int q) { return q ^ ((q >> 4) & 3); };
    constexpr int CHUNKS = LDS ? EV_KEEP / EV_CHUNK : 1;
    uint32_t keys[CHUNKS][4];
    if constexpr (LDS) {
        float4 x[CHUNKS];
        #pragma unroll
        for (int c = 0; c < CHUNKS; c++) x[c] = load(c * EV_NT + t);   // (all on their way at once)
        #pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            kept_in[place(c * EV_NT + t)] = x[c];
            keys[c][0] = ev_key(x[c].x);
            keys[c][1] = ev_key(x[c].y);
            keys[c][2] = ev_key(x[c].z);
            keys[c][3] = ev_key(x[c].w);
        }
    }

    // the want-th largest key among the old positions, in the bits of mask: all
    // keys above it there are kept, and `ties` of those equal to it
    uint32_t key = 0, mask = 0, ties = 0;
    const bool some = want > 0 && want < old;
    // a thread's two digits, 2 t from the top
    const int digit = EV_DIGITS - 2 - 2 * t;
    #pragma unroll
    for (int u = 0; u < EV_COLS; u++) *reinterpret_cast<uint2*>(&hist[u][digit]) = make_uint2(0, 0);
    __syncthreads();
    if (some) {
        ties = (uint32_t)want;
        for (int shift = 21; mask != 0xFFFFFFFFu; shift = shift > 11 ? shift - 11 : 0) {
            const uint32_t digits = shift ? 2047u : 1023u;   // 11, 11 and 10 bits
            const auto add = [&](int c, const uint32_t (&k)[4]) {
                #pragma unroll
                for (int u = 0; u < 4; u++)
                    if (c * EV_CHUNK + 4 * t + u < old && (k[u] & mask) == key)
                        atomicAdd(&hist[t % EV_COLS][(k[u] >> shift) & digits], 1u);
            };
            if constexpr (LDS) {
                #pragma unroll
                for (int c = 0; c < CHUNKS; c++)
                    if (c < chunks) add(c, keys[c]);
            } else {
                for (int c = 0; c < chunks; c++) {
                    const float4 x = load(c * EV_NT + t);
                    const uint32_t k[4] = {ev_key(x.x), ev_key(x.y), ev_key(x.z), ev_key(x.w)};
                    add(c, k);
                }
            }
            __syncthreads();
            // the thread's two digits, and those above them
            uint32_t s[2] = {0, 0};
            #pragma unroll
            for (int u = 0; u < EV_COLS; u++) {
                uint2& p = *reinterpret_cast<uint2*>(&hist[u][digit]);
                s[0] += p.y;
                s[1] += p.x;
                p = make_uint2(0, 0);   // (for the next pass)
            }
            uint32_t all;
            const uint32_t before = wave_scan(s[0] + s[1], all);
            if (l == 0) part[w] = all;
            __syncthreads();
            uint32_t above = before + waves_before(part, w, all);
            #pragma unroll
            for (int i = 0; i < 2; i++) {
                if (above < ties && ties <= above + s[i]) {
                    found[0] = (uint32_t)(digit + 1 - i);
                    found[1] = ties - above;
                    found[2] = s[i];
                }
                above += s[i];
            }
            __syncthreads();
            key |= found[0] << shift;
            mask |= digits << shift;
            ties = found[1];
            if (ties == found[2]) break;   // all that share the bits
        }
    }

    // numbering: of each position the kept ones before it; larger keys and
    // keys equal to the last one counted side by side (16 bits each a stretch)
    const auto flag = [&](int j, float x) {
        const uint32_t k = ev_key(x) & mask;
        const bool gt = (j >= old && j < a.n) || (j < old && (some ? k > key : want > 0));
        return gt ? 1u : some && j < old && k == key ? 0x10000u : 0u;
    };
    if constexpr (LDS) {
        // a stretch of 4 * chunks positions for each thread, as bits
        uint32_t gt = 0, eq = 0;
        for (int c = 0; c < chunks; c++) {
            const float4 x = kept_in[place(t * chunks + c)];
            const float v[4] = {x.x, x.y, x.z, x.w};
            #pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint32_t f = flag(4 * (t * chunks + c) + u, v[u]);
                gt |= (f & 1u) << (4 * c + u);
                eq |= (f >> 16) << (4 * c + u);
            }
        }
        uint32_t all, sum;
        const uint32_t before = wave_scan(__builtin_popcount(gt) | __builtin_popcount(eq) << 16, all);
        if (l == 0) part[w] = all;
        __syncthreads();   // (every mass is in LDS: in place they are overwritten from here on; hist is free)
        const uint32_t b = before + waves_before(part, w, sum), eq_at = b >> 16;
        uint32_t at = (b & 0xFFFFu) + (eq_at < ties ? eq_at : ties);
        // of the equal ones the first ties - eq_at
        uint32_t bits = gt, left = eq_at < ties ? ties - eq_at : 0;
        if (left >= (uint32_t)__builtin_popcount(eq)) bits |= eq;
        else
            for (; left; left--, eq &= eq - 1) bits |= eq & -eq;
        uint16_t* list = reinterpret_cast<uint16_t*>(&hist[0][0]);   // the kept positions, in order
        static_assert(sizeof(hist) >= EV_KEEP * sizeof(uint16_t) && EV_KEEP <= 65536, "room for all");
        for (; bits; bits &= bits - 1) list[at++] = (uint16_t)(4 * t * chunks + __builtin_ctz(bits));
        __syncthreads();
        typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));
        const float* vals = reinterpret_cast<const float*>(kept_in);
        const auto mass = [&](int j) { return vals[4 * place(j >> 2) + (j & 3)]; };
        for (int j = 4 * t; j < a.n; j += EV_CHUNK) {
            int p[4];
            float x[4];
            const uint2 four = *reinterpret_cast<const uint2*>(list + j);   // (behind the last: anything)
            #pragma unroll
            for (int u = 0; u < 4; u++) {
                p[u] = (int)((u < 2 ? four.x : four.y) >> (16 * (u & 1)) & 0xFFFFu);
                x[u] = j + u < a.m ? mass(p[u]) : 0.0f;
            }
            if (j + 4 <= a.m) *reinterpret_cast<i32x4u*>(kept + j) = i32x4u{p[0], p[1], p[2], p[3]};
            else
                #pragma unroll
                for (int u = 0; u < 4; u++)
                    if (j + u < a.m) kept[j + u] = p[u];
            if (!out) continue;
            if (j + 4 <= a.n) *reinterpret_cast<f32x4u*>(out + j) = f32x4u{x[0], x[1], x[2], x[3]};
            else
                #pragma unroll
                for (int u = 0; u < 4; u++)
                    if (j + u < a.n) out[j + u] = x[u];
        }
    } else {
        uint32_t gt0 = 0, eq0 = 0;
        for (int c = 0; c < chunks; c++) {
            const int q = c * EV_NT + t;
            const float4 x = load(q);
            const float v[4] = {x.x, x.y, x.z, x.w};
            uint32_t f[4], n = 0;
            #pragma unroll
            for (int u = 0; u < 4; u++) n += f[u] = flag(4 * q + u, v[u]);
            uint32_t all, sum;
            uint32_t b = wave_scan(n, all);
            __syncthreads();   // part is free (and, in place, this chunk's masses are read by all)
            if (l == 0) part[w] = all;
            __syncthreads();
            b += waves_before(part, w, sum);
            uint32_t gt = gt0 + (b & 0xFFFFu), eq = eq0 + (b >> 16);
            #pragma unroll
            for (int u = 0; u < 4; u++) {
                if (f[u] == 1u || (f[u] && eq < ties)) {
                    const uint32_t at = gt + (eq < ties ? eq : ties);
                    kept[at] = 4 * q + u;
                    if (out) out[at] = v[u];
                }
                gt += f[u] & 0xFFFFu;
                eq += f[u] >> 16;
            }
            gt0 += sum & 0xFFFFu;
            eq0 += sum >> 16;
        }
        __syncthreads();   // in place: the tail is read
        if (out)
            for (int j = a.m + t; j < a.n; j += EV_NT) out[j] = 0.0f;
    }
}

hipError_t evict_select_launch(const float* mass_in, float* mass_out, size_t stride, size_t n_kv, size_t n, size_t m,
                               size_t recent, int32_t* kept, hipStream_t s) {
    EvictArgs a{mass_in, mass_out, stride, (int)n, (int)m, (int)(recent < n ? recent : n), kept};
    const dim3 grid((unsigned)n_kv), block(EV_NT);
    // kept in LDS / read again, us, 8 heads cut to a quarter: 1000 positions 7.5 /
    // 6.5, 4097 9.0 / 9.1, 16384 14.5 / 17.7 (16385 19.6, 32768 29.0)
    if (n > (size_t)EV_CHUNK && n <= (size_t)EV_KEEP) hipLaunchKernelGGL(evict_select_kernel<true>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(evict_select_kernel<false>, grid, block, 0, s, a);
    return hipGetLastError();
}

// ---- f32 rows ----------------------------------------------------------------------

// One thread per V of a row: out[h][j] = in[h][kept[h][j]], K and V.
template <class V>
__global__ __launch_bounds__(256)
void gather_rows_kernel(const V* __restrict__ k, const V* __restrict__ v, size_t src_head, V* __restrict__ ko, V* __restrict__ vo,
                        size_t dst_head, int n_kv, int per_row, int m, const int32_t* __restrict__ kept) {
    size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int i = (int)(t % per_row);
    t /= per_row;
    const int j = (int)(t % m);
    t /= m;
    const int h = (int)(t % n_kv);
    t /= n_kv;
    if (t >= 2) return;
    const size_t from = (size_t)h * src_head + (size_t)kept[(size_t)h * m + j] * per_row + i;
    (t ? vo : ko)[(size_t)h * dst_head + (size_t)j * per_row + i] = (t ? v : k)[from];
}

hipError_t gather_rows_launch(const float* k, const float* v, size_t src_head, float* ko, float* vo, size_t dst_head,
                              size_t n_kv, size_t hd, size_t m, const int32_t* kept, hipStream_t s) {
    const size_t per = evict_heads(false, n_kv, m, hd);
    if (per == 0) return hipErrorInvalidValue;
    for (size_t h = 0; h < n_kv; h += per) {
        const size_t heads = per < n_kv - h ? per : n_kv - h;
        const float *k0 = k + h * src_head, *v0 = v + h * src_head;
        float *k1 = ko + h * dst_head, *v1 = vo + h * dst_head;
        if (hd % 4 == 0) {   // (every row then starts at a multiple of 16 bytes)
            const size_t n = 2 * heads * m * (hd / 4);
            hipLaunchKernelGGL(gather_rows_kernel<float4>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s,
                               reinterpret_cast<const float4*>(k0), reinterpret_cast<const float4*>(v0), src_head / 4,
                               reinterpret_cast<float4*>(k1), reinterpret_cast<float4*>(v1), dst_head / 4, (int)heads,
                               (int)(hd / 4), (int)m, kept + h * m);
        } else {
            const size_t n = 2 * heads * m * hd;
            hipLaunchKernelGGL(gather_rows_kernel<float>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, k0, v0, src_head,
                               k1, v1, dst_head, (int)heads, (int)hd, (int)m, kept + h * m);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ---- 4-bit rows ----------------------------------------------------------------------

// Three kinds of workgroups: V codes (a thread per tile and HD / 16 dims),
// K codes (a thread per 16 bytes of a row), scales (a thread per tile and block, K's and V's).
template <int HD>
__global__ __launch_bounds__(256)
void gather_q4_kernel(Q4View src, Q4View dst, int n_kv, int m, int tiles, const int32_t* __restrict__ kept, unsigned v_blocks,
                      unsigned k_blocks) {
    constexpr int NB = HD / 32, CT = HD / 16;
    if (blockIdx.x < v_blocks) {
        size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
        const int i = (int)(t % 16);
        t /= 16;
        const int tile = (int)(t % tiles), h = (int)(t / tiles);
        if (h >= n_kv) return;
        const int32_t* id = kept + (size_t)h * m;
        uint32_t w[CT] = {};
        #pragma unroll
        for (int e = 0; e < KV_TILE; e++) {
            if (tile * KV_TILE + e < m) {
                const int p = id[tile * KV_TILE + e], from = p % KV_TILE;
                const int down = q4_bit(from), up = q4_bit(e);
                const uint4* x = reinterpret_cast<const uint4*>(src.vc + (size_t)h * src.code_head +
                                                                (size_t)(p / KV_TILE) * (KV_TILE * HD / 2) + i * (CT * 4));
                #pragma unroll
                for (int c = 0; c < CT / 4; c++) {
                    const uint4 q = x[c];
                    w[4 * c] |= ((q.x >> down) & 15u) << up;
                    w[4 * c + 1] |= ((q.y >> down) & 15u) << up;
                    w[4 * c + 2] |= ((q.z >> down) & 15u) << up;
                    w[4 * c + 3] |= ((q.w >> down) & 15u) << up;
                }
            }
        }
        uint4* y = reinterpret_cast<uint4*>(dst.vc + (size_t)h * dst.code_head + (size_t)tile * (KV_TILE * HD / 2) + i * (CT * 4));
        #pragma unroll
        for (int c = 0; c < CT / 4; c++) y[c] = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
    } else if (blockIdx.x < v_blocks + k_blocks) {
        size_t t = (size_t)(blockIdx.x - v_blocks) * 256 + threadIdx.x;
        const int i = (int)(t % NB);
        t /= NB;
        const int j = (int)(t % m), h = (int)(t / m);
        if (h >= n_kv) return;
        const int p = kept[(size_t)h * m + j];
        reinterpret_cast<uint4*>(dst.kc + (size_t)h * dst.code_head + (size_t)j * (HD / 2))[i] =
            reinterpret_cast<const uint4*>(src.kc + (size_t)h * src.code_head + (size_t)p * (HD / 2))[i];
    } else {
        size_t t = (size_t)(blockIdx.x - v_blocks - k_blocks) * 256 + threadIdx.x;
        const int b = (int)(t % NB);
        t /= NB;
        const bool is_v = t % 2;
        t /= 2;
        const int tile = (int)(t % tiles), h = (int)(t / tiles);
        if (h >= n_kv) return;
        const uint16_t* x = reinterpret_cast<const uint16_t*>((is_v ? src.vs : src.ks) + (size_t)h * src.scale_head);
        uint32_t w[4] = {};
        #pragma unroll
        for (int e = 0; e < KV_TILE; e++)
            if (tile * KV_TILE + e < m) {
                const int p = kept[(size_t)h * m + tile * KV_TILE + e];
                w[e / 2] |= (uint32_t)x[((size_t)(p / KV_TILE) * NB + b) * KV_TILE + p % KV_TILE] << (16 * (e & 1));
            }
        reinterpret_cast<uint4*>((is_v ? dst.vs : dst.ks) + (size_t)h * dst.scale_head)[(size_t)tile * NB + b] =
            make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int HD>
static hipError_t gather_q4_t(const Q4View& src, const Q4View& dst, size_t n_kv, size_t m, const int32_t* kept, hipStream_t s) {
    const size_t tiles = q4_tiles(m), per = evict_heads(true, n_kv, m, HD);
    if (per == 0) return hipErrorInvalidValue;
    for (size_t h = 0; h < n_kv; h += per) {
        const size_t heads = per < n_kv - h ? per : n_kv - h;
        const auto from = [&](Q4View w) {   // its heads from h on
            w.kc += h * w.code_head;
            w.vc += h * w.code_head;
            w.ks += h * w.scale_head;
            w.vs += h * w.scale_head;
            return w;
        };
        const unsigned vb = (unsigned)((heads * tiles * 16 + 255) / 256), kb = (unsigned)((heads * m * (HD / 32) + 255) / 256),
                       sb = (unsigned)((heads * tiles * 2 * (HD / 32) + 255) / 256);
        hipLaunchKernelGGL(gather_q4_kernel<HD>, dim3(vb + kb + sb), dim3(256), 0, s, from(src), from(dst), (int)heads, (int)m,
                           (int)tiles, kept + h * m, vb, kb);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t gather_q4_launch(const Q4View& src, const Q4View& dst, size_t n_kv, size_t hd, size_t m, const int32_t* kept,
                            hipStream_t s) {
    switch (hd) {
    case 64: return gather_q4_t<64>(src, dst, n_kv, m, kept, s);
    case 128: return gather_q4_t<128>(src, dst, n_kv, m, kept, s);
    case 256: return gather_q4_t<256>(src, dst, n_kv, m, kept, s);
    default: return hipErrorInvalidValue;
    }
}

// ---- back from the staging area ----------------------------------------------------------

template <class V>
__global__ __launch_bounds__(256)
void copy_planes_kernel(CopyPlanes p, int heads) {
    const int plane = blockIdx.z, h = blockIdx.y;
    const size_t n = p.bytes[plane] / sizeof(V);
    const V* x = reinterpret_cast<const V*>(p.src[plane] + (size_t)h * p.src_head[plane]);
    V* y = reinterpret_cast<V*>(p.dst[plane] + (size_t)h * p.dst_head[plane]);
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) y[i] = x[i];
}

hipError_t copy_planes_launch(const CopyPlanes& p, size_t heads, hipStream_t s) {
    bool wide = true;
    size_t most = 0;
    for (int i = 0; i < p.n; i++) {
        wide = wide && p.bytes[i] % 16 == 0 && p.src_head[i] % 16 == 0 && p.dst_head[i] % 16 == 0 &&
               (reinterpret_cast<uintptr_t>(p.src[i]) | reinterpret_cast<uintptr_t>(p.dst[i])) % 16 == 0;
        most = most > p.bytes[i] ? most : p.bytes[i];
    }
    size_t blocks = (most / (wide ? 16 : 4) + 255) / 256;
    blocks = blocks < 1 ? 1 : blocks > 1024 ? 1024 : blocks;
    const dim3 grid((unsigned)blocks, (unsigned)heads, (unsigned)p.n);
    if (wide) hipLaunchKernelGGL(copy_planes_kernel<uint4>, grid, dim3(256), 0, s, p, (int)heads);
    else hipLaunchKernelGGL(copy_planes_kernel<uint32_t>, grid, dim3(256), 0, s, p, (int)heads);
    return hipGetLastError();
}

}  // namespace barq
