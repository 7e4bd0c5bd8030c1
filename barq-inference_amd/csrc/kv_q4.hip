// Writing and reading the rows of a 4-bit KV cache (kv_q4.hpp has
// the layout and the quantizer's definition).
//
// Both move a few bytes per element once: bound by memory at a prompt's length
// and by the launch for a token.  A thread forms whole dwords of codes in its
// registers (K: 8 dims of one position; V: 8 positions of one dim); the threads
// of a block of 32 dims are neighbouring lanes, which find its scale by lane
// exchanges.  2048 positions of 8 heads of 128 dims (19.1 MB): append 7.6 us
// (2.5 TB/s; append and read with half the threads 15.5 us in all, now 13.4), read
// back 6.6; one position 3.7 and 2.5.
#include "common.hpp"
#include "kv_q4.hpp"
#include "launch.hpp"

namespace barq {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // rows at any 4-byte address

// ---- the quantizer ---------------------------------------------------------------

// Over aligned groups of N = 4 or 8 lanes.
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true)));
    if constexpr (N == 8)
        v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true)));
    return v;
}

// A block's scale from its 32 / D lanes' D elements each.
template <int D>
__device__ __forceinline__ _Float16 q4_scale(const float (&x)[D], int lane) {
    constexpr int N = 32 / D;
    float hi = x[0], lo = x[0], z = x[0] * 0.0f;
    #pragma unroll
    for (int e = 1; e < D; e++) {
        hi = fmaxf(hi, x[e]);
        lo = fminf(lo, x[e]);
        z = __builtin_fmaf(x[e], 0.0f, z);   // NaN after an infinity or a NaN
    }
    hi = lanes_max<N>(hi);
    lo = -lanes_max<N>(-lo);
    const float bad = lanes_max<N>(z != z ? 1.0f : 0.0f);
    float t = hi > -lo ? hi : lo;   // the element of the largest |x|
    if (__any(hi == -lo && hi != 0.0f)) {
        // of both signs: the first one counts (as the largest of 64 - 2 * place - sign)
        float first = 0.0f;
        #pragma unroll
        for (int e = 0; e < D; e++)
            first = fmaxf(first, __builtin_fabsf(x[e]) == hi ? (float)(65 - 2 * ((lane & (N - 1)) * D + e) - (x[e] < 0.0f)) : 0.0f);
        first = lanes_max<N>(first);
        t = hi == -lo ? ((int)first & 1 ? hi : lo) : t;
    }
    if (bad != 0.0f) return __builtin_bit_cast(_Float16, (uint16_t)0x7E00);
    const _Float16 d = (_Float16)(t * -0.125f);   // (a power of two: one rounding)
    const float m = (float)d;
    return m > Q4_D_MAX ? (_Float16)Q4_D_MAX : m < -Q4_D_MAX ? (_Float16)-Q4_D_MAX : d;
}

// The codes of D elements under scale d: floor(x / d + 8.5) within 0 .. 15,
// exactly.  In f32 the quotient plus 8.5 is off by less than 2^-18 (three
// roundings of at most 17); where an element is that near a border, the code's
// own borders (c - 8.5) d, which have 16 bits, settle it by comparison.
template <int D>
__device__ __forceinline__ void q4_codes(const float (&x)[D], float d, uint32_t (&c)[D]) {
    const float inv = d != 0.0f ? 1.0f / d : 0.0f;   // NaN: as 0, all codes 8
    const float by = inv == inv ? inv : 0.0f;
    float f[D], low = 1.0f, high = 0.0f;
    #pragma unroll
    for (int e = 0; e < D; e++) {
        const float y = __builtin_fmaf(x[e], by, 8.5f);
        f[e] = __builtin_amdgcn_fmed3f(y, 0.0f, 15.0f);
        c[e] = (uint32_t)f[e];
        const float r = y - (float)c[e];
        low = fminf(low, __builtin_fabsf(r));
        high = fmaxf(high, y < 15.0f ? r : 0.0f);
    }
    if (__any(low < 0x1p-16f || high > 1.0f - 0x1p-16f)) {
        const float ad = __builtin_fabsf(d);
        #pragma unroll
        for (int e = 0; e < D; e++) {
            const float xs = d < 0.0f ? -x[e] : x[e];
            float k = (float)c[e];
            if (xs < (k - 8.5f) * ad) k -= 1.0f;
            else if (xs >= (k - 7.5f) * ad && ad > 0.0f) k += 1.0f;
            c[e] = (uint32_t)__builtin_amdgcn_fmed3f(k, 0.0f, 15.0f);
        }
    }
}

// ---- append ------------------------------------------------------------------------

constexpr int ROPE_NONE = -1;

struct Q4Append {
    const float *k, *v;         // element (head, position, dim) at head * src_head + position * src_pos + dim
    size_t src_head, src_pos;
    Q4View dst;
    int n_kv, hd;
    long long first, n;         // positions first .. first + n of the cache
    // RoPE of K (ROPE != ROPE_NONE), and of q in the blocks past the cache's
    const float* inv_freq;
    float freq_scale;
    long long start_pos;
    const float* q;             // [n][n_q * hd] -> q_out [n_q][n][hd]
    float* q_out;
    int n_q;
    unsigned kv_blocks;         // workgroups of the cache's part
};

template <int ROPE>
__device__ __forceinline__ void q4_rope8(float (&x)[8], const float* src, int d0, int hd, float pos, const float* inv_freq) {
    // the rotation of rope_kernel (attention.hip), to the bit
    if constexpr (ROPE == ROPE_INTERLEAVED) {
        #pragma unroll
        for (int u = 0; u < 4; u++) {
            float sn, cs;
            sincosf(pos * inv_freq[d0 / 2 + u], &sn, &cs);
            const float x0 = x[2 * u], x1 = x[2 * u + 1];
            x[2 * u] = x0 * cs - x1 * sn;
            x[2 * u + 1] = x0 * sn + x1 * cs;
        }
    } else {
        const int half = hd / 2;
        const bool up = d0 >= half;
        #pragma unroll
        for (int u = 0; u < 8; u++) {
            const int i = d0 - (up ? half : 0) + u;
            float sn, cs;
            sincosf(pos * inv_freq[i], &sn, &cs);
            const float o = src[up ? i : i + half];   // the pair's other element
            x[u] = up ? o * sn + x[u] * cs : x[u] * cs - o * sn;
        }
    }
}

// Grid: x = threads of the tiles, then of q; y = K, V.
template <int ROPE>
__global__ __launch_bounds__(256)
void q4_append_kernel(Q4Append a) {
    const bool is_v = blockIdx.y != 0;
    if (ROPE != ROPE_NONE && blockIdx.x >= a.kv_blocks) {   // q: one thread per pair, as rope_kernel
        if (is_v) return;
        const int half = a.hd / 2;
        const size_t t = (size_t)(blockIdx.x - a.kv_blocks) * 256 + threadIdx.x;
        if (t >= (size_t)a.n * a.n_q * half) return;
        const int i = (int)(t % half);
        const size_t ph = t / half;
        const int h = (int)(ph % a.n_q);
        const long long p = (long long)(ph / a.n_q);
        float sn, cs;
        sincosf(((float)(a.start_pos + p) * a.freq_scale) * a.inv_freq[i], &sn, &cs);
        const float* src = a.q + ((size_t)p * a.n_q + h) * a.hd;
        float* dst = a.q_out + ((size_t)h * a.n + p) * a.hd;
        const int i0 = ROPE == ROPE_INTERLEAVED ? 2 * i : i, i1 = ROPE == ROPE_INTERLEAVED ? 2 * i + 1 : i + half;
        const float x0 = src[i0], x1 = src[i1];
        dst[i0] = x0 * cs - x1 * sn;
        dst[i1] = x0 * sn + x1 * cs;
        return;
    }
    // K: a thread takes 8 dims (a dword) of 4 positions; V: 4 dims of a tile's 8 (a dword each)
    const int nb = a.hd / 32, lane = threadIdx.x & 63, per_tile = nb * 8;
    const long long t0 = a.first / KV_TILE, tiles = (a.first + a.n - 1) / KV_TILE + 1 - t0;
    size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)a.n_kv * tiles * per_tile) return;   // (whole groups of 8 lanes agree)
    const int u = (int)(t % per_tile);
    t /= per_tile;
    const long long tile = t0 + (long long)(t % tiles);
    const int h = (int)(t / tiles);
    const int e0 = (int)(a.first > tile * KV_TILE ? a.first - tile * KV_TILE : 0);   // the tile's positions in the call
    const int e1 = (int)(a.first + a.n < (tile + 1) * KV_TILE ? a.first + a.n - tile * KV_TILE : KV_TILE);
    const float* src = (is_v ? a.v : a.k) + (size_t)h * a.src_head;
    const auto row = [&](int e) { return src + (size_t)(tile * KV_TILE + e - a.first) * a.src_pos; };
    uint8_t* codes = (is_v ? a.dst.vc : a.dst.kc) + (size_t)h * a.dst.code_head;
    const auto scales = [&](int b) {
        return reinterpret_cast<_Float16*>((is_v ? a.dst.vs : a.dst.ks) + (size_t)h * a.dst.scale_head + ((size_t)tile * nb + b) * (2 * KV_TILE));
    };
    if (!is_v) {
        const int kq = u % 4, b = u / 4 % nb, half = u / 4 / nb, d0 = 32 * b + 8 * kq;
        float x[4][8];
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = 4 * half + i;
            f32x4u lo = {}, hi = {};
            if (e >= e0 && e < e1) {
                lo = *reinterpret_cast<const f32x4u*>(row(e) + d0);
                hi = *reinterpret_cast<const f32x4u*>(row(e) + d0 + 4);
            }
            x[i][0] = lo.x; x[i][1] = lo.y; x[i][2] = lo.z; x[i][3] = lo.w;
            x[i][4] = hi.x; x[i][5] = hi.y; x[i][6] = hi.z; x[i][7] = hi.w;
        }
        if constexpr (ROPE != ROPE_NONE) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = 4 * half + i;
                if (e >= e0 && e < e1)
                    q4_rope8<ROPE>(x[i], row(e), d0, a.hd, (float)(a.start_pos + tile * KV_TILE + e - a.first) * a.freq_scale, a.inv_freq);
            }
        }
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = 4 * half + i;
            const _Float16 d = q4_scale(x[i], lane);
            if (e < e0 || e >= e1) continue;
            uint32_t c[8], w = 0;
            q4_codes(x[i], (float)d, c);
            #pragma unroll
            for (int j = 0; j < 8; j++) w |= c[j] << q4_bit(j);
            *reinterpret_cast<uint32_t*>(codes + (size_t)(tile * KV_TILE + e) * (a.hd / 2) + 4 * (kq * nb + b)) = w;
            if (kq == 0) scales(b)[e] = d;
        }
        return;
    }
    const int b = u / 8, d0 = 4 * u;
    float x[8][4];
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        f32x4u v = {};
        if (e >= e0 && e < e1) v = *reinterpret_cast<const f32x4u*>(row(e) + d0);
        x[e][0] = v.x; x[e][1] = v.y; x[e][2] = v.z; x[e][3] = v.w;
    }
    uint32_t w[4] = {};
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        const _Float16 d = q4_scale(x[e], lane);
        if (e < e0 || e >= e1) continue;
        uint32_t c[4];
        q4_codes(x[e], (float)d, c);
        #pragma unroll
        for (int j = 0; j < 4; j++) w[j] |= c[j] << q4_bit(e);
        if (u % 8 == 0) scales(b)[e] = d;
    }
    // the tile's earlier positions keep their nibbles
    uint32_t keep = 0;
    for (int e = 0; e < e0; e++) keep |= 0xFu << q4_bit(e);
    #pragma unroll
    for (int j = 0; j < 4; j++) {
        uint32_t* p = reinterpret_cast<uint32_t*>(codes + (size_t)tile * KV_TILE * (a.hd / 2)) + ((d0 + j) % 16) * (a.hd / 16) + d0 / 16;
        *p = keep ? (*p & keep) | w[j] : w[j];
    }
}

// ---- read --------------------------------------------------------------------------

// One thread per 4 dims of a tile (whole rows of 16-byte stores side by
// side).  Grid: x = threads, y = K, V.
__global__ __launch_bounds__(256)
void q4_read_kernel(Q4View w, int n_kv, int hd, long long first, long long n, float* __restrict__ k, float* __restrict__ v) {
    const bool is_v = blockIdx.y != 0;
    float* out = is_v ? v : k;
    if (!out) return;
    const int nb = hd / 32, quads = hd / 4;
    const long long t0 = first / KV_TILE, tiles = (first + n - 1) / KV_TILE + 1 - t0;
    size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int d0 = 4 * (int)(t % quads);
    t /= quads;
    const long long tile = t0 + (long long)(t % tiles);
    const int h = (int)(t / tiles);
    if (h >= n_kv) return;
    const uint8_t* codes = (is_v ? w.vc : w.kc) + (size_t)h * w.code_head + (size_t)tile * KV_TILE * (hd / 2);
    const uint4 sc = *reinterpret_cast<const uint4*>((is_v ? w.vs : w.ks) + (size_t)h * w.scale_head +
                                                     ((size_t)tile * nb + d0 / 32) * (2 * KV_TILE));
    const uint32_t scw[4] = {sc.x, sc.y, sc.z, sc.w};
    uint32_t word[8];   // V: of the 4 dims; K: of the 8 positions
    #pragma unroll
    for (int j = 0; j < 8; j++)
        if (!is_v || j < 4)
            word[j] = is_v ? reinterpret_cast<const uint32_t*>(codes)[((d0 + j) % 16) * (hd / 16) + d0 / 16]
                           : reinterpret_cast<const uint32_t*>(codes + (size_t)j * (hd / 2))[(d0 / 8 % 4) * nb + d0 / 32];
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        const long long p = tile * KV_TILE + e - first;
        if (p < 0 || p >= n) continue;
        const float d = f16_bits_to_f32((scw[e / 2] >> (16 * (e & 1))) & 0xFFFFu);
        float y[4];
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t c = is_v ? word[j] >> q4_bit(e) : word[e] >> ((d0 & 4) ? q4_bit(4 + j) : q4_bit(j));
            y[j] = (float)((int)(c & 15u) - 8) * d;
        }
        *reinterpret_cast<f32x4u*>(out + ((size_t)h * n + p) * hd + d0) = f32x4u{y[0], y[1], y[2], y[3]};
    }
}

// ---- launch ------------------------------------------------------------------------

// workgroups of K's (or V's) tiles, a thread per `dims` dims of one
static unsigned q4_grid(size_t n_kv, size_t hd, size_t first, size_t n, size_t dims) {
    const size_t tiles = (first + n - 1) / KV_TILE + 1 - first / KV_TILE;
    return (unsigned)((n_kv * tiles * (hd / dims) + 255) / 256);
}

hipError_t q4_append_launch(const Q4View& dst, const float* k, const float* v, size_t src_head, size_t src_pos,
                            size_t n_kv, size_t hd, size_t first, size_t n, hipStream_t s) {
    Q4Append a{};
    a.k = k;
    a.v = v;
    a.src_head = src_head;
    a.src_pos = src_pos;
    a.dst = dst;
    a.n_kv = (int)n_kv;
    a.hd = (int)hd;
    a.first = (long long)first;
    a.n = (long long)n;
    a.kv_blocks = q4_grid(n_kv, hd, first, n, 4);
    hipLaunchKernelGGL(q4_append_kernel<ROPE_NONE>, dim3(a.kv_blocks, 2), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t q4_append_rope_launch(int layout, const Q4View& dst, const float* q, size_t n_q, float* q_out, const float* k,
                                 const float* v, size_t n_kv, size_t hd, size_t first, size_t n, size_t start_pos,
                                 float freq_scale, const float* inv_freq, hipStream_t s) {
    Q4Append a{};
    a.k = k;
    a.v = v;
    a.src_head = hd;
    a.src_pos = n_kv * hd;
    a.dst = dst;
    a.n_kv = (int)n_kv;
    a.hd = (int)hd;
    a.first = (long long)first;
    a.n = (long long)n;
    a.inv_freq = inv_freq;
    a.freq_scale = freq_scale;
    a.start_pos = (long long)start_pos;
    a.q = q;
    a.q_out = q_out;
    a.n_q = q ? (int)n_q : 0;
    a.kv_blocks = q4_grid(n_kv, hd, first, n, 4);
    const unsigned grid = a.kv_blocks + (unsigned)((n * a.n_q * (hd / 2) + 255) / 256);
    if (layout == ROPE_INTERLEAVED)
        hipLaunchKernelGGL(q4_append_kernel<ROPE_INTERLEAVED>, dim3(grid, 2), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(q4_append_kernel<ROPE_SPLIT_HALF>, dim3(grid, 2), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t q4_read_launch(const Q4View& w, size_t n_kv, size_t hd, size_t first, size_t n, float* k, float* v,
                          hipStream_t s) {
    hipLaunchKernelGGL(q4_read_kernel, dim3(q4_grid(n_kv, hd, first, n, 4), 2), dim3(256), 0, s, w, (int)n_kv, (int)hd,
                       (long long)first, (long long)n, k, v);
    return hipGetLastError();
}

}  // namespace barq
