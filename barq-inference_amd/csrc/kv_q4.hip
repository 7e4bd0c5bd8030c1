// Writing, reading and gathering the rows of a 4-bit KV cache (kv_q4.hpp has
// the layout and the quantizer's definition).
//
// All three move a few bytes per element once: bound by memory at a prompt's
// length and by the launch for a token.  A thread owns 8 dims of a block at
// the 8 positions of a tile, for K and V alike, so K's dwords (8 dims of one
// position) and V's (8 positions of one dim) both form in its registers; the
// 4 threads of a block are neighbouring lanes and find its scale with two
// quad exchanges.
#include "common.hpp"
#include "kv_q4.hpp"
#include "launch.hpp"

namespace barq {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // rows at any 4-byte address

// ---- the quantizer ---------------------------------------------------------------

// Of (abs bits, value) pairs the larger abs, the lower lane's where equal.
template <int STEP>   // exchanged with lane ^ STEP (a quad's)
__device__ __forceinline__ void q4_top(uint32_t& a, float& x, int lane) {
    constexpr int CTL = STEP == 1 ? 0xB1 : 0x4E;
    const uint32_t oa = (uint32_t)__builtin_amdgcn_mov_dpp((int)a, CTL, 0xF, 0xF, true);
    const float ox = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTL, 0xF, 0xF, true));
    const bool theirs = oa > a || (oa == a && (lane & STEP));
    a = theirs ? oa : a;
    x = theirs ? ox : x;
}

// The block's scale from its 4 lanes' 8 elements each.
__device__ __forceinline__ _Float16 q4_scale(const float (&x)[8], int lane) {
    uint32_t a = __builtin_bit_cast(uint32_t, x[0]) & 0x7FFFFFFFu;
    float t = x[0];
    #pragma unroll
    for (int e = 1; e < 8; e++) {
        const uint32_t b = __builtin_bit_cast(uint32_t, x[e]) & 0x7FFFFFFFu;   // orders |x|, NaN above infinity
        t = b > a ? x[e] : t;
        a = b > a ? b : a;
    }
    q4_top<1>(a, t, lane);
    q4_top<2>(a, t, lane);
    if (a >= 0x7F800000u) return __builtin_bit_cast(_Float16, (uint16_t)0x7E00);
    const _Float16 d = (_Float16)(t * -0.125f);   // (a power of two: one rounding)
    const float m = (float)d;
    return m > Q4_D_MAX ? (_Float16)Q4_D_MAX : m < -Q4_D_MAX ? (_Float16)-Q4_D_MAX : d;
}

// The code of x under scale d: floor(x / d + 8.5) within 0 .. 15, exactly.
// The quotient from f32 can be off by one where x is next to a border; the
// borders (c - 8.5) d have 16 bits, so comparing with them settles it.
__device__ __forceinline__ uint32_t q4_code(float x, float ad, float inv, bool neg) {
    const float xs = neg ? -x : x;
    const float y = fminf(fmaxf(xs * inv, -9.0f), 8.0f);
    float c = fminf(fmaxf(floorf(y + 8.5f), 0.0f), 15.0f);
    if (xs < (c - 8.5f) * ad) c -= 1.0f;
    else if (xs >= (c - 7.5f) * ad) c += 1.0f;
    return (uint32_t)(int)fminf(fmaxf(c, 0.0f), 15.0f);
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

template <int ROPE>
__global__ __launch_bounds__(256)
void q4_append_kernel(Q4Append a) {
    if (ROPE != ROPE_NONE && blockIdx.x >= a.kv_blocks) {   // q: one thread per pair, as rope_kernel
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
    const int nb = a.hd / 32, lane = threadIdx.x & 63;
    const long long t0 = a.first / KV_TILE, tiles = (a.first + a.n - 1) / KV_TILE + 1 - t0;
    size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    const bool live = t < (size_t)2 * a.n_kv * tiles * nb * 4;   // whole quads: every lane of a quad agrees
    if (!live) return;
    const int kq = (int)(t % 4);
    t /= 4;
    const int b = (int)(t % nb);
    t /= nb;
    const long long tile = t0 + (long long)(t % tiles);
    t /= tiles;
    const int h = (int)(t % a.n_kv);
    const bool is_v = t / a.n_kv != 0;
    const int d0 = 32 * b + 8 * kq;
    const float* src = (is_v ? a.v : a.k) + (size_t)h * a.src_head;
    const int e0 = (int)(a.first > tile * KV_TILE ? a.first - tile * KV_TILE : 0);   // the tile's positions in the call
    const int e1 = (int)(a.first + a.n < (tile + 1) * KV_TILE ? a.first + a.n - tile * KV_TILE : KV_TILE);

    float x[8][8];
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        if (e >= e0 && e < e1) {
            const float* p = src + (size_t)(tile * KV_TILE + e - a.first) * a.src_pos + d0;
            const f32x4u u = *reinterpret_cast<const f32x4u*>(p), w = *reinterpret_cast<const f32x4u*>(p + 4);
            x[e][0] = u.x; x[e][1] = u.y; x[e][2] = u.z; x[e][3] = u.w;
            x[e][4] = w.x; x[e][5] = w.y; x[e][6] = w.z; x[e][7] = w.w;
        } else {
            #pragma unroll
            for (int j = 0; j < 8; j++) x[e][j] = 0.0f;
        }
    }
    if constexpr (ROPE != ROPE_NONE) {
        if (!is_v) {
            #pragma unroll
            for (int e = 0; e < 8; e++)
                if (e >= e0 && e < e1) {
                    const long long p = tile * KV_TILE + e - a.first;
                    q4_rope8<ROPE>(x[e], src + (size_t)p * a.src_pos, d0, a.hd, (float)(a.start_pos + p) * a.freq_scale,
                                   a.inv_freq);
                }
        }
    }
    uint8_t* sc = (is_v ? a.dst.vs : a.dst.ks) + (size_t)h * a.dst.scale_head + ((size_t)tile * nb + b) * (2 * KV_TILE);
    uint8_t* codes = (is_v ? a.dst.vc : a.dst.kc) + (size_t)h * a.dst.code_head;
    uint32_t vw[8] = {};   // V: one dword per dim
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        const _Float16 d = q4_scale(x[e], lane);
        if (e < e0 || e >= e1) continue;
        const float m = (float)d, ad = fabsf(m);
        const float inv = 1.0f / ad;
        uint32_t kw = 0;
        #pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t c = ad > 0.0f ? q4_code(x[e][j], ad, inv, m < 0.0f) : 8u;   // 8 under zero and NaN
            kw |= (c ^ 8u) << (4 * j);
            vw[j] |= c << (4 * (e >> 1) + 16 * (e & 1));
        }
        if (!is_v) *reinterpret_cast<uint32_t*>(codes + (size_t)(tile * KV_TILE + e) * (a.hd / 2) + 4 * (kq * nb + b)) = kw;
        if (kq == 0) reinterpret_cast<_Float16*>(sc)[e] = d;
    }
    if (is_v) {
        uint32_t* w = reinterpret_cast<uint32_t*>(codes + (size_t)tile * KV_TILE * (a.hd / 2));
        // the tile's earlier positions keep their nibbles
        uint32_t keep = 0;
        for (int e = 0; e < e0; e++) keep |= 0xFu << (4 * (e >> 1) + 16 * (e & 1));
        #pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t* p = w + ((d0 + j) % 16) * (a.hd / 16) + d0 / 16;
            *p = keep ? (*p & keep) | vw[j] : vw[j];
        }
    }
}

// ---- read --------------------------------------------------------------------------

__global__ __launch_bounds__(256)
void q4_read_kernel(Q4View w, int n_kv, int hd, long long first, long long n, float* __restrict__ k, float* __restrict__ v) {
    const int nb = hd / 32;
    const long long t0 = first / KV_TILE, tiles = (first + n - 1) / KV_TILE + 1 - t0;
    size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)2 * n_kv * tiles * nb * 4) return;
    const int kq = (int)(t % 4);
    t /= 4;
    const int b = (int)(t % nb);
    t /= nb;
    const long long tile = t0 + (long long)(t % tiles);
    t /= tiles;
    const int h = (int)(t % n_kv);
    const bool is_v = t / n_kv != 0;
    float* out = is_v ? v : k;
    if (!out) return;
    const int d0 = 32 * b + 8 * kq;
    const uint8_t* codes = (is_v ? w.vc : w.kc) + (size_t)h * w.code_head + (size_t)tile * KV_TILE * (hd / 2);
    const _Float16* sc = reinterpret_cast<const _Float16*>((is_v ? w.vs : w.ks) + (size_t)h * w.scale_head +
                                                           ((size_t)tile * nb + b) * (2 * KV_TILE));
    uint32_t word[8];
    #pragma unroll
    for (int j = 0; j < 8; j++)
        word[j] = is_v ? reinterpret_cast<const uint32_t*>(codes)[((d0 + j) % 16) * (hd / 16) + d0 / 16]
                       : reinterpret_cast<const uint32_t*>(codes + (size_t)j * (hd / 2))[kq * nb + b];
    #pragma unroll
    for (int e = 0; e < 8; e++) {
        const long long p = tile * KV_TILE + e - first;
        if (p < 0 || p >= n) continue;
        const float d = (float)sc[e];
        float y[8];
        #pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t c = is_v ? word[j] >> (4 * (e >> 1) + 16 * (e & 1)) : (word[e] >> (4 * j)) ^ 8u;
            y[j] = (float)((int)(c & 15u) - 8) * d;
        }
        float* o = out + ((size_t)h * n + p) * hd + d0;
        *reinterpret_cast<f32x4u*>(o) = f32x4u{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<f32x4u*>(o + 4) = f32x4u{y[4], y[5], y[6], y[7]};
    }
}

// ---- launch ------------------------------------------------------------------------

static unsigned q4_grid(size_t n_kv, size_t hd, size_t first, size_t n) {
    const size_t tiles = (first + n - 1) / KV_TILE + 1 - first / KV_TILE;
    return (unsigned)((2 * n_kv * tiles * (hd / 32) * 4 + 255) / 256);
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
    a.kv_blocks = q4_grid(n_kv, hd, first, n);
    hipLaunchKernelGGL(q4_append_kernel<ROPE_NONE>, dim3(a.kv_blocks), dim3(256), 0, s, a);
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
    a.kv_blocks = q4_grid(n_kv, hd, first, n);
    const unsigned grid = a.kv_blocks + (unsigned)((n * a.n_q * (hd / 2) + 255) / 256);
    if (layout == ROPE_INTERLEAVED)
        hipLaunchKernelGGL(q4_append_kernel<ROPE_INTERLEAVED>, dim3(grid), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(q4_append_kernel<ROPE_SPLIT_HALF>, dim3(grid), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t q4_read_launch(const Q4View& w, size_t n_kv, size_t hd, size_t first, size_t n, float* k, float* v,
                          hipStream_t s) {
    hipLaunchKernelGGL(q4_read_kernel, dim3(q4_grid(n_kv, hd, first, n)), dim3(256), 0, s, w, (int)n_kv, (int)hd,
                       (long long)first, (long long)n, k, v);
    return hipGetLastError();
}

}  // namespace barq
