// Writing new tokens' rows into a paged KV cache, with the norm and the position
// rotation of the heads on the way, and reading them back; the norm and rotation of
// one tensor by itself.
//
// Bound by the bytes: q is read and written in f32, K and V read in f32 and written
// in the cache's type.  A workgroup has some heads of one token, so that a pair's
// cos and sin (64-bit angles) are formed once for all of them; HD / 8 lanes a head.
#include "paged.hpp"
#include "rotary.hpp"

namespace barq {

namespace {

// f32 to the cache's f16: nearest, the finite ones kept within its range, the others NaN.
__device__ __forceinline__ uint32_t cache_f16(float x) {
    const uint32_t h = f32_to_f16_bits(fminf(fmaxf(x, -65504.0f), 65504.0f));
    return (__builtin_bit_cast(uint32_t, x) & 0x7F800000u) == 0x7F800000u ? 0x7E00u : h;
}
__device__ __forceinline__ uint32_t cache_f32(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return (b & 0x7F800000u) == 0x7F800000u ? 0x7FC00000u : b;
}

// Where a row of the pool lies: the byte of its kv head's block.
template <bool H, int HD>
__device__ __forceinline__ size_t block_of(int row, int hk, int n_kv, int log_page) {
    const size_t page = (size_t)row >> log_page, slot = (size_t)row & ((1u << log_page) - 1);
    return (((page * n_kv + hk) << (log_page - 4)) + (slot >> 4)) * (PAGE_BLOCK * HD * (H ? 2 : 4));
}

template <bool H, int HD>
__global__ __launch_bounds__(256)
void paged_append_kernel(PagedAppend a) {
    constexpr int LANES = HD / 8, ROWS = 256 / LANES;
    __shared__ float2 turn[HD / 2];
    const int n_tokens = a.n_tokens < 0 ? a.counts->n_tokens : a.n_tokens;
    const int heads = a.n_q + 2 * a.n_kv, sub = threadIdx.x / LANES, d0 = 8 * (threadIdx.x % LANES);
    for (int t = blockIdx.x; t < n_tokens; t += gridDim.x) {
        const PagedToken tok = a.tokens[t];
        __syncthreads();
        for (int i = threadIdx.x; i < a.rotary.rot / 2; i += 256) turn[i] = rotary_turn(tok.pos, a.rotary, i);
        __syncthreads();
        for (int r = blockIdx.y * ROWS + sub; r < heads; r += gridDim.y * ROWS) {
            float y[8];
            if (r < a.n_q) {
                norm_turn8<HD>(a.q + ((size_t)t * a.n_q + r) * HD, d0, a.q_norm, a.eps, a.rotary, turn, y);
                float4* out = reinterpret_cast<float4*>(a.q_out + ((size_t)r * n_tokens + t) * HD + d0);
                out[0] = make_float4(y[0], y[1], y[2], y[3]);
                out[1] = make_float4(y[4], y[5], y[6], y[7]);
            } else if (r < a.n_q + a.n_kv) {
                const int hk = r - a.n_q;
                norm_turn8<HD>(a.k + ((size_t)t * a.n_kv + hk) * HD, d0, a.k_norm, a.eps, a.rotary, turn, y);
                if (tok.row < 0) continue;
                uint8_t* b = a.k_pool + block_of<H, HD>(tok.row, hk, a.n_kv, a.log_page);
                const int slot = tok.row & 15;
                if constexpr (H) {
                    uint4 h;
                    h.x = cache_f16(y[0]) | cache_f16(y[1]) << 16;
                    h.y = cache_f16(y[2]) | cache_f16(y[3]) << 16;
                    h.z = cache_f16(y[4]) | cache_f16(y[5]) << 16;
                    h.w = cache_f16(y[6]) | cache_f16(y[7]) << 16;
                    *reinterpret_cast<uint4*>(b + ((d0 / 8) * 16 + slot) * 16) = h;
                } else {
                    #pragma unroll
                    for (int u = 0; u < 2; u++)
                        *reinterpret_cast<uint4*>(b + ((d0 / 4 + u) * 16 + slot) * 16) =
                            make_uint4(cache_f32(y[4 * u]), cache_f32(y[4 * u + 1]), cache_f32(y[4 * u + 2]), cache_f32(y[4 * u + 3]));
                }
            } else {
                if (tok.row < 0) continue;
                const int hk = r - a.n_q - a.n_kv;
                const float4* src = reinterpret_cast<const float4*>(a.v + ((size_t)t * a.n_kv + hk) * HD + d0);
                const float4 v0 = src[0], v1 = src[1];
                const float x[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                uint8_t* b = a.v_pool + block_of<H, HD>(tok.row, hk, a.n_kv, a.log_page);
                const int slot = tok.row & 15;
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    if constexpr (H)
                        reinterpret_cast<uint16_t*>(b)[((slot >> 3) * HD + d0 + e) * 8 + (slot & 7)] = (uint16_t)cache_f16(x[e]);
                    else
                        reinterpret_cast<uint32_t*>(b)[((slot >> 2) * HD + d0 + e) * 4 + (slot & 3)] = cache_f32(x[e]);
                }
            }
        }
    }
}

// The tokens' rows of K and V as they lie in the cache, [n_tokens, n_kv, HD] of its type (zeros where they have none).
template <bool H, int HD>
__global__ __launch_bounds__(256)
void paged_read_kernel(PagedAppend a, uint8_t* k_out, uint8_t* v_out) {
    constexpr int E = H ? 8 : 4, LANES = HD / E;   // 16 bytes a lane
    const int n_tokens = a.n_tokens < 0 ? a.counts->n_tokens : a.n_tokens;
    const size_t n = (size_t)n_tokens * a.n_kv * LANES;
    for (size_t w = (size_t)blockIdx.x * 256 + threadIdx.x; w < n; w += (size_t)gridDim.x * 256) {
        const int c = (int)(w % LANES), hk = (int)(w / LANES % a.n_kv), t = (int)(w / LANES / a.n_kv);
        const int row = a.tokens[t].row, slot = row & 15;
        const size_t at = row < 0 ? 0 : block_of<H, HD>(row, hk, a.n_kv, a.log_page);
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (row >= 0) {
            x = *reinterpret_cast<const uint4*>(a.k_pool + at + (c * 16 + slot) * 16);
            if constexpr (H) {
                const uint16_t* b = reinterpret_cast<const uint16_t*>(a.v_pool + at) + ((slot >> 3) * HD + 8 * c) * 8 + (slot & 7);
                y.x = b[0] | (uint32_t)b[8] << 16;
                y.y = b[16] | (uint32_t)b[24] << 16;
                y.z = b[32] | (uint32_t)b[40] << 16;
                y.w = b[48] | (uint32_t)b[56] << 16;
            } else {
                const uint32_t* b = reinterpret_cast<const uint32_t*>(a.v_pool + at) + ((slot >> 2) * HD + 4 * c) * 4 + (slot & 3);
                y = make_uint4(b[0], b[4], b[8], b[12]);
            }
        }
        if (k_out) reinterpret_cast<u32x4_a4*>(k_out)[w] = u32x4_a4{x.x, x.y, x.z, x.w};
        if (v_out) reinterpret_cast<u32x4_a4*>(v_out)[w] = u32x4_a4{y.x, y.y, y.z, y.w};
    }
}

// Neighbouring 16-byte words of pinned host memory by neighbouring lanes.
__global__ __launch_bounds__(256)
void paged_upload_kernel(PagedPieces p) {
    for (int i = 0; i < p.n; i++) {
        const uint4* from = reinterpret_cast<const uint4*>(p.src + p.from[i]);
        uint4* to = reinterpret_cast<uint4*>(p.dst[i]);
        for (uint32_t w = blockIdx.x * 256 + threadIdx.x; w < p.bytes[i] / 16; w += gridDim.x * 256) to[w] = from[w];
    }
}

// x [seq, heads, HD] -> [heads, seq, HD], normed and rotated.
template <int HD>
__global__ __launch_bounds__(256)
void norm_rope_kernel(const float* x, float* out, int seq, int heads, int start_pos, const float* w, float eps, Rotary r) {
    constexpr int LANES = HD / 8, ROWS = 256 / LANES;
    __shared__ float2 turn[HD / 2];
    const int t = blockIdx.x, sub = threadIdx.x / LANES, d0 = 8 * (threadIdx.x % LANES);
    for (int i = threadIdx.x; i < r.rot / 2; i += 256) turn[i] = rotary_turn(start_pos + t, r, i);
    __syncthreads();
    for (int h = blockIdx.y * ROWS + sub; h < heads; h += gridDim.y * ROWS) {
        float y[8];
        norm_turn8<HD>(x + ((size_t)t * heads + h) * HD, d0, w, eps, r, turn, y);
        float4* o = reinterpret_cast<float4*>(out + ((size_t)h * seq + t) * HD + d0);
        o[0] = make_float4(y[0], y[1], y[2], y[3]);
        o[1] = make_float4(y[4], y[5], y[6], y[7]);
    }
}

}  // namespace

hipError_t paged_append_launch(const PagedAppend& a, bool f16, size_t hd, hipStream_t s) {
    const unsigned rows = (unsigned)(256 / (hd / 8)), heads = (unsigned)(a.n_q + 2 * a.n_kv), per = (heads + rows - 1) / rows;
    // (a captured call goes round its tokens)
    const dim3 g(a.n_tokens < 0 ? 256u : (unsigned)a.n_tokens, per);
    #define BARQ_APPEND(H, D) if (f16 == H && hd == D) hipLaunchKernelGGL((paged_append_kernel<H, D>), g, dim3(256), 0, s, a);
    BARQ_APPEND(true, 64) BARQ_APPEND(true, 128) BARQ_APPEND(true, 256)
    BARQ_APPEND(false, 64) BARQ_APPEND(false, 128) BARQ_APPEND(false, 256)
    #undef BARQ_APPEND
    return hipGetLastError();
}

hipError_t paged_read_launch(const PagedAppend& a, bool f16, size_t hd, void* k_out, void* v_out, hipStream_t s) {
    const size_t n = (size_t)(a.n_tokens < 0 ? 256 : a.n_tokens) * a.n_kv * (hd / (f16 ? 8 : 4));
    const dim3 g((unsigned)((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096));
    uint8_t *k = static_cast<uint8_t*>(k_out), *v = static_cast<uint8_t*>(v_out);
    #define BARQ_READ(H, D) if (f16 == H && hd == D) hipLaunchKernelGGL((paged_read_kernel<H, D>), g, dim3(256), 0, s, a, k, v);
    BARQ_READ(true, 64) BARQ_READ(true, 128) BARQ_READ(true, 256)
    BARQ_READ(false, 64) BARQ_READ(false, 128) BARQ_READ(false, 256)
    #undef BARQ_READ
    return hipGetLastError();
}

hipError_t paged_upload_launch(const PagedPieces& p, hipStream_t s) {
    uint64_t most = 0;
    for (int i = 0; i < p.n; i++) most = p.bytes[i] > most ? p.bytes[i] : most;
    const uint64_t g = (most / 16 + 255) / 256;
    hipLaunchKernelGGL(paged_upload_kernel, dim3((unsigned)(g < 1 ? 1 : g < 256 ? g : 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t norm_rope_launch(const float* x, float* out, size_t seq, size_t heads, size_t hd, size_t start_pos,
                            const float* w, float eps, const Rotary& r, hipStream_t s) {
    const unsigned rows = (unsigned)(256 / (hd / 8)), per = (unsigned)((heads + rows - 1) / rows);
    const dim3 g((unsigned)seq, per < 65535u ? per : 65535u);
    if (hd == 64) hipLaunchKernelGGL(norm_rope_kernel<64>, g, dim3(256), 0, s, x, out, (int)seq, (int)heads, (int)start_pos, w, eps, r);
    if (hd == 128) hipLaunchKernelGGL(norm_rope_kernel<128>, g, dim3(256), 0, s, x, out, (int)seq, (int)heads, (int)start_pos, w, eps, r);
    if (hd == 256) hipLaunchKernelGGL(norm_rope_kernel<256>, g, dim3(256), 0, s, x, out, (int)seq, (int)heads, (int)start_pos, w, eps, r);
    return hipGetLastError();
}

}  // namespace barq
