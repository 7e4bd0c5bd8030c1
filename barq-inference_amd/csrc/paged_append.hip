// Writing new tokens' rows into a paged KV cache, with the norm and the position
// rotation of the heads on the way, and reading them back; the norm and rotation of
// one tensor by itself.
//
// Bound by the bytes: q is read and written in f32, K and V read in f32 and written
// in the cache's type: 2048 tokens of 32 + 8 heads of 128 dims, 92 MB, in 19.7 us (4.7 TB/s; a copy has 8.0 within the
// last-level cache's size, as here, 5.2 beyond it), 17.2 of them without the launch.  A workgroup has up to 16 tokens of one block and some of their
// heads: HD / 8 lanes a row of q or K, the next rows in flight while these are rotated; of
// V eight tokens (four in f32) of a dim a lane, which are 16 bytes there.  The pairs' cos and
// sin (64-bit angles) are formed once for a workgroup's tokens, while its first rows come.
#include "paged.hpp"
#include "rotary.hpp"

namespace barq {

namespace {

constexpr size_t TURN_WORKGROUPS = 1024;   // (a 2048-token append: 20.2 us; 512: 22.3, 2048: 22.1)
constexpr int TURN_AHEAD = 1;   // rows of a lane in flight besides the one at hand (2 and 3 are no faster)

// f32 to the cache's f16: nearest, the finite ones kept within its range, the others NaN.
__device__ __forceinline__ uint32_t cache_f16(float x) {
    const uint32_t h = f32_to_f16_bits(__builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f));
    return __builtin_fabsf(x) < INFINITY ? h : 0x7E00u;
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

// The workgroups' rows: of a group of n tokens (or a quarter of them), 2^s at most, row r is token r % 2^s (if there is one) of
// head r / 2^s; the workgroups of the same tokens take ROWS of them each in turn.
__device__ __forceinline__ int log_tokens(int n) { return n < 2 ? 0 : 32 - __builtin_clz(n - 1); }

template <bool H, int HD, bool ODD>
__global__ __launch_bounds__(256)
void paged_append_kernel(PagedAppend a, int per, int per_v, int parts) {
    constexpr int LANES = HD / 8, ROWS = 256 / LANES;
    __shared__ __align__(16) float2 turn[TURN_TOKENS][HD / 2];
    const int n_tokens = a.n_tokens < 0 ? a.counts->n_tokens : a.n_tokens, n_groups = a.n_tokens < 0 ? a.counts->groups : a.n_groups;
    const int sub = threadIdx.x / LANES, d0 = 8 * (threadIdx.x % LANES), heads = a.n_q + a.n_kv;
    for (int w = blockIdx.x; w < n_groups; w += gridDim.x) {
        PagedGroup gr = a.groups[w];
        if ((int)blockIdx.y < per) {
            if (parts > 1) {   // these tokens of the group
                const int t = TURN_TOKENS / parts * (blockIdx.y % parts);
                gr.t0 += t, gr.pos += t, gr.n = min(gr.n - t, TURN_TOKENS / parts), gr.row += gr.row < 0 ? 0 : t;
                if (gr.n <= 0) continue;
            }
            const int log_n = log_tokens(gr.n), mask = (1 << log_n) - 1, rows = heads << log_n;
            const auto from = [&](int r) {   // (a token that is not there: the last one)
                const int head = r >> log_n, t = gr.t0 + min(r & mask, gr.n - 1);
                return head < a.n_q ? a.q + ((size_t)t * a.n_q + head) * HD : a.k + ((size_t)t * a.n_kv + head - a.n_q) * HD;
            };
            const int step = per / parts * ROWS;
            int r = blockIdx.y / parts * ROWS + sub;
            TurnRow<HD, ODD> ahead[TURN_AHEAD];
            #pragma unroll
            for (int k = 0; k < TURN_AHEAD; k++)
                if (r + k * step < rows) ahead[k].load(from(r + k * step), d0);
            __syncthreads();   // (the table of an earlier group has been read)
            turn_table<HD>(turn, gr.pos, gr.n, a.rotary);
            __syncthreads();
            while (r < rows) {
                #pragma unroll
                for (int k = 0; k < TURN_AHEAD; k++, r += step) {
                    if (r >= rows) break;
                    TurnRow<HD, ODD> x = ahead[k];
                    if (r + TURN_AHEAD * step < rows) ahead[k].load(from(r + TURN_AHEAD * step), d0);
                    const int head = r >> log_n, t = r & mask;
                    x.turn(d0, head < a.n_q ? a.q_norm : a.k_norm, a.eps, a.rotary, turn[min(t, gr.n - 1)]);
                    if (t >= gr.n) {
                    } else if (head < a.n_q) {
                        float4* out = reinterpret_cast<float4*>(a.q_out + ((size_t)head * n_tokens + gr.t0 + t) * HD + d0);
                        out[0] = make_float4(x.x[0], x.x[1], x.x[2], x.x[3]);
                        out[1] = make_float4(x.x[4], x.x[5], x.x[6], x.x[7]);
                    } else if (gr.row >= 0) {
                        uint8_t* b = a.k_pool + block_of<H, HD>(gr.row, head - a.n_q, a.n_kv, a.log_page);
                        const int slot = (gr.row & 15) + t;
                        if constexpr (H) {
                            uint4 h;
                            h.x = cache_f16(x.x[0]) | cache_f16(x.x[1]) << 16;
                            h.y = cache_f16(x.x[2]) | cache_f16(x.x[3]) << 16;
                            h.z = cache_f16(x.x[4]) | cache_f16(x.x[5]) << 16;
                            h.w = cache_f16(x.x[6]) | cache_f16(x.x[7]) << 16;
                            *reinterpret_cast<uint4*>(b + ((d0 / 8) * 16 + slot) * 16) = h;
                        } else {
                            #pragma unroll
                            for (int u = 0; u < 2; u++)
                                *reinterpret_cast<uint4*>(b + ((d0 / 4 + u) * 16 + slot) * 16) =
                                    make_uint4(cache_f32(x.x[4 * u]), cache_f32(x.x[4 * u + 1]), cache_f32(x.x[4 * u + 2]), cache_f32(x.x[4 * u + 3]));
                        }
                    }
                }
            }
        } else if (gr.row >= 0) {
            constexpr int E = H ? 8 : 4, PARTS = PAGE_BLOCK / E;
            const int slot0 = gr.row & 15, y = blockIdx.y - per;
            for (int u = y * 256 + threadIdx.x; u < a.n_kv * PARTS * HD; u += per_v * 256) {
                const int d = u % HD, part = u / HD % PARTS, hk = u / HD / PARTS;
                // the slots of the part that are the group's
                const int first = max(slot0, E * part) - E * part, last = min(slot0 + gr.n, E * part + E) - E * part;
                if (first >= last) continue;
                const ptrdiff_t next = (ptrdiff_t)a.n_kv * HD;   // (token's row)
                const float* src = a.v + (gr.t0 + E * part - slot0) * next + hk * HD + d;   // of the part's first slot
                uint8_t* to = a.v_pool + block_of<H, HD>(gr.row, hk, a.n_kv, a.log_page) + (part * HD + d) * 16;
                uint32_t x[E];
                if (last - first == E) {
                    #pragma unroll
                    for (int e = 0; e < E; e++) x[e] = __builtin_bit_cast(uint32_t, src[e * next]);
                    #pragma unroll
                    for (int e = 0; e < E; e++) x[e] = H ? cache_f16(__builtin_bit_cast(float, x[e])) : cache_f32(__builtin_bit_cast(float, x[e]));
                    if constexpr (H) *reinterpret_cast<uint4*>(to) = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
                    else *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
                } else {
                    for (int e = first; e < last; e++) {
                        const float v = src[e * next];
                        if constexpr (H) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)cache_f16(v);
                        else reinterpret_cast<uint32_t*>(to)[e] = cache_f32(v);
                    }
                }
            }
        }
    }
}

// The tokens' rows of K and V as they lie in the cache, [n_tokens, n_kv, HD] of its type (zeros where they have none):
// 16 bytes of a row a lane.
template <bool H, int HD>
__global__ __launch_bounds__(256)
void paged_read_kernel(PagedAppend a, uint8_t* k_out, uint8_t* v_out) {
    constexpr int E = H ? 8 : 4, LANES = HD / E;
    const int n_groups = a.n_tokens < 0 ? a.counts->groups : a.n_groups;
    for (int w = blockIdx.x; w < n_groups; w += gridDim.x) {
        const PagedGroup gr = a.groups[w];
        for (int u = blockIdx.y * 256 + threadIdx.x; u < gr.n * a.n_kv * LANES; u += gridDim.y * 256) {
            const int c = u % LANES, hk = u / LANES % a.n_kv, t = u / LANES / a.n_kv, slot = (gr.row & 15) + t;
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (gr.row >= 0) {
                const size_t at = block_of<H, HD>(gr.row, hk, a.n_kv, a.log_page);
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
            const size_t to = ((size_t)(gr.t0 + t) * a.n_kv + hk) * LANES + c;
            if (k_out) reinterpret_cast<u32x4_a4*>(k_out)[to] = u32x4_a4{x.x, x.y, x.z, x.w};
            if (v_out) reinterpret_cast<u32x4_a4*>(v_out)[to] = u32x4_a4{y.x, y.y, y.z, y.w};
        }
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

// x [seq, heads, HD] -> [heads, seq, HD], normed and rotated; the rows of a workgroup as for the append.
template <int HD, bool ODD>
__global__ __launch_bounds__(256)
void norm_rope_kernel(const float* x, float* out, int seq, int heads, int tokens, int start_pos, const float* w, float eps, Rotary rotary) {
    constexpr int LANES = HD / 8, ROWS = 256 / LANES;
    __shared__ __align__(16) float2 turn[TURN_TOKENS][HD / 2];
    const int t0 = blockIdx.x * tokens, n = min(tokens, seq - t0), log_n = log_tokens(n), mask = (1 << log_n) - 1, rows = heads << log_n;
    const int sub = threadIdx.x / LANES, d0 = 8 * (threadIdx.x % LANES), step = gridDim.y * ROWS;
    const auto from = [&](int r) { return x + ((size_t)(t0 + min(r & mask, n - 1)) * heads + (r >> log_n)) * HD; };
    int r = blockIdx.y * ROWS + sub;
    TurnRow<HD, ODD> ahead[TURN_AHEAD];
    #pragma unroll
    for (int k = 0; k < TURN_AHEAD; k++)
        if (r + k * step < rows) ahead[k].load(from(r + k * step), d0);
    turn_table<HD>(turn, start_pos + t0, n, rotary);
    __syncthreads();
    while (r < rows) {
        #pragma unroll
        for (int k = 0; k < TURN_AHEAD; k++, r += step) {
            if (r >= rows) break;
            TurnRow<HD, ODD> y = ahead[k];
            if (r + TURN_AHEAD * step < rows) ahead[k].load(from(r + TURN_AHEAD * step), d0);
            const int t = r & mask;
            y.turn(d0, w, eps, rotary, turn[min(t, n - 1)]);
            if (t < n) {
                float4* o = reinterpret_cast<float4*>(out + ((size_t)(r >> log_n) * seq + t0 + t) * HD + d0);
                o[0] = make_float4(y.x[0], y.x[1], y.x[2], y.x[3]);
                o[1] = make_float4(y.x[4], y.x[5], y.x[6], y.x[7]);
            }
        }
    }
}

// Workgroups for `groups` groups of at most `passes` passes each: enough to fill the card, with at most all of a group's.
unsigned shares(size_t groups, size_t passes) {
    const size_t want = (TURN_WORKGROUPS + groups - 1) / groups;
    return (unsigned)(want < 1 ? 1 : want < passes ? want : passes);
}

}  // namespace

hipError_t paged_append_launch(const PagedAppend& a, bool f16, size_t hd, hipStream_t s) {
    const bool captured = a.n_tokens < 0;   // (a captured call goes round the groups)
    const size_t groups = captured ? 256 : (size_t)a.n_groups, most = captured || a.n_tokens > a.n_groups ? TURN_TOKENS : 1;
    const size_t rows = 256 / (hd / 8), heads = (size_t)a.n_q + a.n_kv;
    // whole groups' tokens in quarters: a token's cos and sin are formed by fewer workgroups, K is still written 64 bytes at a
    // time (append and read of 2048 tokens of 16 + 2 heads of 256 dims 24.5 -> 22.4 us, of 32 + 8 of 128 27.6 -> 27.0, of
    // 4000 of 8 + 8 32.5 -> 33.2)
    const int parts = !captured && 8 * groups <= (size_t)a.n_tokens ? 4 : 1;
    const unsigned per = (shares(groups, (heads * most + rows - 1) / rows) + parts - 1) / parts * parts;
    const unsigned per_v = shares(groups, ((size_t)a.n_kv * (f16 ? 2 : 4) * hd + 255) / 256);
    const dim3 g((unsigned)groups, per + per_v);
    const bool odd = rotary_odd(a.rotary);
    #define BARQ_APPEND(H, D, O) \
        if (f16 == H && hd == D && odd == O) \
            hipLaunchKernelGGL((paged_append_kernel<H, D, O>), g, dim3(256), 0, s, a, (int)per, (int)per_v, parts);
    BARQ_APPEND(true, 64, false) BARQ_APPEND(true, 128, false) BARQ_APPEND(true, 256, false)
    BARQ_APPEND(false, 64, false) BARQ_APPEND(false, 128, false) BARQ_APPEND(false, 256, false)
    BARQ_APPEND(true, 64, true) BARQ_APPEND(true, 128, true) BARQ_APPEND(true, 256, true)
    BARQ_APPEND(false, 64, true) BARQ_APPEND(false, 128, true) BARQ_APPEND(false, 256, true)
    #undef BARQ_APPEND
    return hipGetLastError();
}

hipError_t paged_read_launch(const PagedAppend& a, bool f16, size_t hd, void* k_out, void* v_out, hipStream_t s) {
    const bool captured = a.n_tokens < 0;
    const size_t groups = captured ? 256 : (size_t)a.n_groups, most = captured || a.n_tokens > a.n_groups ? TURN_TOKENS : 1;
    const dim3 g((unsigned)groups, shares(groups, (most * a.n_kv * (hd / (f16 ? 8 : 4)) + 255) / 256));
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
    // tokens of a workgroup: 16, fewer while there are few of those, so that several workgroups form the same cos and sin only
    // where one token's heads are many (2048 tokens of 32 heads of 128 dims 13.7 us, 15.5 with 16 tokens each; 4000 of 64
    // dims 14.4 and 13.9)
    size_t tokens = TURN_TOKENS;
    while (tokens > 1 && (seq + tokens - 1) / tokens < TURN_WORKGROUPS / 2) tokens /= 2;
    const size_t groups = (seq + tokens - 1) / tokens, rows = 256 / (hd / 8);
    const dim3 g((unsigned)groups, shares(groups, (heads * tokens + rows - 1) / rows));
    const bool odd = rotary_odd(r);
    #define BARQ_TURN(D, O) \
        if (hd == D && odd == O) hipLaunchKernelGGL((norm_rope_kernel<D, O>), g, dim3(256), 0, s, x, out, (int)seq, (int)heads, (int)tokens, (int)start_pos, w, eps, r);
    BARQ_TURN(64, false) BARQ_TURN(128, false) BARQ_TURN(256, false)
    BARQ_TURN(64, true) BARQ_TURN(128, true) BARQ_TURN(256, true)
    #undef BARQ_TURN
    return hipGetLastError();
}

}  // namespace barq
