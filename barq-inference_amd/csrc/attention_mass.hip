// The weight that attention gives each cached position, added up over the
// query rows and the query heads that share a kv head:
//
//   mass_out[hk][j] = mass_in[hk][j] + sum over heads h of hk and rows i of
//                     exp2(score(h, i, j) - M(h, i)) / L(h, i)
//
// with the scores (log2 units) and the partial maxima and sums that attention
// left behind.  Bound by the scores' bytes (written once and read once; K need
// not be read again).  A workgroup takes 64 positions, its four waves every
// fourth row each; the sums run in a fixed order and need no atomics.
#include "common.hpp"
#include "launch.hpp"

namespace barq {

constexpr int MASS_INLINE = 16;   // rows of a kv head whose statistics a workgroup finds itself

// Maximum M and 1 / sum L of row `at`'s partial states, in all 16 lanes of its group.
__device__ __forceinline__ float2 mass_stat(const MassArgs& a, size_t at, int lane16) {
    const float* p = a.part + at * a.ns * (a.head_dim + 2);
    float M = -INFINITY, L = 0.0f;
    for (int s = lane16; s < a.ns; s += 16) {
        const float m = p[(size_t)s * (a.head_dim + 2)], l = p[(size_t)s * (a.head_dim + 2) + 1];
        const float mn = fmaxf(M, m);
        if (mn != -INFINITY) L = L * __builtin_amdgcn_exp2f(M - mn) + l * __builtin_amdgcn_exp2f(m - mn);
        M = mn;
    }
    const float all = row16_max(M);
    L = row16_sum(M == -INFINITY ? 0.0f * L : L * __builtin_amdgcn_exp2f(M - all));
    return make_float2(all, 1.0f / L);
}

__global__ __launch_bounds__(256)
void mass_stat_kernel(MassArgs a) {
    const size_t at = (size_t)blockIdx.x * 16 + threadIdx.x / 16;
    const size_t n = (size_t)a.q_len * a.n_head;
    const float2 st = mass_stat(a, at < n ? at : n - 1, threadIdx.x & 15);
    if (at < n && (threadIdx.x & 15) == 0) reinterpret_cast<float2*>(a.stat)[at] = st;
}

// Grid: x = 64 positions, y = kv head.  INLINE: at most MASS_INLINE rows.
template <bool INLINE>
__global__ __launch_bounds__(256)
void mass_kernel(MassArgs a) {
    __shared__ float2 stat[INLINE ? MASS_INLINE : 1];
    __shared__ float red[4][64];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = blockIdx.y;
    const int j = blockIdx.x * 64 + l;
    // query heads h with h * n_head_kv / n_head = hk
    const int h0 = (int)(((long long)hk * a.n_head + a.n_head_kv - 1) / a.n_head_kv);
    const int h1 = (int)(((long long)(hk + 1) * a.n_head + a.n_head_kv - 1) / a.n_head_kv);
    const int G = h1 - h0, rows = G * a.q_len;
    if constexpr (INLINE) {
        const int r = threadIdx.x / 16;
        if (r < rows) {
            const float2 st = mass_stat(a, (size_t)(r / G) * a.n_head + h0 + r % G, threadIdx.x & 15);
            if ((threadIdx.x & 15) == 0) stat[r] = st;
        }
        __syncthreads();
    }
    float total = 0.0f;
    // (a position past the row's last is not seen; scores behind it are undefined)
    for (int base = w; base < rows; base += 4 * 32) {   // in runs of 32 rows: short sums added to a long one
        float sum = 0.0f;
        #pragma unroll 8
        for (int u = 0; u < 32; u++) {
            const int r = base + 4 * u;
            if (r >= rows) break;
            const int i = r / G, h = h0 + r - i * G;
            const size_t at = (size_t)i * a.n_head + h;
            const float2 st = INLINE ? stat[INLINE ? r : 0] : reinterpret_cast<const float2*>(a.stat)[at];
            const bool seen = j < a.kv_len && j <= a.start_pos + i;
            if (seen) sum += __builtin_amdgcn_exp2f(a.scores[at * a.score_stride + j] - st.x) * st.y;
        }
        total += sum;
    }
    red[w][l] = total;
    __syncthreads();
    if (w == 0 && j < a.kv_len) {
        const float m = a.mass_in ? a.mass_in[(size_t)hk * a.mass_stride + j] : 0.0f;
        a.mass_out[(size_t)hk * a.mass_stride + j] = m + ((red[0][l] + red[1][l]) + (red[2][l] + red[3][l]));
    }
}

static bool mass_inline(size_t n_head, size_t n_head_kv, size_t q_len) {
    return q_len * ((n_head + n_head_kv - 1) / n_head_kv) <= (size_t)MASS_INLINE;
}

size_t attention_mass_stat(size_t n_head, size_t n_head_kv, size_t q_len) {
    return mass_inline(n_head, n_head_kv, q_len) ? 0 : q_len * n_head * sizeof(float2);
}

hipError_t attention_mass_launch(const MassArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.kv_len + 63) / 64), (unsigned)a.n_head_kv);
    if (mass_inline(a.n_head, a.n_head_kv, a.q_len)) {
        hipLaunchKernelGGL(mass_kernel<true>, grid, dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL(mass_stat_kernel, dim3((unsigned)(((size_t)a.q_len * a.n_head + 15) / 16)), dim3(256), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(mass_kernel<false>, grid, dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace barq
