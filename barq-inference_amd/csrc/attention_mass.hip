// The weight that attention gives each cached position, added up over the
// query rows and the query heads that share a kv head:
//
//   mass_out[hk][j] = mass_in[hk][j] + sum over heads h of hk and rows i of
//                     exp2(score(h, i, j) - M(h, i)) / L(h, i)
//
// with the scores (log2 units) and the partial maxima and sums that attention
// left behind.  Bound by the scores' bytes (written once and read once; K need
// not be read again).  The sums run in a fixed order and need no atomics: a
// wave takes positions of its own, and where the rows are shared out over
// workgroups each leaves partial sums that another launch adds.
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

// query heads h with h * n_head_kv / n_head = hk: first, and behind the last
__device__ __forceinline__ int mass_head(const MassArgs& a, int hk) {
    return (int)(((long long)hk * a.n_head + a.n_head_kv - 1) / a.n_head_kv);
}

// Few rows: a workgroup of four waves takes 64 positions, every wave a fourth
// of the rows, whose statistics they find themselves.  Grid: x = 64 positions, y = kv head.
__global__ __launch_bounds__(256)
void mass_few_kernel(MassArgs a) {
    __shared__ float2 stat[MASS_INLINE];
    __shared__ float red[4][64];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = blockIdx.y;
    const int j = blockIdx.x * 64 + l;
    const int h0 = mass_head(a, hk), G = mass_head(a, hk + 1) - h0, rows = G * a.q_len;
    // the scores are on their way while the statistics are found
    float s[MASS_INLINE / 4];
    #pragma unroll
    for (int u = 0; u < MASS_INLINE / 4; u++) {
        const int r = w + 4 * u, i = r < rows ? r / G : 0;
        // (a position behind the row's last is not seen: its score is undefined)
        const bool seen = r < rows && j < a.kv_len && j <= a.start_pos + i;
        s[u] = seen ? a.scores[((size_t)i * a.n_head + h0 + r - i * G) * a.score_stride + j] : -INFINITY;
    }
    const float before = a.mass_in && j < a.kv_len ? a.mass_in[(size_t)hk * a.mass_stride + j] : 0.0f;
    if ((int)threadIdx.x / 16 < rows) {
        const int r = threadIdx.x / 16;
        const float2 st = mass_stat(a, (size_t)(r / G) * a.n_head + h0 + r % G, threadIdx.x & 15);
        if ((threadIdx.x & 15) == 0) stat[r] = st;
    }
    __syncthreads();
    float sum = 0.0f;
    #pragma unroll
    for (int u = 0; u < MASS_INLINE / 4; u++) {
        const int r = w + 4 * u, i = r < rows ? r / G : 0;
        if (r < rows && j <= a.start_pos + i) sum += __builtin_amdgcn_exp2f(s[u] - stat[r].x) * stat[r].y;
    }
    red[w][l] = sum;
    __syncthreads();
    if (w == 0 && j < a.kv_len)
        a.mass_out[(size_t)hk * a.mass_stride + j] = before + ((red[0][l] + red[1][l]) + (red[2][l] + red[3][l]));
}

// Many rows: a wave takes 256 positions, four in a row per lane, and
// MASS_RUN rows; its sums go to sums[run][hk][position].
// Grid: x = 1024 positions (four waves), y = kv head, z = run of rows.
constexpr int MASS_RUN = 64;

__global__ __launch_bounds__(256)
void mass_run_kernel(MassArgs a) {
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = blockIdx.y;
    const int j = (blockIdx.x * 4 + w) * 256 + 4 * l;
    const int h0 = mass_head(a, hk), G = mass_head(a, hk + 1) - h0, rows = G * a.q_len;
    const int r0 = blockIdx.z * MASS_RUN, r1 = min(rows, r0 + MASS_RUN);
    if (j >= (int)a.score_stride) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int i = r0 / G, g = r0 - i * G;
    #pragma unroll 4
    for (int r = r0; r < r1; r++) {
        const size_t at = (size_t)i * a.n_head + h0 + g;
        const float2 st = reinterpret_cast<const float2*>(a.stat)[at];
        const float4 s = *reinterpret_cast<const float4*>(a.scores + at * a.score_stride + j);   // (whole rows of 32)
        const long long seen = (a.start_pos + i + 1 < a.kv_len ? a.start_pos + i + 1 : a.kv_len) - j;
        const float p[4] = {__builtin_amdgcn_exp2f(s.x - st.x) * st.y, __builtin_amdgcn_exp2f(s.y - st.x) * st.y,
                            __builtin_amdgcn_exp2f(s.z - st.x) * st.y, __builtin_amdgcn_exp2f(s.w - st.x) * st.y};
        #pragma unroll
        for (int u = 0; u < 4; u++) sum[u] += u < seen ? p[u] : 0.0f;   // (undefined behind what the row sees)
        if (++g == G) {
            g = 0;
            i++;
        }
    }
    *reinterpret_cast<float4*>(a.sums + ((size_t)blockIdx.z * a.n_head_kv + hk) * a.score_stride + j) =
        make_float4(sum[0], sum[1], sum[2], sum[3]);
}

__global__ __launch_bounds__(256)
void mass_sum_kernel(MassArgs a, int runs) {
    const int j = blockIdx.x * 256 + threadIdx.x, hk = blockIdx.y;
    if (j >= a.kv_len) return;
    float sum = 0.0f;
    #pragma unroll 8
    for (int z = 0; z < runs; z++) sum += a.sums[((size_t)z * a.n_head_kv + hk) * a.score_stride + j];
    a.mass_out[(size_t)hk * a.mass_stride + j] = (a.mass_in ? a.mass_in[(size_t)hk * a.mass_stride + j] : 0.0f) + sum;
}

static size_t mass_rows(size_t n_head, size_t n_head_kv, size_t q_len) { return q_len * ((n_head + n_head_kv - 1) / n_head_kv); }

size_t attention_mass_stat(size_t n_head, size_t n_head_kv, size_t q_len) {
    return mass_rows(n_head, n_head_kv, q_len) <= (size_t)MASS_INLINE ? 0 : q_len * n_head * sizeof(float2);
}

size_t attention_mass_sums(size_t n_head, size_t n_head_kv, size_t q_len, size_t stride) {
    const size_t rows = mass_rows(n_head, n_head_kv, q_len);
    return rows <= (size_t)MASS_INLINE ? 0 : (rows + MASS_RUN - 1) / MASS_RUN * n_head_kv * stride * sizeof(float);
}

hipError_t attention_mass_launch(const MassArgs& a, hipStream_t s) {
    const size_t rows = mass_rows(a.n_head, a.n_head_kv, a.q_len);
    const unsigned heads = (unsigned)a.n_head_kv;
    if (rows <= (size_t)MASS_INLINE) {
        hipLaunchKernelGGL(mass_few_kernel, dim3((unsigned)((a.kv_len + 63) / 64), heads), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    const unsigned runs = (unsigned)((rows + MASS_RUN - 1) / MASS_RUN);
    hipLaunchKernelGGL(mass_stat_kernel, dim3((unsigned)(((size_t)a.q_len * a.n_head + 15) / 16)), dim3(256), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(mass_run_kernel, dim3((unsigned)((a.score_stride + 1023) / 1024), heads, runs), dim3(256), 0, s, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(mass_sum_kernel, dim3((unsigned)((a.kv_len + 255) / 256), heads), dim3(256), 0, s, a, (int)runs);
    return hipGetLastError();
}

}  // namespace barq
