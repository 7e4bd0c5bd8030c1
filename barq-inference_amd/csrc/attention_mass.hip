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
#include <type_traits>

#include "attention_combine.hpp"
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
        // (pieces that saw nothing leave -infinity and 0, pieces that saw only NaN -infinity and NaN, which stays in the sum)
        if (mn != -INFINITY) L = L * __builtin_amdgcn_exp2f(M - mn) + l * __builtin_amdgcn_exp2f(m - mn);
        else L += l;
        M = mn;
    }
    const float all = row16_max(M);
    L = row16_sum(M == -INFINITY ? 0.0f * L : L * __builtin_amdgcn_exp2f(M - all));
    return make_float2(all, 1.0f / L);
}

// query heads h with h * n_head_kv / n_head = hk: first, and behind the last
__device__ __forceinline__ int mass_head(const MassArgs& a, int hk) {
    return (int)(((long long)hk * a.n_head + a.n_head_kv - 1) / a.n_head_kv);
}

// Few rows, and their merge, in one launch (both need the partial states
// only): workgroups x < merges merge a row and head (or with Q8 a block of a
// row); each of the others takes 256 positions of a kv head at a time, a wave 64 of them
// and a fourth of the rows, whose statistics the workgroup finds itself (once: in a
// long cache it takes several 256).  One decoded token of 32/8 heads against 4096
// positions, with the attention: 11.5 to 12.4 us (4-bit) and 14.2 (f32); the launches
// for many rows took 16.2 and 17.3.
struct MassLds {
    float2 stat[MASS_INLINE];
    float red[4][256];
};
template <int HD, bool Q8>
union FinishLds {
    MassLds mass;
    typename std::conditional<Q8, CombineQ8Lds<HD>, CombineLds<HD>>::type merge;
};

template <int HD, bool Q8>
__global__ __launch_bounds__(1024)
void mass_finish_kernel(MassArgs a, int merges, void* __restrict__ out) {
    __shared__ FinishLds<HD, Q8> lds;
    if ((int)blockIdx.x < merges) {
        const int per = Q8 ? a.n_head * HD / 256 : a.n_head, x = (int)blockIdx.x % per, i = (int)blockIdx.x / per;
        if constexpr (Q8) attn_combine_q8k_block<HD>(a.part, a.ns, a.n_head, x, i, lds.merge, static_cast<uint8_t*>(out));
        else attn_combine_row<HD>(a.part, a.ns, a.n_head, x, i, lds.merge, static_cast<float*>(out));
        return;
    }
    const int blk = (int)blockIdx.x - merges, hk = blk % a.n_head_kv;
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = w / 4;
    const int step = ((int)gridDim.x - merges) / a.n_head_kv * 256;
    int j = blk / a.n_head_kv * 256 + w % 4 * 64 + l;
    const int h0 = mass_head(a, hk), G = mass_head(a, hk + 1) - h0, rows = G * a.q_len;
    // the scores are on their way while the statistics are found
    float s[MASS_INLINE / 4], before;
    const auto load = [&]() {
        #pragma unroll
        for (int u = 0; u < MASS_INLINE / 4; u++) {
            const int r = wr + 4 * u, i = r < rows ? r / G : 0;
            // (a position behind the row's last is not seen: its score is undefined)
            const bool seen = r < rows && j < a.kv_len && j <= a.start_pos + i;
            s[u] = seen ? a.scores[((size_t)i * a.n_head + h0 + r - i * G) * a.score_stride + j] : -INFINITY;
        }
        before = wr == 0 && a.mass_in && j < a.kv_len ? a.mass_in[(size_t)hk * a.mass_stride + j] : 0.0f;
    };
    load();
    if ((int)threadIdx.x / 16 < rows) {   // (whole rows of 16 lanes)
        const int r = threadIdx.x / 16;
        const float2 st = mass_stat(a, (size_t)(r / G) * a.n_head + h0 + r % G, threadIdx.x & 15);
        if ((threadIdx.x & 15) == 0) lds.mass.stat[r] = st;
    }
    __syncthreads();
    for (;;) {
        float sum = 0.0f;
        #pragma unroll
        for (int u = 0; u < MASS_INLINE / 4; u++) {
            const int r = wr + 4 * u, i = r < rows ? r / G : 0;
            if (r < rows && j <= a.start_pos + i) sum += __builtin_amdgcn_exp2f(s[u] - lds.mass.stat[r].x) * lds.mass.stat[r].y;
        }
        lds.mass.red[wr][64 * (w % 4) + l] = sum;
        __syncthreads();
        if (wr == 0 && j < a.kv_len) {
            const int q = 64 * w + l;
            a.mass_out[(size_t)hk * a.mass_stride + j] =
                before + ((lds.mass.red[0][q] + lds.mass.red[1][q]) + (lds.mass.red[2][q] + lds.mass.red[3][q]));
        }
        if (a.kv_len - (j - (w % 4 * 64 + l)) <= step) break;   // (the same for the whole workgroup)
        j += step;
        load();
        __syncthreads();   // the sums are read
    }
}

template <int HD>
static hipError_t mass_finish_t(const MassArgs& a, float* out, uint8_t* out_q8, hipStream_t s) {
    const int merges = (out_q8 ? a.n_head * HD / 256 : a.n_head) * a.q_len;
    // about two workgroups a CU
    const int blocks = (a.kv_len + 255) / 256, most = (512 + a.n_head_kv - 1) / a.n_head_kv;
    const dim3 grid((unsigned)merges + (unsigned)(blocks < most ? blocks : most) * (unsigned)a.n_head_kv);
    if (out_q8) hipLaunchKernelGGL((mass_finish_kernel<HD, true>), grid, dim3(1024), 0, s, a, merges, out_q8);
    else hipLaunchKernelGGL((mass_finish_kernel<HD, false>), grid, dim3(1024), 0, s, a, merges, out);
    return hipGetLastError();
}

// Many rows: a wave takes 256 positions, four in a row per lane, and a run of
// rows; its sums go to sums[run][hk][position].
// Grid: x = 1024 positions (four waves), y = kv head, z = run.
// 512 rows of 32/8 heads against 2048 positions: 21.6 us for 134 MB of scores, 6.2 TB/s.
__global__ __launch_bounds__(256)
void mass_run_kernel(MassArgs a, int run) {
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hk = blockIdx.y;
    const int j = (blockIdx.x * 4 + w) * 256 + 4 * l;
    const int h0 = mass_head(a, hk), G = mass_head(a, hk + 1) - h0, rows = G * a.q_len;
    const int r0 = blockIdx.z * run, r1 = min(rows, r0 + run);
    if (j >= (int)a.score_stride) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int i = r0 / G, g = r0 - i * G;
    #pragma unroll 4
    for (int r = r0; r < r1; r++) {
        const size_t at = (size_t)i * a.n_head + h0 + g;
        const float2 st = a.stat[at];
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

bool attention_mass_few(size_t n_head, size_t n_head_kv, size_t q_len) {
    return mass_rows(n_head, n_head_kv, q_len) <= (size_t)MASS_INLINE;
}

// Rows of a run: 16 to 64, about two workgroups a CU in all.  With 64 always /
// 32 always, us with the attention: 32/8 heads, 64 rows after 1000 39.6 / 34.4, 16
// after 4000 36.1 / 31.0, 512 after 1536 100 / 111.
static size_t mass_run(size_t rows, size_t n_head_kv, size_t stride) {
    const size_t run = rows * n_head_kv * ((stride + 1023) / 1024) / 512;
    return run < 16 ? 16 : run > 64 ? 64 : run;
}

size_t attention_mass_sums(size_t n_head, size_t n_head_kv, size_t q_len, size_t stride) {
    const size_t rows = mass_rows(n_head, n_head_kv, q_len), run = mass_run(rows, n_head_kv, stride);
    return (rows + run - 1) / run * n_head_kv * stride * sizeof(float);
}

hipError_t attention_mass_few_launch(const MassArgs& a, const AttnArgs& attn, uint8_t* out_q8, hipStream_t s) {
    switch (a.head_dim) {
    case 64: return mass_finish_t<64>(a, attn.out, out_q8, s);
    case 128: return mass_finish_t<128>(a, attn.out, out_q8, s);
    case 256: return mass_finish_t<256>(a, attn.out, out_q8, s);
    default: return hipErrorInvalidValue;
    }
}

hipError_t attention_mass_launch(const MassArgs& a, hipStream_t s) {
    const unsigned heads = (unsigned)a.n_head_kv;
    const size_t rows = mass_rows(a.n_head, a.n_head_kv, a.q_len), run = mass_run(rows, a.n_head_kv, a.score_stride);
    const unsigned runs = (unsigned)((rows + run - 1) / run);
    hipLaunchKernelGGL(mass_run_kernel, dim3((unsigned)((a.score_stride + 1023) / 1024), heads, runs), dim3(256), 0, s, a, (int)run);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(mass_sum_kernel, dim3((unsigned)((a.kv_len + 255) / 256), heads), dim3(256), 0, s, a, (int)runs);
    return hipGetLastError();
}

}  // namespace barq
