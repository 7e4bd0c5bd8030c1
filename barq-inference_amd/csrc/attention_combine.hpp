// Merging the partial states that a row's splits of the positions leave:
// [n_split][HD + 2] floats, the reference maximum (log2 units), the sum, the
// unnormalised outputs.
#pragma once
#include "common.hpp"
#include "q8k_block.hpp"

namespace barq {

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int ATT_MAX_SPLIT = 1024;

// One output head: out value of dim t (t < HD) from the n_split partial
// states at pp (and unless null its maximum and 1 / sum to stat), by NT threads t = 0 .. NT - 1 (all of them call it: it
// synchronises the workgroup).  The split maxima and weights are spread over
// the threads; the output sums run over SUB = 1024 / HD subsets of the splits
// (split s in subset s % SUB, in increasing order), then are added in LDS in
// subset order.  With NT < 1024 each thread runs 1024 / NT subsets one after
// another, so the sums and their order do not depend on NT: the Q8_K merge
// (heads side by side) quantizes exactly the f32 merge's values.
template <int HD>
struct CombineLds {
    float w[ATT_MAX_SPLIT];
    float red[1024 / HD][HD];
    float wred[2][1024 / 64];
};

template <int HD, int NT>
__device__ __forceinline__ float attn_combine_head(const float* __restrict__ pp, int n_split, CombineLds<HD>& sm,
                                                   int t, float2* stat = nullptr) {
    constexpr int NWV = NT / 64, SUB = 1024 / HD, K = 1024 / NT, STEP = NT / HD, PRE = 8;
    static_assert(NT % HD == 0 && 1024 % NT == 0, "threads per head");
    const int lane = t & 63, wave = t >> 6;
    const int sub = t / HD, d = t % HD;   // subsets sub + STEP j, j < K
    // every load of the first PRE rounds is issued before any reduction
    float ov[K][PRE];
    #pragma unroll
    for (int j = 0; j < K; j++)
        #pragma unroll
        for (int u = 0; u < PRE; u++) {
            const int s = sub + STEP * j + SUB * u;
            ov[j][u] = s < n_split ? pp[(size_t)s * (HD + 2) + 2 + d] : 0.0f;
        }
    // the maximum and sum of the splits t + NT j (j < K), loaded with the
    // output sums above (n_split <= ATT_MAX_SPLIT = 1024, so these are all of
    // this thread's splits): no load waits once the reductions start
    static_assert(ATT_MAX_SPLIT <= 1024, "one split per virtual lane");
    float Msj[K], Lsj[K];
    #pragma unroll
    for (int j = 0; j < K; j++) {
        const int s = t + NT * j;
        Msj[j] = s < n_split ? pp[(size_t)s * (HD + 2)] : -INFINITY;
        Lsj[j] = s < n_split ? pp[(size_t)s * (HD + 2) + 1] : 0.0f;
    }
    float M = Msj[0];
    #pragma unroll
    for (int j = 1; j < K; j++) M = fmaxf(M, Msj[j]);
    M = wave_max_all(M);
    if (lane == 0) sm.wred[0][wave] = M;
    __syncthreads();
    M = sm.wred[0][0];
    #pragma unroll
    for (int u = 1; u < NWV; u++) M = fmaxf(M, sm.wred[0][u]);
    // The denominator in the 1024-thread merge's order whatever NT is: thread
    // t plays the 1024 lanes t + NT j (j < K), each holding its one split; a
    // reduction per 64 of those lanes (a real wave holds 64 consecutive ones);
    // then the 16 wave partials in lane order.  So the Q8_K merge's rows are
    // the f32 merge's to the bit.
    float Lj[K];
    #pragma unroll
    for (int j = 0; j < K; j++) {
        const int s = t + NT * j;
        float L = 0.0f;
        if (s < n_split) {
            const float ws = Msj[j] == -INFINITY ? 0.0f : fast_exp2(Msj[j] - M);
            sm.w[s] = ws;
            L = Lsj[j] * ws;
        }
        L = wave_sum_all(L);
        Lj[j] = L;
    }
    if (lane == 0) {
        #pragma unroll
        for (int j = 0; j < K; j++) sm.wred[1][NWV * j + wave] = Lj[j];
    }
    __syncthreads();
    float L = sm.wred[1][0];
    #pragma unroll
    for (int u = 1; u < 1024 / 64; u++) L += sm.wred[1][u];
    if (stat && t == 0) *stat = make_float2(M, 1.0f / L);
    #pragma unroll
    for (int j = 0; j < K; j++) {
        const int sj = sub + STEP * j;
        float O = 0.0f;
        #pragma unroll
        for (int u = 0; u < PRE; u++) {
            const int s = sj + SUB * u;
            if (s < n_split) O = __builtin_fmaf(ov[j][u], sm.w[s], O);
        }
        for (int s = sj + SUB * PRE; s < n_split; s += SUB) O = __builtin_fmaf(pp[(size_t)s * (HD + 2) + 2 + d], sm.w[s], O);
        sm.red[sj][d] = O;
    }
    __syncthreads();
    float acc = 0.0f;
    if (t < HD) {
        acc = sm.red[0][t];
        #pragma unroll
        for (int u = 1; u < SUB; u++) acc += sm.red[u][t];
        acc = acc / L;
    }
    return acc;
}

// out[i, h, :] by a workgroup of 1024 threads.
template <int HD>
__device__ __forceinline__ void attn_combine_row(const float* __restrict__ part, int n_split, int n_head, int h, int i,
                                                 CombineLds<HD>& sm, float* __restrict__ out, float2* stat = nullptr) {
    const int t = threadIdx.x;
    const size_t at = (size_t)i * n_head + h;
    const float v = attn_combine_head<HD, 1024>(part + at * n_split * (HD + 2), n_split, sm, t, stat ? stat + at : nullptr);
    if (t < HD) out[((size_t)i * n_head + h) * HD + t] = v;
}

// Block b of row i as Q8_K by a workgroup of 1024 threads: the block's 256 /
// HD heads side by side (1024 / (256 / HD) threads each), then one wave
// quantizes it (q8_k_block: the bytes quantize_q8_k_kernel writes for the same values).
template <int HD>
struct CombineQ8Lds {
    CombineLds<HD> head[256 / HD];
    __align__(16) float vals[256];
};
template <int HD>
__device__ __forceinline__ void attn_combine_q8k_block(const float* __restrict__ part, int n_split, int n_head, int b, int i,
                                                       CombineQ8Lds<HD>& sm, uint8_t* __restrict__ out,
                                                       float2* stat = nullptr) {
    constexpr int NH = 256 / HD, NT = 1024 / NH;
    const int t = threadIdx.x, hh = t / NT, tg = t % NT, h = b * NH + hh;
    const size_t at = (size_t)i * n_head + h;
    const float v = attn_combine_head<HD, NT>(part + at * n_split * (HD + 2), n_split, sm.head[hh], tg, stat ? stat + at : nullptr);
    if (tg < HD) sm.vals[hh * HD + tg] = v;
    __syncthreads();
    if (t < 64) {
        const float4 v4 = reinterpret_cast<const float4*>(sm.vals)[t];
        const float vv[4] = {v4.x, v4.y, v4.z, v4.w};
        q8_k_block(vv, t, out + ((size_t)i * (n_head * HD / 256) + b) * Q8_K_BYTES);
    }
}

}  // namespace barq
