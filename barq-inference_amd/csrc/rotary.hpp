// Position rotation as the paged cache's append and norm_rope use it: pairs of the
// first `rot` dims of a head turn by position * freq_scale * inv_freq, cos and sin
// times a magnitude; the dims behind them stay.
#pragma once
#include "common.hpp"
#include "launch.hpp"

namespace barq {

// cos and sin of a pair's angle.  In 64 bits up to the fraction of a turn: an f32
// angle of position 100000 is off by 0.004.  The rest is an eighth of a turn at most.
__device__ __forceinline__ float2 rotary_turn(int pos, const Rotary& r, int i) {
    const double turns = (double)pos * (double)r.freq_scale * (double)r.inv_freq[i] * 0.15915494309189533577;
    const double quarter = rint(4.0 * turns);
    float s, c;
    sincospif(2.0f * (float)(turns - 0.25 * quarter), &s, &c);
    const int k = (int)((long long)quarter & 3);
    const float cs = k == 0 ? c : k == 1 ? -s : k == 2 ? -c : s;
    const float sn = k == 0 ? s : k == 1 ? c : k == 2 ? -s : -c;
    return make_float2(cs * r.magnitude, sn * r.magnitude);
}

// The lane's eight dims d0 .. d0 + 7 of a head (a row of HD / 8 neighbouring lanes, 16-byte aligned): loaded, then
// normed where w is not null and rotated where r.rot is not zero, with cos and sin of pair i at turn[i].
template <int HD>
struct TurnRow {
    float x[8];
    __device__ __forceinline__ void load(const float* __restrict__ row, int d0) {
        #pragma unroll
        for (int u = 0; u < 2; u++) {
            const float4 v = *reinterpret_cast<const float4*>(row + d0 + 4 * u);
            x[4 * u] = v.x, x[4 * u + 1] = v.y, x[4 * u + 2] = v.z, x[4 * u + 3] = v.w;
        }
    }
    __device__ __forceinline__ void turn(const float* __restrict__ row, int d0, const float* __restrict__ w, float eps, const Rotary& r,
                                         const float2* turn) {
        float f = 1.0f;
        if (w) {   // (the sum in the same order whatever the grid)
            float ss = 0.0f;
            #pragma unroll
            for (int e = 0; e < 8; e++) ss = __builtin_fmaf(x[e], x[e], ss);
            ss = group_sum<HD / 8>(ss);
            f = 1.0f / sqrtf(ss / (float)HD + fmaxf(eps, 1.1920929e-7f));
            #pragma unroll
            for (int e = 0; e < 8; e++) x[e] = (x[e] * f) * w[d0 + e];
        }
        if (r.layout == ROPE_INTERLEAVED) {
            #pragma unroll
            for (int e = 0; e < 8; e += 2) {
                if (d0 + e < r.rot) {
                    const float2 t = turn[(d0 + e) / 2];
                    const float a = x[e] * t.x - x[e + 1] * t.y, b = x[e] * t.y + x[e + 1] * t.x;
                    x[e] = a;
                    x[e + 1] = b;
                }
            }
        } else {
            // the pairs' other halves: whole lanes of the row, or read once more
            const int half = r.rot / 2, to = d0 < half ? half : -half;
            float z[8];
            if (half % 8 == 0) {
                const int lane = (threadIdx.x & 63) + (d0 < r.rot ? to / 8 : 0);
                #pragma unroll
                for (int e = 0; e < 8; e++) z[e] = __shfl(x[e], lane);
            } else {
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int d = d0 + e, other = d < half ? d + half : d - half;
                    z[e] = d < r.rot ? row[other] : 0.0f;
                    if (w && d < r.rot) z[e] = (z[e] * f) * w[other];
                }
            }
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = d0 + e;
                if (d < r.rot) {
                    const bool low = d < half;
                    const float2 t = turn[low ? d : d - half];
                    x[e] = low ? x[e] * t.x - z[e] * t.y : z[e] * t.y + x[e] * t.x;
                }
            }
        }
    }
};

constexpr int TURN_TOKENS = 16;   // tokens of a workgroup

// cos and sin of tokens pos .. pos + n - 1: turn[token][HD / 2]
template <int HD>
__device__ __forceinline__ void turn_table(float2 (*turn)[HD / 2], int pos, int n, const Rotary& r) {
    const int half = r.rot / 2;
    for (int u = threadIdx.x; u < n * half; u += 256) turn[u / half][u % half] = rotary_turn(pos + u / half, r, u % half);
}

}  // namespace barq
