// Position rotation as the paged cache's append and norm_rope use it: pairs of the
// first `rot` dims of a head turn by position * freq_scale * inv_freq, cos and sin
// times a magnitude; the dims behind them stay.
#pragma once
#include "common.hpp"
#include "launch.hpp"

namespace barq {

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// cos and sin of a pair's angle.  In 64 bits up to the fraction of a turn: an f32
// angle of position 100000 is off by 0.004.  What is left of it is x, an eighth of a turn at
// most, where Taylor's series with 5 terms of the sine and 6 of the cosine are off by 2e-9 and 2e-10 of
// 1: far below f32's rounding, and a seventh of the instructions of a general sine and cosine
// (1024 pairs of a workgroup were half of all it executed).
__device__ __forceinline__ float2 rotary_turn(int pos, const Rotary& r, int i) {
    const double turns = (double)pos * (double)r.freq_scale * (double)r.inv_freq[i] * 0.15915494309189533577;
    const double quarter = rint(4.0 * turns);
    const float x = (float)((turns - 0.25 * quarter) * 6.28318530717958647693), z = x * x;
    float s = __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040), c = __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320);
    s = __builtin_fmaf(z, s, 1.0f / 120);
    s = __builtin_fmaf(z, s, -1.0f / 6);
    s = __builtin_fmaf(z * x, s, x);
    c = __builtin_fmaf(z, c, -1.0f / 720);
    c = __builtin_fmaf(z, c, 1.0f / 24);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.0f);
    const int k = (int)((long long)quarter & 3);
    const float cs = k & 1 ? s : c, sn = k & 1 ? c : s;
    return make_float2((k == 1 || k == 2 ? -cs : cs) * r.magnitude, (k & 2 ? -sn : sn) * r.magnitude);
}

// The lane's eight dims d0 .. d0 + 7 of a head (a row of HD / 8 neighbouring lanes, 16-byte aligned): loaded, then
// normed where w is not null and rotated where r.rot is not zero, with cos and sin of pair i at turn[i].
// ODD: split halves that are no multiple of 8, in a kernel of their own, beside which the others stay 3 % faster (2048 rows of 32
// heads of 128 dims, 90 of them rotated: norm_rope 14.4 us, 23.5 when the other halves were read once more).
template <int HD, bool ODD>
struct TurnRow {
    float x[8];
    __device__ __forceinline__ void load(const float* __restrict__ row, int d0) {
        #pragma unroll
        for (int u = 0; u < 2; u++) {
            const float4 v = *reinterpret_cast<const float4*>(row + d0 + 4 * u);
            x[4 * u] = v.x, x[4 * u + 1] = v.y, x[4 * u + 2] = v.z, x[4 * u + 3] = v.w;
        }
    }
    __device__ __forceinline__ void turn(int d0, const float* __restrict__ w, float eps, const Rotary& r, const float2* turn) {
        float f = 1.0f;
        if (w) {   // (the sum in the same order whatever the grid)
            float ss = 0.0f;
            #pragma unroll
            for (int e = 0; e < 8; e++) ss = __builtin_fmaf(x[e], x[e], ss);
            ss = group_sum<HD / 8>(ss);
            f = 1.0f / sqrtf(ss / (float)HD + fmaxf(eps, 1.1920929e-7f));
            #pragma unroll
            for (int u = 0; u < 2; u++) {
                const f32x4_a4 v = *reinterpret_cast<const f32x4_a4*>(w + d0 + 4 * u);
                #pragma unroll
                for (int e = 0; e < 4; e++) x[4 * u + e] = (x[4 * u + e] * f) * v[e];
            }
        }
        // (no branch on an element: a pair behind the rotated dims is not turned, or what it gives not taken)
        if constexpr (ODD) {
            turn_odd(d0, r, turn);
        } else if (r.layout == ROPE_INTERLEAVED) {
            #pragma unroll
            for (int u = 0; u < 2; u++) {
                const float4 t = *reinterpret_cast<const float4*>(turn + d0 / 2 + 2 * u);
                float* y = x + 4 * u;
                const float a = y[0] * t.x - y[1] * t.y, b = y[0] * t.y + y[1] * t.x;
                const float c = y[2] * t.z - y[3] * t.w, d = y[2] * t.w + y[3] * t.z;
                const bool one = d0 + 4 * u < r.rot, two = d0 + 4 * u + 2 < r.rot;
                y[0] = one ? a : y[0];
                y[1] = one ? b : y[1];
                y[2] = two ? c : y[2];
                y[3] = two ? d : y[3];
            }
        } else {   // the pairs' other halves: whole lanes of the row
            const int half = r.rot / 2;
            const bool low = d0 < half, in = d0 < r.rot;
            const int lane = (threadIdx.x & 63) + (!in ? 0 : low ? half / 8 : -half / 8);
            const float sign = low ? -1.0f : 1.0f;
            const float4* t4 = reinterpret_cast<const float4*>(turn + (!in ? 0 : low ? d0 : d0 - half));
            #pragma unroll
            for (int u = 0; u < 4; u++) {
                const float4 t = t4[u];
                const float a = x[2 * u], b = x[2 * u + 1], za = __shfl(a, lane) * sign, zb = __shfl(b, lane) * sign;
                x[2 * u] = in ? a * t.x + za * t.y : a;
                x[2 * u + 1] = in ? b * t.z + zb * t.w : b;
            }
        }
    }
    // A lane's other halves lie in two lanes: its own values in those lanes' order, from each of them.
    __device__ __forceinline__ void turn_odd(int d0, const Rotary& r, const float2* turn) {
        const int half = r.rot / 2, lanes = half / 8, by = half % 8, lane = threadIdx.x & 63;
        float up[8], down[8];
        turned_round(x, by, up);
        turned_round(x, 8 - by, down);
        #pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = d0 + e;
            const float above = __shfl(up[e], lane + lanes + (e + by >= 8 ? 1 : 0)), below = __shfl(down[e], lane - lanes - (e < by ? 1 : 0));
            const bool low = d < half, in = d < r.rot;
            const float2 t = turn[!in ? 0 : low ? d : d - half];
            const float y = x[e] * t.x + (low ? -above : below) * t.y;
            x[e] = in ? y : x[e];
        }
    }
    // to[e] = from[(e + by) % 8]
    __device__ __forceinline__ static void turned_round(const float (&from)[8], int by, float (&to)[8]) {
        typedef float f8 __attribute__((ext_vector_type(8)));
        f8 v = {from[0], from[1], from[2], from[3], from[4], from[5], from[6], from[7]};
        const f8 a = __builtin_shufflevector(v, v, 1, 2, 3, 4, 5, 6, 7, 0);
        v = by & 1 ? a : v;
        const f8 b = __builtin_shufflevector(v, v, 2, 3, 4, 5, 6, 7, 0, 1);
        v = by & 2 ? b : v;
        const f8 c = __builtin_shufflevector(v, v, 4, 5, 6, 7, 0, 1, 2, 3);
        v = by & 4 ? c : v;
        #pragma unroll
        for (int e = 0; e < 8; e++) to[e] = v[e];
    }
};

inline bool rotary_odd(const Rotary& r) { return r.layout == ROPE_SPLIT_HALF && r.rot % 16 != 0; }

constexpr int TURN_TOKENS = 16;   // tokens of a workgroup

// cos and sin of the rotated pairs of tokens pos .. pos + n - 1: turn[token][pair].  (The others' are not written, nor is
// anything kept of what they turn.)
template <int HD>
__device__ __forceinline__ void turn_table(float2 (*turn)[HD / 2], int pos, int n, const Rotary& r) {
    const int half = r.rot / 2;
    for (int u = threadIdx.x; u < n * half; u += 256) turn[u / half][u % half] = rotary_turn(pos + u / half, r, u % half);
}

}  // namespace barq
