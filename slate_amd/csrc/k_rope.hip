// k_rope.hip -- rotary positions: pairs in halves or interleaved, part of a
// head, angles from frequencies given per pair.
//
//   y_j = m (x_j cos a - x_k sin a),  y_k = m (x_k cos a + x_j sin a),
//   a = 2 pi * frac(pos * w_i),  (j, k) the pair's elements
//
// The product pos * w_i (w_i in turns per position) and its reduction to half
// a turn are done in f64: in f32 the angle of position p is off by about
// p * 2^-24 radians.  What is left goes to sincospif.
#include "packed.h"

namespace slate_hip {

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes at any float

// VEC = 4: a thread turns four neighbouring pairs by 16-byte loads and
// stores, which needs rot % 8 == 0; VEC = 1 takes any even rot.  A thread
// keeps its pairs' cosines for all the heads that it walks over, and a
// workgroup takes one row, or a part of its heads.
template <int VEC>
__global__ __launch_bounds__(256) void rope_scaled_kernel(float* y, const float* x,
                                                          const int32_t* __restrict__ pos, int n_heads, int hd,
                                                          int64_t ld, int layout, int rot, float magnitude,
                                                          int heads_per_wg, const RopeTurns turns) {
    const int row = blockIdx.x;
    const int h0 = blockIdx.y * heads_per_wg, h1 = min(n_heads, h0 + heads_per_wg);
    const float* xr = x + (int64_t)row * ld;
    float* yr = y + (int64_t)row * ld;
    const int half = rot / 2;
    const int units = half / VEC;                      // threads that share a head
    const int step = (int)blockDim.x / units;          // heads side by side (units <= blockDim.x)
    const int u = threadIdx.x % units, hh = threadIdx.x / units;
    const int i0 = u * VEC;
    if (hh < step) {
        const double p = (double)pos[row];
        float c[VEC], s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const double t = p * turns.w[i0 + e];
            sincospif((float)(2.0 * (t - rint(t))), &s[e], &c[e]);
            c[e] *= magnitude;
            s[e] *= magnitude;
        }
        for (int h = h0 + hh; h < h1; h += step) {
            const float* xh = xr + (int64_t)h * hd;
            float* yh = yr + (int64_t)h * hd;
            if constexpr (VEC == 4) {
                const int ja = layout == 0 ? i0 : 2 * i0, jb = layout == 0 ? half + i0 : 2 * i0 + 4;
                const float4u a = *(const float4u*)(xh + ja), b = *(const float4u*)(xh + jb);
                float4u ya, yb;
                if (layout == 0) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ya[e] = a[e] * c[e] - b[e] * s[e];
                        yb[e] = b[e] * c[e] + a[e] * s[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        ya[2 * e] = a[2 * e] * c[e] - a[2 * e + 1] * s[e];
                        ya[2 * e + 1] = a[2 * e + 1] * c[e] + a[2 * e] * s[e];
                        yb[2 * e] = b[2 * e] * c[e + 2] - b[2 * e + 1] * s[e + 2];
                        yb[2 * e + 1] = b[2 * e + 1] * c[e + 2] + b[2 * e] * s[e + 2];
                    }
                }
                *(float4u*)(yh + ja) = ya;
                *(float4u*)(yh + jb) = yb;
            } else {
                const int j = layout == 0 ? i0 : 2 * i0, k = layout == 0 ? half + i0 : 2 * i0 + 1;
                const float a = xh[j], b = xh[k];
                yh[j] = a * c[0] - b * s[0];
                yh[k] = b * c[0] + a * s[0];
            }
        }
    }
    const int tail = hd - rot;
    if (tail > 0 && y != x) {
        for (int e = threadIdx.x; e < (h1 - h0) * tail; e += blockDim.x) {
            const int64_t at = (int64_t)(h0 + e / tail) * hd + rot + e % tail;
            yr[at] = xr[at];
        }
    }
}

int launch_rope_scaled(float* y, const float* x, const int32_t* pos, int n_rows, int n_heads, int hd, int64_t ld,
                       int layout, int rot, float magnitude, const RopeTurns& turns, hipStream_t s) {
    const bool vec = rot % 8 == 0;
    const int step = 256 / (rot / 2 / (vec ? 4 : 1));
    // few rows: a workgroup takes as many heads as it has threads for
    const int per = n_rows < 512 ? step : n_heads;
    const dim3 grid(n_rows, (n_heads + per - 1) / per);
    if (vec)
        hipLaunchKernelGGL(rope_scaled_kernel<4>, grid, dim3(256), 0, s, y, x, pos, n_heads, hd, ld, layout, rot,
                           magnitude, per, turns);
    else
        hipLaunchKernelGGL(rope_scaled_kernel<1>, grid, dim3(256), 0, s, y, x, pos, n_heads, hd, ld, layout, rot,
                           magnitude, per, turns);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
