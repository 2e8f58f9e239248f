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

// A thread owns four neighbouring pairs (VEC = 4, rot % 8 == 0) or one (VEC = 1,
// any even rot) and walks over heads with their cosines and sines: two
// 16-byte loads and stores a head, two heads' loads at a time (of single pairs
// four heads').  Where the rest of the head is copied (y != x), the threads
// after the pairs' copy it the same way.  A workgroup takes one
// row, or a part of its heads where rows are few.
// Memory bound: 4096 rows of 72 heads of 128 (302 MB) take 60.3 us, 5.0 TB/s
// (a 4 GiB copy reaches 4.7); one pass over heads at a time and scalar copies
// of the rest took 66.9.  Single pairs: 7438 rows of 40 heads of
// 116, 42 of them turned (276 MB), 58.8 us, 4.7 TB/s (89.7 with the rest
// copied after the pairs).  16 rows of 40 heads: 3 us, the launch and two
// rounds of load latency.
template <int VEC>
__global__ __launch_bounds__(256) void rope_scaled_kernel(float* y, const float* x, const int32_t* __restrict__ pos,
                                                          int n_heads, int hd, int64_t ld, int layout, int rot,
                                                          float magnitude, int units, int heads_per_wg,
                                                          const RopeTurns turns) {
    constexpr int N = VEC == 4 ? 4 : 1, HEADS = VEC == 4 ? 2 : 4;   // loads at a time
    typedef float vec __attribute__((ext_vector_type(N), aligned(4)));
    typedef float float4a __attribute__((ext_vector_type(4), aligned(4)));
    const int row = blockIdx.x;
    const int h0 = blockIdx.y * heads_per_wg, h1 = min(n_heads, h0 + heads_per_wg);
    const float* xr = x + (int64_t)row * ld;
    float* yr = y + (int64_t)row * ld;
    const int half = rot / 2, pairs = half / VEC;      // units that turn
    const int step = (int)blockDim.x / units;          // heads side by side (units <= blockDim.x)
    const int u = threadIdx.x % units, hh = threadIdx.x / units;
    if (hh < step) {
        const bool turn = u < pairs;
        const int i0 = u * VEC;
        // the unit's two places in a head
        const int ja = !turn || layout ? 2 * i0 : i0, jb = turn && !layout ? half + i0 : 2 * i0 + VEC;
        float c[VEC], s[VEC];
        if (turn) {
            const double p = (double)pos[row];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const double t = p * turns.w[i0 + e];
                sincospif((float)(2.0 * (t - rint(t))), &s[e], &c[e]);
                c[e] *= magnitude;
                s[e] *= magnitude;
            }
        }
        for (int h = h0 + hh; h < h1; h += HEADS * step) {
            vec a[HEADS], b[HEADS];
#pragma unroll
            for (int k = 0; k < HEADS; ++k) {
                if (VEC == 1 && k > 0 && h + k * step >= h1) break;
                const float* xh = xr + (int64_t)min(h + k * step, h1 - 1) * hd;
                a[k] = *(const vec*)(xh + ja);
                b[k] = *(const vec*)(xh + jb);
            }
#pragma unroll
            for (int k = 0; k < HEADS; ++k) {
                if (h + k * step >= h1) break;
                vec ya = a[k], yb = b[k];
                if (turn) {
                    if constexpr (VEC == 1) {
                        ya[0] = a[k][0] * c[0] - b[k][0] * s[0];
                        yb[0] = b[k][0] * c[0] + a[k][0] * s[0];
                    } else if (layout == 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ya[e] = a[k][e] * c[e] - b[k][e] * s[e];
                            yb[e] = b[k][e] * c[e] + a[k][e] * s[e];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            ya[e] = a[k][e] * c[e / 2] - a[k][e + 1] * s[e / 2];
                            ya[e + 1] = a[k][e + 1] * c[e / 2] + a[k][e] * s[e / 2];
                            yb[e] = b[k][e] * c[2 + e / 2] - b[k][e + 1] * s[2 + e / 2];
                            yb[e + 1] = b[k][e + 1] * c[2 + e / 2] + b[k][e] * s[2 + e / 2];
                        }
                    }
                }
                float* yh = yr + (int64_t)(h + k * step) * hd;
                *(vec*)(yh + ja) = ya;
                *(vec*)(yh + jb) = yb;
            }
        }
    }
    const int done = 2 * VEC * units, tail = hd - done;   // what the units leave of a head
    if (tail > 0 && y != x) {
        const int each = (tail + 3) / 4;               // four floats a thread, the last of a head up to four
        for (int e = threadIdx.x; e < (h1 - h0) * each; e += blockDim.x) {
            const int c = 4 * (e % each);
            const int64_t at = (int64_t)(h0 + e / each) * hd + done + c;
            if (c + 4 <= tail)
                *(float4a*)(yr + at) = *(const float4a*)(xr + at);
            else
                for (int k = 0; k < tail - c; ++k) yr[at + k] = xr[at + k];
        }
    }
}

int launch_rope_scaled(float* y, const float* x, const int32_t* pos, int n_rows, int n_heads, int hd, int64_t ld,
                       int layout, int rot, float magnitude, const RopeTurns& turns, hipStream_t s) {
    const bool vec = rot % 8 == 0;
    const int wide = vec ? 8 : 2;
    const int units = y != x && hd <= 256 * wide ? hd / wide : rot / wide;
    const int step = 256 / units;
    // few rows: a workgroup takes as many heads as it has threads for
    const int per = n_rows < 512 ? max(step, n_heads / 32768) : n_heads;
    const dim3 grid(n_rows, (n_heads + per - 1) / per);
    if (vec)
        hipLaunchKernelGGL(rope_scaled_kernel<4>, grid, dim3(256), 0, s, y, x, pos, n_heads, hd, ld, layout, rot,
                           magnitude, units, per, turns);
    else
        hipLaunchKernelGGL(rope_scaled_kernel<1>, grid, dim3(256), 0, s, y, x, pos, n_heads, hd, ld, layout, rot,
                           magnitude, units, per, turns);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
