// attn_rows.h -- a wave's 16 query rows: the part of the MFMA
// attention kernels that does not go by how K and V are stored.
//
//   S^T [32 keys x 16 rows] = K Q^T,   O^T [hd x 16 rows] += V^T P^T
//
// K and V come as f16 numbers times a power of two or a step each (per key, or
// per key and 32 elements).  Q and P are split into two halves, hi = f16(x)
// and lo = f16(x - hi), 22 bits in all.  Softmax, sums and steps are f32 (but
// V's steps of 32 keys that all rows see, f16 relative to the largest of them: 11
// bits like the steps themselves down to 2^-14 of it, and 2^-25 of it below).
// A row's running maximum moves only when a score passes it by 2^4, so weights
// reach 2^4; weight times step carries a power of two by the largest V step seen,
// so that it stays inside f16's range whatever V's size is.
#pragma once
#include "lanes.h"
#include "mfma.h"
#include "packed.h"

namespace slate_hip {

constexpr int AR_TILE = 16;            // query rows of an MFMA
constexpr int AR_KEYS = 32;            // keys of a step
constexpr float AR_SLACK = 4.0f;       // log2 of the largest weight before the maximum moves
constexpr int AR_PEXP = 11;            // weight 1 times the largest V step is scaled to [2^10, 2^11)

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef int int2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes at any float

// Over the four lanes that hold one row (j, j + 16, j + 32, j + 48).
__device__ __forceinline__ float cols_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float cols_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Zeros to start sums of products from, in registers that the MFMA leaves as
// they are (as a constant the compiler writes them out for every chain).
__device__ __forceinline__ floatx4 zeros() {
    floatx4 z = {0.f, 0.f, 0.f, 0.f};
    asm("" : "+v"(z));
    return z;
}

// p times an f16 step in one operation (v_fma_mix_f32).
__device__ __forceinline__ float times(float p, _Float16 d) { return fmaf(p, (float)d, 0.f); }

// x = hi + lo to 22 bits.
__device__ __forceinline__ void halves(const float* x, half8_t& hi, half8_t& lo) {
    float minus = -1.0f;               // the compiler does not see that it could subtract
    asm("" : "+s"(minus));
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float2v v = {x[e], x[e + 1]};
        const half2_t h = __builtin_convertvector(v, half2_t);
        // x - hi, exact, in one operation that takes hi as it is (v_fma_mix_f32)
        const float2v r = {fmaf((float)h[0], minus, x[e]), fmaf((float)h[1], minus, x[e + 1])};
        const half2_t l = __builtin_convertvector(r, half2_t);
        hi[e] = h[0];
        hi[e + 1] = h[1];
        lo[e] = l[0];
        lo[e + 1] = l[1];
    }
}

// Bits of the drafts that a token sees (bit d: draft d of its sequence) as
// bits of the keys k0 .. k0 + 31: committed keys (below p0) are seen.
__device__ __forceinline__ uint32_t seen_keys(uint32_t drafts, int k0, int p0) {
    const int d = k0 - p0;
    if (d <= -32) return 0xffffffffu;
    if (d < 0) return drafts << -d | ((1u << -d) - 1);
    return d < 32 ? drafts >> d : 0;
}

// Lane (g, j) = (lane / 16, lane % 16) holds row j.
template <int HD>
struct AttnRows {
    static constexpr int NB = HD / 32, ND = HD / 16;
    half8_t qh[NB], ql[NB];    // Q^T as the B operand: elements 32t + 8g .. +7 of row j
    floatx4 o[ND];                 // O^T: columns 16n + 4g .. +3 of row j
    float unq;                     // what undoes Q's scale
    float m, l;                // running maximum (log2), the lane's part of the sum
    float pexp;                    // o is 2^pexp times what l and m say
    int lim;                       // the largest V step seen, as the caller orders them (0: none)

    // Rows from q (raw: elements 32t + 8g .. +7 of row j; not live: no row),
    // scaled by `scale` and then to [2^13, 2^14) at the row's largest element:
    // lo keeps its 11 bits for any element within 2^-14 of that one.
    __device__ __forceinline__ void start(const float4u (*raw)[2], bool live, float scale) {
        float v[NB][8], top = 0.f;
#pragma unroll
        for (int t = 0; t < NB; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[t][e] = live ? raw[t][e >> 2][e & 3] * scale : 0.f;
                top = fmaxf(top, fabsf(v[t][e]));
            }
        top = cols_max(top);
        const int e2 = top > 0.f ? min(126, 14 - __builtin_amdgcn_frexp_expf(top)) : 0;   // unq is not 0
        unq = ldexpf(1.0f, -e2);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[t][e] = ldexpf(v[t][e], e2);
            halves(v[t], qh[t], ql[t]);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] = floatx4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.f;
        pexp = 0.f;
        lim = 0;
    }

    // The weights p = 2^(score - m) of the lane's 4 H scores s (keys 16 hf + 4g + i of row j;
    // -inf: not seen).  big: the largest V step, in the lane's own keys
    // (EACH) or in any lane; exponent(big): e with that step in [2^(e-1), 2^e).
    // The caller multiplies them, or the steps, by 2^pexp: an exponent of 64 or
    // more (V may be of any size, pexp is up to 100) would keep but 17 bits behind
    // its point.  Or p has the powers of two pexp + shift[i] in it, 11 at most,
    // for each 32 keys.
    template <int H, bool EACH, class Exponent>
    __device__ __forceinline__ void weights(const floatx4* s, int big, const Exponent& exponent, float* p,
                                            const int* shift = nullptr) {
        float mx = s[0][0];
#pragma unroll
        for (int e = 1; e < 4 * H; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
        mx *= unq;
        if (__builtin_amdgcn_ballot_w64(mx > m + AR_SLACK || big > lim)) {
            const float mn = fmaxf(m, cols_max(mx));
            float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
            if (__builtin_amdgcn_ballot_w64(big > lim)) {
                if (!EACH)
#pragma unroll
                    for (int off = 1; off < 16; off <<= 1) big = max(big, __shfl_xor(big, off));
                big = max(big, __shfl_xor(big, 16));
                big = max(big, __shfl_xor(big, 32));
                if (big > lim) {
                    lim = big;
                    const float pe = (float)(AR_PEXP - exponent(big));
                    f *= __builtin_amdgcn_exp2f(pe - pexp);
                    pexp = pe;
                }
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) o[n] *= f;
        }
        const float mref = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int b = 0; b < H / 2; ++b) {
            const float k = shift ? pexp + (float)shift[b] : 0.f;
            const float by = mref + k;
            float sum = 0.f;
#pragma unroll
            for (int e = 8 * b; e < 8 * b + 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], unq, by));
                (shift ? sum : l) += p[e];
            }
            if (shift) l += ldexpf(sum, -(int)k);
        }
    }

    // What undoes o's scale, and the sum of the weights over the keys.
    __device__ __forceinline__ float back() const { return __builtin_amdgcn_exp2f(-pexp); }
    __device__ __forceinline__ float sum() const { return cols_sum(l); }
};

}  // namespace slate_hip
