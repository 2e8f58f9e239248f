// attn_q8.h -- the step of the 8-bit attention kernels: 32 keys against tiles
// of 16 query rows, operands in LDS and registers.
//
//   S^T [32 keys x 16 rows] = K Q^T, one MFMA K step per 32-element block, the
//       block's f32 result weighted by the key's step for it;
//   O^T [hd x 16 rows] += V^T P^T, with P weighted by the steps of V, block by
//       block of 32 output columns.
//
// The codes are exact in f16.  Q and P are split into two halves, hi = f16(x)
// and lo = f16(x - hi), 22 bits in all, so a product costs two f16 MFMAs and
// nothing is rounded to fewer bits than that.  Softmax, sums and steps are
// f32.  A row's running maximum moves only when a score passes it by 2^4, so
// weights reach 2^4; they carry a power of two by the largest V step seen, so
// that weight times step stays inside f16's range whatever V's size is.
#pragma once
#include "lanes.h"
#include "mfma.h"
#include "packed.h"

namespace slate_hip {

constexpr float A8_SLACK = 4.0f;       // log2 of the largest weight before the maximum moves
constexpr int A8_PEXP = 11;            // weight 1 times the largest V step is scaled to [2^10, 2^11)

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef int int2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes at any float

template <int HD>
struct Q8Geom {
    static constexpr int NB = HD / 32;                 // steps (blocks) of a row
    static constexpr int ND = HD / 16;                 // 16-column tiles of V
    static constexpr int CH = HD / 16;                 // 16-byte chunks of a row of codes
    static constexpr int SH = HD == 128 ? 1 : HD == 64 ? 2 : 3;
};
template <int HD>
struct alignas(HD / 16) Q8Steps {
    _Float16 s[HD / 32];
};

// Where chunk c of key k (0 .. 31) sits in its LDS row, at place c ^ swz(k):
// 256 / HD rows share a round of the banks, the ones after them are shifted,
// and keys 16 apart, which the transposing read takes together, too.
template <int HD>
__device__ __forceinline__ int swz(int k) {
    using G = Q8Geom<HD>;
    return ((k >> G::SH) ^ ((k >> 4) << (3 - G::SH))) & (G::CH - 1);
}

// Eight codes as f16: 0x6400 | (code + 128) is the number 1152 + code.
__device__ __forceinline__ half8_t codes_f16(uint2v x) {
    const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    half8_t r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const uint32_t u = x[w] ^ 0x80808080u;
        const half2_t a = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
        const half2_t b = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
        r[4 * w] = a[0];
        r[4 * w + 1] = a[1];
        r[4 * w + 2] = b[0];
        r[4 * w + 3] = b[1];
    }
    return r;
}

// Transposing LDS read of bytes: the 16 lanes of a group name eight rows of 16
// bytes, lane i half i % 2 of row i / 2; lane i gets byte i of each row.
__device__ __forceinline__ uint2v read_columns(const unsigned char* p) {
    return __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                          (__attribute__((address_space(3))) int2v*)(p)));
}

// Over the four lanes that hold one row (j, j + 16, j + 32, j + 48).
__device__ __forceinline__ float cols_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float cols_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// x = hi + lo to 22 bits.
__device__ __forceinline__ void halves(const float* x, half8_t& hi, half8_t& lo) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float2v v = {x[e], x[e + 1]};
        const half2_t h = __builtin_convertvector(v, half2_t);
        const half2_t l = __builtin_convertvector(v - __builtin_convertvector(h, float2v), half2_t);
        hi[e] = h[0];
        hi[e + 1] = h[1];
        lo[e] = l[0];
        lo[e + 1] = l[1];
    }
}

// A step's bits, ordered as its size is; 0 for one that is not finite.
__device__ __forceinline__ int step_bits(_Float16 d) {
    const int b = __builtin_bit_cast(uint16_t, d) & 0x7fff;
    return b < 0x7c00 ? b : 0;
}

// Bits of the drafts that a token sees (bit d: draft d of its sequence) as
// bits of the keys k0 .. k0 + 31: committed keys (below p0) are seen.
__device__ __forceinline__ uint32_t seen_keys(uint32_t drafts, int k0, int p0) {
    const int d = k0 - p0;
    if (d <= -32) return 0xffffffffu;
    if (d < 0) return drafts << -d | ((1u << -d) - 1);
    return d < 32 ? drafts >> d : 0;
}

// NT tiles of 16 query rows of a wave: lane (g, j) = (lane / 16, lane % 16)
// holds row j of each tile.
template <int HD, int NT>
struct Q8Rows {
    static constexpr int NB = HD / 32, ND = HD / 16;
    half8_t qh[NT][NB], ql[NT][NB];    // Q^T as the B operand: elements 32t + 8g .. +7 of row j
    floatx4 o[NT][ND];                 // O^T: columns 16n + 4g .. +3 of row j
    float unq[NT];                     // what undoes Q's scale
    float m[NT], l[NT];                // running maximum (log2), the lane's part of the sum
    float pexp[NT];                    // the weights are 2^(score - m + pexp)
    int lim[NT];                       // bits of the largest V step seen

    // Tile i's rows from q (row j at qp, or nothing there), scaled by `scale`
    // and then to [2^13, 2^14) at the row's largest element: lo keeps its 11
    // bits for any element within 2^-14 of that one.
    __device__ __forceinline__ void start(int i, const float* qp, bool live, float scale) {
        const int g = (threadIdx.x & 63) >> 4;
        float4u raw[NB][2];
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            raw[t][0] = *(const float4u*)(qp + 32 * t + 8 * g);
            raw[t][1] = *(const float4u*)(qp + 32 * t + 8 * g + 4);
        }
        start(i, raw, live, scale);
    }
    __device__ __forceinline__ void start(int i, const float4u (*raw)[2], bool live, float scale) {
        float v[NB][8], top = 0.f;
#pragma unroll
        for (int t = 0; t < NB; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[t][e] = live ? raw[t][e >> 2][e & 3] * scale : 0.f;
                top = fmaxf(top, fabsf(v[t][e]));
            }
        top = cols_max(top);
        const int e2 = top > 0.f ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        unq[i] = ldexpf(1.0f, -e2);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[t][e] = ldexpf(v[t][e], e2);
            halves(v[t], qh[i][t], ql[i][t]);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) o[i][n] = floatx4{0.f, 0.f, 0.f, 0.f};
        m[i] = -INFINITY;
        l[i] = 0.f;
        pexp[i] = 0.f;
        lim[i] = 0;
    }

    // 32 keys: k, v their codes in LDS (rows of HD bytes, permuted), ks, vs
    // their steps.  MASKED: tile i's row sees the keys of its bits seen[i];
    // otherwise every row sees them all.
    template <bool MASKED>
    __device__ __forceinline__ void keys32(const unsigned char* k, const unsigned char* v, const Q8Steps<HD>* ks,
                                           const Q8Steps<HD>* vs, const uint32_t* seen) {
        const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
        // scores: lane (g, j) has keys 16 hf + 4g + i of row j
        floatx4 s[NT][2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            Q8Steps<HD> d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = ks[16 * hf + 4 * g + i];
#pragma unroll
            for (int i = 0; i < NT; ++i) s[i][hf] = floatx4{0.f, 0.f, 0.f, 0.f};
            const int key = 16 * hf + j;
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                const int c = 2 * t + (g >> 1);
                const half8_t kc =
                    codes_f16(*(const uint2v*)(k + key * HD + 16 * (c ^ swz<HD>(key)) + 8 * (g & 1)));
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    floatx4 r = {0.f, 0.f, 0.f, 0.f};
                    r = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[i][t], r, 0, 0, 0);
                    r = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[i][t], r, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][hf][e] = fmaf((float)d[e].s[t], r[e], s[i][hf][e]);
                }
            }
        }
        Q8Steps<HD> dv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] = vs[16 * (e >> 2) + 4 * g + (e & 3)];
        int top_step = 0;
        if (!MASKED) {                                 // a lane looks at one key's V steps
            const Q8Steps<HD> one = vs[lane & 31];
#pragma unroll
            for (int t = 0; t < NB; ++t) top_step = max(top_step, step_bits(one.s[t]));
        }
        float p[NT][8];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint32_t bits = MASKED ? seen[i] >> (4 * g) : 0;
            int big = top_step;
            if (MASKED) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(bits >> (16 * (e >> 2) + (e & 3)) & 1)) {
                        s[i][e >> 2][e & 3] = -INFINITY;
                    } else {
#pragma unroll
                        for (int t = 0; t < NB; ++t) big = max(big, step_bits(dv[e].s[t]));
                    }
            }
            float mx = s[i][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[i][e >> 2][e & 3]);
            mx *= unq[i];
            if (__builtin_amdgcn_ballot_w64(mx > m[i] + A8_SLACK || big > lim[i])) {
                const float mn = fmaxf(m[i], cols_max(mx));
                float f = m[i] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[i] - mn);
                m[i] = mn;
                if (__builtin_amdgcn_ballot_w64(big > lim[i])) {
                    if (!MASKED)
#pragma unroll
                        for (int off = 1; off < 16; off <<= 1) big = max(big, __shfl_xor(big, off));
                    big = max(big, __shfl_xor(big, 16));
                    big = max(big, __shfl_xor(big, 32));
                    if (big > lim[i]) {
                        lim[i] = big;
                        const float top = (float)__builtin_bit_cast(_Float16, (uint16_t)big);
                        const float pe = (float)(A8_PEXP - __builtin_amdgcn_frexp_expf(top));
                        f *= __builtin_amdgcn_exp2f(pe - pexp[i]);
                        pexp[i] = pe;
                    }
                }
                l[i] *= f;
#pragma unroll
                for (int n = 0; n < ND; ++n) o[i][n] *= f;
            }
            const float mref = pexp[i] - (m[i] == -INFINITY ? 0.f : m[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e >> 2][e & 3], unq[i], mref));
                l[i] += p[i][e];
            }
        }
        // the transposing read: lane j of a group names half (j & 1) of the 16
        // columns of the key of slot 8g + j / 2 (slot 8g + e is the lane's e-th key)
        const int tkey = 16 * (j >> 3) + 4 * g + ((j >> 1) & 3);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            half8_t ph[NT], pl[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint32_t bits = MASKED ? seen[i] >> (4 * g) : 0;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float d = (float)dv[e].s[t];
                    // a step that the row does not see may be anything
                    if (MASKED) d = bits >> (16 * (e >> 2) + (e & 3)) & 1 ? d : 0.f;
                    x[e] = p[i][e] * d;
                }
                halves(x, ph[i], pl[i]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int n = 2 * t + u;
                const half8_t vc = codes_f16(read_columns(v + tkey * HD + 16 * (n ^ swz<HD>(tkey)) + 8 * (j & 1)));
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    o[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pl[i], o[i][n], 0, 0, 0);
                    o[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, ph[i], o[i][n], 0, 0, 0);
                }
            }
        }
    }

    // Tile i's sum over its keys, and what undoes the weights' scale.
    __device__ __forceinline__ float back(int i) const { return __builtin_amdgcn_exp2f(-pexp[i]); }
    __device__ __forceinline__ float sum(int i) const { return cols_sum(l[i]) * back(i); }
};

}  // namespace slate_hip
