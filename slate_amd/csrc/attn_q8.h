// attn_q8.h -- 32 keys of the 8-bit cache against a wave's 16 query rows, the
// codes in LDS as they are stored.
//
// A code is exact in f16.  S: one MFMA K step (two, for Q's halves) per block
// of 32 elements, the block's f32 result weighted by the key's step for it.
// O: P is weighted by the steps of V, block by block of 32 output columns.
#pragma once
#include "attn_rows.h"

namespace slate_hip {

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

// A step's bits, ordered as its size is; 0 for one that is not finite.
__device__ __forceinline__ int step_bits(_Float16 d) {
    const int b = __builtin_bit_cast(uint16_t, d) & 0x7fff;
    return b < 0x7c00 ? b : 0;
}

__device__ __forceinline__ int step_exponent(int bits) {
    return __builtin_amdgcn_frexp_expf((float)__builtin_bit_cast(_Float16, (uint16_t)bits));
}

template <int HD>
struct Q8Rows : AttnRows<HD> {
    using AttnRows<HD>::qh;
    using AttnRows<HD>::ql;
    using AttnRows<HD>::o;
    static constexpr int NB = HD / 32;

    // 32 keys: k, v their codes in LDS (rows of HD bytes, permuted), ks, vs
    // their steps.  MASKED: the row sees the keys of its bits `seen`;
    // otherwise every row sees them all.
    template <bool MASKED>
    __device__ __forceinline__ void keys32(const unsigned char* k, const unsigned char* v, const Q8Steps<HD>* ks,
                                           const Q8Steps<HD>* vs, uint32_t seen) {
        const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
        // scores: lane (g, j) has keys 16 hf + 4g + i of row j
        floatx4 s[2];
        const floatx4 zero = zeros();
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            Q8Steps<HD> d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = ks[16 * hf + 4 * g + i];
            s[hf] = floatx4{0.f, 0.f, 0.f, 0.f};
            const int key = 16 * hf + j;
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                const int c = 2 * t + (g >> 1);
                const half8_t kc =
                    codes_f16(*(const uint2v*)(k + key * HD + 16 * (c ^ swz<HD>(key)) + 8 * (g & 1)));
                floatx4 r = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[t], zero, 0, 0, 0);
                r = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[t], r, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[hf][e] = fmaf((float)d[e].s[t], r[e], s[hf][e]);
            }
        }
        Q8Steps<HD> dv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) dv[e] = vs[16 * (e >> 2) + 4 * g + (e & 3)];
        // bit 16 (e / 4) + e % 4 of `bits`: the row sees the lane's key e
        const uint32_t bits = MASKED ? seen >> (4 * g) : 0;
        int big = 0;
        if (MASKED) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (!(bits >> (16 * (e >> 2) + (e & 3)) & 1)) {
                    s[e >> 2][e & 3] = -INFINITY;
                } else {
#pragma unroll
                    for (int t = 0; t < NB; ++t) big = max(big, step_bits(dv[e].s[t]));
                }
        } else {                                       // a lane looks at one key's V steps
            const Q8Steps<HD> one = vs[lane & 31];
#pragma unroll
            for (int t = 0; t < NB; ++t) big = max(big, step_bits(one.s[t]));
        }
        float p[8];
        this->template weights<2, MASKED>(s, big, step_exponent, p);
        const float by = __builtin_amdgcn_exp2f(this->pexp);
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] *= by;
        // the transposing read: lane j of a group names half (j & 1) of the 16
        // columns of the key of slot 8g + j / 2 (slot 8g + e is the lane's e-th key)
        const int tkey = 16 * (j >> 3) + 4 * g + ((j >> 1) & 3);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = times(p[e], dv[e].s[t]);
                // a step that the row does not see may be anything
                if (MASKED) x[e] = bits >> (16 * (e >> 2) + (e & 3)) & 1 ? x[e] : 0.f;
            }
            half8_t ph, pl;
            halves(x, ph, pl);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int n = 2 * t + u;
                const half8_t vc = codes_f16(read_columns(v + tkey * HD + 16 * (n ^ swz<HD>(tkey)) + 8 * (j & 1)));
                o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pl, o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, ph, o[n], 0, 0, 0);
            }
        }
    }
};

}  // namespace slate_hip
