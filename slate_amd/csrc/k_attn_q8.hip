// k_attn_q8.hip -- attention of few query rows per sequence (a decode step,
// small trees) over the 8-bit cache.
//
// The rows of a (sequence, kv head) -- its tokens times the query heads that
// share the kv head, at most 16 -- are the columns of 16 x 16 x 32 f16 MFMAs:
//   S^T [32 keys x 16 rows] = K Q^T, one MFMA K step per 32-element block, the
//       block's f32 result weighted by the key's step for it;
//   O^T [hd x 16 rows] += V^T P^T, with P weighted by the steps of V, block by
//       block of 32 output columns.
// The codes are exact in f16; Q and P are split into two halves, hi = f16(x)
// and lo = f16(x - hi), 22 bits in all, so a product costs two MFMAs and
// nothing is rounded to fewer bits than that.  Softmax, sums and steps are
// f32; the running maximum moves only when a score passes it by 2^4 (weights
// up to 16 stay well inside f16's range).
//
// Memory bound: 2.125 bytes per key and element against two f16 MFMAs and about
// 400 VALU operations per 32 keys and wave.  So the whole design is about
// loads: each wave copies its next 32 keys' K and V rows straight into LDS
// (16 bytes per lane, no registers) while it works on the last 32, by itself,
// with no barrier until its range ends; four waves of a workgroup take a granule of 128
// keys.  Rows of 16-byte chunks are stored in LDS permuted, chunk c of key k
// at place c ^ swz(k), so that both kinds of reads spread over the banks: K
// by key (8 bytes a lane), V by the transposing byte read, which hands a lane
// one column of eight keys.
#include "attn_plan.h"
#include "lanes.h"
#include "mfma.h"

namespace slate_hip {

constexpr int AQ_ROWS = 16;            // query rows of a block
constexpr int AQ_KEYS = 32;            // keys of a wave's step
constexpr int AQ_GRAN = 4 * AQ_KEYS;   // keys of a workgroup's step
constexpr int AQ_WGS = 512;            // two workgroups per CU (LDS)
constexpr float AQ_SLACK = 4.0f;       // log2 of the largest weight before the maximum moves
constexpr int AQ_PEXP = 11;            // weights are scaled so that weight 1 times the largest V step is in [2^10, 2^11]

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef int int2v __attribute__((ext_vector_type(2)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float float8v __attribute__((ext_vector_type(8)));

template <int HD>
struct Q8Geom {
    static constexpr int NB = HD / 32;                 // steps (blocks) of a row
    static constexpr int ND = HD / 16;                 // 16-column tiles of V
    static constexpr int ROWB = HD;                    // bytes of a row of codes
    static constexpr int TILE = AQ_KEYS * HD;          // bytes of a wave's K (or V) codes
    static constexpr int STEPS = AQ_KEYS * NB * 2;     // bytes of their steps
    static constexpr int BUF = 2 * TILE + 2 * STEPS;
    static constexpr int CH = HD / 16;                 // 16-byte chunks of a row
    static constexpr int SH = HD == 128 ? 1 : HD == 64 ? 2 : 3;
};

// Where chunk c of key k sits in its LDS row: 256 / HD rows share a round of
// the banks, the ones after them are shifted; keys 16 apart, which the
// transposing read takes together, too.
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

__device__ __forceinline__ float cols_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float cols_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// A step's bits, ordered as its size is; 0 for one that is not finite.
__device__ __forceinline__ int step_bits(_Float16 d) {
    const int b = __builtin_bit_cast(uint16_t, d) & 0x7fff;
    return b < 0x7c00 ? b : 0;
}

// Granules of a sequence whose rows fit a block.
struct FewCount {
    int G, Hkv;
    __device__ __forceinline__ int64_t operator()(const SeqView& s) const {
        if (s.n < 1 || (int64_t)s.n * G > AQ_ROWS) return 0;
        return (int64_t)Hkv * ((s.p0 + s.n + AQ_GRAN - 1) / AQ_GRAN);
    }
};

// Partial slot: AQ_ROWS rows of HD outputs, then AQ_ROWS pairs (m, l).
__host__ __device__ constexpr int64_t few_slot_floats(int hd) { return (int64_t)AQ_ROWS * (hd + 2); }

template <int HD>
__global__ __launch_bounds__(256, 2) void attn_q8_few_kernel(PackedAttn a, PackedBatch pb) {
    using Geo = Q8Geom<HD>;
    constexpr int NB = Geo::NB, ND = Geo::ND;
    constexpr int OS = HD + 4;                         // row stride of the waves' results in LDS
    __shared__ __attribute__((aligned(16))) unsigned char smem[8 * Geo::BUF];
    __shared__ float s_m[4][AQ_ROWS], s_l[4][AQ_ROWS];
    static_assert(8 * Geo::BUF >= 4 * AQ_ROWS * OS * (int)sizeof(float), "results fit");
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, j = lane & 15;
    const int G = a.Hq / a.Hkv;
    const Plan<FewCount> plan(pb, FewCount{G, a.Hkv});
    const int64_t x0 = plan.begin(blockIdx.x, AQ_WGS), x1 = plan.begin(blockIdx.x + 1, AQ_WGS);
    const float scale2 = (1.0f / sqrtf((float)HD)) * LOG2E;
    unsigned char* buf0 = smem + w * 2 * Geo::BUF;

    for (int64_t x = x0; x < x1;) {
        const Place pl = plan.find(x);
        const SeqView sv = seq_view(pb, pl.b);
        const int keys = sv.p0 + sv.n;
        const int gran = (keys + AQ_GRAN - 1) / AQ_GRAN;
        const int h = (int)(pl.at / gran), g0 = (int)(pl.at % gran);
        const int g1 = (int)min((int64_t)gran, g0 + (x1 - x));
        const int64_t row0 = (pb.kv_base[pl.b] + h * a.head_stride) / HD;
        const int8_t *kq = a.kv8.kq + row0 * HD, *vq = a.kv8.vq + row0 * HD;
        const _Float16 *ks = a.kv8.ks + row0 * NB, *vs = a.kv8.vs + row0 * NB;

        // K and V rows of the wave's 32 keys from k0 on, into buffer `to`;
        // rows past the last key repeat it (their weights are zero)
        struct alignas(2 * NB) Steps { _Float16 s[NB]; };
        Steps st;
        auto issue = [&](int k0, int to) {
            const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(buf0 + to * Geo::BUF));
            const int8_t *kb = uniform(kq + (int64_t)k0 * HD), *vb = uniform(vq + (int64_t)k0 * HD);
#pragma unroll
            for (int i = 0; i < Geo::TILE / 1024; ++i) {
                const int at = 64 * i + lane, key = at / Geo::CH, c = at % Geo::CH;
                const uint32_t off = (uint32_t)min(key, keys - 1 - k0) * HD + 16 * (c ^ swz<HD>(key));
                lds_copy16(kb, off, dst + 1024 * i);
                lds_copy16(vb, off, dst + Geo::TILE + 1024 * i);
            }
            // lanes 0..31 carry the steps of a K row each, 32..63 of a V row
            const int64_t r = min(k0 + (lane & 31), keys - 1);
            st = *(const Steps*)((lane < 32 ? ks : vs) + r * NB);
        };
        auto key0 = [&](int gr) { return gr * AQ_GRAN + w * AQ_KEYS; };
        int to = 0;
        if (key0(g0) < keys) issue(key0(g0), 0);

        // Q^T as the B operand: lane (g, j) holds row j, elements 32t + 8g .. +7,
        // scaled to [2^13, 2^14) at its largest so that lo keeps 11 bits of
        // any element within 2^-14 of it
        const int rows = sv.n * G;
        const int tok = j / G, hq = h * G + j % G;
        const bool live = j < rows;
        float qv[NB][8];
        float top = 0.f;
        const float* qp = a.q + ((int64_t)(sv.t0 + (live ? tok : 0)) * a.Hq + (live ? hq : 0)) * HD + 8 * g;
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            const float4u u0 = *(const float4u*)(qp + 32 * t), u1 = *(const float4u*)(qp + 32 * t + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                qv[t][e] = live ? u0[e] * scale2 : 0.f;
                qv[t][4 + e] = live ? u1[e] * scale2 : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(qv[t][e]));
        }
        top = cols_max(top);
        const int qe = top > 0.f ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        const float unq = ldexpf(1.0f, -qe);
        half8_t qh[NB], ql[NB];
#pragma unroll
        for (int t = 0; t < NB; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = ldexpf(qv[t][e], qe);
                const _Float16 hi = (_Float16)v;
                qh[t][e] = hi;
                ql[t][e] = (_Float16)(v - (float)hi);
            }
        // the drafts that row j's token sees (n <= 16): itself and, causal,
        // all before it, or its ancestors
        uint32_t seen = (2u << tok) - 1;
        if (a.parent) {
            const int par = a.parent[sv.t0 + min(lane, sv.n - 1)];
            seen = 0;
            int cur = live ? tok : -1;
            while (__builtin_amdgcn_ballot_w64(cur >= 0)) {
                const int up = __shfl(par, max(cur, 0));
                if (cur >= 0) seen |= 1u << cur;
                cur = up >= 0 && up < cur ? up : -1;
            }
        }
        if (!live) seen = 0;

        floatx4 o[ND];
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] = floatx4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        int lim = 0;                                   // f16 bits of the largest V step seen so far
        float pexp = 0.f;                              // the row's weights are 2^(score - m + pexp)

        for (int gr = g0; gr < g1; ++gr) {
            const int k0 = key0(gr);
            if (k0 >= keys) break;                     // only in the last granule
            unsigned char* buf = buf0 + to * Geo::BUF;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            const Steps mine = st;
            *(Steps*)(buf + 2 * Geo::TILE + lane * (int)sizeof(Steps)) = mine;
            const int kn = key0(gr + 1);
            if (gr + 1 < g1 && kn < keys) issue(kn, to ^ 1);
            to ^= 1;

            // scores of 32 keys: lane (g, j) has keys 16 hf + 4g + i of row j
            const _Float16* sk = (const _Float16*)(buf + 2 * Geo::TILE);
            floatx4 s[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                s[hf] = floatx4{0.f, 0.f, 0.f, 0.f};
                alignas(2 * NB) _Float16 d[4][NB];
#pragma unroll
                for (int i = 0; i < 4; ++i) *(Steps*)d[i] = *(const Steps*)(sk + (16 * hf + 4 * g + i) * NB);
                const int key = 16 * hf + j;
#pragma unroll
                for (int t = 0; t < NB; ++t) {
                    const int c = 2 * t + (g >> 1);
                    const uint2v raw = *(const uint2v*)(buf + key * HD + 16 * (c ^ swz<HD>(key)) + 8 * (g & 1));
                    const half8_t k = codes_f16(raw);
                    floatx4 r = {0.f, 0.f, 0.f, 0.f};
                    r = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[t], r, 0, 0, 0);
                    r = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[t], r, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[hf][i] = fmaf((float)d[i][t], r[i], s[hf][i]);
                }
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = s[e >> 2][e & 3] * unq;
            const _Float16* svs = sk + AQ_KEYS * NB;
            alignas(2 * NB) _Float16 dv[8][NB];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                *(Steps*)dv[e] = *(const Steps*)(svs + (16 * (e >> 2) + 4 * g + (e & 3)) * NB);
            // the largest V step that the row sees: the weights' scale goes by it
            int big = 0;
            if (k0 + AQ_KEYS > sv.p0) {                // drafts among the keys, or past the last one
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = k0 + 16 * (e >> 2) + 4 * g + (e & 3) - sv.p0;
                    const bool sees = d < 0 || (d < 32 && (seen >> d & 1));
                    v[e] = sees ? v[e] : -INFINITY;
#pragma unroll
                    for (int t = 0; t < NB; ++t) big = max(big, sees ? step_bits(dv[e][t]) : 0);
                }
            } else {                                   // all rows see all keys: a lane looks at one key's
#pragma unroll
                for (int t = 0; t < NB; ++t) big = max(big, lane >= 32 ? step_bits(mine.s[t]) : 0);
            }
            float mx = v[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, v[e]);
            if (__builtin_amdgcn_ballot_w64(mx > m + AQ_SLACK || big > lim)) {
                const float mn = fmaxf(m, cols_max(mx));
                float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                if (__builtin_amdgcn_ballot_w64(big > lim)) {
                    big = max(big, __shfl_xor(big, 16));
                    big = max(big, __shfl_xor(big, 32));
                    if (k0 + AQ_KEYS <= sv.p0)
#pragma unroll
                        for (int off = 1; off < 16; off <<= 1) big = max(big, __shfl_xor(big, off));
                    if (big > lim) {
                        lim = big;
                        const float top = (float)__builtin_bit_cast(_Float16, (uint16_t)lim);
                        const float pe = (float)(AQ_PEXP - __builtin_amdgcn_frexp_expf(top));
                        f *= __builtin_amdgcn_exp2f(pe - pexp);
                        pexp = pe;
                    }
                }
                l *= f;
#pragma unroll
                for (int n = 0; n < ND; ++n) o[n] *= f;
            }
            const float mref = (m == -INFINITY ? 0.f : m) - pexp;
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(v[e] - mref);
                l += p[e];
            }
            // O^T += V^T P^T; MFMA slots 8g + e are the lane's keys
            const unsigned char* sv8 = buf + Geo::TILE;
            // the transposing read: lane j of a group names half (j & 1) of
            // the 16 columns of the key of slot 8g + j / 2
            const int tkey = 16 * (j >> 3) + 4 * g + ((j >> 1) & 3);
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                half8_t ph, pl8;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = p[e] == 0.f ? 0.f : p[e] * (float)dv[e][t];
                    const _Float16 hi = (_Float16)x;
                    ph[e] = hi;
                    pl8[e] = (_Float16)(x - (float)hi);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int n = 2 * t + u;
                    const half8_t vv =
                        codes_f16(read_columns(sv8 + tkey * HD + 16 * (n ^ swz<HD>(tkey)) + 8 * (j & 1)));
                    o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pl8, o[n], 0, 0, 0);
                    o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, ph, o[n], 0, 0, 0);
                }
            }
        }

        // the four waves' results joined through LDS
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();                               // nobody still reads its rows
        l = cols_sum(l);
        const float back = __builtin_amdgcn_exp2f(-pexp);
        float* so = (float*)smem;
        if (g == 0) {
            s_m[w][j] = m;
            s_l[w][j] = l * back;
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) *(floatx4*)(so + (w * AQ_ROWS + j) * OS + 16 * n + 4 * g) = o[n] * back;
        __syncthreads();
        const bool whole = g0 == 0 && g1 == gran;
        float* slot = (float*)a.ws + (2 * (int64_t)blockIdx.x + (x == x0 ? 0 : 1)) * few_slot_floats(HD);
        for (int u = threadIdx.x; u < rows * (HD / 4); u += 256) {
            const int r = u / (HD / 4), c = 4 * (u % (HD / 4));
            const float mt = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            floatx4 sum = {0.f, 0.f, 0.f, 0.f};
            float lt = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = s_m[k][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[k][r] - mt);
                lt += f * s_l[k][r];
                const floatx4 ok = *(const floatx4*)(so + (k * AQ_ROWS + r) * OS + c);
                sum += f == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : f * ok;
            }
            if (whole) {
                const int64_t at = ((int64_t)(sv.t0 + r / G) * a.Hq + h * G + r % G) * HD + c;
                const float inv = 1.0f / lt;
#pragma unroll
                for (int e = 0; e < 4; ++e) a.out[at + e] = sum[e] * inv;
            } else {
                *(floatx4*)(slot + r * HD + c) = sum;
                if (c == 0) *(float2*)(slot + AQ_ROWS * HD + 2 * r) = make_float2(mt, lt);
            }
        }
        __syncthreads();                               // before the next piece's copies land
        x += g1 - g0;
    }
}

// Joins the partials of a block that lies in several workgroups' ranges.
// Workgroup m - 1 looks at the boundary N m / P: where it is the first one
// inside a block, the block's pieces are joined here, a wave per row.
template <int HD>
__global__ __launch_bounds__(256) void attn_q8_few_join_kernel(PackedAttn a, PackedBatch pb) {
    constexpr int P = AQ_WGS;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int G = a.Hq / a.Hkv;
    const Plan<FewCount> plan(pb, FewCount{G, a.Hkv});
    const int64_t x = plan.begin(blockIdx.x + 1, P), before = plan.begin(blockIdx.x, P);
    if (x >= plan.total) return;
    const Place pl = plan.find(x);
    const SeqView sv = seq_view(pb, pl.b);
    const int gran = (sv.p0 + sv.n + AQ_GRAN - 1) / AQ_GRAN;
    const int h = (int)(pl.at / gran), in = (int)(pl.at % gran);
    const int64_t start = x - in, end = start + gran;
    if (in == 0 || before > start) return;             // no block is cut here, or an earlier boundary cuts it
    const int first = blockIdx.x;                      // the pieces: this workgroup's last, then whole first slots
    int pieces = 1;
    while (first + pieces < P && plan.begin(first + pieces, P) < end) ++pieces;
    const float* ws = (const float*)a.ws;
    auto slot = [&](int k) {
        return ws + (2 * (int64_t)(first + k) + (k == 0 && before != start ? 1 : 0)) * few_slot_floats(HD);
    };
    auto some = [&](int k) { return plan.begin(first + k + 1, P) > plan.begin(first + k, P); };
    for (int r = w; r < sv.n * G; r += 4) {
        float mt = -INFINITY;
        for (int k = lane; k < pieces; k += 64)
            if (some(k)) mt = fmaxf(mt, slot(k)[AQ_ROWS * HD + 2 * r]);
        mt = wave_max(mt);
        float lt = 0.f, acc[2] = {0.f, 0.f};
        for (int k0 = 0; k0 < pieces; k0 += 64) {
            float f = 0.f;
            if (k0 + lane < pieces && some(k0 + lane)) {
                const float2 ml = *(const float2*)(slot(k0 + lane) + AQ_ROWS * HD + 2 * r);
                f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mt);
                lt += f * ml.y;
            }
            const int n = min(64, pieces - k0);
            for (int k = 0; k < n; ++k) {
                const float fk = lane_read(f, k);
                if (fk == 0.f) continue;
                const float* op = slot(k0 + k) + r * HD;
#pragma unroll
                for (int e = 0; e < (HD + 63) / 64; ++e)
                    if (64 * e + lane < HD) acc[e] += fk * op[64 * e + lane];
            }
        }
        lt = wave_sum(lt);
        const int64_t at = ((int64_t)(sv.t0 + r / G) * a.Hq + h * G + r % G) * HD;
#pragma unroll
        for (int e = 0; e < (HD + 63) / 64; ++e)
            if (64 * e + lane < HD) a.out[at + 64 * e + lane] = acc[e] / lt;
    }
}

bool attention_q8_few_shape(int hd, int G) { return (hd == 32 || hd == 64 || hd == 128) && G <= AQ_ROWS; }
int64_t attention_q8_few_bytes(int hd) { return 2 * AQ_WGS * few_slot_floats(hd) * (int64_t)sizeof(float); }

template <int HD>
static void launch_few(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    hipLaunchKernelGGL(attn_q8_few_kernel<HD>, dim3(AQ_WGS), dim3(256), 0, s, a, pb);
    if (pb.max_seq > AQ_GRAN)          // a block of one granule is never cut
        hipLaunchKernelGGL(attn_q8_few_join_kernel<HD>, dim3(AQ_WGS - 1), dim3(256), 0, s, a, pb);
}

int launch_attention_q8_few(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    if (a.hd == 128)
        launch_few<128>(a, pb, s);
    else if (a.hd == 64)
        launch_few<64>(a, pb, s);
    else
        launch_few<32>(a, pb, s);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
