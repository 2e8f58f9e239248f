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
constexpr int AQ_KEEP = 4;             // blocks of up to this many granules are not cut
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
    static constexpr int OS = HD + 4;                  // row stride of a wave's results in LDS (floats)
    static constexpr int USED = 2 * TILE + 2 * STEPS;
    static constexpr int BUF = USED > AQ_ROWS * OS * 4 ? USED : AQ_ROWS * OS * 4;
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

__host__ __device__ inline int few_granules(int keys) { return (keys + AQ_GRAN - 1) / AQ_GRAN; }

// Granules of a sequence whose rows fit a block (one block per kv head).
struct FewCount {
    int G, Hkv;
    __device__ __forceinline__ int operator()(const SeqView& s) const {
        return s.n < 1 || (int64_t)s.n * G > AQ_ROWS ? 0 : Hkv * few_granules(s.p0 + s.n);
    }
};
using FewPlan = Plan<FewCount>;

// Where workgroup w's range begins: N w / P, or the start of the block there
// if it is short (it is not cut: the last workgroup that would begin in it
// takes it whole).
__device__ __forceinline__ int few_begin(const FewPlan& plan, int w) {
    const int x = plan.begin(w, AQ_WGS);
    if (x >= plan.total) return plan.total;
    const Place pl = plan.find(x);
    const int gran = few_granules(pl.seq.p0 + pl.seq.n), in = pl.at % gran;
    return gran <= AQ_KEEP ? x - in : x;
}

// Workspace: a JoinEntry per workgroup, then two slots each of AQ_ROWS rows
// of HD outputs and AQ_ROWS pairs (m, l).
__host__ __device__ constexpr int64_t few_slot_floats(int hd) { return (int64_t)AQ_ROWS * (hd + 2); }
constexpr int64_t FEW_ENTRIES = (int64_t)AQ_WGS * 32;  // bytes
__device__ __forceinline__ float* few_slot(void* ws, int i, int hd) {
    return (float*)((char*)ws + FEW_ENTRIES) + i * few_slot_floats(hd);
}

template <int HD>
__global__ __launch_bounds__(256, 2) void attn_q8_few_kernel(PackedAttn a, PackedBatch pb) {
    using Geo = Q8Geom<HD>;
    constexpr int NB = Geo::NB, ND = Geo::ND, OS = Geo::OS;
    struct alignas(2 * NB) Steps { _Float16 s[NB]; };
    __shared__ __attribute__((aligned(16))) unsigned char smem[8 * Geo::BUF];
    __shared__ float s_m[4][AQ_ROWS], s_l[4][AQ_ROWS];
    __shared__ int s_at[4];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, j = lane & 15;
    const int G = a.Hq / a.Hkv;
    const FewPlan plan(pb, FewCount{G, a.Hkv});
    const int x0 = few_begin(plan, blockIdx.x), x1 = few_begin(plan, blockIdx.x + 1);
    JoinEntry* entry = (JoinEntry*)((char*)a.ws + 32 * blockIdx.x);
    if (x0 >= x1) {
        if (threadIdx.x == 0) entry->rows = 0;
        return;
    }
    const float scale2 = (1.0f / sqrtf((float)HD)) * LOG2E;
    unsigned char* buf0 = smem + w * 2 * Geo::BUF;

    // the piece being worked on, and the loads that are under way for one
    struct Piece {
        SeqView seq;
        int h, gran, g0, g1;
        const int8_t *kq, *vq;
        const _Float16 *ks, *vs;
    };
    auto piece_at = [&](int x) {
        const Place pl = plan.find(x);
        Piece p;
        p.seq = pl.seq;
        p.gran = few_granules(pl.seq.p0 + pl.seq.n);
        p.h = pl.at / p.gran;
        p.g0 = pl.at % p.gran;
        p.g1 = min(p.gran, p.g0 + (x1 - x));
        const int64_t row0 = pl.base / HD + p.h * (a.head_stride / HD);
        p.kq = a.kv8.kq + row0 * HD;
        p.vq = a.kv8.vq + row0 * HD;
        p.ks = a.kv8.ks + row0 * NB;
        p.vs = a.kv8.vs + row0 * NB;
        return p;
    };
    Steps st;
    // K and V rows of the wave's 32 keys of granule gr, into buffer `to`;
    // rows past the last key repeat it (their weights are zero)
    auto key0 = [&](int gr) { return gr * AQ_GRAN + w * AQ_KEYS; };
    auto issue = [&](const Piece& p, int gr, int to) {
        const int k0 = key0(gr), last = p.seq.p0 + p.seq.n - 1;
        if (k0 > last) return;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(buf0 + to * Geo::BUF));
        const int8_t *kb = uniform(p.kq + (int64_t)k0 * HD), *vb = uniform(p.vq + (int64_t)k0 * HD);
#pragma unroll
        for (int i = 0; i < Geo::TILE / 1024; ++i) {
            const int at = 64 * i + lane, key = at / Geo::CH, c = at % Geo::CH;
            const uint32_t off = (uint32_t)min(key, last - k0) * HD + 16 * (c ^ swz<HD>(key));
            lds_copy16(kb, off, dst + 1024 * i);
            lds_copy16(vb, off, dst + Geo::TILE + 1024 * i);
        }
        // lanes 0..31 carry the steps of a K row each, 32..63 of a V row
        const int64_t r = min(k0 + (lane & 31), last);
        st = *(const Steps*)((lane < 32 ? p.ks : p.vs) + r * NB);
    };
    // q of row j, elements 32t + 8g .. +7
    float4u qraw[NB][2];
    auto load_q = [&](const Piece& p) {
        const bool live = j < p.seq.n * G;
        const float* qp =
            a.q + ((int64_t)(p.seq.t0 + (live ? j / G : 0)) * a.Hq + p.h * G + (live ? j % G : 0)) * HD + 8 * g;
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            qraw[t][0] = *(const float4u*)(qp + 32 * t);
            qraw[t][1] = *(const float4u*)(qp + 32 * t + 4);
        }
    };

    Piece pc = piece_at(x0);
    int to = 0;
    issue(pc, pc.g0, 0);
    load_q(pc);
    if (w == 0) {                                      // is the boundary x0 a block's first cut?
        // (all lanes work it out: the plan's searches are the wave's)
        const int start = x0 - pc.g0, end = start + pc.gran, before = (int)blockIdx.x - 1;
        const int from = pc.g0 > 0 ? few_begin(plan, before) : 0;
        int pieces = 0;
        if (pc.g0 > 0 && from <= start) {
            pieces = 2;
            while (before + pieces < AQ_WGS && plan.begin(before + pieces, AQ_WGS) < end) ++pieces;
        }
        if (lane == 0)
            *entry = JoinEntry{pc.seq.t0, pieces ? pc.seq.n * G : 0, 0, pc.h, pieces, 2 * before + (from != start)};
    }

    for (int x = x0;;) {
        const SeqView sv = pc.seq;
        const int keys = sv.p0 + sv.n, h = pc.h;
        // Q^T as the B operand: lane (g, j) holds row j, elements 32t + 8g .. +7,
        // scaled to [2^13, 2^14) at its largest so that lo keeps 11 bits of
        // any element within 2^-14 of it
        const int rows = sv.n * G;
        const int tok = j / G;
        const bool live = j < rows;
        float qv[NB][8];
        float top = 0.f;
#pragma unroll
        for (int t = 0; t < NB; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                qv[t][e] = live ? qraw[t][e >> 2][e & 3] * scale2 : 0.f;
                top = fmaxf(top, fabsf(qv[t][e]));
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

        for (int gr = pc.g0; gr < pc.g1; ++gr) {
            const int k0 = key0(gr);
            if (k0 >= keys) break;                     // only in the last granule
            unsigned char* buf = buf0 + to * Geo::BUF;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            const Steps mine = st;
            *(Steps*)(buf + 2 * Geo::TILE + lane * (int)sizeof(Steps)) = mine;
            to ^= 1;
            if (gr + 1 < pc.g1) issue(pc, gr + 1, to);

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

        // the next piece's first loads go out, then the four waves' results
        // are joined through LDS: each leaves them where its last keys were
        const int xn = x + pc.g1 - pc.g0;
        const bool more = xn < x1, whole = pc.g0 == 0 && pc.g1 == pc.gran;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) {
            pc = piece_at(xn);
            issue(pc, pc.g0, to);
            load_q(pc);
        }
        l = cols_sum(l);
        const float back = __builtin_amdgcn_exp2f(-pexp);
        float* mine = (float*)(buf0 + (to ^ 1) * Geo::BUF);
        if (g == 0) {
            s_m[w][j] = m;
            s_l[w][j] = l * back;
            s_at[w] = (int)((unsigned char*)mine - smem);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) *(floatx4*)(mine + j * OS + 16 * n + 4 * g) = o[n] * back;
        __syncthreads();
        float* slot = few_slot(a.ws, 2 * blockIdx.x + (x == x0 ? 0 : 1), HD);
        for (int u = threadIdx.x; u < rows * (HD / 4); u += 256) {
            const int r = u / (HD / 4), c = 4 * (u % (HD / 4));
            const float mt = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
            floatx4 sum = {0.f, 0.f, 0.f, 0.f};
            float lt = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = s_m[k][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[k][r] - mt);
                lt += f * s_l[k][r];
                const floatx4 ok = *(const floatx4*)((const float*)(smem + s_at[k]) + r * OS + c);
                sum += f == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : f * ok;
            }
            if (whole) {
                const float inv = 1.0f / lt;
                *(float4u*)(a.out + ((int64_t)(sv.t0 + r / G) * a.Hq + h * G + r % G) * HD + c) = sum * inv;
            } else {
                *(floatx4*)(slot + r * HD + c) = sum;
                if (c == 0) *(float2*)(slot + AQ_ROWS * HD + 2 * r) = make_float2(mt, lt);
            }
        }
        if (!more) break;
        __syncthreads();                               // before these rows' places are copied over
        x = xn;
    }
}

// Joins the partials of a block that lies in several workgroups' ranges, a
// wave per row: workgroup b takes the block that is first cut before
// workgroup b + 1.
template <int HD>
__global__ __launch_bounds__(256) void attn_q8_few_join_kernel(PackedAttn a) {
    constexpr int EL = (HD + 63) / 64;                 // outputs per lane
    const JoinEntry en = *(const JoinEntry*)((const char*)a.ws + 32 * (blockIdx.x + 1));
    if (en.rows == 0) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int G = a.Hq / a.Hkv;
    // the first part's slot, then the first slot of each workgroup after it
    auto slot = [&](int k) { return few_slot(a.ws, k == 0 ? en.slot0 : 2 * ((int)blockIdx.x + k), HD); };
    for (int r = w; r < en.rows; r += 4) {
        float m = -INFINITY, l = 0.f, o[EL];
#pragma unroll
        for (int e = 0; e < EL; ++e) o[e] = 0.f;
        for (int k0 = 0; k0 < en.pieces; k0 += 8) {
            float2 ml[8];
            float v[8][EL];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float* sl = slot(min(k0 + k, en.pieces - 1));
                ml[k] = *(const float2*)(sl + AQ_ROWS * HD + 2 * r);
#pragma unroll
                for (int e = 0; e < EL; ++e) v[k][e] = sl[r * HD + min(64 * e + lane, HD - 1)];
            }
            float mt = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) mt = fmaxf(mt, ml[k].x);
            if (mt == -INFINITY) continue;             // nothing seen yet
            const float f = __builtin_amdgcn_exp2f(m - mt);
            m = mt;
            l *= f;
#pragma unroll
            for (int e = 0; e < EL; ++e) o[e] *= f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float fk = k0 + k < en.pieces ? __builtin_amdgcn_exp2f(ml[k].x - mt) : 0.f;
                l += fk * ml[k].y;
#pragma unroll
                for (int e = 0; e < EL; ++e) o[e] += fk * v[k][e];
            }
        }
        const int64_t at = ((int64_t)(en.t0 + r / G) * a.Hq + en.h * G + r % G) * HD;
#pragma unroll
        for (int e = 0; e < EL; ++e)
            if (64 * e + lane < HD) a.out[at + 64 * e + lane] = o[e] / l;
    }
}

bool attention_q8_few_shape(int hd, int G) { return (hd == 32 || hd == 64 || hd == 128) && G <= AQ_ROWS; }
int64_t attention_q8_few_bytes(int hd) {
    return FEW_ENTRIES + 2 * AQ_WGS * few_slot_floats(hd) * (int64_t)sizeof(float);
}

template <int HD>
static void launch_few(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    hipLaunchKernelGGL(attn_q8_few_kernel<HD>, dim3(AQ_WGS), dim3(256), 0, s, a, pb);
    if (few_granules(pb.max_seq) > AQ_KEEP)            // else no block is cut
        hipLaunchKernelGGL(attn_q8_few_join_kernel<HD>, dim3(AQ_WGS - 1), dim3(256), 0, s, a);
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
