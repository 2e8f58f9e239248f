// k_attn_many.hip -- attention of packed batches with more than a few query
// rows per (sequence, kv head), over the 8-bit cache or f32 pools: prompt
// chunks, mixed steps, drafted trees.  The arithmetic: attn_rows.h, how the
// keys are shared out: attn_plan.h.
//
// A workgroup of eight waves takes a block of 128 query rows over a range of
// keys: a wave 16 rows, or, where the block has fewer rows, several waves the
// same 16 rows and a part of the keys each.  A stage of keys is brought into
// LDS as f16 once for all waves, while the stage before is worked on and the
// one after is on its way in registers; one barrier a stage.
//   8-bit: the codes (exact in f16); a key's scores and weights go by its
//       steps, block by block of 32 elements.  Two MFMAs a product.
//   f32: a row of K or V is scaled by a power of two to [2^13, 2^14) at its
//       largest element and split into halves hi + lo of 22 bits; three MFMAs
//       a product (lo * lo is below what f32 sums keep).
// What bounds it: over the 8-bit cache no unit by itself.  The vector unit is
// busy in 57 % of the cycles (products by steps, the weights and their halves,
// the conversion), the matrix unit in 27 % (causal) and 30 % (trees), LDS in 41
// and 43 %, and a wave waits in 36 % of its cycles, most for the stage's barrier.
// Over f32 pools it is the bytes.  Head_dim 128, 8 kv heads: a mixed step of 13
// decoding users and three chunks of 714 to 839 tokens 347 us (251 TFLOP/s), a
// whole prompt of 4096 tokens 478 us (287 TFLOP/s), 4 users' trees of 32 to 61
// drafts over 48000 keys 230 us (319 TFLOP/s); 16 users' trees of 14 to 24
// drafts over 645 MB of f32 caches 164 us (3.9 TB/s; 158 on the fastest of the
// machines it was timed on).  12 or 16 waves, or two tiles a wave, do not fit
// the registers.
// Rows stay as they are stored, [key][element]: V^T comes out of LDS by the
// transposing read.  16-byte chunks of a row are permuted, chunk c of key k
// at place c ^ turn(k), so that both kinds of reads spread over the banks.
#include "attn_plan.h"
#include "attn_q8.h"

namespace slate_hip {

constexpr int AM_WGS = 256;            // one workgroup per CU
constexpr int AM_TH = 512;
constexpr int AM_ROWS = 8 * AR_TILE;   // query rows of a block
constexpr int AM_KEYS = 64;            // keys of a stage
constexpr int AM_KEEP = 512;           // blocks of up to this many keys are not cut
static_assert(AM_KEYS <= 128 && PK_MAX_KEYS + AM_KEYS > 0, "a count of keys passes 32 bits");

typedef short short4v __attribute__((ext_vector_type(4)));

// Transposing LDS read of 16-bit numbers: the 16 lanes of a group name four
// rows of 32 bytes, lane i quarter i % 4 of row i / 4; lane i gets number i of
// each row.
__device__ __forceinline__ half4_t read_columns16(const _Float16* p) {
    return __builtin_bit_cast(half4_t,
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(p)));
}

template <int HD>
__device__ __forceinline__ int turn(int key) {
    if (HD == 128) return ((key << 1) | (key >> 3 & 1)) & 15;
    if (HD == 64) return ((key & 6) | (key >> 3 & 1)) & 7;
    return key >> 2 & 3;
}

// Where element 8c of key k sits in a stage's plane (in halves).
template <int HD>
__device__ __forceinline__ int place(int key, int c) {
    return key * HD + 8 * (c ^ turn<HD>(key));
}

template <int HD, bool F32>
struct ManyGeom {
    static constexpr int PLANE = AM_KEYS * HD;         // halves
    static constexpr int PLANES = F32 ? 4 : 2;         // K hi (lo), V hi (lo)
    // what a thread brings in: 16 codes of a row, or 8 f32
    static constexpr int UNIT = F32 ? 8 : 16;
    static constexpr int UNITS = AM_KEYS * HD / UNIT;  // of K, and of V
    static constexpr int EACH = (UNITS + AM_TH - 1) / AM_TH;   // a thread's
};

// Blocks of a sequence and their granules (stages).
struct ManyCount {
    int G, Hkv, rows;                  // rows of a block
    bool causal;
    __device__ __forceinline__ int blocks(const SeqView& s) const { return (s.n * G + rows - 1) / rows; }
    // keys that block i's rows see
    __device__ __forceinline__ int seen(const SeqView& s, int i) const {
        return s.p0 + (causal ? (min(s.n * G, (i + 1) * rows) - 1) / G + 1 : s.n);
    }
    __device__ __forceinline__ int granules(const SeqView& s, int i) const { return (seen(s, i) + AM_KEYS - 1) / AM_KEYS; }
    // granules of a sequence, counted by the one lane that holds it: the keys
    // that a block sees step by rows / G and carry the rest
    __device__ __forceinline__ int operator()(const SeqView& s) const {
        if (s.n < 1) return 0;
        const int nb = blocks(s);
        if (!causal) return Hkv * nb * granules(s, 0);
        const int step = rows / G, rest = rows - step * G;
        int sum = granules(s, nb - 1);
        for (int i = 1, r = rest - 1, t = s.p0 + step; i < nb; ++i, t += step, r += rest) {
            if (r >= G) r -= G, ++t;                   // (i rows - 1) / G = t - p0 + floor(r / G), r < 2 G
            sum += (t + (r >= 0) + AM_KEYS - 1) / AM_KEYS;
        }
        return Hkv * sum;
    }
};
using ManyPlan = Plan<ManyCount>;

struct ManyPlace {
    SeqView seq;
    int64_t base;
    int h, block, gran, in;            // kv head, block, its granules, granule of it
};
__device__ __forceinline__ ManyPlace many_find(const ManyPlan& plan, const ManyCount& c, int x) {
    const Place pl = plan.find(x);
    ManyPlace r{pl.seq, pl.base, 0, 0, 0, 0};
    const int nb = c.blocks(pl.seq);
    if (!c.causal || nb <= 1) {
        r.gran = c.granules(pl.seq, 0);
        const int b = pl.at / r.gran;
        r.h = b / nb;
        r.block = b % nb;
        r.in = pl.at % r.gran;
        return r;
    }
    const int lane = threadIdx.x & 63;
    auto scan_from = [&](int i0, int& own) {           // blocks i0 .., a lane each
        own = i0 + lane < nb ? c.granules(pl.seq, i0 + lane) : 0;
        return wave_scan(own);
    };
    int own, per = 0;                                  // granules of a kv head
    for (int i0 = 0; i0 < nb; i0 += 64) per += __builtin_amdgcn_readlane(scan_from(i0, own), 63);
    r.h = pl.at / per;
    r.in = pl.at % per;
    for (int i0 = 0;; i0 += 64) {
        const int upto = scan_from(i0, own);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > r.in);
        if (past) {
            const int l = __builtin_ctzll(past);
            r.block = i0 + l;
            r.gran = __builtin_amdgcn_readlane(own, l);
            r.in -= __builtin_amdgcn_readlane(upto - own, l);
            return r;
        }
        r.in -= __builtin_amdgcn_readlane(upto, 63);
    }
}
__device__ __forceinline__ int many_begin(const ManyPlan& plan, const ManyCount& c, int w, int P) {
    const int x = plan.begin(w, P);
    if (x >= plan.total) return plan.total;
    const ManyPlace p = many_find(plan, c, x);
    return p.gran * AM_KEYS <= AM_KEEP ? x - p.in : x;
}

// Keys of a stage against the wave's rows.
template <int HD, bool F32>
struct ManyRows : AttnRows<HD> {
    using AttnRows<HD>::qh;
    using AttnRows<HD>::ql;
    using AttnRows<HD>::o;
    static constexpr int NB = HD / 32, ND = HD / 16;
    using Steps = Q8Steps<HD>;
    int koff[NB], voff[ND];            // where the lane reads K's and V's operands in a plane (halves)

    __device__ __forceinline__ void offsets() {
        const int g = (threadIdx.x & 63) >> 4, j = threadIdx.x & 15;
#pragma unroll
        for (int t = 0; t < NB; ++t) koff[t] = place<HD>(j, 4 * t + g);
        // lane i of a group names quarter i % 4 of the 16 columns of the
        // i / 4-th of its four keys (slots 8g .. +3 hold keys 4g + i, slots
        // 8g + 4 .. +7 keys 16 + 4g + i)
#pragma unroll
        for (int n = 0; n < ND; ++n) voff[n] = place<HD>(4 * g + (j >> 2), 2 * n + ((j & 3) >> 1)) + 4 * (j & 1);
    }

    // 16 H keys from key `at` of the stage on.  planes: K hi (lo), V hi (lo);
    // ks, vs: the keys' steps (Steps, or the power of two of a row as a
    // float).  MASKED as in Q8Rows (H = 2).  8-bit, all keys seen: top, the
    // bits of the largest V step of each 32 keys, vnorm, the V steps by the
    // inverse of its power of two, [block][key].  bad: keys whose V row has an element that
    // is not finite (it is 0 in the plane), vrow the first key's row (f32).
    template <int H, bool MASKED>
    __device__ __forceinline__ void keys(const _Float16* planes, int at, const unsigned char* steps, int2 top,
                                         const _Float16* vnorm, uint32_t seen, uint32_t bad, const float* vrow) {
        constexpr int PLANE = AM_KEYS * HD;
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const _Float16 *k = planes + at * HD, *v = k + (F32 ? 2 : 1) * PLANE;
        const Steps *ks = (const Steps*)steps + at, *vs = ks + AM_KEYS;
        const float *kf = (const float*)steps + at, *vf = kf + AM_KEYS;
        floatx4 s[H];
        const floatx4 zero = zeros();
        // Operands come out of LDS one group of MFMAs ahead; the fences keep
        // the order, which the scheduler gives up where registers get scarce
        // (mixed step 405 -> 368 us, trees over f32 172 -> 158 us).  8-bit: what
        // a group leaves to the vector unit goes between the MFMAs of the next
        // (368 -> 360 us).
        // A group of K: 16 keys, for f32 at most 64 elements of them.
        constexpr int KT = F32 && NB > 2 ? 2 : NB, KG = NB / KT, LO = F32 ? KT : 0;
        half8_t kr[2][KT + LO];
        auto read_k = [&](int q) {
            const _Float16* kh = k + 16 * (q / KG) * HD;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                kr[q & 1][t] = *(const half8_t*)(kh + koff[q % KG * KT + t]);
                if constexpr (F32) kr[q & 1][LO + t] = *(const half8_t*)(kh + PLANE + koff[q % KG * KT + t]);
            }
        };
        auto columns = [&](const _Float16* plane, int n) {
            const half4_t a = read_columns16(plane + voff[n]), b = read_columns16(plane + 16 * HD + voff[n]);
            return half8_t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        };
        // A group of V: 32 keys, 16 or 32 elements.
        constexpr int VU = F32 ? 1 : 2, VG = ND / VU, GROUPS = H / 2 * VG;
        half8_t vr[2][2];
        auto read_v = [&](int q) {
            const _Float16* vb = v + 32 * (q / VG) * HD;
#pragma unroll
            for (int u = 0; u < 2; ++u)
                vr[q & 1][u] = columns(F32 ? vb + u * PLANE : vb, F32 ? q % VG : VU * (q % VG) + u);
        };
        // 8-bit: a group's products, by the keys' steps
        floatx4 kp[2][NB];
        Steps kd[2][4];
        auto by_steps = [&](int hf) {
#pragma unroll
            for (int t = 0; t < NB; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[hf][e] = t == 0 ? times(kp[hf & 1][0][e], kd[hf & 1][e].s[0])
                                      : fmaf((float)kd[hf & 1][e].s[t], kp[hf & 1][t][e], s[hf][e]);
        };
        read_k(0);
#pragma unroll
        for (int q = 0; q < H * KG; ++q) {
            const int hf = q / KG, t0 = q % KG * KT;
            if (q + 1 < H * KG)
                read_k(q + 1);
            else
                read_v(0);
            __builtin_amdgcn_sched_barrier(0);
            const half8_t* kc = kr[q & 1];
            if constexpr (F32) {
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    s[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[LO + t], qh[t0 + t], t0 + t == 0 ? zero : s[hf], 0,
                                                                   0, 0);
                    s[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[t], ql[t0 + t], s[hf], 0, 0, 0);
                    s[hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[t], qh[t0 + t], s[hf], 0, 0, 0);
                }
                if (q % KG == KG - 1) s[hf] *= *(const floatx4*)(kf + 16 * hf + 4 * g);
            } else {
                floatx4* r = kp[q & 1];
#pragma unroll
                for (int i = 0; i < 4; ++i) kd[q & 1][i] = ks[16 * hf + 4 * g + i];
#pragma unroll
                for (int t = 0; t < NB; ++t) r[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[t], ql[t], zero, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < NB; ++t) r[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[t], qh[t], r[t], 0, 0, 0);
                if (hf > 0) {
                    by_steps(hf - 1);
#pragma unroll
                    for (int i = 0; i < 2 * NB; ++i) {  // a MFMA, then what the group before left to the vector unit
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!F32) by_steps(H - 1);
        // bit 16 (e / 4) + e % 4 of `bits`: the row sees the lane's key e
        const uint32_t bits = MASKED ? seen >> (4 * g) : 0;
        auto sees = [&](int e) { return !MASKED || (bits >> (16 * (e >> 2) + (e & 3)) & 1) != 0; };
        float p[4 * H], x[8];
        half8_t ph, pl;
        if constexpr (F32) {
            floatx4 d[H];
            int big = 0;
#pragma unroll
            for (int hf = 0; hf < H; ++hf) d[hf] = *(const floatx4*)(vf + 16 * hf + 4 * g);
#pragma unroll
            for (int e = 0; e < 4 * H; ++e) {
                const float step = d[e >> 2][e & 3];   // (a bit cast of the element itself reads the vector's first)
                if (!sees(e)) s[e >> 2][e & 3] = -INFINITY;
                if (sees(e)) big = max(big, __builtin_bit_cast(int, step));
            }
            this->template weights<H, true>(s, big, [](int b) { return (b >> 23) - 126; }, p);
            const float by = __builtin_amdgcn_exp2f(this->pexp);
#pragma unroll
            for (int b = 0; b < H / 2; ++b) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = p[8 * b + e] * (sees(e) ? d[2 * b + (e >> 2)][e & 3] * by : 0.f);
                halves(x, ph, pl);
#pragma unroll
                for (int n = 0; n < ND; ++n) {
                    const int q = b * ND + n;
                    if (q + 1 < GROUPS) read_v(q + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vr[q & 1][1], ph, o[n], 0, 0, 0);
                    o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vr[q & 1][0], pl, o[n], 0, 0, 0);
                    o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vr[q & 1][0], ph, o[n], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (MASKED)
                for (uint32_t left = bad; left; left &= left - 1) {   // for the rows that do see such a row
                    const int key = __builtin_ctz(left);
                    if (!(seen >> key & 1)) continue;
#pragma unroll
                    for (int n = 0; n < ND; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float val = vrow[(int64_t)key * HD + 16 * n + 4 * g + e];
                            if (!(fabsf(val) < INFINITY)) o[n][e] += val;
                        }
                }
        } else {
            int big = max(top.x, top.y);
            // V steps of 0 in all 32 keys: the smallest step's exponent, so that weights stay in f16's range
            // whatever the largest step elsewhere is (their products are 0, infinity's would be NaN)
            const int shift[2] = {step_exponent(max(top.x, 1)), step_exponent(max(top.y, 1))};
            if (MASKED) {
                big = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const Steps d = vs[16 * (e >> 2) + 4 * g + (e & 3)];
                    if (!sees(e)) {
                        s[e >> 2][e & 3] = -INFINITY;
                    } else {
#pragma unroll
                        for (int t = 0; t < NB; ++t) big = max(big, step_bits(d.s[t]));
                    }
                }
            }
            // Group q's weights are p times its steps as halves, hi + lo to 22
            // bits, made while group q - 1 is multiplied.
            half8_t wh[2], wl[2];
            auto multiply = [&](int q, int k) {            // k: the tile in bit 0, hi in bit 1
                o[2 * (q % NB) + (k & 1)] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    vr[q & 1][k & 1], k & 2 ? wh[q & 1] : wl[q & 1], o[2 * (q % NB) + (k & 1)], 0, 0, 0);
            };
            if constexpr (MASKED) {
                this->template weights<H, true>(s, big, step_exponent, p);
                const float by = __builtin_amdgcn_exp2f(this->pexp);
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] *= by;
                Steps dv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) dv[e] = vs[16 * (e >> 2) + 4 * g + (e & 3)];
#pragma unroll
                for (int q = 0; q < GROUPS; ++q) {
                    if (q + 1 < GROUPS) read_v(q + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = sees(e) ? times(p[e], dv[e].s[q]) : 0.f;   // an unseen step may be anything
                    halves(x, wh[q & 1], wl[q & 1]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) multiply(q, k);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                // All keys are seen: their steps come as f16 d by the power of
                // two of the largest of the 32, in (0, 1), and p = a + b, by
                // the inverse power, is split but once.  hi = f16(a d), its
                // remainder a d - hi is exact (or below 2^-25 where a weight of
                // 1 stands for 2^10 or more), lo = b d + that: packed f16
                // operations, half of what f32 products and their halves take
                // (mixed step 373 -> 341 us).
                this->template weights<H, true>(s, big, step_exponent, p, shift);
                half8_t ph[H / 2], pl[H / 2], d[2];
#pragma unroll
                for (int b = 0; b < H / 2; ++b) halves(p + 8 * b, ph[b], pl[b]);
                auto read_d = [&](int q) {
                    const _Float16* at = vnorm + q % NB * AM_KEYS + 32 * (q / NB) + 4 * g;
                    const half4_t lo = *(const half4_t*)at, hi = *(const half4_t*)(at + 16);
                    d[q & 1] = half8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                };
                half8_t rest;
                auto split = [&](int q, int k) {           // in three steps
                    const half8_t a = ph[q / NB], dq = d[q & 1];
                    if (k == 0) wh[q & 1] = a * dq;
                    if (k == 1) rest = __builtin_elementwise_fma(a, dq, -wh[q & 1]);
                    if (k == 2) wl[q & 1] = __builtin_elementwise_fma(pl[q / NB], dq, rest);
                };
                read_d(0);
                if (GROUPS > 1) read_d(1);
#pragma unroll
                for (int k = 0; k < 3; ++k) split(0, k);
#pragma unroll
                for (int q = 0; q < GROUPS; ++q) {
                    if (q + 1 < GROUPS) read_v(q + 1);
                    if (q + 2 < GROUPS) read_d(q + 2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        multiply(q, k);
                        if (q + 1 < GROUPS) split(q + 1, k);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    }
};

// The largest of the lanes that share a row (16, 8 or 4 of them).
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
    if (N == 16) return row16_max(v);
    if (N == 8) return group8_max(v);
    v = fmaxf(v, dpp_mov<DPP_QUAD_XOR1>(v));
    return fmaxf(v, dpp_mov<DPP_QUAD_XOR2>(v));
}

// TREE: rows see their ancestors, else what lies before them (one kernel for
// both holds the registers of both: 418 against 406 us for the mixed step).
template <int HD, bool F32, bool TREE>
__global__ __launch_bounds__(AM_TH, 2) void attn_many_kernel(PackedAttn a, PackedBatch pb) {
    using Geo = ManyGeom<HD, F32>;
    constexpr int TH = AM_TH, W = AM_TH / 64, ROWS = AM_ROWS, WGS = AM_WGS;
    using Steps = Q8Steps<HD>;
    constexpr int NB = HD / 32, ND = HD / 16, KEYS = AM_KEYS, PLANE = Geo::PLANE, EACH = Geo::EACH;
    constexpr int STEP = F32 ? 4 : (int)sizeof(Steps);   // bytes
    __shared__ __attribute__((aligned(16))) _Float16 s_rows[2][Geo::PLANES * PLANE];
    __shared__ __attribute__((aligned(16))) unsigned char s_step[2][2 * KEYS * STEP];
    __shared__ uint32_t s_seen[PK_MAX_DRAFT / 32][ROWS];   // the drafts that a block's token sees
    __shared__ int16_t s_par[PK_MAX_DRAFT];
    __shared__ ManyPlan::Lane s_plan[64];
    __shared__ uint32_t s_bad[4][2];                  // f32: keys whose V row has an element that is not finite
    __shared__ int s_top[2][2];                       // 8-bit: the largest V step of each 32 keys
    __shared__ __attribute__((aligned(16))) _Float16 s_vnorm[2][F32 ? 1 : NB * KEYS];   // [block][key]: V steps by 2^-shift
    // what the waves that share rows leave for each other: where the stage
    // that is worked through was, if it fits
    constexpr int OS = HD + 4;
    constexpr int JOIN_FLOATS = (W - 1) * AR_TILE * OS;
    constexpr bool JOIN_IN_ROWS = JOIN_FLOATS * 4 <= Geo::PLANES * PLANE * 2;
    __shared__ __attribute__((aligned(16))) float s_join[JOIN_IN_ROWS ? 4 : JOIN_FLOATS];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, j = lane & 15;
    const int G = a.Hq / a.Hkv;
    // neighbouring ranges on one XCD: blocks that share keys find them in its L2
    const int wg = (blockIdx.x % 8) * (WGS / 8) + blockIdx.x / 8;
    const ManyCount count{G, a.Hkv, ROWS, !TREE};
    const ManyPlan plan(pb, count);
    auto begin = [&](int v) { return many_begin(plan, count, v, WGS); };
    const int x0 = begin(wg), x1 = begin(wg + 1);
    if (x0 >= x1) {
        if (tid == 0) entry_of(a.ws, wg)->rows = 0;
        return;
    }
    const float scale2 = (1.0f / sqrtf((float)HD)) * LOG2E;
    if (tid < 8) s_bad[tid >> 1][tid & 1] = 0;

    struct Piece {
        int x;                         // its place on the line; >= x1: none
        SeqView seq;
        int h, block, gran, g0, g1, last;
        int open;                      // keys below it are seen by all rows of the block
        int64_t at;                    // first element of the head's rows
    };
    auto piece_in = [&](const ManyPlan& plan, int x) {
        const ManyPlace pl = many_find(plan, count, x);
        const int64_t base = F32 ? pl.base : pl.base / HD * HD;
        return Piece{x, pl.seq, pl.h, pl.block, pl.gran, pl.in, min(pl.gran, pl.in + (x1 - x)),
                     count.seen(pl.seq, pl.block) - 1,
                     TREE ? pl.seq.p0 : pl.seq.p0 + pl.block * ROWS / G + 1, base + pl.h * a.head_stride};
    };
    const int total = plan.total, end = plan.end;
    auto piece_after = [&](const Piece& p) {
        const int x = p.x + p.g1 - p.g0;
        return x < x1 ? piece_in(ManyPlan(pb, count, total, end, s_plan[lane]), x) : Piece{x1};
    };
    // a stage's rows on their way: the thread's unit of K and of V, and steps
    // (rows past the last key repeat it: nobody sees them)
    typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
    uint4v raw[2][EACH];                               // 8-bit: K's and V's codes
    float4u f32[2][EACH][2];
    Steps st;
    // key and element of the thread's unit u
    auto unit_key = [&](int u) { return (tid + TH * u) * Geo::UNIT / HD; };
    auto unit_elem = [&](int u) { return (tid + TH * u) * Geo::UNIT % HD; };
    const bool mine = Geo::UNITS >= TH || tid < Geo::UNITS;
    auto load = [&](const Piece& p, int gr) {
        const int k0 = gr * KEYS;
        if (mine) {
#pragma unroll
            for (int u = 0; u < EACH; ++u) {
                const int64_t e = p.at + (int64_t)min(k0 + unit_key(u), p.last) * HD + unit_elem(u);
                if constexpr (F32) {
                    f32[0][u][0] = *(const float4u*)(a.kf + e);
                    f32[0][u][1] = *(const float4u*)(a.kf + e + 4);
                    f32[1][u][0] = *(const float4u*)(a.vf + e);
                    f32[1][u][1] = *(const float4u*)(a.vf + e + 4);
                } else {
                    raw[0][u] = *(const uint4v*)(a.kv8.kq + e);
                    raw[1][u] = *(const uint4v*)(a.kv8.vq + e);
                }
            }
        }
        if (!F32 && tid < 2 * KEYS) {
            const int64_t r = p.at / KV8_BLOCK + (int64_t)min(k0 + tid % KEYS, p.last) * NB;
            st = *(const Steps*)((tid < KEYS ? a.kv8.ks : a.kv8.vs) + r);
        }
    };
    // and into LDS; some row may not see its keys from `all` on
    auto put = [&](int to, int ring, int all) {
        _Float16* rows = s_rows[to];
        if (mine) {
#pragma unroll
            for (int u = 0; u < EACH; ++u) {
                const int key = unit_key(u), elem = unit_elem(u);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    _Float16* at = rows + kv * (Geo::PLANES / 2) * PLANE;
                    if constexpr (F32) {
                        float x[8], top = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = f32[kv][u][e >> 2][e & 3];
                        if (kv == 1 && key >= all) {
                            bool bad = false;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const bool fine = fabsf(x[e]) < INFINITY;
                                bad |= !fine;
                                x[e] = fine ? x[e] : 0.f;
                            }
                            if (bad) atomicOr(&s_bad[ring][key >> 5], 1u << (key & 31));
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
                        top = lanes_max<HD / 8>(top);
                        // K: a step's inverse stays a normal number.  V: weights carry 2^(11 - 14 + e2) (AR_PEXP),
                        // and their sum over the keys stays finite; rows below 2^-92 are kept to 2^-114.
                        const int e2 = top > 0.f && top < INFINITY
                                           ? min(kv ? 90 : 126, 14 - __builtin_amdgcn_frexp_expf(top))
                                           : 0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = ldexpf(x[e], e2);
                        half8_t hi, lo;
                        halves(x, hi, lo);
                        *(half8_t*)(at + place<HD>(key, elem / 8)) = hi;
                        *(half8_t*)(at + PLANE + place<HD>(key, elem / 8)) = lo;
                        // a V row of zeros has a step of 0: it does not count among the largest steps
                        if (elem == 0)
                            ((float*)s_step[to])[kv * KEYS + key] = kv == 1 && top == 0.f ? 0.f : ldexpf(1.0f, -e2);
                    } else {
                        const uint4v r = raw[kv][u];
                        *(half8_t*)(at + place<HD>(key, elem / 8)) = codes_f16(uint2v{r[0], r[1]});
                        *(half8_t*)(at + place<HD>(key, elem / 8 + 1)) = codes_f16(uint2v{r[2], r[3]});
                    }
                }
            }
        }
        if (!F32 && tid < 2 * KEYS) {
            ((Steps*)s_step[to])[tid] = st;
            if (tid >= KEYS) {                         // wave 1: a V row's steps per lane
                int top = 0;
#pragma unroll
                for (int t = 0; t < NB; ++t) top = max(top, step_bits(st.s[t]));
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) top = max(top, __shfl_xor(top, off));
                if ((lane & 31) == 0) s_top[to][lane >> 5] = top;
#pragma unroll
                for (int t = 0; t < NB; ++t)
                    s_vnorm[to][t * KEYS + lane] = (_Float16)ldexpf((float)st.s[t], -step_exponent(top));
            }
        }
    };
    auto put_piece = [&](const Piece& p, int gr, int to, int ring) { put(to, ring, p.open - gr * KEYS); };

    // How a block's rows go to the waves: tiles of 16 rows, each taken by
    // W / tiles waves, which share the keys 32 by 32.
    struct Share {
        int part, parts, r;            // the wave's part of the keys, and how many there are; its first row in the block
    };
    auto share_of = [&](const Piece& p) {
        const int rows = min(ROWS, p.seq.n * G - p.block * ROWS);
        const int tiles = rows <= AR_TILE ? 1 : rows <= 2 * AR_TILE ? 2 : rows <= 4 * AR_TILE ? 4 : W;
        return Share{w / tiles, W / tiles, AR_TILE * (w % tiles)};
    };
    // The piece worked on and the two after it: the stage being loaded is two
    // ahead, so in one of them, and no search stands in the loop over stages.
    Piece pc = piece_in(plan, x0);
    load(pc, pc.g0);
    if (w == 0)
        leave_entry(a.ws, WGS, wg, x0, pc.g0, pc.gran, plan, begin,
                    JoinEntry{pc.seq.t0, min(ROWS, pc.seq.n * G - pc.block * ROWS), pc.block * ROWS, pc.h, 0,
                              0});
    if (w == 0) s_plan[lane] = plan.first();
    __syncthreads();                                   // (s_bad is clear, too)
    Piece p1 = piece_after(pc), p2 = piece_after(p1);
    Piece nx = pc;                                     // the piece of the stage being loaded
    int ngr = pc.g0, ahead = 0;                        // that stage; the piece is pc, p1 or p2
    // the next stage after the one being loaded; false at the range's end
    auto advance = [&]() {
        if (ngr + 1 < nx.g1) {
            ++ngr;
            return true;
        }
        nx = ahead == 0 ? p1 : p2;
        ++ahead;
        ngr = nx.g0;
        return nx.x < x1;
    };
    bool coming = true;
    int to = 0, ring = 0;

    for (;;) {
        const SeqView sv = pc.seq;
        const int h = pc.h, r0 = pc.block * ROWS, rows = min(ROWS, sv.n * G - r0);
        const Share sh = share_of(pc);
        const int rw = sh.r, tok0 = r0 / G;            // the wave's first row in the block, the block's first token
        const int row = r0 + rw + j;
        const bool live = rw + j < rows;
        const int tok = row / G;
        ManyRows<HD, F32> R;
        R.offsets();
        float4u qraw[NB][2];
        const float* qp =
            a.q + ((int64_t)(sv.t0 + (live ? tok : 0)) * a.Hq + h * G + (live ? row % G : 0)) * HD + 8 * g;
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            qraw[t][0] = *(const float4u*)(qp + 32 * t);
            qraw[t][1] = *(const float4u*)(qp + 32 * t + 4);
        }
        if (pc.x == x0) {                               // the first stage, once q is on its way too
            put_piece(nx, ngr, 0, 0);
            if ((coming = advance())) load(nx, ngr);
        }
        R.start(qraw, live, scale2);
        // keys below `open` are seen by all of the wave's rows, from `end` on by none
        const int open = TREE ? sv.p0 : sv.p0 + (r0 + min(rw, rows - 1)) / G + 1;
        const int end = rw >= rows ? 0 : TREE ? sv.p0 + sv.n : sv.p0 + (r0 + min(rw + AR_TILE, rows) - 1) / G + 1;
        const int words = (sv.n + 31) / 32;
        if (TREE && pc.g1 * KEYS > sv.p0) {        // the block's tokens' ancestors
            __syncthreads();
            for (int i = tid; i < sv.n; i += TH) {
                const int up = a.parent[sv.t0 + i];
                s_par[i] = (int16_t)(up >= 0 && up < i ? up : -1);
            }
            __syncthreads();
            if (tid < (r0 + rows - 1) / G - tok0 + 1) {
                int cur = tok0 + tid;
                for (int wd = words - 1; wd >= 0; --wd) {
                    uint32_t bits = 0;
                    while (cur >= 32 * wd) {
                        bits |= 1u << (cur & 31);
                        cur = s_par[cur];
                    }
                    s_seen[wd][tid] = bits;
                }
            }
        }
        for (int gr = pc.g0; gr < pc.g1; ++gr) {
            __syncthreads();                           // the stage is in LDS; the other buffer is read through
            const int now = to, now_ring = ring;
            to ^= 1;
            ring = (ring + 1) & 3;
            if (F32 && tid < 2) s_bad[(ring + 1) & 3][tid] = 0;   // last read two stages ago, next set after a barrier
            // The next stage goes into LDS now in the first half of the waves,
            // after this one's work in the other half: the two waves of a SIMD are then
            // in different phases (8-bit 430 -> 416 and 262 -> 244 us, f32 211 -> 194).
            const bool had = coming, early = w < W / 2;
            auto bring = [&]() {
                put_piece(nx, ngr, to, ring);
                if ((coming = advance())) load(nx, ngr);
            };
            if (had && early) bring();
            const int k0 = gr * KEYS;
            const _Float16* planes = s_rows[now];
            const unsigned char* steps = s_step[now];
            const int top0 = F32 ? 0 : s_top[now][0], top1 = F32 ? 0 : s_top[now][1];
            const bool all = sh.parts == 1 && k0 + KEYS <= open && k0 < end;
            if (all) R.template keys<4, false>(planes, 0, steps, make_int2(top0, top1), s_vnorm[now], 0, 0, nullptr);
#pragma unroll 1
            for (int at = 0; !all && at < KEYS && k0 + at < end; at += AR_KEYS) {
                if (((2 * gr + at / AR_KEYS) & (sh.parts - 1)) != sh.part) continue;
                if (k0 + at + AR_KEYS <= open) {
                    R.template keys<2, false>(planes, at, steps, make_int2(at ? top1 : top0, 0), s_vnorm[now] + (F32 ? 0 : at), 0, 0,
                                                nullptr);
                    continue;
                }
                uint32_t seen = 0;
                if (live && !TREE) {
                    const int n = min(32, max(0, sv.p0 + tok + 1 - k0 - at));
                    seen = n == 32 ? 0xffffffffu : (1u << n) - 1;
                } else if (live) {
                    const int d = k0 + at - sv.p0, wd = d >> 5;
                    const uint32_t lo = wd < 0 ? 0xffffffffu : wd < words ? s_seen[wd][tok - tok0] : 0;
                    const uint32_t hi = wd + 1 < 0 ? 0xffffffffu : wd + 1 < words ? s_seen[wd + 1][tok - tok0] : 0;
                    seen = (uint32_t)(((uint64_t)hi << 32 | lo) >> (d & 31));
                }
                R.template keys<2, true>(planes, at, steps, make_int2(0, 0), nullptr, seen, F32 ? s_bad[now_ring][at >> 5] : 0,
                                         F32 ? a.vf + pc.at + (int64_t)(k0 + at) * HD : nullptr);
            }
            if (had && !early) bring();
        }
        const bool whole = pc.g0 == 0 && pc.g1 == pc.gran;
        const float back = R.back();
        float l = R.sum();
#pragma unroll
        for (int n = 0; n < ND; ++n) R.o[n] *= back;
        if (sh.parts > 1) {                            // the parts of the keys joined
            float* area = JOIN_IN_ROWS ? (float*)s_rows[to ^ 1] : s_join;
            const int tiles = W / sh.parts, tile = rw / AR_TILE;
            __syncthreads();
            if (sh.part > 0) {
                float* at = area + ((sh.part - 1) * tiles + tile) * AR_TILE * OS + j * OS;
#pragma unroll
                for (int n = 0; n < ND; ++n) *(floatx4*)(at + 16 * n + 4 * g) = R.o[n];
                if (g == 0) *(float2*)(at + HD) = make_float2(R.m, l);
            }
            __syncthreads();
            for (int k = 1; k < sh.parts && sh.part == 0; ++k) {
                const float* at = area + ((k - 1) * tiles + tile) * AR_TILE * OS + j * OS;
                const float2 ml = *(const float2*)(at + HD);
                const float mt = fmaxf(R.m, ml.x);
                // (a part that saw no key is left out; any other, if its factor is 0, still has its NaN and infinities)
                const bool none0 = R.m == -INFINITY, none1 = ml.x == -INFINITY;
                const float f0 = none0 ? 0.f : __builtin_amdgcn_exp2f(R.m - mt);
                const float f1 = none1 ? 0.f : __builtin_amdgcn_exp2f(ml.x - mt);
                R.m = mt;
                l = l * f0 + ml.y * f1;
#pragma unroll
                for (int n = 0; n < ND; ++n) {
                    const floatx4 other = *(const floatx4*)(at + 16 * n + 4 * g);
                    R.o[n] = (none0 ? floatx4{0.f, 0.f, 0.f, 0.f} : R.o[n] * f0) +
                             (none1 ? floatx4{0.f, 0.f, 0.f, 0.f} : other * f1);
                }
            }
        }
        if (live && sh.part == 0) {
            if (whole) {
                float* op = a.out + ((int64_t)(sv.t0 + tok) * a.Hq + h * G + row % G) * HD + 4 * g;
                const float inv = 1.0f / l;
#pragma unroll
                for (int n = 0; n < ND; ++n) *(float4u*)(op + 16 * n) = R.o[n] * inv;
            } else {
                float* slot = slot_of(a.ws, WGS, 2 * wg + (pc.x == x0 ? 0 : 1), ROWS, HD);
                const int r = rw + j;
                if (g == 0) *(float2*)(slot + ROWS * HD + 2 * r) = make_float2(R.m, l);
#pragma unroll
                for (int n = 0; n < ND; ++n) *(floatx4*)(slot + r * HD + 16 * n + 4 * g) = R.o[n];
            }
        }
        if (p1.x >= x1) break;
        pc = p1;
        p1 = p2;
        p2 = piece_after(p2);
        --ahead;
    }
}

int64_t attention_many_bytes(int hd) { return plan_bytes(AM_WGS, AM_ROWS, hd); }
bool attention_many_takes(const PackedAttn& a) { return a.hd == 32 || a.hd == 64 || a.hd == 128; }
double attention_many_most(const PackedAttn& a, const PackedBatch& pb) {
    return a.Hkv * ((double)pb.T * (a.Hq / a.Hkv) / AM_ROWS + pb.B) * ((pb.max_seq + AM_KEYS - 1) / AM_KEYS);
}

template <int HD>
static void launch_many(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    auto kernel = a.kf ? attn_many_kernel<HD, true, true>
                       : a.parent ? attn_many_kernel<HD, false, true> : attn_many_kernel<HD, false, false>;
    hipLaunchKernelGGL(kernel, dim3(AM_WGS), dim3(AM_TH), 0, s, a, pb);
    if (pb.max_seq > AM_KEEP)                          // else no block is cut
        launch_attn_join(a.out, a.ws, a.Hq, a.Hkv, HD, AM_ROWS, AM_WGS, s);
}

int launch_attention_many(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    if (a.hd == 128)
        launch_many<128>(a, pb, s);
    else if (a.hd == 64)
        launch_many<64>(a, pb, s);
    else
        launch_many<32>(a, pb, s);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
