// k_attn_q8.hip -- attention over the 8-bit cache (the arithmetic: attn_q8.h,
// how the keys are shared out: attn_plan.h).
//
// Two kernels.  Few rows per (sequence, kv head) -- a decode step's tokens
// times the query heads of a kv head, small trees --: each of a workgroup's
// four waves takes every fourth 32 keys, for all rows.  Many rows (prompt
// chunks, larger trees): all four waves take all keys, each for its own rows.
#include "attn_plan.h"
#include "attn_q8.h"

namespace slate_hip {

constexpr int A8_TILE = 16;            // query rows of an MFMA
constexpr int A8_KEYS = 32;            // keys of a step

// ---------------------------------------------------------------------------
// Few rows.  Memory bound: 2.125 bytes per key and element against two f16 MFMAs
// and about 400 VALU operations per 32 keys and wave.  So the design is about
// loads: each wave copies its next 32 keys' rows straight into LDS (16 bytes
// per lane, no registers) while it works on the last 32, with no barrier
// until its range ends; 70 KB are on their way per CU.

constexpr int AF_GRAN = 4 * A8_KEYS;   // keys of a granule
constexpr int AF_KEEP = 4;             // blocks of up to this many granules are not cut

__host__ __device__ inline int few_granules(int keys) { return (keys + AF_GRAN - 1) / AF_GRAN; }

// Granules of a sequence: one block of at most `rows` rows per kv head.
struct FewCount {
    int G, Hkv, rows;
    __device__ __forceinline__ int operator()(const SeqView& s) const {
        return s.n < 1 || (int64_t)s.n * G > rows ? 0 : Hkv * few_granules(s.p0 + s.n);
    }
};
using FewPlan = Plan<FewCount>;

// Where workgroup w's range begins: N w / P, or the start of the block there
// if it is short (it is not cut: the last workgroup that would begin in it
// takes it whole).
__device__ __forceinline__ int few_begin(const FewPlan& plan, int w) {
    const int x = plan.begin(w, AP_WGS);
    if (x >= plan.total) return plan.total;
    const Place pl = plan.find(x);
    const int gran = few_granules(pl.seq.p0 + pl.seq.n), in = pl.at % gran;
    return gran <= AF_KEEP ? x - in : x;
}

template <int HD, int NT>
__global__ __launch_bounds__(256, 2) void attn_q8_few_kernel(PackedAttn a, PackedBatch pb) {
    using Geo = Q8Geom<HD>;
    using Steps = Q8Steps<HD>;
    constexpr int NB = Geo::NB, ND = Geo::ND;
    constexpr int ROWS = A8_TILE * NT;
    constexpr int CODES = A8_KEYS * HD;                // bytes of a wave's K (or V) codes
    constexpr int OS = HD + 4;                         // row stride of a wave's results in LDS (floats)
    constexpr int USED = 2 * CODES + 2 * A8_KEYS * (int)sizeof(Steps);
    constexpr int BUF = USED > A8_TILE * OS * 4 ? USED : A8_TILE * OS * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[8 * BUF];
    __shared__ float s_m[4][A8_TILE], s_l[4][A8_TILE];
    __shared__ int s_at[4];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, j = lane & 15;
    const int G = a.Hq / a.Hkv;
    const FewPlan plan(pb, FewCount{G, a.Hkv, ROWS});
    const int x0 = few_begin(plan, blockIdx.x), x1 = few_begin(plan, blockIdx.x + 1);
    if (x0 >= x1) {
        if (threadIdx.x == 0) entry_of(a.ws, blockIdx.x)->rows = 0;
        return;
    }
    const float scale2 = (1.0f / sqrtf((float)HD)) * LOG2E;
    unsigned char* buf0 = smem + w * 2 * BUF;

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
    auto key0 = [&](int gr) { return gr * AF_GRAN + w * A8_KEYS; };
    auto issue = [&](const Piece& p, int gr, int to) {
        const int k0 = key0(gr), last = p.seq.p0 + p.seq.n - 1;
        if (k0 > last) return;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(buf0 + to * BUF));
        const int8_t *kb = uniform(p.kq + (int64_t)k0 * HD), *vb = uniform(p.vq + (int64_t)k0 * HD);
#pragma unroll
        for (int i = 0; i < CODES / 1024; ++i) {
            const int at = 64 * i + lane, key = at / Geo::CH, c = at % Geo::CH;
            const uint32_t off = (uint32_t)min(key, last - k0) * HD + 16 * (c ^ swz<HD>(key));
            lds_copy16(kb, off, dst + 1024 * i);
            lds_copy16(vb, off, dst + CODES + 1024 * i);
        }
        // lanes 0..31 carry the steps of a K row each, 32..63 of a V row
        const int64_t r = min(k0 + (lane & 31), last);
        st = *(const Steps*)((lane < 32 ? p.ks : p.vs) + r * NB);
    };
    // q of row j of the first tile, elements 32t + 8g .. +7
    float4u qraw[NB][2];
    auto q_row = [&](const Piece& p, int r) {
        const bool live = r < p.seq.n * G;
        return a.q + ((int64_t)(p.seq.t0 + (live ? r / G : 0)) * a.Hq + p.h * G + (live ? r % G : 0)) * HD;
    };
    auto load_q = [&](const Piece& p) {
        const float* qp = q_row(p, j) + 8 * g;
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
    if (w == 0)
        leave_entry(a.ws, blockIdx.x, x0, pc.g0, pc.gran, [&](int v) { return few_begin(plan, v); },
                    JoinEntry{pc.seq.t0, pc.seq.n * G, 0, pc.h, 0, 0});

    for (int x = x0;;) {
        const SeqView sv = pc.seq;
        const int keys = sv.p0 + sv.n, h = pc.h, rows = sv.n * G;
        Q8Rows<HD, NT> R;
        uint32_t drafts[NT];                           // the drafts that row j's token sees (n <= 32)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = A8_TILE * i + j, tok = r / G;
            const bool live = r < rows;
            if (i == 0)
                R.start(i, qraw, live, scale2);
            else
                R.start(i, q_row(pc, r), live, scale2);
            drafts[i] = (2u << min(tok, 31)) - 1;      // causal: itself and all before it
            if (a.parent) {
                const int par = a.parent[sv.t0 + min(lane, sv.n - 1)];
                drafts[i] = 0;
                int cur = live ? tok : -1;
                while (__builtin_amdgcn_ballot_w64(cur >= 0)) {
                    const int up = __shfl(par, max(cur, 0));
                    if (cur >= 0) drafts[i] |= 1u << cur;
                    cur = up >= 0 && up < cur ? up : -1;
                }
            }
            if (!live) drafts[i] = 0;
        }

        for (int gr = pc.g0; gr < pc.g1; ++gr) {
            const int k0 = key0(gr);
            if (k0 >= keys) break;                     // only in the last granule
            unsigned char* buf = buf0 + to * BUF;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            Steps* steps = (Steps*)(buf + 2 * CODES);
            steps[lane] = st;
            to ^= 1;
            if (gr + 1 < pc.g1) issue(pc, gr + 1, to);
            uint32_t seen[NT];
            if (k0 + A8_KEYS <= sv.p0) {
                R.template keys32<false>(buf, buf + CODES, steps, steps + A8_KEYS, seen);
            } else {                                   // drafts among the keys, or past the last one
#pragma unroll
                for (int i = 0; i < NT; ++i) seen[i] = seen_keys(drafts[i], k0, sv.p0);
                R.template keys32<true>(buf, buf + CODES, steps, steps + A8_KEYS, seen);
            }
        }

        // the next piece's first loads go out, then the four waves' results
        // are joined through LDS, a tile at a time: each wave leaves them where its last keys were
        const int xn = x + pc.g1 - pc.g0;
        const bool more = xn < x1, whole = pc.g0 == 0 && pc.g1 == pc.gran;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) {
            pc = piece_at(xn);
            issue(pc, pc.g0, to);
            load_q(pc);
        }
        float* slot = slot_of(a.ws, 2 * blockIdx.x + (x == x0 ? 0 : 1), ROWS, HD);
        float* mine = (float*)(buf0 + (to ^ 1) * BUF);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if (i > 0) {
                if (A8_TILE * i >= rows) break;
                __syncthreads();
            }
            const float back = R.back(i), l = R.sum(i);
            if (g == 0) {
                s_m[w][j] = R.m[i];
                s_l[w][j] = l;
                s_at[w] = (int)((unsigned char*)mine - smem);
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) *(floatx4*)(mine + j * OS + 16 * n + 4 * g) = R.o[i][n] * back;
            __syncthreads();
            const int here = min(A8_TILE, rows - A8_TILE * i);
            for (int u = threadIdx.x; u < here * (HD / 4); u += 256) {
                const int r = u / (HD / 4), c = 4 * (u % (HD / 4)), row = A8_TILE * i + r;
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
                    *(float4u*)(a.out + ((int64_t)(sv.t0 + row / G) * a.Hq + h * G + row % G) * HD + c) = sum * inv;
                } else {
                    *(floatx4*)(slot + row * HD + c) = sum;
                    if (c == 0) *(float2*)(slot + ROWS * HD + 2 * row) = make_float2(mt, lt);
                }
            }
        }
        if (!more) break;
        __syncthreads();                               // before these rows' places are copied over
        x = xn;
    }
}

// ---------------------------------------------------------------------------
// Many rows.  A workgroup takes a block of 64 NT rows (16 NT a wave) over a
// range of keys, 64 at a time: the waves copy them into LDS together while
// they work on the last 64, one barrier per 64 keys.  VALU bound: about 230
// operations per 16 rows and 32 keys (softmax, splitting and weighting P four
// blocks wide), 160 per 32 keys to convert the codes, against 32 MFMAs a tile.

constexpr int AM_KEYS = 64;            // keys of a granule
constexpr int AM_KEEP = 4;

// Blocks of a sequence and their granules.
struct ManyCount {
    int G, Hkv, rows;                  // rows of a block
    bool causal;
    __device__ __forceinline__ int blocks(const SeqView& s) const { return (s.n * G + rows - 1) / rows; }
    // keys that block i's rows see
    __device__ __forceinline__ int keys(const SeqView& s, int i) const {
        return s.p0 + (causal ? (min(s.n * G, (i + 1) * rows) - 1) / G + 1 : s.n);
    }
    __device__ __forceinline__ int granules(const SeqView& s, int i) const {
        return (keys(s, i) + AM_KEYS - 1) / AM_KEYS;
    }
    __device__ __forceinline__ int per_head(const SeqView& s) const {
        const int nb = blocks(s);
        if (!causal || nb <= 1) return nb * granules(s, 0);
        int sum = 0;
        for (int i = 0; i < nb; ++i) sum += granules(s, i);
        return sum;
    }
    __device__ __forceinline__ int operator()(const SeqView& s) const { return s.n < 1 ? 0 : Hkv * per_head(s); }
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
    const int per = c.per_head(pl.seq);
    r.h = pl.at / per;
    r.in = pl.at % per;
    for (int i0 = 0;; i0 += 64) {                      // 64 blocks at a time
        const int i = i0 + (int)(threadIdx.x & 63);
        const int own = i < nb ? c.granules(pl.seq, i) : 0, upto = wave_scan(own);
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
__device__ __forceinline__ int many_begin(const ManyPlan& plan, const ManyCount& c, int w) {
    const int x = plan.begin(w, AP_WGS);
    if (x >= plan.total) return plan.total;
    const ManyPlace p = many_find(plan, c, x);
    return p.gran <= AM_KEEP ? x - p.in : x;
}

template <int HD, int NT>
__global__ __launch_bounds__(256, 2) void attn_q8_many_kernel(PackedAttn a, PackedBatch pb) {
    using Geo = Q8Geom<HD>;
    using Steps = Q8Steps<HD>;
    constexpr int NB = Geo::NB, ND = Geo::ND;
    constexpr int ROWS = 4 * A8_TILE * NT;
    constexpr int CODES = AM_KEYS * HD;
    constexpr int BUF = 2 * CODES + 2 * AM_KEYS * (int)sizeof(Steps);
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * BUF];
    __shared__ uint32_t s_seen[PK_MAX_DRAFT / 32][ROWS];   // the drafts that a block's token sees
    __shared__ int16_t s_par[PK_MAX_DRAFT];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, j = lane & 15;
    const int G = a.Hq / a.Hkv;
    // neighbouring ranges on one XCD: blocks that share keys find them in its L2
    const int wg = (blockIdx.x % 8) * (AP_WGS / 8) + blockIdx.x / 8;
    const ManyCount count{G, a.Hkv, ROWS, a.parent == nullptr};
    const ManyPlan plan(pb, count);
    auto begin = [&](int v) { return many_begin(plan, count, v); };
    const int x0 = begin(wg), x1 = begin(wg + 1);
    if (x0 >= x1) {
        if (threadIdx.x == 0) entry_of(a.ws, wg)->rows = 0;
        return;
    }
    const float scale2 = (1.0f / sqrtf((float)HD)) * LOG2E;

    struct Piece {
        SeqView seq;
        int h, block, gran, g0, g1, last;
        const int8_t *kq, *vq;
        const _Float16 *ks, *vs;
    };
    auto piece_at = [&](int x) {
        const ManyPlace pl = many_find(plan, count, x);
        const int64_t row0 = pl.base / HD + pl.h * (a.head_stride / HD);
        return Piece{pl.seq, pl.h, pl.block, pl.gran, pl.in, min(pl.gran, pl.in + (x1 - x)),
                     count.keys(pl.seq, pl.block) - 1, a.kv8.kq + row0 * HD, a.kv8.vq + row0 * HD,
                     a.kv8.ks + row0 * NB, a.kv8.vs + row0 * NB};
    };
    Steps st;
    auto issue = [&](const Piece& p, int gr, int to) {
        const int k0 = gr * AM_KEYS;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(smem + to * BUF));
        const int8_t *kb = uniform(p.kq + (int64_t)k0 * HD), *vb = uniform(p.vq + (int64_t)k0 * HD);
        constexpr int EACH = 2 * CODES / 1024 / 4;     // a wave's copies of 1 KB
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int u = w * EACH + i;                // K's first
            const bool isv = u >= CODES / 1024;
            const int at = 64 * (isv ? u - CODES / 1024 : u) + lane, key = at / Geo::CH, c = at % Geo::CH;
            const uint32_t off = (uint32_t)min(key, p.last - k0) * HD + 16 * (c ^ swz<HD>(key & 31));
            lds_copy16(isv ? vb : kb, off, dst + 1024 * u);
        }
        // waves 0 and 1 carry the steps of a K and a V row per lane
        const int64_t r = min(k0 + lane, p.last);
        if (w < 2) st = *(const Steps*)((w == 0 ? p.ks : p.vs) + r * NB);
    };

    Piece pc = piece_at(x0);
    int to = 0;
    issue(pc, pc.g0, 0);
    if (w == 0)
        leave_entry(a.ws, wg, x0, pc.g0, pc.gran, begin,
                    JoinEntry{pc.seq.t0, min(ROWS, pc.seq.n * G - pc.block * ROWS), pc.block * ROWS, pc.h, 0, 0});

    for (int x = x0;;) {
        const SeqView sv = pc.seq;
        const int h = pc.h, r0 = pc.block * ROWS, rows = min(ROWS, sv.n * G - r0);
        const int rw = A8_TILE * NT * w;               // the wave's first row in the block
        const int tok0 = r0 / G;
        Q8Rows<HD, NT> R;
        int tok[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = rw + A8_TILE * i + j;
            const bool live = r < rows;
            tok[i] = live ? (r0 + r) / G : -1;
            R.start(i, a.q + ((int64_t)(sv.t0 + (live ? tok[i] : 0)) * a.Hq + h * G + (live ? (r0 + r) % G : 0)) * HD,
                    live, scale2);
        }
        // keys below `open` are seen by all of the wave's rows, from `end` on by none
        const int first = (r0 + min(rw, rows - 1)) / G, lastr = (r0 + min(rw + A8_TILE * NT, rows) - 1) / G;
        const int open = a.parent ? sv.p0 : sv.p0 + first + 1;
        const int end = rw >= rows ? 0 : a.parent ? sv.p0 + sv.n : sv.p0 + lastr + 1;
        const int words = (sv.n + 31) / 32;
        if (a.parent && pc.g1 * AM_KEYS > sv.p0) {     // the block's tokens' ancestors
            __syncthreads();
            for (int i = threadIdx.x; i < sv.n; i += 256) {
                const int up = a.parent[sv.t0 + i];
                s_par[i] = (int16_t)(up >= 0 && up < i ? up : -1);
            }
            __syncthreads();
            const int ntok = (r0 + rows - 1) / G - tok0 + 1;
            if ((int)threadIdx.x < ntok) {
                int cur = tok0 + threadIdx.x;
                for (int wd = words - 1; wd >= 0; --wd) {
                    uint32_t bits = 0;
                    while (cur >= 32 * wd) {
                        bits |= 1u << (cur & 31);
                        cur = s_par[cur];
                    }
                    s_seen[wd][threadIdx.x] = bits;
                }
            }
            __syncthreads();
        }
        const int xn = x + pc.g1 - pc.g0;
        const bool more = xn < x1, whole = pc.g0 == 0 && pc.g1 == pc.gran;
        const int g0 = pc.g0, g1 = pc.g1;
        for (int gr = g0; gr < g1; ++gr) {
            unsigned char* buf = smem + to * BUF;
            Steps* steps = (Steps*)(buf + 2 * CODES);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (w < 2) steps[w * AM_KEYS + lane] = st;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __syncthreads();                           // the rows are there; the other buffer is read through
            to ^= 1;
            if (gr + 1 < g1) {
                issue(pc, gr + 1, to);
            } else if (more) {
                pc = piece_at(xn);
                issue(pc, pc.g0, to);
            }
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
                const int k0 = gr * AM_KEYS + A8_KEYS * hf;
                if (k0 >= end) break;
                const unsigned char *kc = buf + A8_KEYS * HD * hf, *vc = kc + CODES;
                const Steps *ks = steps + A8_KEYS * hf, *vs = ks + AM_KEYS;
                uint32_t seen[NT];
                if (k0 + A8_KEYS <= open) {
                    R.template keys32<false>(kc, vc, ks, vs, seen);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    seen[i] = 0;
                    if (tok[i] < 0) continue;
                    if (!a.parent) {
                        const int n = min(32, max(0, sv.p0 + tok[i] + 1 - k0));
                        seen[i] = n == 32 ? 0xffffffffu : (1u << n) - 1;
                    } else {
                        const int d = k0 - sv.p0, wd = d >> 5;
                        const uint32_t lo = wd < 0 ? 0xffffffffu : wd < words ? s_seen[wd][tok[i] - tok0] : 0;
                        const uint32_t hi =
                            wd + 1 < 0 ? 0xffffffffu : wd + 1 < words ? s_seen[wd + 1][tok[i] - tok0] : 0;
                        seen[i] = (uint32_t)(((uint64_t)hi << 32 | lo) >> (d & 31));
                    }
                }
                R.template keys32<true>(kc, vc, ks, vs, seen);
            }
        }
        float* slot = slot_of(a.ws, 2 * wg + (x == x0 ? 0 : 1), ROWS, HD);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = rw + A8_TILE * i + j;
            const float back = R.back(i), l = R.sum(i);
            if (r >= rows) continue;
            if (whole) {
                float* op = a.out + ((int64_t)(sv.t0 + tok[i]) * a.Hq + h * G + (r0 + r) % G) * HD + 4 * g;
                const float inv = back / l;
#pragma unroll
                for (int n = 0; n < ND; ++n) *(float4u*)(op + 16 * n) = R.o[i][n] * inv;
            } else {
                if (g == 0) *(float2*)(slot + ROWS * HD + 2 * r) = make_float2(R.m[i], l);
#pragma unroll
                for (int n = 0; n < ND; ++n) *(floatx4*)(slot + r * HD + 16 * n + 4 * g) = R.o[i][n] * back;
            }
        }
        if (!more) break;
        x = xn;
    }
}

// ---------------------------------------------------------------------------
bool attention_q8_shape(int hd) { return hd == 32 || hd == 64 || hd == 128; }
int64_t attention_q8_bytes(int hd) { return plan_bytes(8 * A8_TILE, hd); }

template <int HD>
static void launch_q8_hd(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    const int64_t rows = (int64_t)pb.max_new * (a.Hq / a.Hkv);
    const dim3 grid(AP_WGS), block(256);
    if (rows <= A8_TILE) {
        hipLaunchKernelGGL((attn_q8_few_kernel<HD, 1>), grid, block, 0, s, a, pb);
        if (few_granules(pb.max_seq) > AF_KEEP)        // else no block is cut
            launch_attn_join(a.out, a.ws, a.Hq, a.Hkv, HD, A8_TILE, s);
        return;
    }
    hipLaunchKernelGGL((attn_q8_many_kernel<HD, 1>), grid, block, 0, s, a, pb);
    if (pb.max_seq > AM_KEEP * AM_KEYS) launch_attn_join(a.out, a.ws, a.Hq, a.Hkv, HD, 4 * A8_TILE, s);
}

int launch_attention_q8(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    if (a.hd == 128)
        launch_q8_hd<128>(a, pb, s);
    else if (a.hd == 64)
        launch_q8_hd<64>(a, pb, s);
    else
        launch_q8_hd<32>(a, pb, s);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
