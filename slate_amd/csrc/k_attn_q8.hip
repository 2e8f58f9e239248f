// k_attn_q8.hip -- attention over the 8-bit cache for few query rows per
// (sequence, kv head): a decode step's tokens times the query heads of a kv
// head, trees of up to 48 rows.  The arithmetic: attn_q8.h, how the keys are
// shared out: attn_plan.h.
//
// A workgroup takes a block of 16 rows over a range of keys, each of its four
// waves every fourth 32 of them.
// Memory bound: 2.125 bytes per key and element against two f16 MFMAs and about
// 400 VALU operations per 32 keys and wave.  So the design is about loads:
// each wave copies its next 32 keys' rows straight into LDS (16 bytes per
// lane, no registers) while it works on the last 32, with no barrier until
// its range ends; 70 KB are on their way per CU.  Head_dim 128, 8 kv heads of
// 4 query heads: decode of 64 users over 1.33 GB in 245 us (5.4 TB/s), of 16
// users over 79 MB in 27.5 us (its loads alone take 22, plan and join the
// rest), trees of 4 to 8 drafts (up to two blocks, the keys read again for the
// second) of 16 users 43.4 us.
#include "attn_plan.h"
#include "attn_q8.h"

namespace slate_hip {

constexpr int AF_WGS = 512;            // two workgroups per CU (LDS)
constexpr int AF_GRAN = 4 * AR_KEYS;   // keys of a granule
constexpr int AF_KEEP = 4;             // blocks of up to this many granules are not cut

__host__ __device__ constexpr int few_granules(int keys) { return (keys + AF_GRAN - 1) / AF_GRAN; }
static_assert(few_granules(PK_MAX_KEYS) == (1 << 24) - 8 && AF_GRAN <= 128, "a count of keys passes 32 bits");

// Granules of a sequence: blocks of 16 rows, of each kv head.
struct FewCount {
    int G, Hkv;
    __device__ __forceinline__ int blocks(const SeqView& s) const { return (s.n * G + AR_TILE - 1) / AR_TILE; }
    __device__ __forceinline__ int operator()(const SeqView& s) const {
        return s.n < 1 ? 0 : Hkv * blocks(s) * few_granules(s.p0 + s.n);
    }
};
using FewPlan = Plan<FewCount>;

// Where workgroup w's range begins: N w / P, or the start of the block there
// if it is short (it is not cut: the last workgroup that would begin in it
// takes it whole).
__device__ __forceinline__ int few_begin(const FewPlan& plan, int w) {
    const int x = plan.begin(w, AF_WGS);
    if (x >= plan.total) return plan.total;
    const Place pl = plan.find(x);
    const int gran = few_granules(pl.seq.p0 + pl.seq.n), in = pl.at % gran;
    return gran <= AF_KEEP ? x - in : x;
}

template <int HD>
__global__ __launch_bounds__(256, 2) void attn_q8_few_kernel(PackedAttn a, PackedBatch pb) {
    using Geo = Q8Geom<HD>;
    using Steps = Q8Steps<HD>;
    constexpr int NB = Geo::NB, ND = Geo::ND;
    constexpr int CODES = AR_KEYS * HD;                // bytes of a wave's K (or V) codes
    constexpr int OS = HD + 4;                         // row stride of a wave's results in LDS (floats)
    constexpr int USED = 2 * CODES + 2 * AR_KEYS * (int)sizeof(Steps);
    constexpr int BUF = USED > AR_TILE * OS * 4 ? USED : AR_TILE * OS * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[8 * BUF];
    __shared__ float s_m[4][AR_TILE], s_l[4][AR_TILE];
    __shared__ int s_at[4];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, j = lane & 15;
    const int G = a.Hq / a.Hkv;
    const FewCount count{G, a.Hkv};
    const FewPlan plan(pb, count);
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
        int h, r0, gran, g0, g1;       // kv head, first row of the block
        const int8_t *kq, *vq;
        const _Float16 *ks, *vs;
    };
    auto piece_at = [&](int x) {
        const Place pl = plan.find(x);
        Piece p;
        p.seq = pl.seq;
        p.gran = few_granules(pl.seq.p0 + pl.seq.n);
        const int nb = count.blocks(pl.seq), b = pl.at / p.gran;
        p.h = b / nb;
        p.r0 = AR_TILE * (b % nb);
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
    auto key0 = [&](int gr) { return gr * AF_GRAN + w * AR_KEYS; };
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
    // q of row j, elements 32t + 8g .. +7
    float4u qraw[NB][2];
    auto load_q = [&](const Piece& p) {
        const int r = p.r0 + j;
        const bool live = r < p.seq.n * G;
        const float* qp =
            a.q + ((int64_t)(p.seq.t0 + (live ? r / G : 0)) * a.Hq + p.h * G + (live ? r % G : 0)) * HD + 8 * g;
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
        leave_entry(a.ws, AF_WGS, blockIdx.x, x0, pc.g0, pc.gran, plan, [&](int v) { return few_begin(plan, v); },
                    JoinEntry{pc.seq.t0, min(AR_TILE, pc.seq.n * G - pc.r0), pc.r0, pc.h, 0, 0});

    for (int x = x0;;) {
        const SeqView sv = pc.seq;
        const int keys = sv.p0 + sv.n, h = pc.h, r0 = pc.r0, rows = min(AR_TILE, sv.n * G - r0);
        const int tok = (r0 + j) / G;
        const bool live = j < rows;
        Q8Rows<HD> R;
        R.start(qraw, live, scale2);
        // the drafts that row j's token sees (n <= 32): itself and, causal,
        // all before it, or its ancestors
        uint32_t drafts = (2u << min(tok, 31)) - 1;
        if (a.parent) {
            const int par = a.parent[sv.t0 + min(lane, sv.n - 1)];
            drafts = 0;
            int cur = live ? tok : -1;
            while (__builtin_amdgcn_ballot_w64(cur >= 0)) {
                const int up = __shfl(par, max(cur, 0));
                if (cur >= 0) drafts |= 1u << cur;
                cur = up >= 0 && up < cur ? up : -1;
            }
        }
        if (!live) drafts = 0;

        for (int gr = pc.g0; gr < pc.g1; ++gr) {
            const int k0 = key0(gr);
            if (k0 >= keys) break;                     // only in the last granule
            unsigned char* buf = buf0 + to * BUF;
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            Steps* steps = (Steps*)(buf + 2 * CODES);
            steps[lane] = st;
            to ^= 1;
            if (gr + 1 < pc.g1) issue(pc, gr + 1, to);
            if (k0 + AR_KEYS <= sv.p0)
                R.template keys32<false>(buf, buf + CODES, steps, steps + AR_KEYS, 0);
            else                                       // drafts among the keys, or past the last one
                R.template keys32<true>(buf, buf + CODES, steps, steps + AR_KEYS, seen_keys(drafts, k0, sv.p0));
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
        float* slot = slot_of(a.ws, AF_WGS, 2 * blockIdx.x + (x == x0 ? 0 : 1), AR_TILE, HD);
        float* mine = (float*)(buf0 + (to ^ 1) * BUF);
        const float back = R.back(), l = R.sum();
        if (g == 0) {
            s_m[w][j] = R.m;
            s_l[w][j] = l;
            s_at[w] = (int)((unsigned char*)mine - smem);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) *(floatx4*)(mine + j * OS + 16 * n + 4 * g) = R.o[n] * back;
        __syncthreads();
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
                const int row = r0 + r;
                *(float4u*)(a.out + ((int64_t)(sv.t0 + row / G) * a.Hq + h * G + row % G) * HD + c) = sum * inv;
            } else {
                *(floatx4*)(slot + r * HD + c) = sum;
                if (c == 0) *(float2*)(slot + AR_TILE * HD + 2 * r) = make_float2(mt, lt);
            }
        }
        if (!more) break;
        __syncthreads();                               // before these rows' places are copied over
        x = xn;
    }
}

// ---------------------------------------------------------------------------
int64_t attention_q8_few_bytes(int hd) { return plan_bytes(AF_WGS, AR_TILE, hd); }
// Blocks of 16 rows read the keys again for every block, but without a
// barrier.  us here and in the many-row kernel (head_dim 128, 4 query heads a kv
// head, trees of max_new drafts each, in brackets of half as many to max_new):
// 16 sequences of up to 4096: 32 rows 49 and 58, 48 rows 64 and 64 (55 and 62),
// 64 rows 81 and 72 (69 and 69), 80 rows 93 and 77 (78 and 76); 64 sequences of up
// to 2000: 32 rows 84 and 111, 48 rows 128 and 126 (108 and 121), 64 rows 148 and
// 127 (121 and 123); head_dim 64: 48 rows 42 and 45, 64 rows 51 and 49.  One
// sequence of 16384 goes faster there at any number of rows but 64 (20 rows 32
// and 31, 48 rows 40 and 34): the rule, which knows a bound on the rows and no
// lengths, leaves that.  A row's drafts are kept in 32 bits.
constexpr int AF_MAX_ROWS = 48, AF_MAX_NEW = 32;
bool attention_q8_few_takes(const PackedAttn& a, const PackedBatch& pb) {
    return !a.kf && (a.hd == 32 || a.hd == 64 || a.hd == 128) && pb.max_new <= AF_MAX_NEW &&
           pb.max_new * (int64_t)(a.Hq / a.Hkv) <= AF_MAX_ROWS;
}
double attention_q8_few_most(const PackedAttn& a, const PackedBatch& pb) {
    return a.Hkv * ((double)pb.T * (a.Hq / a.Hkv) / AR_TILE + pb.B) * few_granules(pb.max_seq);
}

template <int HD>
static void launch_few(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    hipLaunchKernelGGL(attn_q8_few_kernel<HD>, dim3(AF_WGS), dim3(256), 0, s, a, pb);
    if (few_granules(pb.max_seq) > AF_KEEP)            // else no block is cut
        launch_attn_join(a.out, a.ws, a.Hq, a.Hkv, HD, AR_TILE, AF_WGS, s);
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
