// k_verify.hip -- which drafted tokens stand, and the token after them.
//
// A draft x with probability q(x) stands where u q(x) < p(x), so it is kept with
// probability min(1, p / q); one that is turned down leaves max(p - q, 0) to the
// next token, and the tokens come out distributed as p (the drafts without
// probabilities: q is 1 on x, the rest of p is divided by what is left of it).
//
// Every logit is read once (softmax sums of all rows at once, a wave per 1024
// logits), then a workgroup per sequence walks its drafts; where a draft was turned
// down by its probability, the rows p and q of that place are read once more.
// Bound by the bytes of the logits, beside an exponential in 64 bits for each: the
// next token is found among sums of up to V terms, and its borders are as near to each
// other as the least likely token is unlikely, so 32 bits would pick a neighbour now
// and then (1e-7 of the whole against 1e-5 for one of 1e5 tokens).
#include "lanes.h"
#include "paged.h"

namespace slate_hip {

constexpr int VF_CHUNK = 1024;         // logits of a wave: 16 a lane
constexpr int VF_TH = 512;             // threads that walk a sequence
// Workgroups of the sums: five waves a SIMD.  254 rows of 128256 logits take 31 to 34 us
// (130 MB, 4 TB/s; 27.5 with no exponentials); where they took 34.4, four waves took 35.8,
// six 38 and eight 47, which leave the compiler fewer registers.
constexpr int VF_SUM_WGS = 1280;
constexpr int VF_ROWS = PK_MAX_DRAFT + 1;

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// 2^t for t < 1000, to 2^-42 of itself: e^(f ln 2) for the part f of t behind the
// point, |f ln 2| <= 0.347, by its series up to the tenth power.
__device__ __forceinline__ double pow2(double t) {
    t = fmax(t, -1100.0);
    const double n = rint(t), f = (t - n) * 0.69314718055994530942;
    double e = 1.0 / 3628800;
    e = fma(e, f, 1.0 / 362880);
    e = fma(e, f, 1.0 / 40320);
    e = fma(e, f, 1.0 / 5040);
    e = fma(e, f, 1.0 / 720);
    e = fma(e, f, 1.0 / 120);
    e = fma(e, f, 1.0 / 24);
    e = fma(e, f, 1.0 / 6);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return ldexp(e, (int)n);
}

// Weight of logit x beside `top`, the largest one or (where all weights fit beside
// it) 0: e^((x - top) / temperature), by = log2(e) / temperature.  0 for -infinity;
// infinite logits share all.
__device__ __forceinline__ double weight(float x, float top, double by) {
    double w = pow2(((double)x - (double)top) * by);   // selects: branches would keep several from overlapping
    w = top == INFINITY || !(x > -INFINITY) ? 0.0 : w;
    return x == top && top > -INFINITY ? 1.0 : w;
}

// The same beside 0 instead of the largest logit, for sums over whole rows: 64 bits hold
// 2^512 as they hold 1.  2^(k / 64 + r / 64), |r| <= 1/2, is 2^(k / 64) from a table (entry
// k % 64 in lane k % 64) times the series of e^(r ln 2 / 64) up to the fourth power, to
// 2^-44 of itself; 13 operations.
class Weights {
  public:
    __device__ __forceinline__ Weights() {
        const int lane = threadIdx.x & 63;
        const uint64_t u = __builtin_bit_cast(uint64_t, exp2(lane * (1.0 / 64)));
        lo_ = (uint32_t)u;
        hi_ = (uint32_t)(u >> 32) - ((uint32_t)lane << 14);    // k << 14 is k / 64 in the exponent, and this
    }
    __device__ __forceinline__ void start(double by) {
        by_ = 64 * by;
        low_ = (float)(-900 / by);
        most_ = (float)(512 / by);
    }
    // Whether a wave's values can be taken so, `top` being the largest that the lane
    // has: none above 2^512 and one above 2^-512, so that what counts as 2^-900
    // below shows in no sum (infinities, NaN, temperatures without an end: no).
    __device__ __forceinline__ bool takes(float top) const {
        return most_ < 1e38f && most_ > 1e-30f && !__builtin_amdgcn_ballot_w64(top > most_) &&
               __builtin_amdgcn_ballot_w64(top > -most_);
    }
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double WHOLE = 6755399441055744.0;   // 1.5 2^52: a sum with it is a whole number in its low bits
        constexpr double L = 0.69314718055994530942 / 64;
        const double d = (double)fmaxf(x, low_);       // NaN counts as the least
        const double kd = fma(d, by_, WHOLE), r = fma(d, by_, WHOLE - kd);
        const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, kd);
        const uint32_t lo = __builtin_amdgcn_ds_bpermute((int)(4 * k), (int)lo_);
        const uint32_t hi = __builtin_amdgcn_ds_bpermute((int)(4 * k), (int)hi_) + (k << 14);
        const double t = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
        const double e = r * fma(r, fma(r, fma(r, L * L * L * L / 24, L * L * L / 6), L * L / 2), L);
        return fma(t, e, t);
    }

  private:
    uint32_t lo_, hi_;
    double by_ = 0;
    float low_ = 0, most_ = INFINITY;
};

struct alignas(16) Part {
    float top;                         // the largest logit, or 0 (Weights); -infinity: no p
    int best;                          // its first place (greedy rows)
    double sum;                        // of the weights beside top
};

// The temperature's inverse times log2(e); 0 stands for greedy here.
struct Heat {
    bool greedy;
    double by;
};
__device__ __forceinline__ Heat heat_of(const float* temperature, int b) {
    const float t = temperature ? temperature[b] : 1.0f;
    return Heat{!(t > 0), t > 0 ? 1.4426950408889634074 / (double)t : 0.0};
}

// A wave's 16 values a lane of chunk c: x[4k + e] is element 256 k + 4 lane + e of
// it, whole lines at a time; `none` behind V.
__device__ __forceinline__ int place(int c, int i) {
    return c * VF_CHUNK + 256 * (i / 4) + 4 * (int)(threadIdx.x & 63) + i % 4;
}
__device__ __forceinline__ void load16(const float* z, int c, int V, float none, float* x) {
    if (V - c * VF_CHUNK >= VF_CHUNK) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4u v = *(const float4u*)(z + place(c, 4 * k));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * k + e] = v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int at = place(c, i);
            x[i] = at < V ? z[at] : none;
        }
    }
}
// Four elements in a row.
__device__ __forceinline__ void load4(const float* z, int at, int V, float none, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = at < V - i ? z[at + i] : none;
}

// Inclusive sum over the wave's lanes (DPP: within rows of 16, then across).
__device__ __forceinline__ double wave_scan_f64(double v) {
#define VF_SCAN_STEP(ctrl, rows)                                                                               \
    {                                                                                                          \
        const uint64_t u = __builtin_bit_cast(uint64_t, v);                                                    \
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, ctrl, rows, 0xF, false);          \
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), ctrl, rows, 0xF, false);            \
        v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                                              \
    }
    VF_SCAN_STEP(0x111, 0xF)           // row_shr:1, 2, 4, 8
    VF_SCAN_STEP(0x112, 0xF)
    VF_SCAN_STEP(0x114, 0xF)
    VF_SCAN_STEP(0x118, 0xF)
    VF_SCAN_STEP(0x142, 0xA)           // row_bcast:15 into rows 1 and 3
    VF_SCAN_STEP(0x143, 0xC)           // row_bcast:31 into rows 2 and 3
#undef VF_SCAN_STEP
    return v;
}
__device__ __forceinline__ double last_lane(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = __builtin_amdgcn_readlane((int)(u >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) { return last_lane(wave_scan_f64(v)); }
__device__ __forceinline__ int wave_min_int(int v) {
    v = min(v, __builtin_amdgcn_update_dpp(0, v, DPP_QUAD_XOR1, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, DPP_QUAD_XOR2, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, DPP_ROW_HALF_MIRROR, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, DPP_ROW_MIRROR, 0xF, 0xF, false));
    return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

__host__ __device__ constexpr int chunks_of(int V) { return (V - 1) / VF_CHUNK + 1; }

// Workspace: a Part per row and chunk, a mass per sequence and chunk, a Next per sequence.
struct Next {
    int row, turned, at;               // the row whose p it is, the draft's row (-1: nothing to do), where it goes
    float top;
    double sum;                        // of the row's weights
    int done, pad;                     // workgroups that have left their chunks' masses
};
struct Space {
    Part* part;
    double* mass;
    Next* next;
};
__host__ __device__ inline Space space_of(const VerifyArgs& a) {
    const int64_t nch = chunks_of(a.V);
    Part* part = (Part*)a.ws;
    double* mass = (double*)(part + a.T * nch);
    return Space{part, mass, (Next*)(mass + a.B * nch)};
}
int64_t verify_drafts_bytes(int B, int T, int V) {
    const int64_t nch = chunks_of(V);
    return T * nch * (int64_t)sizeof(Part) + B * nch * (int64_t)sizeof(double) + B * (int64_t)sizeof(Next);
}

// The weights of a lane's 16 logits, four at a time (in few instructions: what runs
// once takes as long as it is fetched).
__device__ __forceinline__ double weights_of(float* x, float top, double by) {
    double s = 0;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        s += (weight(x[0], top, by) + weight(x[1], top, by)) + (weight(x[2], top, by) + weight(x[3], top, by));
#pragma unroll
        for (int k = 0; k < 12; ++k) x[k] = x[k + 4];
    }
    return s;
}

// Softmax sums (greedy rows: the largest logit) of all rows, a wave per chunk of a
// stretch of rows, the next row's logits under way while it works on the last.
__global__ __launch_bounds__(256, 5) void verify_sums_kernel(VerifyArgs a) {
    const int lane = threadIdx.x & 63, nch = chunks_of(a.V);
    const int c = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (c >= nch) return;
    const int r0 = (int)((int64_t)a.T * blockIdx.y / gridDim.y), r1 = (int)((int64_t)a.T * (blockIdx.y + 1) / gridDim.y);
    const Space sp = space_of(a);
    float next[16];
    load16(a.logits + (int64_t)r0 * a.ld, c, a.V, -INFINITY, next);
    // the first row's sequence, for its temperature (a row that belongs to none has some)
    int b = 0;
    if (a.temperature)
        for (int b0 = 0; b0 < a.B; b0 += 64) {
            const int i = b0 + lane;
            uint64_t begun = __builtin_amdgcn_ballot_w64(i < a.B && a.tok_off[i] <= r0);
            const uint64_t falls = __builtin_amdgcn_ballot_w64(i < a.B && a.tok_off[i + 1] < a.tok_off[i]);
            if (falls) begun &= (falls & -falls) - 1;
            b += __popcll(begun);
            if (falls) break;
        }
    b = max(0, b - 1);
    Heat heat = heat_of(a.temperature, b);
    Weights weights;
    if (!heat.greedy) weights.start(heat.by);
    for (int t = r0; t < r1; ++t) {
        float x[16], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = next[i];
            top = fmaxf(top, x[i]);                    // (not NaN)
        }
        if (t + 1 < r1) load16(a.logits + (int64_t)(t + 1) * a.ld, c, a.V, -INFINITY, next);
        // (behind a fall of tok_off no row's sums are looked at)
        if (a.temperature && b + 1 < a.B && a.tok_off[b + 1] <= t) {
            while (b + 1 < a.B && a.tok_off[b + 1] <= t) ++b;
            heat = heat_of(a.temperature, b);
            if (!heat.greedy) weights.start(heat.by);
        }
        Part p{0.f, -1, 0};
        if (!heat.greedy && weights.takes(top)) {
            double s = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += weights(x[i]);
            p.sum = wave_sum_f64(s);
        } else {
            p.top = top = wave_max(top);
            if (heat.greedy) {
                int at = INT32_MAX;
#pragma unroll
                for (int i = 15; i >= 0; --i)
                    if (x[i] == top) at = place(c, i);
                p.best = wave_min_int(at);
            } else {
                p.sum = wave_sum_f64(weights_of(x, top, heat.by));
            }
        }
        if (lane == 0) sp.part[(int64_t)t * nch + c] = p;
    }
}

// A row's parts joined by a wave.
__device__ __forceinline__ Part row_part(const Part* part, int nch, const Heat& heat) {
    const int lane = threadIdx.x & 63;
    Part p{-INFINITY, INT32_MAX, 0};
    for (int c = lane; c < nch; c += 64) {
        const Part o = part[c];
        if (!(o.top > -INFINITY)) continue;
        if (o.top > p.top) {
            p.sum = p.sum * weight(p.top, o.top, heat.by) + o.sum;
            p.top = o.top;
            p.best = o.best;
        } else {
            p.sum += o.sum * weight(o.top, p.top, heat.by);
        }
    }
    const float top = wave_max(p.top);
    p.sum = wave_sum_f64(p.sum * weight(p.top, top, heat.by));
    p.best = top > -INFINITY ? wave_min_int(p.top == top ? p.best : INT32_MAX) : -1;
    p.top = top;
    return p;
}

// Inclusive sum over the workgroup in thread order, and the whole.
struct Sums {
    double upto, total;
};
template <int TH>
__device__ __forceinline__ Sums block_sums(double v, double* s_part) {
    const int w = threadIdx.x >> 6;
    v = wave_scan_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s_part[w] = v;
    __syncthreads();
    double before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) {
        before += i < w ? s_part[i] : 0;
        total += s_part[i];
    }
    return Sums{before + v, total};
}

// The first thread of the workgroup that says `is`, or (none) the last that says
// `some`; -1 if none does.  By ballots: that many atomics on one place of LDS take
// 4 us.
template <int TH>
__device__ __forceinline__ int first_or_last(bool is, bool some, int* s_first, int* s_last) {
    const int w = threadIdx.x >> 6;
    const uint64_t a = __builtin_amdgcn_ballot_w64(is), b = __builtin_amdgcn_ballot_w64(some);
    if ((threadIdx.x & 63) == 0) {
        s_first[w] = a ? 64 * w + __builtin_ctzll(a) : -1;
        s_last[w] = b ? 64 * w + 63 - __builtin_clzll(b) : -1;
    }
    __syncthreads();
    int first = -1, last = -1;
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) {
        first = first < 0 ? s_first[i] : first;
        last = max(last, s_last[i]);
    }
    return first >= 0 ? first : last < 0 ? -1 : last + TH;     // TH and more: of the last kind
}

// The token at which the sums of the chunks' masses pass u times the whole: mass(c)
// is a chunk's, values(at, m) are those of the tokens at .. at + 3.  -1 where there is
// no mass.  Called by a workgroup of TH threads.
template <int TH, class Mass, class Values>
__device__ int pick_token(int nch, float u, const Mass& mass, const Values& values, double* s_part) {
    static_assert(TH >= VF_CHUNK / 4, "four tokens a thread");
    __shared__ int s_first[TH / 64], s_last[TH / 64], s_pick;
    __shared__ double s_before;
    // up to a chunk a thread: one round of sums
    const bool one = nch <= TH;
    double own = (int)threadIdx.x < nch ? mass(threadIdx.x) : 0;
    Sums s = block_sums<TH>(own, s_part);
    double total = s.total;
    for (int c0 = TH; c0 < nch; c0 += TH) {
        const int c = c0 + threadIdx.x;
        total += block_sums<TH>(c < nch ? mass(c) : 0, s_part).total;
    }
    const double at = total * (double)u;
    double before = 0;
    int chunk = -1;
    for (int c0 = 0; c0 < nch; c0 += TH) {
        if (!one) {
            own = c0 + (int)threadIdx.x < nch ? mass(c0 + threadIdx.x) : 0;
            s = block_sums<TH>(own, s_part);
        }
        const int who = first_or_last<TH>(own > 0 && before + s.upto > at, own > 0, s_first, s_last);
        if (who >= 0) {                                // of the last kind: while none of the first follows
            chunk = c0 + who % TH;
            if ((int)threadIdx.x == who % TH) s_before = before + (s.upto - own);
            if (who < TH) break;
        }
        before += s.total;
        __syncthreads();                               // before the next round's numbers
    }
    if (chunk < 0) return -1;
    const int first = chunk * VF_CHUNK + 4 * (int)threadIdx.x;
    double m[4] = {0, 0, 0, 0};
    if (threadIdx.x < VF_CHUNK / 4) values(first, m);
    own = (m[0] + m[1]) + (m[2] + m[3]);
    s = block_sums<TH>(own, s_part);                   // its barriers: s_before is there, s_first is read
    double run = s_before + (s.upto - own);
    int here = -1, last = -1;                          // the thread's first that passes `at`, its last one
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        run += m[i];
        if (m[i] > 0) {
            last = first + i;
            if (here < 0 && run > at) here = last;
        }
    }
    const int who = first_or_last<TH>(here >= 0, last >= 0, s_first, s_last);
    if (who >= 0 && (int)threadIdx.x == who % TH) s_pick = who < TH ? here : last;
    __syncthreads();
    return who < 0 ? -1 : s_pick;
}

// One workgroup per sequence: its rows' sums joined, its drafts' chances, the walk,
// and the next token where no draft's probability has to be taken off.  Latency: 4.4 us
// for one sequence, 8.4 for 64 of four drafts, 10.5 for 16 trees of eight, whose
// tokens turned down have a chunk each summed again.
__global__ __launch_bounds__(VF_TH) void verify_walk_kernel(VerifyArgs a) {
    __shared__ double s_sum[VF_ROWS], s_p[VF_ROWS], s_u[VF_ROWS];
    __shared__ float s_top[VF_ROWS], s_z[VF_ROWS];
    __shared__ int s_best[VF_ROWS], s_parent[VF_ROWS], s_tok[VF_ROWS];
    __shared__ double s_part[VF_TH / 64], s_mass[VF_TH];
    __shared__ int s_node, s_acc, s_turned, s_n_out;
    int* const s_out = (int*)s_z;                      // the node's tokens that were turned down, once s_z was read
    const int b = blockIdx.x, lane = threadIdx.x & 63, V = a.V, nch = chunks_of(V);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Space sp = space_of(a);
    const int t0 = a.tok_off[b], t1 = a.tok_off[b + 1];
    bool falls = false;                                // before this sequence: its rows' sums may be another's
    for (int i = threadIdx.x; i < b; i += VF_TH) falls |= a.tok_off[i + 1] < a.tok_off[i];
    if (__syncthreads_or(falls) || t0 < 0 || t1 > a.T || t1 <= t0 || t1 - t0 > VF_ROWS) {
        if (threadIdx.x == 0) {
            a.n_accepted[b] = -1;
            sp.next[b].turned = -1;
        }
        return;
    }
    const int n = t1 - t0;
    const Heat heat = heat_of(a.temperature, b);
    const float u_next = a.u_next[b];
    // the drafts' numbers by the first waves, the rows' sums from the last wave on: side by side for few rows
    for (int i = threadIdx.x; i < n; i += VF_TH) {
        const int x = a.token[t0 + i];
        int up = a.parent ? a.parent[t0 + i] : i - 1;
        up = up >= 0 && up < i ? up : -1;
        s_tok[i] = x;
        s_parent[i] = up;
        const bool in = up >= 0 && x >= 0 && x < V;
        s_z[i] = in ? a.logits[(int64_t)(t0 + up) * a.ld + x] : -INFINITY;
        const double q = in && a.q ? (double)a.q[(int64_t)(t0 + i) * a.q_ld + x] : 1.0;
        s_u[i] = in ? a.u[t0 + i] * q : INFINITY;      // infinite: never
    }
    for (int i = VF_TH / 64 - 1 - w; i < n; i += VF_TH / 64) {
        const Part p = row_part(sp.part + (int64_t)(t0 + i) * nch, nch, heat);
        if (lane == 0) {
            s_sum[i] = p.sum;
            s_top[i] = p.top;
            s_best[i] = p.best;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += VF_TH) {
        const int up = s_parent[i], x = s_tok[i];
        const bool in = x >= 0 && x < V;
        double p = 0;
        if (up >= 0 && in) {
            // a token that an earlier child of the same row has was turned down before this one is tried
            bool again = false;
            if (a.parent)
                for (int j = up + 1; j < i; ++j) again |= s_parent[j] == up && s_tok[j] == x;
            if (heat.greedy)
                p = s_best[up] == x;
            else if (!again && s_sum[up] > 0)
                p = weight(s_z[i], s_top[up], heat.by) / s_sum[up];
            if (heat.greedy) s_u[i] = 0.5;
        }
        s_p[i] = p;
    }
    __syncthreads();
    if (w == 0) {
        // drafts in order, 64 at a time: a row's children lie behind it
        int node = 0, acc = 0, turned = -1, n_out = 0;
        double rest = 1;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int i = i0 + lane, up = i < n && i > 0 ? s_parent[i] : -1;
            uint64_t left = __builtin_amdgcn_ballot_w64(up == node);
            while (left) {
                const int l = __builtin_ctzll(left), c = i0 + l;
                const double p = s_p[c], u = s_u[c];
                if (u * (a.q || heat.greedy ? 1.0 : rest) < p) {
                    if (lane == 0) {
                        a.out_tok[t0 + acc] = s_tok[c];
                        if (a.out_row) a.out_row[t0 + acc] = c;
                    }
                    ++acc;
                    node = c;
                    rest = 1;
                    turned = -1;
                    n_out = 0;
                    left = __builtin_amdgcn_ballot_w64(up == node) & ~((2ull << l) - 1);
                } else {
                    rest -= p;
                    turned = c;
                    if (p > 0) {                       // (a token outside the vocabulary or a second time: no p)
                        if (lane == 0) s_out[n_out] = s_tok[c];
                        ++n_out;
                    }
                    left &= left - 1;
                }
            }
        }
        if (lane == 0) {
            s_node = node;
            s_acc = acc;
            s_turned = turned;
            s_n_out = n_out;
            a.n_accepted[b] = acc;
        }
    }
    __syncthreads();
    const int node = s_node, acc = s_acc, turned = s_turned;
    for (int i = acc + threadIdx.x; i < n; i += VF_TH) {
        if (i > acc) a.out_tok[t0 + i] = -1;
        if (a.out_row) a.out_row[t0 + i] = -1;
    }
    const bool less = a.q && turned >= 0 && !heat.greedy && s_sum[node] > 0;
    if (threadIdx.x == 0)
        sp.next[b] = Next{t0 + node, less ? t0 + turned : -1, t0 + acc, s_top[node], s_sum[node], 0, 0};
    if (less) return;                                  // the next kernels'
    if (heat.greedy || !(s_top[node] > -INFINITY)) {
        if (threadIdx.x == 0) a.out_tok[t0 + acc] = s_best[node];     // -1 where the row has no p
        return;
    }
    // p without the tokens that were turned down: their chunks are summed again
    const float* z = a.logits + (int64_t)(t0 + node) * a.ld;
    const Part* part = sp.part + (int64_t)(t0 + node) * nch;
    const float top = s_top[node];
    double* own = nch <= VF_TH ? s_mass : sp.mass + (int64_t)b * nch;
    int pick = -1;
    // the second pass, where nothing was left, is from p itself
    for (int without = !a.q && s_n_out > 0; without >= 0 && pick < 0; --without) {
        const int n_out = without ? s_n_out : 0;
        auto values = [&](int at, double* m) {
            float x[4];
            load4(z, at, V, -INFINITY, x);
            for (int k = 0; k < n_out; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (s_out[k] == at + i) x[i] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = weight(x[i], top, heat.by);
        };
        for (int c = threadIdx.x; c < nch; c += VF_TH) own[c] = part[c].sum * weight(part[c].top, top, heat.by);
        if (n_out > 0) {
            __syncthreads();
            for (int j = w; j < n_out; j += VF_TH / 64) {
                const int c = s_out[j] / VF_CHUNK;     // of two tokens in a chunk either writes the same
                float x[16];
                load16(z, c, V, -INFINITY, x);
                for (int k = 0; k < n_out; ++k)
                    if (s_out[k] / VF_CHUNK == c)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (s_out[k] == place(c, i)) x[i] = -INFINITY;
                const double s = wave_sum_f64(weights_of(x, top, heat.by));
                if (lane == 0) own[c] = s;
            }
        }
        __syncthreads();
        pick = pick_token<VF_TH>(nch, u_next, [&](int c) { return own[c]; }, values, s_part);
        __syncthreads();
    }
    if (threadIdx.x == 0) a.out_tok[t0 + acc] = pick;
}

// What p has more than q: the chunks' masses, a wave each, and by the last workgroup
// of a sequence the token.  The masses pass between workgroups of other XCDs, so they
// and the count of workgroups are written and read past the L2 (relaxed atomics of the
// device's scope; a workgroup's count follows its masses by the wait between them).
// 8 us for one sequence (latency), 13 for 64 (66 MB, 5 TB/s).
constexpr int VL_TH = 256;
__global__ __launch_bounds__(VL_TH) void verify_less_kernel(VerifyArgs a) {
    __shared__ double s_part[VL_TH / 64];
    __shared__ int s_done;
    const int nch = chunks_of(a.V), b = blockIdx.y;
    const int c = __builtin_amdgcn_readfirstlane(blockIdx.x * (VL_TH / 64) + (threadIdx.x >> 6));
    const Space sp = space_of(a);
    const Next nx = sp.next[b];
    if (nx.turned < 0) return;
    const double by = heat_of(a.temperature, b).by, share = 1.0 / nx.sum;
    const float *z = a.logits + (int64_t)nx.row * a.ld, *q = a.q + (int64_t)nx.turned * a.q_ld;
    double* own = sp.mass + (int64_t)b * nch;
    auto more = [&](double w, float y) { return fmax(fma(w, share, -(double)y), 0.0); };
    if (c < nch) {
        float x[16], y[16], top = -INFINITY;
        load16(z, c, a.V, -INFINITY, x);
        load16(q, c, a.V, INFINITY, y);
        double s = 0;
        Weights weights;
        weights.start(by);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, x[i]);
        if (nx.top == 0.f && weights.takes(top)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const double wt = weights(x[i]);       // by all lanes
                s += more(x[i] > -INFINITY ? wt : 0.0, y[i]);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
                s += more(weight(x[0], nx.top, by), y[0]);
#pragma unroll
                for (int k = 0; k < 15; ++k) {
                    x[k] = x[k + 1];
                    y[k] = y[k + 1];
                }
            }
        }
        s = wave_sum_f64(s);
        if ((threadIdx.x & 63) == 0) __hip_atomic_store(own + c, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
        s_done = __hip_atomic_fetch_add(&sp.next[b].done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_done != (int)gridDim.x - 1) return;
    const Part* part = sp.part + (int64_t)nx.row * nch;
    int pick = -1;
    for (int less = 1; less >= 0 && pick < 0; --less) {        // where p has nothing more than q: from p
        __syncthreads();
        pick = pick_token<VL_TH>(
            nch, a.u_next[b],
            [&](int i) {
                return less ? __hip_atomic_load(own + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                            : part[i].sum * weight(part[i].top, nx.top, by);
            },
            [&](int at, double* m) {
                float x[4], y[4];
                load4(z, at, a.V, -INFINITY, x);
                load4(q, at, a.V, INFINITY, y);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    m[i] = weight(x[i], nx.top, by);
                    if (less) m[i] = more(m[i], y[i]);
                }
            },
            s_part);
    }
    if (threadIdx.x == 0) a.out_tok[nx.at] = pick;
}

int launch_verify_drafts(const VerifyArgs& a, hipStream_t s) {
    const int groups = (chunks_of(a.V) + 3) / 4;
    // a wave's rows follow each other
    const int stretches = max(1, min(min(a.T, 65535), VF_SUM_WGS / groups));
    hipLaunchKernelGGL(verify_sums_kernel, dim3(groups, stretches), dim3(256), 0, s, a);
    hipLaunchKernelGGL(verify_walk_kernel, dim3(a.B), dim3(VF_TH), 0, s, a);
    if (a.q) hipLaunchKernelGGL(verify_less_kernel, dim3(groups, a.B), dim3(VL_TH), 0, s, a);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
