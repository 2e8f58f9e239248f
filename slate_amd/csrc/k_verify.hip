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
constexpr int VF_ROWS = PK_MAX_DRAFT + 1;

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// 2^t for t <= 0, to 2^-42 of itself: e^(f ln 2) for the part f of t behind the
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

// Weight of logit x beside the largest one: e^((x - top) / temperature), by =
// log2(e) / temperature.  0 for -infinity; infinite logits share all.
__device__ __forceinline__ double weight(float x, float top, double by) {
    if (!(x > -INFINITY)) return 0;
    if (x == top) return 1;
    return top == INFINITY ? 0 : pow2(((double)x - (double)top) * by);
}

struct alignas(16) Part {
    float top;                         // -infinity: none
    int best;                          // its first place (greedy rows)
    double sum;                        // of the weights beside it
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

__device__ __forceinline__ int place(int c, int k, int lane) { return c * VF_CHUNK + 256 * k + 4 * lane; }

// A wave's 16 values a lane of chunk c: x[4k + e] is element 256 k + 4 lane + e of
// it; `none` behind V.
__device__ __forceinline__ void load16(const float* z, int c, int V, float none, float* x) {
    const int lane = threadIdx.x & 63;
    if (V - c * VF_CHUNK >= VF_CHUNK) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4u v = *(const float4u*)(z + place(c, k, lane));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * k + e] = v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int at = place(c, i / 4, lane) + i % 4;
            x[i] = at < V ? z[at] : none;
        }
    }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = min(v, __shfl_xor(v, o));
    return v;
}

__host__ __device__ constexpr int chunks_of(int V) { return (V - 1) / VF_CHUNK + 1; }

// Workspace: a Part per row and chunk, a mass per sequence and chunk, a Next per sequence.
struct Next {
    int row, turned, at;               // the row whose p it is, the draft's row (-1: nothing to do), where it goes
    float top;
    double sum;                        // of the row's weights
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

// Softmax sums (greedy rows: the largest logit) of all rows, a wave per chunk.
__global__ __launch_bounds__(256) void verify_sums_kernel(VerifyArgs a) {
    const int lane = threadIdx.x & 63, nch = chunks_of(a.V);
    const int c = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (c >= nch) return;
    const Space sp = space_of(a);
    for (int t = blockIdx.y; t < a.T; t += gridDim.y) {
        float x[16];
        load16(a.logits + (int64_t)t * a.ld, c, a.V, -INFINITY, x);
        // the sequence, for its temperature (a row that belongs to none has some)
        int b = 0;
        if (a.temperature)
            for (int b0 = 0; b0 < a.B; b0 += 64) {
                const int i = b0 + lane;
                uint64_t begun = __builtin_amdgcn_ballot_w64(i < a.B && a.tok_off[i] <= t);
                const uint64_t falls = __builtin_amdgcn_ballot_w64(i < a.B && a.tok_off[i + 1] < a.tok_off[i]);
                if (falls) begun &= (falls & -falls) - 1;
                b += __popcll(begun);
                if (falls) break;
            }
        const Heat heat = heat_of(a.temperature, max(0, b - 1));
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = x[i] > -INFINITY ? x[i] : -INFINITY;        // NaN too
            top = fmaxf(top, x[i]);
        }
        top = wave_max(top);
        Part p{top, -1, 0};
        if (heat.greedy) {
            int at = INT32_MAX;
#pragma unroll
            for (int i = 15; i >= 0; --i)
                if (x[i] == top) at = place(c, i / 4, lane) + i % 4;
            p.best = wave_min_int(at);
        } else {
            double s = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += weight(x[i], top, heat.by);
            p.sum = wave_sum_f64(s);
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
__device__ __forceinline__ Sums block_sums(double v, double* s_part) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(v, o);
        if (lane >= o) v += up;
    }
    __syncthreads();
    if (lane == 63) s_part[w] = v;
    __syncthreads();
    double before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < VF_TH / 64; ++i) {
        before += i < w ? s_part[i] : 0;
        total += s_part[i];
    }
    return Sums{before + v, total};
}

// The token at which the sums of the chunks' masses pass u times the whole: mass(c)
// is a chunk's, values(c, m) a wave's 16 elements of it a lane, in load16's places.
// -1 where there is no mass.  Called by the workgroup; thread 0's answer counts.
template <class Mass, class Values>
__device__ int pick_token(int nch, float u, const Mass& mass, const Values& values, double* s_part) {
    __shared__ int s_chunk, s_last, s_pick;
    __shared__ double s_before;
    double total = 0;
    for (int c0 = 0; c0 < nch; c0 += VF_TH) {
        const int c = c0 + threadIdx.x;
        total += block_sums(c < nch ? mass(c) : 0, s_part).total;
    }
    const double at = total * (double)u;
    if (threadIdx.x == 0) {
        s_chunk = INT32_MAX;
        s_last = -1;
        s_pick = -1;
    }
    double before = 0;
    for (int c0 = 0; c0 < nch; c0 += VF_TH) {
        const int c = c0 + threadIdx.x;
        const double m = c < nch ? mass(c) : 0;
        const Sums s = block_sums(m, s_part);          // its barriers order the writes above
        if (m > 0) {
            if (before + s.upto > at) atomicMin(&s_chunk, c);
            atomicMax(&s_last, c);
        }
        __syncthreads();
        const bool found = s_chunk != INT32_MAX;       // none at all: the last one with any mass
        if ((found ? s_chunk : s_last) == c) s_before = before + (s.upto - m);
        if (found) break;
        before += s.total;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, chunk = s_chunk != INT32_MAX ? s_chunk : s_last;
    if (threadIdx.x < 64 && chunk >= 0) {
        double m[16], sum = s_before;
        values(chunk, m);
        int pick = -1, last = -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            double v = (m[4 * k] + m[4 * k + 1]) + (m[4 * k + 2] + m[4 * k + 3]);
            const double own = v;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(v, o);
                if (lane >= o) v += up;
            }
            double run = sum + (v - own);
            int here = INT32_MAX, some = -1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                run += m[4 * k + e];
                if (m[4 * k + e] > 0) {
                    some = place(chunk, k, lane) + e;
                    if (run > at && here == INT32_MAX) here = some;
                }
            }
            here = wave_min_int(here);
            last = max(last, -wave_min_int(-some));
            if (pick < 0 && here != INT32_MAX) pick = here;
            sum += __shfl(v, 63);
        }
        if (lane == 0) s_pick = pick >= 0 ? pick : last;
    }
    __syncthreads();
    return s_pick;
}

// One workgroup per sequence: its rows' sums joined, its drafts' chances, the walk,
// and the next token where no draft's probability has to be taken off.
__global__ __launch_bounds__(VF_TH) void verify_walk_kernel(VerifyArgs a) {
    __shared__ double s_sum[VF_ROWS], s_p[VF_ROWS], s_u[VF_ROWS];
    __shared__ float s_top[VF_ROWS];
    __shared__ int s_best[VF_ROWS], s_parent[VF_ROWS], s_tok[VF_ROWS];
    __shared__ double s_part[VF_TH / 64];
    __shared__ int s_node, s_acc, s_turned;
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
    for (int i = threadIdx.x; i < n; i += VF_TH) {
        s_tok[i] = a.token[t0 + i];
        const int up = a.parent ? a.parent[t0 + i] : i - 1;
        s_parent[i] = up >= 0 && up < i ? up : -1;
    }
    for (int i = w; i < n; i += VF_TH / 64) {
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
        double p = 0, u = INFINITY;                    // u infinite: never
        if (up >= 0 && in) {
            // a token that an earlier child of the same row has was turned down before this one is tried
            bool again = false;
            if (a.parent)
                for (int j = up + 1; j < i; ++j) again |= s_parent[j] == up && s_tok[j] == x;
            if (heat.greedy)
                p = s_best[up] == x;
            else if (!again && s_sum[up] > 0)
                p = weight(a.logits[(int64_t)(t0 + up) * a.ld + x], s_top[up], heat.by) / s_sum[up];
            u = heat.greedy ? 0.5 : a.u[t0 + i] * (a.q ? (double)a.q[(int64_t)(t0 + i) * a.q_ld + x] : 1.0);
        }
        s_p[i] = p;
        s_u[i] = u;
    }
    __syncthreads();
    if (w == 0) {
        // drafts in order, 64 at a time: a row's children lie behind it
        int node = 0, acc = 0, turned = -1;
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
                    left = __builtin_amdgcn_ballot_w64(up == node) & ~((2ull << l) - 1);
                } else {
                    rest -= p;
                    turned = c;
                    left &= left - 1;
                }
            }
        }
        if (lane == 0) {
            s_node = node;
            s_acc = acc;
            s_turned = turned;
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
        sp.next[b] = Next{t0 + node, less ? t0 + turned : -1, t0 + acc, s_top[node], s_sum[node]};
    if (less) return;                                  // the next kernels'
    if (heat.greedy || !(s_top[node] > -INFINITY)) {
        if (threadIdx.x == 0) a.out_tok[t0 + acc] = s_best[node];     // -1 where the row has no p
        return;
    }
    // p without the tokens that were turned down: their chunks are summed again
    const float* z = a.logits + (int64_t)(t0 + node) * a.ld;
    const Part* part = sp.part + (int64_t)(t0 + node) * nch;
    const float top = s_top[node];
    const bool without = !a.q && turned >= 0;
    auto values = [&](int c, double* m) {
        float x[16];
        load16(z, c, V, -INFINITY, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) m[i] = weight(x[i], top, heat.by);
    };
    auto values_without = [&](int c, double* m) {
        values(c, m);
        for (int j = node + 1; j <= turned; ++j) {
            if (s_parent[j] != node || s_tok[j] < 0 || s_tok[j] >= V || s_tok[j] / VF_CHUNK != c) continue;
            const int x = s_tok[j] % VF_CHUNK;
            if (lane == (x >> 2 & 63))
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i == (x >> 8) * 4 + (x & 3)) m[i] = 0;
        }
    };
    auto mass = [&](int c) { return part[c].sum * weight(part[c].top, top, heat.by); };
    int pick = -1;
    if (without) {
        double* own = sp.mass + (int64_t)b * nch;
        for (int c = threadIdx.x; c < nch; c += VF_TH) own[c] = mass(c);
        __syncthreads();
        for (int j = node + 1 + w; j <= turned; j += VF_TH / 64) {
            if (s_parent[j] != node || s_tok[j] < 0 || s_tok[j] >= V) continue;
            const int c = s_tok[j] / VF_CHUNK;
            double m[16], s = 0;
            values_without(c, m);                      // of two tokens in a chunk either writes the same
#pragma unroll
            for (int i = 0; i < 16; ++i) s += m[i];
            s = wave_sum_f64(s);
            if (lane == 0) own[c] = s;
        }
        __syncthreads();
        pick = pick_token(nch, a.u_next[b], [&](int c) { return own[c]; }, values_without, s_part);
        __syncthreads();
    }
    if (pick < 0) pick = pick_token(nch, a.u_next[b], mass, values, s_part);
    if (threadIdx.x == 0) a.out_tok[t0 + acc] = pick;
}
// What p has more than q, a wave per chunk: the sums.
__device__ __forceinline__ void more_than(const VerifyArgs& a, const Next& nx, double by, int c, double* m) {
    float x[16], y[16];
    load16(a.logits + (int64_t)nx.row * a.ld, c, a.V, -INFINITY, x);
    load16(a.q + (int64_t)nx.turned * a.q_ld, c, a.V, 0.f, y);
    const double share = 1.0 / nx.sum;
#pragma unroll
    for (int i = 0; i < 16; ++i) m[i] = fmax(fma(weight(x[i], nx.top, by), share, -(double)y[i]), 0.0);
}
__global__ __launch_bounds__(256) void verify_less_kernel(VerifyArgs a) {
    const int nch = chunks_of(a.V), b = blockIdx.y;
    const int c = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const Space sp = space_of(a);
    const Next nx = sp.next[b];
    if (c >= nch || nx.turned < 0) return;
    double m[16], s = 0;
    more_than(a, nx, heat_of(a.temperature, b).by, c, m);
#pragma unroll
    for (int i = 0; i < 16; ++i) s += m[i];
    s = wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) sp.mass[(int64_t)b * nch + c] = s;
}
__global__ __launch_bounds__(VF_TH) void verify_pick_kernel(VerifyArgs a) {
    __shared__ double s_part[VF_TH / 64];
    const int nch = chunks_of(a.V), b = blockIdx.x;
    const Space sp = space_of(a);
    const Next nx = sp.next[b];
    if (nx.turned < 0) return;
    const double by = heat_of(a.temperature, b).by;
    const double* own = sp.mass + (int64_t)b * nch;
    int pick = pick_token(nch, a.u_next[b], [&](int c) { return own[c]; },
                          [&](int c, double* m) { more_than(a, nx, by, c, m); }, s_part);
    if (pick < 0) {                                    // p has nothing more than q: from p
        __syncthreads();
        const Part* part = sp.part + (int64_t)nx.row * nch;
        pick = pick_token(nch, a.u_next[b], [&](int c) { return part[c].sum * weight(part[c].top, nx.top, by); },
                          [&](int c, double* m) {
                              float x[16];
                              load16(a.logits + (int64_t)nx.row * a.ld, c, a.V, -INFINITY, x);
#pragma unroll
                              for (int i = 0; i < 16; ++i) m[i] = weight(x[i], nx.top, by);
                          },
                          s_part);
    }
    if (threadIdx.x == 0) a.out_tok[nx.at] = pick;
}

int launch_verify_drafts(const VerifyArgs& a, hipStream_t s) {
    const int groups = (chunks_of(a.V) + 3) / 4;
    hipLaunchKernelGGL(verify_sums_kernel, dim3(groups, min(a.T, 65535)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(verify_walk_kernel, dim3(a.B), dim3(VF_TH), 0, s, a);
    if (a.q) {
        hipLaunchKernelGGL(verify_less_kernel, dim3(groups, a.B), dim3(256), 0, s, a);
        hipLaunchKernelGGL(verify_pick_kernel, dim3(a.B), dim3(VF_TH), 0, s, a);
    }
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
