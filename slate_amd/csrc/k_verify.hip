// k_verify.hip -- which drafted tokens stand, and the token after them.
//
// A draft x with probability q(x) stands where u q(x) < p(x), so it is kept with
// probability min(1, p / q); one that is turned down leaves max(p - q, 0) to the
// next token, and the tokens come out distributed as p (the drafts without
// probabilities: q is 1 on x, the rest of p is divided by what is left of it).
#include "lanes.h"
#include "paged.h"

namespace slate_hip {

constexpr int VF_TH = 1024;

// Sum over the workgroup in a fixed order; every thread gets it.
__device__ __forceinline__ double block_total(double v, double* s_part) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0;
    for (int i = 0; i < VF_TH / 64; ++i) t += s_part[i];
    return t;
}

// A row's p up to its sum: w(i) = exp((z_i - top) / temperature), or 1 on the
// first largest logit.
struct Weights {
    const float* z;
    float top;
    int best;                          // -1: the row has no p
    double temp;                       // 0: greedy
    __device__ __forceinline__ double operator()(int i) const {
        const float x = z[i];
        if (!(x > -INFINITY) || best < 0) return 0;    // NaN too
        if (temp == 0) return i == best ? 1 : 0;
        return x == top ? 1 : top == INFINITY ? 0 : exp(((double)x - (double)top) / temp);
    }
};

__device__ __forceinline__ Weights row_weights(const float* z, int V, double temp, float* s_v, int* s_i) {
    float v = -INFINITY;
    int at = -1;
    for (int i = threadIdx.x; i < V; i += VF_TH)
        if (z[i] > v) {
            v = z[i];
            at = i;
        }
    __syncthreads();
    s_v[threadIdx.x] = v;
    s_i[threadIdx.x] = at;
    __syncthreads();
    for (int o = VF_TH / 2; o > 0; o >>= 1) {
        if (threadIdx.x < o) {
            const float v2 = s_v[threadIdx.x + o];
            const int i2 = s_i[threadIdx.x + o];
            if (i2 >= 0 && (s_i[threadIdx.x] < 0 || v2 > s_v[threadIdx.x] ||
                            (v2 == s_v[threadIdx.x] && i2 < s_i[threadIdx.x]))) {
                s_v[threadIdx.x] = v2;
                s_i[threadIdx.x] = i2;
            }
        }
        __syncthreads();
    }
    return Weights{z, s_v[0], s_i[0], temp};
}

// One workgroup per sequence, row after row.
__global__ __launch_bounds__(VF_TH) void verify_kernel(VerifyArgs a) {
    __shared__ float s_v[VF_TH];
    __shared__ int s_i[VF_TH];
    __shared__ double s_part[VF_TH / 64], s_sum[VF_TH];
    __shared__ int s_next;
    const int b = blockIdx.x;
    const int t0 = a.tok_off[b], t1 = a.tok_off[b + 1];
    if (t0 < 0 || t1 > a.T || t1 <= t0) {
        if (threadIdx.x == 0) a.n_accepted[b] = -1;
        return;
    }
    const int n = t1 - t0, V = a.V;
    const float tf = a.temperature ? a.temperature[b] : 1.0f;
    const double temp = tf > 0 ? (double)tf : 0.0;
    int node = 0, n_acc = 0, turned = -1;
    Weights w;
    double Z;
    auto parent = [&](int i) { return a.parent ? a.parent[t0 + i] : i - 1; };
    // turned down before i among the children of the node
    auto tried = [&](int tok, int i) {
        for (int j = node + 1; j < i; ++j)
            if (parent(j) == node && a.token[t0 + j] == tok) return true;
        return false;
    };
    for (;;) {
        w = row_weights(a.logits + (int64_t)(t0 + node) * a.ld, V, temp, s_v, s_i);
        double z = 0;
        for (int i = threadIdx.x; i < V; i += VF_TH) z += w(i);
        Z = block_total(z, s_part);
        double rest = 1;
        int next = -1;
        turned = -1;
        for (int c = node + 1; c < n && next < 0; ++c) {
            if (parent(c) != node) continue;
            const int x = a.token[t0 + c];
            double p = x >= 0 && x < V && Z > 0 && !tried(x, c) ? w(x) / Z : 0;
            bool yes;
            if (temp == 0)
                yes = p > 0;
            else if (a.q)
                yes = x >= 0 && x < V && (double)a.u[t0 + c] * (double)a.q[(int64_t)(t0 + c) * a.q_ld + x] < p;
            else
                yes = (double)a.u[t0 + c] * rest < p;
            if (yes) {
                next = c;
            } else {
                turned = c;
                rest -= p;
            }
        }
        if (next < 0) break;
        if (threadIdx.x == 0) {
            a.out_tok[t0 + n_acc] = a.token[t0 + next];
            if (a.out_row) a.out_row[t0 + n_acc] = next;
        }
        ++n_acc;
        node = next;
    }
    // the next token: thread after thread over stretches of the row
    const int step = (V + VF_TH - 1) / VF_TH, i0 = min(V, (int)threadIdx.x * step), i1 = min(V, i0 + step);
    const float* q = a.q && turned >= 0 && temp != 0 ? a.q + (int64_t)(t0 + turned) * a.q_ld : nullptr;
    const bool without = !a.q && turned >= 0 && temp != 0;
    int pick = -1;
    for (int pass = 0; pass < 2 && pick < 0; ++pass) { // the second without anything taken off
        auto mass = [&](int i) {
            double p = w(i);
            if (pass == 0 && q) p = fmax(p / Z - (double)q[i], 0.0);
            if (pass == 0 && without && p > 0 && tried(i, n)) p = 0;
            return p;
        };
        double s = 0;
        for (int i = i0; i < i1; ++i) s += mass(i);
        __syncthreads();
        s_sum[threadIdx.x] = s;
        if (threadIdx.x == 0) s_next = VF_TH;
        __syncthreads();
        double before = 0, total = 0;
        for (int j = 0; j < VF_TH; ++j) {
            if (j == (int)threadIdx.x) before = total;
            total += s_sum[j];
        }
        if (!(total > 0)) continue;
        const double at = total * (double)a.u_next[b];
        // the first stretch that passes `at`, or the last with any mass
        if (s > 0 && before + s > at) atomicMin(&s_next, (int)threadIdx.x);
        __syncthreads();
        if (s_next == VF_TH && threadIdx.x == 0)
            for (int j = VF_TH - 1; j >= 0 && s_next == VF_TH; --j)
                if (s_sum[j] > 0) s_next = j;
        __syncthreads();
        const int who = s_next;
        __syncthreads();
        if ((int)threadIdx.x == who) {
            int last = -1;
            for (int i = i0; i < i1; ++i) {
                const double p = mass(i);
                before += p;
                if (p > 0) last = i;
                if (p > 0 && before > at) break;
            }
            s_next = last;
        }
        __syncthreads();
        pick = s_next;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        a.n_accepted[b] = n_acc;
        a.out_tok[t0 + n_acc] = pick;
    }
    for (int i = n_acc + threadIdx.x; i < n; i += VF_TH) {
        if (i > n_acc) a.out_tok[t0 + i] = -1;
        if (a.out_row) a.out_row[t0 + i] = -1;
    }
}

int64_t verify_drafts_bytes(int, int, int) { return 16; }

int launch_verify_drafts(const VerifyArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(verify_kernel, dim3(a.B), dim3(VF_TH), 0, s, a);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
