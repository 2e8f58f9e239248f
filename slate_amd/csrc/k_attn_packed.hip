// k_attn_packed.hip -- attention of packed batches over an 8-bit or f32 K/V
// cache, causal or over trees of drafted tokens.
//
// out = sum_k exp(s_k - m) V_k / sum_k exp(s_k - m), s_k = q.K_k / sqrt(hd),
// over the keys that the token sees.
#include "attn_plan.h"
#include "lanes.h"

namespace slate_hip {

// One workgroup per (token, query head), its four waves taking every fourth
// key: a wave's lanes share the key's elements, with an online softmax per
// wave, joined at the end.  For head_dims of the other kernels' range this is
// the plain one to check them against.
__global__ __launch_bounds__(256) void attn_packed_rows_kernel(PackedAttn a, PackedBatch pb) {
    __shared__ uint32_t s_seen[PK_MAX_DRAFT / 32];
    __shared__ float s_o[4][PK_MAX_HD], s_m[4], s_l[4];
    constexpr int NE = PK_MAX_HD / 64;
    const int t = blockIdx.x, hq = blockIdx.y, h = hq / (a.Hq / a.Hkv);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int b = find_seq(pb, t);
    if (b < 0) return;
    const SeqView sv = seq_view(pb, b);
    const int i = t - sv.t0;
    if (i < 0 || i >= sv.n) return;
    const int hd = a.hd;
    if (a.parent) {                                    // the token's ancestors among the drafts, itself included
        for (int j = threadIdx.x; j < PK_MAX_DRAFT / 32; j += 256) s_seen[j] = 0;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int j = i;;) {
                s_seen[j >> 5] |= 1u << (j & 31);
                const int up = a.parent[sv.t0 + j];
                if (up < 0 || up >= j) break;
                j = up;
            }
        __syncthreads();
    }
    const int64_t kvb = a.kf ? pb.kv_base[b] : pb.kv_base[b] / hd * hd;
    const int64_t head = kvb + h * a.head_stride;
    const float scale2 = (1.0f / sqrtf((float)hd)) * LOG2E;
    const float* qr = a.q + ((int64_t)t * a.Hq + hq) * hd;
    float q[NE], o[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        q[e] = lane + 64 * e < hd ? qr[lane + 64 * e] : 0.f;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int key = w; key <= sv.p0 + i; key += 4) {
        if (a.parent && key >= sv.p0 && !(s_seen[(key - sv.p0) >> 5] >> ((key - sv.p0) & 31) & 1)) continue;
        const int64_t at = head + (int64_t)key * hd;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int j = lane + 64 * e;
            if (j >= hd) break;
            s += q[e] * (a.kf ? a.kf[at + j] : (float)a.kv8.ks[(at + j) / KV8_BLOCK] * (float)a.kv8.kq[at + j]);
        }
        s = wave_sum(s) * scale2;
        const float mn = fmaxf(m, s);
        const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(s - mn);
        l = l * alpha + p;
        m = mn;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int j = lane + 64 * e;
            if (j >= hd) break;
            o[e] = o[e] * alpha +
                   p * (a.kf ? a.vf[at + j] : (float)a.kv8.vs[(at + j) / KV8_BLOCK] * (float)a.kv8.vq[at + j]);
        }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e)
        if (lane + 64 * e < hd) s_o[w][lane + 64 * e] = o[e];
    if (lane == 0) {
        s_m[w] = m;
        s_l[w] = l;
    }
    __syncthreads();
    const float mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float f[4], lt = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[k] = s_l[k] == 0.f ? 0.f : __builtin_amdgcn_exp2f(s_m[k] - mx);
        lt += f[k] * s_l[k];
    }
    for (int j = threadIdx.x; j < hd; j += 256) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) v += f[k] * s_o[k][j];
        a.out[((int64_t)t * a.Hq + hq) * hd + j] = v / lt;
    }
}

int64_t attention_packed_bytes(int Hq, int Hkv, int hd) {
    return attention_q8_few_shape(hd, Hq / Hkv) ? attention_q8_few_bytes(hd) : 0;
}

int launch_attention_packed(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    const int G = a.Hq / a.Hkv;
    if (!a.kf && attention_q8_few_shape(a.hd, G) && pb.max_new * (int64_t)G <= 16)
        return launch_attention_q8_few(a, pb, s);
    hipLaunchKernelGGL(attn_packed_rows_kernel, dim3(pb.T, a.Hq), dim3(256), 0, s, a, pb);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
