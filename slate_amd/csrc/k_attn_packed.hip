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
// wave, joined at the end.  It serves the head_dims that the matrix kernels do
// not take (other than 32, 64, 128).  Every query row reads its keys for
// itself, out of L2: a decode step of 16 users at head_dim 128 took it 1155 us
// where the few-row kernel takes 27.5.
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

// Joins the parts of a block that lies in several workgroups' ranges:
// workgroup b takes the block that is first cut before workgroup b + 1 of the
// attention kernel, HD / 4 lanes a row, eight parts' loads at a time.
constexpr int JOIN_TH = 512;
template <int HD>
__global__ __launch_bounds__(JOIN_TH) void attn_join_kernel(float* __restrict__ out, void* ws, int Hq, int G,
                                                       int slot_rows, int P) {
    const JoinEntry en = *entry_of(ws, blockIdx.x + 1);
    const int c = 4 * (threadIdx.x % (HD / 4));
    // the first part's slot, then the first slot of each workgroup after it
    auto slot = [&](int k) { return slot_of(ws, P, k == 0 ? en.slot0 : 2 * ((int)blockIdx.x + k), slot_rows, HD); };
    const int r = blockIdx.y * (JOIN_TH / (HD / 4)) + threadIdx.x / (HD / 4);
    if (r < en.rows) {
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < en.pieces; k0 += 8) {
            float2 ml[8];
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                ml[k] = make_float2(-INFINITY, 0.f);
                if (k0 + k >= en.pieces) continue;     // the same for the whole workgroup
                const float* sl = slot(k0 + k);
                ml[k] = *(const float2*)(sl + slot_rows * HD + 2 * r);
                v[k] = *(const float4*)(sl + r * HD + c);
            }
            float mt = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) mt = fmaxf(mt, ml[k].x);
            if (mt == -INFINITY) continue;             // nothing seen yet
            const float f = __builtin_amdgcn_exp2f(m - mt);
            m = mt;
            l *= f;
            o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float fk = __builtin_amdgcn_exp2f(ml[k].x - mt);
                if (fk == 0.f) continue;
                l += fk * ml[k].y;
                o.x += fk * v[k].x;
                o.y += fk * v[k].y;
                o.z += fk * v[k].z;
                o.w += fk * v[k].w;
            }
        }
        const float inv = 1.0f / l;
        float* op = out + ((int64_t)(en.t0 + (en.r0 + r) / G) * Hq + en.h * G + (en.r0 + r) % G) * HD + c;
        op[0] = o.x * inv;
        op[1] = o.y * inv;
        op[2] = o.z * inv;
        op[3] = o.w * inv;
    }
}

template <int HD>
static void launch_join_hd(float* out, void* ws, int Hq, int Hkv, int slot_rows, int P, hipStream_t s) {
    constexpr int AT_ONCE = JOIN_TH / (HD / 4);        // rows of a workgroup
    hipLaunchKernelGGL(attn_join_kernel<HD>, dim3(P - 1, (slot_rows + AT_ONCE - 1) / AT_ONCE), dim3(JOIN_TH), 0, s, out,
                       ws, Hq, Hq / Hkv, slot_rows, P);
}

void launch_attn_join(float* out, void* ws, int Hq, int Hkv, int hd, int slot_rows, int P, hipStream_t s) {
    if (hd == 128)
        launch_join_hd<128>(out, ws, Hq, Hkv, slot_rows, P, s);
    else if (hd == 64)
        launch_join_hd<64>(out, ws, Hq, Hkv, slot_rows, P, s);
    else
        launch_join_hd<32>(out, ws, Hq, Hkv, slot_rows, P, s);
}

int64_t attention_packed_bytes(int Hq, int Hkv, int hd) {
    if (hd != 32 && hd != 64 && hd != 128) return 0;
    return max(attention_q8_few_bytes(hd), attention_many_bytes(hd));
}

bool attention_packed_fits(const PackedAttn& a, const PackedBatch& pb) {
    const double most = attention_q8_few_takes(a, pb) ? attention_q8_few_most(a, pb)
                        : attention_many_takes(a)     ? attention_many_most(a, pb)
                                                      : 0;
    return most < 2147483648.0;
}

int launch_attention_packed(const PackedAttn& a, const PackedBatch& pb, hipStream_t s) {
    if (attention_q8_few_takes(a, pb)) return launch_attention_q8_few(a, pb, s);
    if (attention_many_takes(a)) return launch_attention_many(a, pb, s);
    hipLaunchKernelGGL(attn_packed_rows_kernel, dim3(pb.T, a.Hq), dim3(256), 0, s, a, pb);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
