// k_attn_paged.hip -- causal attention of new tokens over a K/V cache in pages.
//
// out = sum_k exp(s_k - m) V_k / sum_k exp(s_k - m), s_k = q.K_k / sqrt(hd),
// over the rows 0 .. pos0 + i of the token's slot.
#include "attn_plan.h"
#include "lanes.h"
#include "paged.h"

namespace slate_hip {

// One workgroup per (token, query head), its four waves taking every fourth
// key: a wave's lanes share the key's elements, with an online softmax per
// wave, joined at the end.
template <class E>
__global__ __launch_bounds__(256) void attn_paged_rows_kernel(PagedAttn a, PagedBatch pb) {
    constexpr int NE = PG_MAX_HD / 64;
    __shared__ float s_o[4][PG_MAX_HD], s_m[4], s_l[4];
    const int t = blockIdx.x, hq = blockIdx.y, h = hq / (a.Hq / a.kv.n_kv_heads);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    // the last sequence, before any fall of tok_off, that begins at or before t
    int b = -1;
    for (int c = lane; c < ((pb.B + 63) & ~63); c += 64) {
        uint64_t begun = __builtin_amdgcn_ballot_w64(c < pb.B && pb.tok_off[c] <= t);
        const uint64_t falls = __builtin_amdgcn_ballot_w64(c < pb.B && pb.tok_off[c + 1] < pb.tok_off[c]);
        if (falls) begun &= (falls & -falls) - 1;
        b += __popcll(begun);
        if (falls) break;
    }
    if (b < 0) return;
    const int t0 = pb.tok_off[b], t1 = pb.tok_off[b + 1], p0 = pb.pos0[b], slot = pb.slot[b];
    if (t0 < 0 || t >= t1 || t1 > pb.T || t1 - t0 > pb.max_new || p0 < 0 || p0 > pb.max_seq - (t1 - t0) || slot < 0 ||
        slot >= pb.n_slots)
        return;
    const int hd = a.kv.head_dim;
    const int32_t* table = a.pg.table + (int64_t)slot * a.pg.max_pages;
    const float scale2 = (1.0f / sqrtf((float)hd)) * LOG2E;
    const float* qr = a.q + ((int64_t)t * a.Hq + hq) * hd;
    float q[NE], o[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) {
        q[e] = lane + 64 * e < hd ? qr[lane + 64 * e] : 0.f;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int key = w; key <= p0 + (t - t0); key += 4) {
        const int i = key / a.pg.page_size, page = table[i];
        if ((unsigned)page >= (unsigned)a.pg.n_pages) continue;
        const int64_t at = page * a.kv.page_stride + h * a.kv.head_stride + (key - i * a.pg.page_size) * a.kv.row_stride;
        const E *kr = (const E*)a.kv.K + at, *vr = (const E*)a.kv.V + at;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int j = lane + 64 * e;
            if (j < hd) s += q[e] * (float)kr[j];
        }
        s = wave_sum(s) * scale2;
        const float mn = fmaxf(m, s);
        const float alpha = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(s - mn);
        l = l * alpha + p;
        m = mn;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int j = lane + 64 * e;
            if (j < hd) o[e] = o[e] * alpha + p * (float)vr[j];
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
        lt += s_l[k] == 0.f ? 0.f : f[k] * s_l[k];
    }
    for (int j = threadIdx.x; j < hd; j += 256) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (s_l[k] != 0.f) v += f[k] * s_o[k][j];
        a.out[((int64_t)t * a.Hq + hq) * hd + j] = lt == 0.f ? 0.f : v / lt;
    }
}

int64_t attention_paged_bytes(int) { return 16; }

int launch_attention_paged(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    const dim3 grid(pb.T, a.Hq);
    if (a.kv.dtype == KV_F32)
        hipLaunchKernelGGL(attn_paged_rows_kernel<float>, grid, dim3(256), 0, s, a, pb);
    else if (a.kv.dtype == KV_F16)
        hipLaunchKernelGGL(attn_paged_rows_kernel<_Float16>, grid, dim3(256), 0, s, a, pb);
    else
        hipLaunchKernelGGL(attn_paged_rows_kernel<__bf16>, grid, dim3(256), 0, s, a, pb);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
