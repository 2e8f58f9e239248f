// k_kv8.hip -- K/V rows of a packed batch quantised into the 8-bit cache, and
// read back.
//
//   step = f16(max |x| / 127),  code = x / step to the nearest, ties to even
//
// Eight lanes share a block of 32 elements, four of them each: the maximum
// stays inside a DPP row, loads and stores are whole lines.  A workgroup
// takes one token's K or V row (grid.y).
#include "lanes.h"
#include "packed.h"

namespace slate_hip {

constexpr int KV8_THREADS = 256;

// x / step (step > 0 an f16 number, |x| at most about 127 step) rounded to
// nearest even, exactly: the quotient by a reciprocal is off by at most one
// in its rounding, and the remainder x - n step, which fma gives without
// error (n has 8 bits, step 11), says on which side of the tie x lies.
__device__ __forceinline__ int code_of(float x, float step, float inv) {
    if (x != x) return 0;
    const float n = rintf(fminf(fmaxf(x * inv, -127.f), 127.f));
    if (fabsf(n) >= 127.f && fabsf(x) >= 127.f * step) return (int)n;   // the end of the range
    const float r = fmaf(-n, step, x), h = 0.5f * step;
    float m = n;
    const bool odd = (int)n & 1;
    if (r > h || (r == h && odd)) m = n + 1.f;
    if (r < -h || (r == -h && odd)) m = n - 1.f;
    return (int)fminf(fmaxf(m, -127.f), 127.f);
}

__global__ __launch_bounds__(KV8_THREADS) void kv_store_q8_kernel(int8_t* __restrict__ kq, _Float16* __restrict__ ks,
                                                                  int8_t* __restrict__ vq, _Float16* __restrict__ vs,
                                                                  const float* __restrict__ k,
                                                                  const float* __restrict__ v, int64_t ld,
                                                                  PackedBatch pb, int n_kv, int hd,
                                                                  int64_t head_stride) {
    const int t = blockIdx.x;
    const int b = find_seq(pb, t);
    if (b < 0) return;
    const SeqView sv = seq_view(pb, b);
    if (t < sv.t0 || t >= sv.t0 + sv.n) return;
    const int64_t base = pb.kv_base[b] / hd * hd + (int64_t)(sv.p0 + t - sv.t0) * hd;
    const float* src = (blockIdx.y ? v : k) + (int64_t)t * ld;
    int8_t* codes = blockIdx.y ? vq : kq;
    _Float16* steps = blockIdx.y ? vs : ks;
    const int n4 = n_kv * hd / 4;                      // a multiple of 8: an octet of lanes is in or out whole
    for (int j = threadIdx.x; j < n4; j += KV8_THREADS) {
        const int h = 4 * j / hd, e = 4 * j - h * hd;
        const float4 x = *(const float4*)(src + 4 * j);
        const float top = group8_max(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fmaxf(fabsf(x.z), fabsf(x.w)), 0.f)));
        const _Float16 step = (_Float16)fminf(top / 127.0f, 65504.0f);
        const float d = (float)step, inv = 1.0f / d;
        uint32_t c = 0;
        if (d > 0.f)
            c = (uint32_t)(code_of(x.x, d, inv) & 255) | (uint32_t)(code_of(x.y, d, inv) & 255) << 8 |
                (uint32_t)(code_of(x.z, d, inv) & 255) << 16 | (uint32_t)code_of(x.w, d, inv) << 24;
        const int64_t at = base + h * head_stride + e;
        *(uint32_t*)(codes + at) = c;
        if ((threadIdx.x & 7) == 0) steps[at / KV8_BLOCK] = step;
    }
}

__global__ __launch_bounds__(KV8_THREADS) void kv_load_q8_kernel(float* __restrict__ k, float* __restrict__ v,
                                                                 int64_t ld, Kv8 kv, PackedBatch pb, int n_kv, int hd,
                                                                 int64_t head_stride) {
    const int t = blockIdx.x;
    const int b = find_seq(pb, t);
    if (b < 0) return;
    const SeqView sv = seq_view(pb, b);
    if (t < sv.t0 || t >= sv.t0 + sv.n) return;
    const int64_t base = pb.kv_base[b] / hd * hd + (int64_t)(sv.p0 + t - sv.t0) * hd;
    float* dst = (blockIdx.y ? v : k) + (int64_t)t * ld;
    const int8_t* codes = blockIdx.y ? kv.vq : kv.kq;
    const _Float16* steps = blockIdx.y ? kv.vs : kv.ks;
    const int n4 = n_kv * hd / 4;
    for (int j = threadIdx.x; j < n4; j += KV8_THREADS) {
        const int h = 4 * j / hd, e = 4 * j - h * hd;
        const int64_t at = base + h * head_stride + e;
        const uint32_t c = *(const uint32_t*)(codes + at);
        const float d = (float)steps[at / KV8_BLOCK];
        *(float4*)(dst + 4 * j) = make_float4(d * (float)(int8_t)(c & 255), d * (float)(int8_t)(c >> 8 & 255),
                                              d * (float)(int8_t)(c >> 16 & 255), d * (float)(int8_t)(c >> 24));
    }
}

int launch_kv_store_q8(int8_t* kq, _Float16* ks, int8_t* vq, _Float16* vs, const float* k, const float* v, int64_t ld,
                       const PackedBatch& pb, int n_kv, int hd, int64_t head_stride, hipStream_t s) {
    hipLaunchKernelGGL(kv_store_q8_kernel, dim3(pb.T, 2), dim3(KV8_THREADS), 0, s, kq, ks, vq, vs, k, v, ld, pb, n_kv,
                       hd, head_stride);
    SH_CHECK_LAUNCH();
    return 0;
}

int launch_kv_load_q8(float* k, float* v, int64_t ld, const Kv8& kv, const PackedBatch& pb, int n_kv, int hd,
                      int64_t head_stride, hipStream_t s) {
    hipLaunchKernelGGL(kv_load_q8_kernel, dim3(pb.T, 2), dim3(KV8_THREADS), 0, s, k, v, ld, kv, pb, n_kv, hd,
                       head_stride);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
