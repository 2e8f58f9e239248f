// k_kv8.hip -- K/V rows of a packed batch quantised into the 8-bit cache, and
// read back.
//
//   step = f16(max |x| / 127),  code = x / step to the nearest, ties to even
//
// Eight lanes share a block of 32 elements, four of them each: the maximum
// stays inside a DPP row, loads and stores are whole lines.  Memory bound: K
// and V rows of 5592 tokens (8 heads of 128) are stored in 16.4 us (58 MB
// read and written, 3.5 TB/s; a store per token and exact divisions took 21)
// and loaded in 13.3 us (4.4 TB/s); rows of 16 tokens in 3 us each, launch and
// two rounds of load latency.
#include "lanes.h"
#include "packed.h"

namespace slate_hip {

constexpr int KV8_THREADS = 256;

// x / step rounded to nearest even within -127 .. 127 (step > 0 an f16 number,
// inv its reciprocal within 2^-23).  |x| is at most 190.5 steps (max / 127 just
// below 1.5 * 2^-24 becomes a step of 2^-24), so x inv is off the quotient by
// less than 2^-14 and rounds the same way unless it lies
// that close to a tie; there the remainder x - n step, which fma gives without
// error (n has 8 bits, step 11), says on which side of the tie x is.  Where the
// step was limited to 65504, or x is infinite, |x| can be anything above: what
// is 127 steps or more ends at the clamp either way.
__device__ __forceinline__ int code_of(float x, float step, float inv) {
    const float t = x * inv;
    float n = rintf(t);
    if (!(fabsf(t - n) <= 0.4999f)) {                  // infinities and NaN come here too
        if (x != x) return 0;
        n = fminf(fmaxf(n, -127.f), 127.f);
        if (fabsf(x) < 127.f * step) {
            const float r = fmaf(-n, step, x), h = 0.5f * step;
            const bool odd = (int)n & 1;
            const float at = n;
            if (r > h || (r == h && odd)) n = at + 1.f;
            if (r < -h || (r == -h && odd)) n = at - 1.f;
        }
    }
    return (int)fminf(fmaxf(n, -127.f), 127.f);
}

// top / 127, rounded to nearest: the product with the rounded 1/127, mended by
// its remainder, is the correctly rounded quotient for every finite f32 (all
// of them were compared).  Infinity gives NaN, which fminf turns into the
// limit.
__device__ __forceinline__ _Float16 step_of(float top) {
    const float c = 1.0f / 127.0f, q = top * c;
    return (_Float16)fminf(fmaf(fmaf(-q, 127.0f, top), c, q), 65504.0f);
}

// The batch's first 64 sequences, one per lane, so that a token's sequence is
// found without a load per token.
class Sequences {
  public:
    __device__ __forceinline__ explicit Sequences(const PackedBatch& pb) : pb_(pb) {
        const int b = threadIdx.x & 63;
        if (b < pb.B) {
            seq_ = seq_view(pb, b);
            base_ = pb.kv_base[b];
        }
    }
    // Element where the token's row of head 0 starts; -1: it is stored nowhere.
    __device__ __forceinline__ int64_t row_of(int t, int hd) const {
        SeqView s;
        int64_t base;
        if (pb_.B <= 64) {
            const int b = __popcll(__builtin_amdgcn_ballot_w64((int)(threadIdx.x & 63) < pb_.B && seq_.t0 <= t)) - 1;
            if (b < 0) return -1;
            s = SeqView{__builtin_amdgcn_readlane(seq_.t0, b), __builtin_amdgcn_readlane(seq_.n, b),
                        __builtin_amdgcn_readlane(seq_.p0, b)};
            base = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)((uint64_t)base_ >> 32), b) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)base_, b));
        } else {
            const int b = find_seq(pb_, t);
            if (b < 0) return -1;
            s = seq_view(pb_, b);
            base = pb_.kv_base[b];
        }
        return t < s.t0 || t >= s.t0 + s.n ? -1 : base / hd * hd + (int64_t)(s.p0 + t - s.t0) * hd;
    }

  private:
    const PackedBatch& pb_;
    SeqView seq_{};
    int64_t base_ = 0;
};

// A workgroup takes TOK tokens' K (grid.y 0) or V rows; the rows' loads go out
// before the descriptors are looked at.
template <int TOK>
__global__ __launch_bounds__(KV8_THREADS) void kv_store_q8_kernel(int8_t* __restrict__ kq, _Float16* __restrict__ ks,
                                                                  int8_t* __restrict__ vq, _Float16* __restrict__ vs,
                                                                  const float* __restrict__ k,
                                                                  const float* __restrict__ v, int64_t ld,
                                                                  PackedBatch pb, int n_kv, int hd,
                                                                  int64_t head_stride) {
    const int t0 = blockIdx.x * TOK;
    const float* src = blockIdx.y ? v : k;
    int8_t* codes = blockIdx.y ? vq : kq;
    _Float16* steps = blockIdx.y ? vs : ks;
    const Sequences seqs(pb);
    const int n4 = n_kv * hd / 4;                      // a multiple of 8: an octet of lanes is in or out whole
    for (int j0 = 0; j0 < n4; j0 += KV8_THREADS) {
        const int j = j0 + threadIdx.x, jj = min(j, n4 - 1);
        float4 x[TOK];
#pragma unroll
        for (int i = 0; i < TOK; ++i) x[i] = *(const float4*)(src + (int64_t)min(t0 + i, pb.T - 1) * ld + 4 * jj);
        const int h = 4 * jj / hd;
        const int64_t in = h * head_stride + (4 * jj - h * hd);
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            const int64_t row = t0 + i < pb.T ? seqs.row_of(t0 + i, hd) : -1;
            if (row < 0) continue;
            const float top =
                group8_max(fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fmaxf(fabsf(x[i].z), fabsf(x[i].w)), 0.f)));
            const _Float16 step = step_of(top);
            const float d = (float)step, inv = __builtin_amdgcn_rcpf(d);
            uint32_t c = 0;
            if (d > 0.f)
                c = (uint32_t)(code_of(x[i].x, d, inv) & 255) | (uint32_t)(code_of(x[i].y, d, inv) & 255) << 8 |
                    (uint32_t)(code_of(x[i].z, d, inv) & 255) << 16 | (uint32_t)code_of(x[i].w, d, inv) << 24;
            if (j < n4) {
                *(uint32_t*)(codes + row + in) = c;
                if ((threadIdx.x & 7) == 0) steps[(row + in) / KV8_BLOCK] = step;
            }
        }
    }
}

template <int TOK>
__global__ __launch_bounds__(KV8_THREADS) void kv_load_q8_kernel(float* __restrict__ k, float* __restrict__ v,
                                                                 int64_t ld, Kv8 kv, PackedBatch pb, int n_kv, int hd,
                                                                 int64_t head_stride) {
    const int t0 = blockIdx.x * TOK;
    float* dst = blockIdx.y ? v : k;
    const int8_t* codes = blockIdx.y ? kv.vq : kv.kq;
    const _Float16* steps = blockIdx.y ? kv.vs : kv.ks;
    const Sequences seqs(pb);
    int64_t row[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) row[i] = t0 + i < pb.T ? seqs.row_of(t0 + i, hd) : -1;
    const int n4 = n_kv * hd / 4;
    for (int j = threadIdx.x; j < n4; j += KV8_THREADS) {
        const int h = 4 * j / hd;
        const int64_t in = h * head_stride + (4 * j - h * hd);
        uint32_t c[TOK];
        float d[TOK];
#pragma unroll
        for (int i = 0; i < TOK; ++i)
            if (row[i] >= 0) {
                c[i] = *(const uint32_t*)(codes + row[i] + in);
                d[i] = (float)steps[(row[i] + in) / KV8_BLOCK];
            }
#pragma unroll
        for (int i = 0; i < TOK; ++i)
            if (row[i] >= 0)
                *(float4*)(dst + (int64_t)(t0 + i) * ld + 4 * j) =
                    make_float4(d[i] * (float)(int8_t)(c[i] & 255), d[i] * (float)(int8_t)(c[i] >> 8 & 255),
                                d[i] * (float)(int8_t)(c[i] >> 16 & 255), d[i] * (float)(int8_t)(c[i] >> 24));
    }
}

// Tokens of a workgroup: few tokens are spread over workgroups, many share the
// descriptors' latency.  Storing and loading 5592 tokens takes 39.4 us with one a
// workgroup, 32.9 with 2, 33.2 with 4 and 38.1 with 8.
constexpr int KV8_TOK = 4;
static bool kv8_one(const PackedBatch& pb) { return pb.T < 1024; }

int launch_kv_store_q8(int8_t* kq, _Float16* ks, int8_t* vq, _Float16* vs, const float* k, const float* v, int64_t ld,
                       const PackedBatch& pb, int n_kv, int hd, int64_t head_stride, hipStream_t s) {
    if (kv8_one(pb))
        hipLaunchKernelGGL(kv_store_q8_kernel<1>, dim3(pb.T, 2), dim3(KV8_THREADS), 0, s, kq, ks, vq, vs, k, v, ld, pb,
                           n_kv, hd, head_stride);
    else
        hipLaunchKernelGGL(kv_store_q8_kernel<KV8_TOK>, dim3((pb.T + KV8_TOK - 1) / KV8_TOK, 2), dim3(KV8_THREADS), 0,
                           s, kq, ks, vq, vs, k, v, ld, pb, n_kv, hd, head_stride);
    SH_CHECK_LAUNCH();
    return 0;
}

int launch_kv_load_q8(float* k, float* v, int64_t ld, const Kv8& kv, const PackedBatch& pb, int n_kv, int hd,
                      int64_t head_stride, hipStream_t s) {
    if (kv8_one(pb))
        hipLaunchKernelGGL(kv_load_q8_kernel<1>, dim3(pb.T, 2), dim3(KV8_THREADS), 0, s, k, v, ld, kv, pb, n_kv, hd,
                           head_stride);
    else
        hipLaunchKernelGGL(kv_load_q8_kernel<KV8_TOK>, dim3((pb.T + KV8_TOK - 1) / KV8_TOK, 2), dim3(KV8_THREADS), 0,
                           s, k, v, ld, kv, pb, n_kv, hd, head_stride);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
