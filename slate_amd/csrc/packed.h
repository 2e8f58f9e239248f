// packed.h -- packed batches of sequences over a K/V cache (the descriptors
// of slate_hip_kv_store_q8 and the attention entries beside it): device
// views of them, and the launchers.
#pragma once
#include "launch.h"

namespace slate_hip {

constexpr int PK_MAX_SEQ = 1024;       // sequences of a batch
constexpr int PK_MAX_DRAFT = 1024;     // drafted tokens of a sequence
constexpr int PK_MAX_HD = 512;
// Keys that a sequence can have in the attention kernels, which round counts of
// them up to 128 and step past the last ones in 32 bits.
constexpr int PK_MAX_KEYS = INT32_MAX - 1023;
constexpr int KV8_BLOCK = 32;          // elements that share a step

struct PackedBatch {
    const int32_t *tok_off, *pos0;
    const int64_t* kv_base;
    int B, T;
    int max_new;                       // tokens of a sequence (T where the call has no bound)
    int max_seq;
};

// A sequence's tokens: n of them from row t0 on (0: none, or numbers that do
// not fit), the first one's cache row p0.
struct SeqView {
    int t0, n, p0;
};
__device__ __forceinline__ SeqView seq_view(const PackedBatch& pb, int b) {
    const int t0 = pb.tok_off[b], t1 = pb.tok_off[b + 1], p0 = pb.pos0[b];
    const bool fits = t0 >= 0 && t1 >= t0 && t1 <= pb.T && t1 - t0 <= pb.max_new && p0 >= 0 &&
                      p0 <= pb.max_seq - (t1 - t0) && pb.kv_base[b] >= 0;
    return SeqView{t0, fits ? t1 - t0 : 0, p0};
}

// The last sequence whose first token is at or before t (tok_off does not
// fall), by one wave: every lane returns it; -1 if there is none.
__device__ __forceinline__ int find_seq(const PackedBatch& pb, int t) {
    int count = 0;
    for (int b = threadIdx.x & 63; b < ((pb.B + 63) & ~63); b += 64)
        count += __popcll(__builtin_amdgcn_ballot_w64(b < pb.B && pb.tok_off[b] <= t));
    return count - 1;
}

// 8-bit pools: codes, and the f16 step of each 32 of them.
struct Kv8 {
    const int8_t *kq, *vq;
    const _Float16 *ks, *vs;
};

// k_rope.hip
constexpr int ROPE_MAX_PAIRS = 256;
struct RopeTurns {
    double w[ROPE_MAX_PAIRS];          // turns per position of each pair
};
int launch_rope_scaled(float* y, const float* x, const int32_t* pos, int n_rows, int n_heads, int hd, int64_t ld,
                       int layout, int rot, float magnitude, const RopeTurns& turns, hipStream_t s);

// k_kv8.hip
int launch_kv_store_q8(int8_t* kq, _Float16* ks, int8_t* vq, _Float16* vs, const float* k, const float* v, int64_t ld,
                       const PackedBatch& pb, int n_kv, int hd, int64_t head_stride, hipStream_t s);
int launch_kv_load_q8(float* k, float* v, int64_t ld, const Kv8& kv, const PackedBatch& pb, int n_kv, int hd,
                      int64_t head_stride, hipStream_t s);

// k_attn_packed.hip.  parent: nullptr for causal attention.
struct PackedAttn {
    float* out;
    const float* q;
    const float *kf, *vf;              // f32 pools, or nullptr
    Kv8 kv8;                           // 8-bit pools where kf is nullptr
    const int32_t* parent;
    int Hq, Hkv, hd;
    int64_t head_stride;
    void* ws;
};
int64_t attention_packed_bytes(int Hq, int Hkv, int hd);
// k_attn_q8.hip: 8-bit pools, few query rows per (sequence, kv head).
bool attention_q8_few_takes(const PackedAttn& a, const PackedBatch& pb);
int64_t attention_q8_few_bytes(int hd);
int launch_attention_q8_few(const PackedAttn& a, const PackedBatch& pb, hipStream_t s);
// k_attn_many.hip: head_dim 32, 64, 128, either kind of pools, any rows.
bool attention_many_takes(const PackedAttn& a);
int64_t attention_many_bytes(int hd);
int launch_attention_many(const PackedAttn& a, const PackedBatch& pb, hipStream_t s);
// The most granules of keys that a call's blocks can have together; the kernels
// count them in 32 bits.
double attention_q8_few_most(const PackedAttn& a, const PackedBatch& pb);
double attention_many_most(const PackedAttn& a, const PackedBatch& pb);
bool attention_packed_fits(const PackedAttn& a, const PackedBatch& pb);
int launch_attention_packed(const PackedAttn& a, const PackedBatch& pb, hipStream_t s);

}  // namespace slate_hip
