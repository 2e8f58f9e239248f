// paged.h -- a K/V cache in pages: device views of the descriptors, and the
// launchers of the page table's upkeep, the row store, the attention over
// pages and the verification of drafted tokens.
#pragma once
#include "packed.h"

namespace slate_hip {

constexpr int PG_MAX_HD = 256;
constexpr int64_t PG_MAX_ROW_STRIDE = 1 << 26;

enum KvType { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

using Pages = slate_hip_pages_t;

// k_pages.hip
int launch_pages_reset(const Pages& pg, hipStream_t s);
int launch_pages_extend(const Pages& pg, const int32_t* slot, const int32_t* pos0, const int32_t* n_new, int B,
                        int T_cap, int32_t* tok_off, int32_t* tok2seq, int32_t* tok_pos, int32_t* tok_row,
                        int32_t* last_tok, int32_t* status, hipStream_t s);
int launch_pages_trim(const Pages& pg, const int32_t* slot, const int32_t* length, int B, int32_t* status,
                      hipStream_t s);
int launch_kv_store_paged(const slate_hip_paged_kv_t& kv, const Pages& pg, const float* k, const float* v, int64_t ld,
                          const int32_t* tok_row, int T, hipStream_t s);

// k_attn_paged.hip
struct PagedAttn {
    float* out;
    const float* q;
    slate_hip_paged_kv_t kv;
    Pages pg;
    int Hq;
    void* ws;
};
struct PagedBatch {
    const int32_t *slot, *tok_off, *pos0;
    int B, T, max_new, n_slots;
    int max_seq;                       // rows that a slot can have
};
__device__ __forceinline__ SeqView seq_view(const PagedBatch& pb, int b) {
    const int t0 = pb.tok_off[b], t1 = pb.tok_off[b + 1], p0 = pb.pos0[b], slot = pb.slot[b];
    const bool fits = t0 >= 0 && t1 >= t0 && t1 <= pb.T && t1 - t0 <= pb.max_new && p0 >= 0 &&
                      p0 <= pb.max_seq - (t1 - t0) && slot >= 0 && slot < pb.n_slots;
    return SeqView{t0, fits ? t1 - t0 : 0, p0};
}
__device__ __forceinline__ int64_t seq_base(const PagedBatch& pb, int b) { return pb.slot[b]; }
int64_t attention_paged_bytes(int hd);
int launch_attention_paged(const PagedAttn& a, const PagedBatch& pb, hipStream_t s);

// k_verify.hip
struct VerifyArgs {
    int32_t *n_accepted, *out_tok, *out_row;
    const float *logits, *q, *temperature, *u, *u_next;
    const int32_t *token, *parent, *tok_off;
    int64_t ld, q_ld;
    int B, T, V;
    void* ws;
};
int64_t verify_drafts_bytes(int B, int T, int V);
int launch_verify_drafts(const VerifyArgs& a, hipStream_t s);

}  // namespace slate_hip
