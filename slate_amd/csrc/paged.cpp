// paged.cpp -- C entries of the K/V cache in pages and of the verification of
// drafted tokens (include/slate_hip.h).  Arguments are checked before the
// device is touched.
#include <mutex>

#include "paged.h"

namespace slate_hip {
extern std::mutex g_enqueue_mu;
}
using namespace slate_hip;

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int pages_check(const char* what, const Pages* pg) {
    SH_REQUIRE(pg && pg->table && pg->held && pg->free_pages && pg->n_free, "%s: null pointer", what);
    SH_REQUIRE(pg->n_slots >= 1 && pg->max_pages >= 1 && pg->n_pages >= 1 && pg->page_size >= 1 &&
                   (int64_t)pg->n_pages * pg->page_size <= PK_MAX_KEYS &&
                   (int64_t)pg->max_pages * pg->page_size <= PK_MAX_KEYS,
               "%s: %d slots of %d pages, %d pages of %d rows", what, pg->n_slots, pg->max_pages, pg->n_pages,
               pg->page_size);
    return 0;
}

int kv_check(const char* what, const slate_hip_paged_kv_t* kv) {
    SH_REQUIRE(kv && kv->K && kv->V, "%s: null pointer", what);
    SH_REQUIRE(kv->dtype >= KV_F32 && kv->dtype <= KV_BF16, "%s: dtype=%d", what, kv->dtype);
    SH_REQUIRE(kv->n_kv_heads >= 1 && kv->n_kv_heads <= 65535 && kv->head_dim >= 8 && kv->head_dim <= PG_MAX_HD &&
                   kv->head_dim % 8 == 0,
               "%s: %d heads of %d", what, kv->n_kv_heads, kv->head_dim);
    SH_REQUIRE(kv->page_stride >= 0 && kv->head_stride >= 0 && kv->row_stride >= kv->head_dim &&
                   kv->row_stride <= PG_MAX_ROW_STRIDE && kv->page_stride % 8 == 0 && kv->head_stride % 8 == 0 &&
                   kv->row_stride % 8 == 0,
               "%s: strides of %lld, %lld and %lld", what, (long long)kv->page_stride, (long long)kv->head_stride,
               (long long)kv->row_stride);
    SH_REQUIRE(aligned16(kv->K) && aligned16(kv->V), "%s: pools are not 16-byte aligned", what);
    return 0;
}

bool overlap(const void* a, size_t n, const void* b, size_t m) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + m && y < x + n;
}

// The caller's workspace, or the backend's where there is none; nullptr with
// *rc set if it can be neither.  Called under g_enqueue_mu.
void* workspace(const char* what, void* ws, size_t need, int slot, int* rc) {
    if (ws) return ws;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    const hipError_t e = hipStreamIsCapturing(stream(), &st);
    if (e != hipSuccess) {
        set_error(-7, "%s: hipStreamIsCapturing failed: %s", what, hipGetErrorString(e));
        *rc = -7;
        return nullptr;
    }
    if (st != hipStreamCaptureStatusNone) {
        set_error(-5, "%s: a captured call needs a workspace of its own", what);
        *rc = -5;
        return nullptr;
    }
    void* p = scratch(slot, need);
    if (!p) *rc = -2;
    return p;
}

bool heads_ok(int Hq, int Hkv, int hd) {
    return Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 65535 && hd >= 8 && hd <= PG_MAX_HD && hd % 8 == 0;
}

}  // namespace

extern "C" {

int slate_hip_pages_reset(const slate_hip_pages_t* pages) {
    const int rc = pages_check("pages_reset", pages);
    if (rc) return rc;
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_pages_reset(*pages, stream());
}

int slate_hip_pages_extend(const slate_hip_pages_t* pages, const int32_t* slot, const int32_t* pos0,
                           const int32_t* n_new, int B, int T_cap, int32_t* tok_off, int32_t* tok2seq,
                           int32_t* tok_pos, int32_t* tok_row, int32_t* last_tok, int32_t* status) {
    const int rc = pages_check("pages_extend", pages);
    if (rc) return rc;
    SH_REQUIRE(slot && pos0 && n_new && tok_off && tok2seq && tok_pos && tok_row && last_tok && status,
               "pages_extend: null pointer");
    SH_REQUIRE(B >= 1 && B <= PK_MAX_SEQ && T_cap >= 0, "pages_extend: bad sizes (B=%d, T_cap=%d)", B, T_cap);
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_pages_extend(*pages, slot, pos0, n_new, B, T_cap, tok_off, tok2seq, tok_pos, tok_row, last_tok,
                               status, stream());
}

int slate_hip_pages_trim(const slate_hip_pages_t* pages, const int32_t* slot, const int32_t* length, int B,
                         int32_t* status) {
    const int rc = pages_check("pages_trim", pages);
    if (rc) return rc;
    SH_REQUIRE(slot && length && status, "pages_trim: null pointer");
    SH_REQUIRE(B >= 1 && B <= PK_MAX_SEQ, "pages_trim: B=%d", B);
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_pages_trim(*pages, slot, length, B, status, stream());
}

int slate_hip_kv_store_paged(const slate_hip_paged_kv_t* kv, const slate_hip_pages_t* pages, const float* k,
                             const float* v, int64_t ld, const int32_t* tok_row, int T) {
    int rc = kv_check("kv_store_paged", kv);
    if (!rc) rc = pages_check("kv_store_paged", pages);
    if (rc) return rc;
    SH_REQUIRE(k && v && tok_row, "kv_store_paged: null pointer");
    SH_REQUIRE(T >= 1 && (int64_t)kv->n_kv_heads * kv->head_dim <= ld && ld % 4 == 0, "kv_store_paged: T=%d, ld=%lld",
               T, (long long)ld);
    SH_REQUIRE(aligned16(k) && aligned16(v), "kv_store_paged: rows are not 16-byte aligned");
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_kv_store_paged(*kv, *pages, k, v, ld, tok_row, T, stream());
}

int64_t slate_hip_attention_paged_bytes(int n_q_heads, int n_kv_heads, int head_dim) {
    return heads_ok(n_q_heads, n_kv_heads, head_dim) ? attention_paged_bytes(head_dim) : -1;
}

int slate_hip_attention_paged(float* out, const float* q, const slate_hip_paged_kv_t* kv,
                              const slate_hip_pages_t* pages, const int32_t* slot, const int32_t* tok_off,
                              const int32_t* pos0, int B, int T, int max_new, int n_q_heads, void* ws,
                              size_t ws_bytes) {
    int rc = kv_check("attention_paged", kv);
    if (!rc) rc = pages_check("attention_paged", pages);
    if (rc) return rc;
    SH_REQUIRE(out && q && slot && tok_off && pos0, "attention_paged: null pointer");
    SH_REQUIRE(B >= 1 && B <= PK_MAX_SEQ && T >= 1 && max_new >= 1, "attention_paged: bad sizes (B=%d, T=%d, max_new=%d)",
               B, T, max_new);
    SH_REQUIRE(heads_ok(n_q_heads, kv->n_kv_heads, kv->head_dim), "attention_paged: %d/%d heads", n_q_heads,
               kv->n_kv_heads);
    const int max_seq = pages->max_pages * pages->page_size;
    const double blocks = (double)T * (n_q_heads / kv->n_kv_heads) / 16 + B;
    SH_REQUIRE((int64_t)T * n_q_heads <= INT32_MAX - 127 &&
                   kv->n_kv_heads * blocks * ((max_seq + 127) / 128) < 2147483648.0,
               "attention_paged: %d tokens over %d rows are too much for one call", T, max_seq);
    const size_t bytes = (size_t)T * n_q_heads * kv->head_dim * sizeof(float);
    SH_REQUIRE(!overlap(out, bytes, q, bytes), "attention_paged: out overlaps q");
    const size_t need = (size_t)attention_paged_bytes(kv->head_dim);
    SH_REQUIRE(!ws || (aligned16(ws) && ws_bytes >= need),
               "attention_paged: workspace of %zu bytes, %zu are needed (aligned)", ws_bytes, need);
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    ws = workspace("attention_paged", ws, need, 8, &rc);
    if (rc) return rc;
    return launch_attention_paged(PagedAttn{out, q, *kv, *pages, n_q_heads, ws},
                                  PagedBatch{slot, tok_off, pos0, B, T, max_new, pages->n_slots, max_seq}, stream());
}

int64_t slate_hip_verify_drafts_bytes(int B, int T, int V) {
    return B < 1 || B > PK_MAX_SEQ || T < 1 || V < 1 || V > PK_MAX_KEYS ? -1 : verify_drafts_bytes(B, T, V);
}

int slate_hip_verify_drafts(int32_t* n_accepted, int32_t* out_tok, int32_t* out_row, const float* logits, int64_t ld,
                            const int32_t* token, const int32_t* parent, const float* draft_probs, int64_t draft_ld,
                            const float* temperature, const float* u, const float* u_next, const int32_t* tok_off,
                            int B, int T, int V, void* ws, size_t ws_bytes) {
    SH_REQUIRE(n_accepted && out_tok && logits && token && u && u_next && tok_off, "verify_drafts: null pointer");
    SH_REQUIRE(B >= 1 && B <= PK_MAX_SEQ && T >= 1 && V >= 1 && V <= PK_MAX_KEYS,
               "verify_drafts: bad sizes (B=%d, T=%d, V=%d)", B, T, V);
    SH_REQUIRE(ld >= V && (!draft_probs || draft_ld >= V), "verify_drafts: rows of %d, ld=%lld, draft_ld=%lld", V,
               (long long)ld, (long long)draft_ld);
    SH_REQUIRE(!draft_probs || !parent, "verify_drafts: draft_probs are for chains (parent NULL)");
    const size_t need = (size_t)verify_drafts_bytes(B, T, V);
    SH_REQUIRE(!ws || (aligned16(ws) && ws_bytes >= need),
               "verify_drafts: workspace of %zu bytes, %zu are needed (aligned)", ws_bytes, need);
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    int rc = 0;
    ws = workspace("verify_drafts", ws, need, 9, &rc);
    if (rc) return rc;
    return launch_verify_drafts(VerifyArgs{n_accepted, out_tok, out_row, logits, draft_probs, temperature, u, u_next,
                                           token, parent, tok_off, ld, draft_ld, B, T, V, ws},
                                stream());
}

}  // extern "C"
