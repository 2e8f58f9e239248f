/*
 * slate_hip.h -- C ABI of the MI355X (gfx950) HIP compute backend for slate.
 *
 * Everything here is plain C: pointers, sizes and ints, no C++ types, no
 * exceptions.  Pointers documented as "device" come from the backend's
 * alloc() (or slate_hip_alloc); "host" pointers are ordinary memory.
 *
 * 1. slate_backend_hip() returns the drop-in vtable.  Its first 14 members
 *    are slate_backend_t exactly as include/slate/backend.h:41-99 declares
 *    it (same order, same signatures, same meaning), so slate's engines call
 *    it unchanged; the extension entries follow `sync`.
 * 2. slate_hip_* functions are the same entry points under stable names for
 *    FFI binders, plus the extensions the vtable appends.
 * 3. slate_hip_llama_* is a device-resident LLaMA engine with the session API
 *    of include/slate/llama.h:124-139 and a ragged continuous-batching step
 *    generalising slate_infer_batch_step (include/slate/infer.h:170-187).
 *
 * Errors: vtable compute entries return void (backend.h:58-98), so failures
 * are recorded in a sticky per-process error that slate_hip_last_error()
 * reports and slate_hip_clear_error() resets; int-returning entries return
 * 0 on success and a negative code: -1 bad argument, -2 cache full /
 * capacity exceeded, -3 bad token (llama_infer.c:144-145), -5 not
 * supported, -7 device/runtime failure.
 *
 * Threading: all work is enqueued on one backend stream created at first
 * use (default priority); entries may be called from several host threads;
 * sync() waits for everything enqueued so far.
 */
#ifndef SLATE_HIP_H
#define SLATE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- slate_backend_t (include/slate/backend.h:41-99) ----------------------
 * When slate's own header is visible -- already included, or reachable as
 * "slate/backend.h" on the include path -- it is used as is, factories
 * (backend.h:104-110) included.  Otherwise the same struct is declared here,
 * member for member, under this header's own guard; slate's guard
 * SLATE_BACKEND_H is never defined here, so a translation unit that later
 * includes slate/backend.h by another path gets a loud redefinition error
 * rather than a silently skipped header.  In a TU that uses both headers,
 * put slate's include/ directory on the include path (or include
 * slate/backend.h first). */
#if !defined(SLATE_BACKEND_H) && defined(__has_include)
#if __has_include("slate/backend.h")
#include "slate/backend.h"
#endif
#endif
#if !defined(SLATE_BACKEND_H) && !defined(SLATE_HIP_BACKEND_T_DECLARED)
#define SLATE_HIP_BACKEND_T_DECLARED 1
typedef struct slate_backend {
    const char* name;
    void* (*alloc)(size_t bytes);
    void  (*release)(void* dev_ptr);
    void  (*copy_h2d)(void* dst_dev, const void* src_host, size_t bytes);
    void  (*copy_d2h)(void* dst_host, const void* src_dev, size_t bytes);
    void  (*matvec)(float* y, const float* A, const float* x, int M, int K);
    void  (*linear_batch)(float* C, const float* X, const float* W, int B, int K, int N);
    void  (*matvec_q4k)(float* y, const void* A_q4k, const float* x, int M, int K);
    void  (*rmsnorm_row)(float* y, const float* x, const float* w, int D, float eps);
    void  (*silu_mul)(float* y, const float* gate, const float* up, int H);
    void  (*add_inplace)(float* y, const float* x, int D);
    void  (*embed_lookup)(float* y, const float* W, int token_id, int D);
    void  (*attention_step)(float* out, const float* q, const float* K_cache,
                            const float* V_cache, float* scores, int L, int D);
    void  (*sync)(void);
} slate_backend_t;
#endif

/* Vtable extended past `sync`.  slate_backend_hip() returns &ext.base. */
typedef struct slate_hip_backend {
    slate_backend_t base;
    /* Y[B,M] = X[B,K] @ dequant(A)[M,K]^T; A is M rows of K/256 Q4_K blocks. */
    int  (*matmul_q4k)(float* Y, const void* A_q4k, const float* X, int B, int M, int K);
    /* Bit-exact dequantisation (quant.c:168-202), n % 256 == 0. */
    int  (*dequant_q4k)(float* dst, const void* A_q4k, int64_t n);
    /* y[b,:] = rmsnorm(x[b,:]) * w for B rows. */
    int  (*rmsnorm_rows)(float* y, const float* x, const float* w, int B, int D, float eps);
    /* Row-wise RoPE (llama_infer.c:77-92) with per-row positions (device
     * int32[n_rows]); |pos| must be < max_pos. */
    int  (*rope_rows)(float* x, const int32_t* pos, int n_rows, int n_heads, int head_dim,
                      float theta_base, int max_pos);
    /* Greedy argmax per row, lowest index on ties (sampling.c:14-18). */
    int  (*argmax_rows)(int32_t* out, const float* logits, int B, int V);
    const char* (*last_error)(void);
} slate_hip_backend_t;

/* NULL when no gfx950 device can be opened (like the reference's stubs). */
const slate_backend_t* slate_backend_hip(void);                 /* replaces backend_cuda_stub.c:33 */
/* The same kernels behind host-visible memory, for callers that treat the
 * backend's memory as host memory (slate's toy engine memcpy's into its KV
 * cache and passes module weights from host memory, src/infer/engine.c:
 * 276-277, 411-412, 586-591): alloc returns pinned host memory the device
 * reads directly, compute entries copy pageable arguments through device
 * buffers and return after their kernel has finished.  Correct, slow; for
 * running slate_infer_engine_new_ex (infer.h:90-96) unchanged.  NULL
 * without a gfx950 device. */
const slate_backend_t* slate_backend_hip_compat(void);

/* ---- errors -------------------------------------------------------------- */
const char* slate_hip_last_error(void);  /* NULL when no error is pending */
void        slate_hip_clear_error(void);

/* ---- the vtable entries under stable names (backend.h:41-99) -------------- */
void* slate_hip_alloc(size_t bytes);                                          /* backend.h:45 */
void  slate_hip_release(void* dev);                                           /* backend.h:46 */
void  slate_hip_copy_h2d(void* dst_dev, const void* src_host, size_t bytes);  /* backend.h:49 */
void  slate_hip_copy_d2h(void* dst_host, const void* src_dev, size_t bytes);  /* backend.h:50 */
void  slate_hip_matvec(float* y, const float* A, const float* x, int M, int K);           /* backend.h:56 */
void  slate_hip_linear_batch(float* C, const float* X, const float* W, int B, int K, int N); /* backend.h:60-61 */
void  slate_hip_matvec_q4k(float* y, const void* A_q4k, const float* x, int M, int K);     /* backend.h:68 */
void  slate_hip_rmsnorm_row(float* y, const float* x, const float* w, int D, float eps);   /* backend.h:71-72 */
void  slate_hip_silu_mul(float* y, const float* gate, const float* up, int H);            /* backend.h:76 */
void  slate_hip_add_inplace(float* y, const float* x, int D);                             /* backend.h:79 */
void  slate_hip_embed_lookup(float* y, const float* W, int token_id, int D);              /* backend.h:82 */
void  slate_hip_attention_step(float* out, const float* q, const float* K_cache,
                               const float* V_cache, float* scores, int L, int D);        /* backend.h:91-93 */
void  slate_hip_sync(void);                                                               /* backend.h:96 */

/* ---- extensions (device pointers, enqueued on the backend stream) -------- */
int   slate_hip_matmul_q4k(float* Y, const void* A_q4k, const float* X, int B, int M, int K);
int   slate_hip_dequant_q4k(float* dst, const void* A_q4k, int64_t n);
/* Tiled Q4_K: the same blocks regrouped into 16-row tiles so that each
 * tile's block kb is 2304 contiguous bytes (16 headers, then the nibbles in
 * the order the matmul lanes read them); rows past M are zero.  It replaces
 * the row layout of quant.c:135-166 only in device memory owned by the
 * caller; the values and results are identical.  q4k_tile converts M rows
 * of K/256 blocks (device src, row layout) into dst of q4k_tiled_bytes. */
int64_t slate_hip_q4k_tiled_bytes(int M, int K);
int   slate_hip_q4k_tile(void* dst_tiled, const void* src_q4k, int M, int K);
int   slate_hip_matmul_q4k_tiled(float* Y, const void* A_tiled, const float* X, int B, int M, int K);
/* slate_hip_matmul_q4k that allocates nothing, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid it); no counterpart in slate.  Same inputs,
 * outputs and results; the activation operand and split-K partials live in
 * a fixed 32 MiB device array of the library, so calls whose operand plus
 * one split of partials ((16-row-padded B) * M * 4 bytes) exceed it return
 * -1 with an error naming the limit.  Calls are serialised on the backend
 * stream; work on that array from another stream (a replay of a captured
 * call next to new calls, say) would race with it. */
int   slate_hip_matmul_q4k_noalloc(float* Y, const void* A_q4k, const float* X, int B, int M, int K);
/* Q8_0 (34-byte blocks [f16 d][32 x int8], quant.h:16-31), device pointers.
 * q8_0_matvec has slate_q8_0_matvec's signature and meaning (quant.c:126-133,
 * y[m] = sum_k d*q[m,k] * x[k], K % 32 == 0); matmul_q8_0 is B such calls in
 * one launch (Y[B,M] = X[B,K] @ dequant(A)[M,K]^T); dequant_q8_0 is
 * slate_dequant_q8_0 (quant.c:12-25), bit-exact, n % 32 == 0.  Sums are in
 * another order than the reference's eight AVX2 lanes (float tolerance). */
void  slate_hip_q8_0_matvec(float* y, const void* A_q8, const float* x, int M, int K);  /* quant.h:31 */
int   slate_hip_matmul_q8_0(float* Y, const void* A_q8, const float* X, int B, int M, int K);
int   slate_hip_dequant_q8_0(float* dst, const void* A_q8, int64_t n);                   /* quant.h:24 */
/* Tiled Q8_0: the same bytes regrouped into 16-row x 256-element tiles of
 * 4352 bytes (the eight d of each row, then the int8 weights in the order
 * the matmul lanes read them); rows past M and blocks past K/32 are zero.
 * From two rows on, matmul_q8_0 regroups into backend scratch on every call;
 * callers that keep weights resident tile them once with q8_0_tile (device
 * src, row layout, into dst of q8_0_tiled_bytes) and call matmul_q8_0_tiled
 * (same results). */
int64_t slate_hip_q8_0_tiled_bytes(int M, int K);
int   slate_hip_q8_0_tile(void* dst_tiled, const void* src_q8, int M, int K);
int   slate_hip_matmul_q8_0_tiled(float* Y, const void* A_tiled, const float* X, int B, int M, int K);
int   slate_hip_rmsnorm_rows(float* y, const float* x, const float* w, int B, int D, float eps);
/* RoPE with the angles of llama_infer.c:83-86 (host powf/cosf/sinf table,
 * so identical inputs rotate bit-identically); rows with |pos| >= max_pos
 * are left unchanged and make the call return -1. */
int   slate_hip_rope_rows(float* x, const int32_t* pos, int n_rows, int n_heads, int head_dim,
                          float theta_base, int max_pos);
/* The host table behind rope_rows: cs[(p*hd/2 + i)*2 + {0,1}] = {cos, sin}. */
void  slate_hip_rope_table(float* cs, int max_pos, int head_dim, float theta_base);
int   slate_hip_argmax_rows(int32_t* out, const float* logits, int B, int V);

/* Ragged-batch packing on the device.  Inputs (device int32[B]): slot,
 * pos0 (positions already cached), n_new (>= 1 tokens this step).  Outputs
 * (device): tok_off[B+1] (exclusive prefix sum of n_new), tok2seq[T],
 * tok_pos[T], kv_base[B] (int64 float offset slot*slot_stride), last_tok[B].
 * Invalid descriptors (n_new < 1, pos0 + n_new > max_seq) are reported in
 * status[0] (0 ok, -1, -2) and produce no index writes. */
int   slate_hip_pack_batch(const int32_t* slot, const int32_t* pos0, const int32_t* n_new,
                           int B, int max_seq, int64_t slot_stride, int T_cap,
                           int32_t* tok_off, int32_t* tok2seq, int32_t* tok_pos,
                           int64_t* kv_base, int32_t* last_tok, int32_t* status);

/* Ragged GQA attention over per-sequence KV caches, split over key chunks.
 * q      : [T, n_q_heads*hd] post-RoPE queries, packed token-major
 * kv     : K and V pools; the cache of kv head h of the sequence that owns
 *          token t starts at kv_base[tok2seq[t]] + h*head_stride and holds
 *          [max_seq, hd] rows (key position-major); any float offset is
 *          taken, rows that start on 16 bytes are read fastest
 * token t attends to key positions 0..tok_pos[t] of its own sequence.
 * out    : [T, n_q_heads*hd].  scale = 1/sqrtf(hd) as llama_infer.c:104. */
int   slate_hip_attention_ragged(float* out, const float* q, const float* Kpool,
                                 const float* Vpool, const int32_t* tok2seq,
                                 const int32_t* tok_pos, const int64_t* kv_base,
                                 int T, int n_q_heads, int n_kv_heads, int head_dim,
                                 int64_t head_stride, int max_pos);

/* Rotary positions beyond rope_rows: pairs in halves or interleaved, part of
 * a head, frequencies rescaled for contexts longer than the trained one, any
 * position.  Pair i < rot_dim/2 turns by pos * w_i and is multiplied by
 * `magnitude`; the elements past rot_dim are copied.  w_i starts as
 * theta_base^(-2i/rot_dim) and `scaling` changes it:
 *   0  not at all;
 *   1  w_i / factor (every position is divided);
 *   2  by how often the pair turns in the trained context, t = orig_ctx * w_i
 *      / 2 pi: t <= low gives w_i / factor, t >= high keeps w_i, in between
 *      the two are mixed linearly in t;
 *   3  (YaRN) by the pair's index: the pairs that turn `high` and `low` times
 *      are x(t) = rot_dim * ln(orig_ctx / (2 pi t)) / (2 ln theta_base); up
 *      to a = max(0, floor x(high)) w_i is kept, from b = min(rot_dim - 1,
 *      ceil x(low)) on it is w_i / factor, in between mixed linearly in i.
 * Angles are formed and reduced to one turn in 64 bits, so far positions are
 * as exact as near ones; the rotation is in f32. */
typedef struct slate_hip_rope {
    int    layout;      /* 0: pairs (i, i + rot_dim/2) as rope_rows, 1: pairs (2i, 2i + 1) */
    int    rot_dim;     /* even, 2 .. min(head_dim, 512) */
    int    scaling;     /* 0 .. 3, above */
    int    orig_ctx;    /* scaling 2 and 3: positions of the trained context, >= 1 */
    double theta_base;  /* > 0 (scaling 3: > 1) */
    double factor;      /* scaling 1 .. 3: > 0 */
    double low, high;   /* scaling 2 and 3: turns, 0 < low < high */
    double magnitude;   /* 0: the default, 0.1 ln(factor) + 1 for scaling 3 (1 where factor <= 1), else 1 */
} slate_hip_rope_t;
/* y[row, head, :] = the rotated x[row, head, :]; rows are ld floats apart in
 * both (ld >= n_heads * head_dim).  pos is device int32[n_rows], any value: a
 * negative position turns backwards (the transpose of the rotation, which is
 * also its gradient; `magnitude` multiplies either way).  y is x (in place)
 * or does not overlap it. */
int   slate_hip_rope_scaled(float* y, const float* x, const int32_t* pos, int n_rows, int n_heads, int head_dim,
                            int64_t ld, const slate_hip_rope_t* rope);
/* The w_i (host double[rot_dim/2]) and the magnitude behind rope_scaled;
 * host only, needs no device.  -1 for a configuration rope_scaled refuses. */
int   slate_hip_rope_frequencies(double* w, double* magnitude, const slate_hip_rope_t* rope);

/* ---- packed batches over an 8-bit K/V cache, and drafted tokens ------------
 * The entries below take a batch as pack_batch lays it out: B sequences
 * (1 .. 1024) of T token rows in all, sequence b's tokens being the rows
 * tok_off[b] .. tok_off[b+1]-1 (device int32[B+1], not falling); pos0[b]
 * (device int32[B]) rows of it are cached already, and its token i belongs to
 * cache row pos0[b] + i.  Row p of kv head h starts at element
 * kv_base[b] + h * head_stride + p * head_dim of a pool (device int64[B];
 * offsets may pass 32 bits).  A sequence may have no token in a call.  One whose
 * numbers do not fit (tok_off falling or outside 0 .. T, more than max_new
 * tokens where the call has that bound, pos0 < 0, pos0 + tokens > max_seq,
 * kv_base < 0) is left out: nothing of it is read or written.  (In attention
 * a max_seq above 2^31 - 1024 counts as that.)  Behind a fall
 * of tok_off sequences may be left out too.  Rows of the outputs that no
 * sequence owns stay as they were.
 * The 8-bit pools: int8 codes (device, 16-byte aligned), and the f16 steps
 * (uint16_t bits, 16-byte aligned) of each 32 codes, the step of element e
 * at index e / 32.  A value is step * code: the values of Q8_0, in two pools
 * so that rows are read in whole 16-byte loads.  In these pools kv_base and
 * head_stride are multiples of head_dim (a kv_base that is not is rounded down
 * to one) and head_dim is a multiple of 32. */

/* Quantise new K and V rows into the cache: k, v [T, n_kv_heads * head_dim]
 * f32 (16-byte aligned), rows ld floats apart (ld % 4 == 0).  Per 32 elements
 * step = f16(max|x| / 127) (at most 65504) and code = x / step to the nearest
 * whole number, ties to even, within -127 .. 127; a block whose step rounds
 * to 0 gets codes 0.  NaN counts as 0.  Rows that two sequences of one call
 * both write (they share cache rows) end up undefined. */
int   slate_hip_kv_store_q8(int8_t* Kq, uint16_t* Ks, int8_t* Vq, uint16_t* Vs, const float* k, const float* v,
                            int64_t ld, const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base, int B,
                            int T, int n_kv_heads, int head_dim, int64_t head_stride, int max_seq);
/* The same rows of the cache back as f32 (step * code, exact in f32). */
int   slate_hip_kv_load_q8(float* k, float* v, int64_t ld, const int8_t* Kq, const uint16_t* Ks, const int8_t* Vq,
                           const uint16_t* Vs, const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base,
                           int B, int T, int n_kv_heads, int head_dim, int64_t head_stride, int max_seq);
/* Causal GQA attention over the 8-bit cache: q, out [T, n_q_heads * head_dim]
 * f32 (out is not q); token i of sequence b attends to rows 0 .. pos0[b] + i
 * (its own is stored before the call).  n_q_heads is a multiple of
 * n_kv_heads; query head g belongs to kv head g / (n_q_heads / n_kv_heads).
 * Scores are q.k / sqrt(head_dim), as attention_ragged's.  max_new bounds the
 * tokens that one sequence brings (1 for a decode step); head_dim is at most
 * 512; 32, 64 and 128 run on the matrix instructions, the others on a plain
 * kernel in f32.  Queries must be finite and, like the cache's values, below
 * 2^100 in size.  On the matrix instructions queries, weights and f32 values
 * have 22 bits, sums are f32, and V counts by what is largest in it: an f32
 * value is resolved to 2^-22 of its row's largest (and to 2^-114), an 8-bit one
 * to 2^-24 of the largest in the 32 cache rows around it, and what a key adds to
 * the sum to 2^-33 of the largest weight times the largest V of all keys seen,
 * also where that V has no weight.  What the cache holds in rows a token does
 * not see never matters.
 * T * n_q_heads <= 2^31 - 128, and the kernels count blocks of query rows times pieces
 * of keys in 32 bits: where n_kv_heads * (T * n_q_heads / n_kv_heads / 128 + B)
 * * max_seq / 64 (or, for max_new * n_q_heads / n_kv_heads <= 48 and max_new
 * <= 32, / 16 and / 128) reaches 2^31 the call is refused.
 * ws: device scratch of slate_hip_attention_packed_bytes, 16-byte aligned,
 * its content of no matter, for calls that run beside each other or are
 * captured into graphs that do; NULL takes the backend's own, which calls on
 * the backend stream share (a call under stream capture is then refused with
 * -5). */
int   slate_hip_attention_ragged_q8(float* out, const float* q, const int8_t* Kq, const uint16_t* Ks,
                                    const int8_t* Vq, const uint16_t* Vs, const int32_t* tok_off,
                                    const int32_t* pos0, const int64_t* kv_base, int B, int T, int max_new,
                                    int n_q_heads, int n_kv_heads, int head_dim, int64_t head_stride, int max_seq,
                                    void* ws, size_t ws_bytes);
/* Attention of drafted tokens that form trees: sequence b's tokens are drafts
 * after its pos0[b] committed rows, K/V of draft i stored in row pos0[b] + i.
 * parent[t] (device int32[T]) is the draft, counted within its sequence, that
 * token t continues, or -1 where it continues the committed text; it comes
 * before its child (parent[t] < the token's own number; any other value is
 * taken as -1).  A token attends to the committed rows, to its ancestors and
 * to itself.  max_new <= 1024.  K/V in f32 pools as attention_ragged's
 * (kv_base and head_stride any), or in the 8-bit pools; head_dim of f32
 * pools is a multiple of 16. */
int   slate_hip_attention_tree(float* out, const float* q, const float* Kpool, const float* Vpool,
                               const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base,
                               const int32_t* parent, int B, int T, int max_new, int n_q_heads, int n_kv_heads,
                               int head_dim, int64_t head_stride, int max_seq, void* ws, size_t ws_bytes);
int   slate_hip_attention_tree_q8(float* out, const float* q, const int8_t* Kq, const uint16_t* Ks,
                                  const int8_t* Vq, const uint16_t* Vs, const int32_t* tok_off,
                                  const int32_t* pos0, const int64_t* kv_base, const int32_t* parent, int B, int T,
                                  int max_new, int n_q_heads, int n_kv_heads, int head_dim, int64_t head_stride,
                                  int max_seq, void* ws, size_t ws_bytes);
/* Bytes of ws that the three take for these heads, whatever the batch; -1 for
 * heads they refuse. */
int64_t slate_hip_attention_packed_bytes(int n_q_heads, int n_kv_heads, int head_dim);

/* ---- a K/V cache in pages, and verification of drafted tokens --------------
 * The cache's rows are given out in pages of page_size rows to n_slots slots (a
 * sequence has one).  All arrays are the caller's (device); pages_reset fills
 * them.  Page table[s * max_pages + i] holds the rows i * page_size .. of slot s,
 * for i < held[s]; entries behind are -1.  free_pages[0 .. n_free[0]-1] are the
 * pages that no slot has, the last is taken first.  n_pages * page_size and
 * max_pages * page_size are at most 2^31 - 1024. */
typedef struct slate_hip_pages {
    int32_t *table, *held, *free_pages, *n_free;   /* [n_slots * max_pages], [n_slots], [n_pages], [1] */
    int n_slots, max_pages, n_pages, page_size;
} slate_hip_pages_t;
/* The pools of K and V (device, 16-byte aligned) and where in them row r (0 ..
 * page_size-1) of page p of head h is: its head_dim elements start at element p *
 * page_stride + h * head_stride + r * row_stride.  Strides are multiples of 8, row_stride
 * at least head_dim and at most 2^26, so any order of page, head and row will do;
 * head_dim is a multiple of 8, at most 256. */
typedef struct slate_hip_paged_kv {
    void *K, *V;
    int dtype;                                     /* 0: f32, 1: f16, 2: bf16 */
    int n_kv_heads, head_dim;
    int64_t page_stride, head_stride, row_stride;
} slate_hip_paged_kv_t;

/* All pages free (page 0 is taken first), no slot has any. */
int   slate_hip_pages_reset(const slate_hip_pages_t* pages);
/* Take the pages that a step's new tokens need, and lay its batch out as
 * pack_batch does.  Sequence b (of B, 1 .. 1024) has slot[b], pos0[b] rows cached
 * and brings n_new[b] >= 0 tokens (device int32[B] each): its slot gets the pages
 * that hold pos0 + n_new rows, if it has fewer, sequence after sequence.  Outputs
 * (device): tok_off[B+1]; of every token its sequence tok2seq[T], position
 * tok_pos[T] and cache row tok_row[T] (page * page_size + row within it, where
 * kv_store_paged puts it; -1 where the table names no page); last_tok[B] (-1 for
 * a sequence without tokens).  status[0] says 0, or, with nothing else written:
 * -1 bad descriptor (a negative number, a slot outside 0 .. n_slots-1 or in two
 * sequences, held or n_free outside their ranges), -2 more rows than a slot can
 * have, more tokens than T_cap or more pages than are free. */
int   slate_hip_pages_extend(const slate_hip_pages_t* pages, const int32_t* slot, const int32_t* pos0,
                             const int32_t* n_new, int B, int T_cap, int32_t* tok_off, int32_t* tok2seq,
                             int32_t* tok_pos, int32_t* tok_row, int32_t* last_tok, int32_t* status);
/* Give back the pages behind the first length[b] rows (device int32[B]; 0: all)
 * of slot[b]: of requests that end, of drafts that did not stand.  The pages
 * that pages_extend just took come back in the order in which they lay there.
 * status as above (-1 also where the stack would hold more than n_pages, or where
 * an entry that would go back names no page).  A page goes back for every slot that
 * names it: of slots that share pages all but one are cleared by the caller. */
int   slate_hip_pages_trim(const slate_hip_pages_t* pages, const int32_t* slot, const int32_t* length, int B,
                           int32_t* status);
/* New K and V rows into their pages: k, v [T, n_kv_heads * head_dim] f32 (16-byte
 * aligned), rows ld floats apart (ld % 4 == 0), rounded to the pools' type to
 * nearest, ties to even.  A row whose tok_row is outside 0 .. n_pages * page_size - 1
 * is stored nowhere; where two rows have the same tok_row each element is either's. */
int   slate_hip_kv_store_paged(const slate_hip_paged_kv_t* kv, const slate_hip_pages_t* pages, const float* k,
                               const float* v, int64_t ld, const int32_t* tok_row, int T);
/* Causal GQA attention of new tokens over the pages: q, out [T, n_q_heads *
 * head_dim] f32 (out is not q).  Sequence b's tokens are the rows tok_off[b] ..
 * tok_off[b+1]-1, at most max_new of them, and token i attends to rows 0 .. pos0[b]
 * + i of slot[b] (its own is stored before the call).  Scores are q.k /
 * sqrt(head_dim); query head g belongs to kv head g / (n_q_heads / n_kv_heads).
 * A sequence whose numbers do not fit (as for the packed batches above; slot
 * outside 0 .. n_slots-1, more than max_pages * page_size rows) is left out; rows
 * of out that no sequence owns stay as they were.  Keys in pages outside 0 ..
 * n_pages-1 count as not seen, and a token that sees none gets zeros.  What the
 * cache holds in rows that a token does not see never matters, not even infinities
 * and NaN; one in V of a row that it sees makes that column of its output not
 * finite, a NaN in K all of it.
 * Queries must be finite and below 2^100 in size, and so must bf16 and f32 K and V (V below
 * 2^90 where slots have more than 2^23 rows); over those the sum of the |q_i k_i| of a token
 * and a row that it sees must be below 2^126.  Sums are f32 (outputs below 2^-100 in size
 * lose bits).  f32 caches are multiplied in f32; over bf16 ones queries and weights have 24
 * bits; over f16 ones 22, where a weight is resolved to 2^-35 of the largest and an element
 * of a query to 2^-37 of its row's largest.
 * Made for few tokens a sequence (decode steps, drafts): K and V are read once for
 * every 16 query rows of a kv head where max_new brings no more, else for every 32 or 64
 * (f32, and head_dim above 128: 32).  T * n_q_heads <= 2^31 - 128, and n_kv_heads * (T *
 * n_q_heads / n_kv_heads / 16 + B) * max_pages * page_size / 128 stays below 2^31.  ws as
 * for attention_ragged_q8, of slate_hip_attention_paged_bytes. */
int   slate_hip_attention_paged(float* out, const float* q, const slate_hip_paged_kv_t* kv,
                                const slate_hip_pages_t* pages, const int32_t* slot, const int32_t* tok_off,
                                const int32_t* pos0, int B, int T, int max_new, int n_q_heads, void* ws,
                                size_t ws_bytes);
/* Bytes of ws for these heads, whatever the batch; -1 for heads it refuses. */
int64_t slate_hip_attention_paged_bytes(int n_q_heads, int n_kv_heads, int head_dim);

/* Which drafted tokens stand, and the token after them.  Sequence b has the rows
 * tok_off[b] .. tok_off[b+1]-1 (device int32[B+1]): the first is its last
 * committed token, the others are drafts; row i continues row parent[i] (device
 * int32[T], counted within the sequence, below i; another value: no row), or row i - 1
 * where parent is NULL.  Row t of logits (f32, rows ld floats apart, V of them
 * count) is the target's distribution after row t, p = softmax(logits /
 * temperature[b]) (device float[B]; NULL: 1; 0, negative or NaN: all of it on the
 * largest logit, the lowest of equal ones).  NaN counts as -infinity, +infinity
 * shares all of p with its like; a row that is all -infinity has no p.  From the first
 * row on, the drafts x that continue the row are tried in order, the first one
 * accepted is the next row:
 *  - with draft_probs (rows draft_ld floats apart; row t is the distribution q that
 *    token[t] was drawn from; chains only, parent NULL): where u[t] q(x) < p(x).  If it is
 *    turned down the next token comes from max(p - q, 0), or from p where that is 0;
 *  - without: where u[t] (1 - the sum of p of those turned down before) < p(x), a
 *    token that was turned down before having p 0.  The next token comes from p
 *    without those turned down (from p where nothing else has any);
 *  - at temperature 0: where x has the largest logit, whatever u and q are.
 * Where none stands the next token is the lowest i with p(i) > 0 and a sum of p up to i above
 * u_next[b] times the whole sum (the last with p > 0 where no sum is).  u (device
 * float[T], at the drafts) and u_next (float[B]) are uniform in [0, 1).  Tokens
 * outside 0 .. V-1 never stand.  q is not negative.  All T rows of logits are read.
 * Outputs (device): n_accepted[b] (-1 for a sequence that is left out: without rows, with
 * more than 1024 drafts, outside 0 .. T, or behind a fall of tok_off); out_tok[T]: in a
 * sequence's rows the accepted tokens, the next one (-1: no p), then -1; out_row[T] (or
 * NULL): the rows that were accepted, counted within the sequence, then -1.  Rows that no
 * sequence owns stay as they were.
 * Probabilities, sums and comparisons are in 64 bits, exponentials good to 2^-42.  V is at
 * most 2^31 - 1024.
 * ws: device scratch of slate_hip_verify_drafts_bytes, as for attention_ragged_q8. */
int   slate_hip_verify_drafts(int32_t* n_accepted, int32_t* out_tok, int32_t* out_row, const float* logits, int64_t ld,
                              const int32_t* token, const int32_t* parent, const float* draft_probs, int64_t draft_ld,
                              const float* temperature, const float* u, const float* u_next, const int32_t* tok_off,
                              int B, int T, int V, void* ws, size_t ws_bytes);
/* Bytes of ws for a batch of that size; -1 for one it refuses. */
int64_t slate_hip_verify_drafts_bytes(int B, int T, int V);

/* Synthetic weights generated on the device (seeded, ~N(0, std)):
 * f32 values, or rows x cols quantised to Q4_K. */
int   slate_hip_synth_f32(float* dst, int64_t n, uint64_t seed, float std);
int   slate_hip_synth_q4k(void* dst, int64_t rows, int64_t cols, uint64_t seed, float std);

/* ---- device-resident LLaMA engine ---------------------------------------- */
/* Mirrors slate_llama_config_t (llama.h:53-65). */
typedef struct slate_hip_llama_config {
    int   n_layers, d_model, ffn_hidden, n_heads, n_kv_heads, head_dim;
    int   max_seq, vocab;
    float theta_base, rms_eps;
    int   tied_output;
} slate_hip_llama_config_t;

/* Mirrors slate_llama_layer_t (llama.h:69-86): host pointers, dtypes are
 * slate_dtype_t values (0 = F32, 16 = Q8_0, 18 = Q4_K).  Unlike the
 * reference's mv_dispatch (llama_infer.c:43-51), which reads a Q8_0 tensor
 * as f32, Q8_0 linears run the Q8_0 matmul. */
typedef struct slate_hip_llama_layer {
    const void *attn_norm, *attn_q, *attn_k, *attn_v, *attn_output;
    const void *ffn_norm, *ffn_gate, *ffn_up, *ffn_down;
    int attn_q_dtype, attn_k_dtype, attn_v_dtype, attn_output_dtype;
    int ffn_gate_dtype, ffn_up_dtype, ffn_down_dtype;
} slate_hip_llama_layer_t;

typedef struct slate_hip_llama slate_hip_llama_t;
typedef struct slate_hip_llama_session slate_hip_llama_session_t;

/* Upload a model from host pointers (e.g. the mmap views slate_llama_open
 * resolves).  max_slots = concurrent sessions (KV slots); max_tokens = the
 * largest number of packed tokens one step may carry. */
slate_hip_llama_t* slate_hip_llama_new(const slate_hip_llama_config_t* cfg,
                                       const float* token_embd, const float* output_norm,
                                       const void* output, int output_dtype,
                                       const slate_hip_llama_layer_t* layers,
                                       int max_slots, int max_tokens);
/* Same engine with seeded synthetic weights generated on the device:
 * linears Q4_K (quant = 18), Q8_0 (quant = 16) or F32 (quant = 0),
 * embeddings f32, norms 1. */
slate_hip_llama_t* slate_hip_llama_new_synthetic(const slate_hip_llama_config_t* cfg,
                                                 uint64_t seed, int quant,
                                                 int max_slots, int max_tokens);
void  slate_hip_llama_free(slate_hip_llama_t* m);
/* The model's config (llama.h:98 slate_llama_config); NULL for NULL. */
const slate_hip_llama_config_t* slate_hip_llama_config(const slate_hip_llama_t* m);
/* Copy a weight tensor back to host ("token_embd", "output", "output_norm",
 * or "blk.N.<name>"); returns bytes written or a negative code. */
int64_t slate_hip_llama_get_tensor(const slate_hip_llama_t* m, const char* name,
                                   void* host_dst, int64_t cap, int* dtype);

/* llama.h:124-139 semantics, device-resident.  A session belongs to its
 * engine: free every session before slate_hip_llama_free (as a slate
 * session must not outlive its model). */
slate_hip_llama_session_t* slate_hip_llama_session_new(slate_hip_llama_t* m);
void  slate_hip_llama_session_free(slate_hip_llama_session_t* s);
int   slate_hip_llama_session_position(const slate_hip_llama_session_t* s);
/* Back to position 0 for a new conversation, keeping the KV slot
 * (slate_infer_session_reset, infer.h:116, engine.c:429-431). */
void  slate_hip_llama_session_reset(slate_hip_llama_session_t* s);
int   slate_hip_llama_prefill(slate_hip_llama_session_t* s, const int32_t* tokens,
                              int n_tokens, float* out_logits);
int   slate_hip_llama_decode_step(slate_hip_llama_session_t* s, int32_t token,
                                  float* out_logits);

/* One ragged continuous-batching step: sessions[i] contributes n_new[i]
 * tokens (tokens packed session-major in `tokens`).  For each session the
 * logits of its last new token go to out_logits[i*V..] (host, may be NULL)
 * and the greedy next token to out_next[i] (host, may be NULL).  Positions
 * advance by n_new[i].  Returns 0 or a negative code; on error no session
 * advances. */
int   slate_hip_llama_step(slate_hip_llama_t* m, slate_hip_llama_session_t** sessions,
                           int n, const int32_t* n_new, const int32_t* tokens,
                           float* out_logits, int32_t* out_next);
/* slate_infer_batch_step (engine.c:543-642) semantics: one token each. */
int   slate_hip_llama_batch_step(slate_hip_llama_t* m, slate_hip_llama_session_t** sessions,
                                 int n, const int32_t* tokens, float* out_logits);

/* KV cache of a session copied to host as [n_layers, max_seq, kv_dim] (the
 * reference session layout, llama_infer.c:57-58) for checking. */
int   slate_hip_llama_session_kv(const slate_hip_llama_session_t* s, float* K, float* V);

/* Kernel-class timing with HIP events recorded on the backend stream around
 * each launch: class 0 = Q4_K matmuls of decode shape (<= 16 rows),
 * 1 = attention in decode-only steps, 2 = decode-only steps, 3 = Q4_K
 * matmuls over more rows, 4 = attention in steps carrying prompt chunks,
 * 5 = steps carrying prompt chunks.
 * profile(m, 1) resets the totals and starts recording, profile(m, 2)
 * resumes recording without a reset, profile(m, 0) stops.  Kernel classes
 * are timed by events the dispatches record themselves (kernel start and
 * end).  Steps run while recording are launched one kernel at a time, not
 * from a graph.  profile_read returns the summed device milliseconds, the
 * summed algorithmic bytes (weights once, K/V once per kv head and sequence,
 * activations in and out) and the launch count of a class. */
int   slate_hip_llama_profile(slate_hip_llama_t* m, int enable);
/* graphs(m, 1) (or SLATE_HIP_GRAPHS=1): decode-only steps (one token per
 * session) are captured once per batch size into a HIP graph and replayed.
 * Default off: every kernel is launched separately.  Same results either
 * way.  Refused (-5, graphs stay off) while a rocprofiler tool is attached
 * (ROCPROF* / ROCP_* in the environment): a graph launch under
 * rocprofv3 --kernel-trace has ended in a crash inside the HIP runtime.
 * No slate counterpart (slate has no device graphs). */
int   slate_hip_llama_graphs(slate_hip_llama_t* m, int enable);
/* 1 when the engine keeps its K/V cache in f16 (opt-in at creation with
 * SLATE_HIP_KV_F16=1, head_dim 32/64/128), 0 for f32 as the reference
 * (llama_infer.c:57-58).  f16 halves the attention bytes; it rounds every
 * cached element to 11 bits, a numerics change measured against the parity
 * tolerance.  slate_hip_llama_session_kv returns f32 either way. */
int   slate_hip_llama_kv_f16(const slate_hip_llama_t* m);
/* 1 while the engine's decode steps merge the attention chunks inside the
 * decode attention kernel (workgroup i takes its work from queue i % 8, the
 * workgroups of a queue share one XCD, and the merging unit reads the
 * partials from that XCD's L2), 0 when they use the separate merge kernel:
 * shapes the in-kernel merge does not take, SLATE_HIP_ATTN_XCD=0, a device
 * where the placement probe failed, or after a merge found a partial
 * written on another XCD (the engine then runs that step again on the merge
 * kernel and keeps to it).  No slate counterpart. */
int   slate_hip_llama_attn_xcd_merge(const slate_hip_llama_t* m);
int   slate_hip_llama_profile_read(slate_hip_llama_t* m, int cls, double* ms, double* bytes,
                                   int64_t* launches);

/* The backend stream as a hipStream_t (for timing with events). */
void* slate_hip_stream(void);

#ifdef __cplusplus
}
#endif
#endif
