// k_pages.hip -- pages of a K/V cache taken and given back, the slot map of a
// step's tokens, and new K/V rows stored by it.
#include "attn_plan.h"
#include "paged.h"

namespace slate_hip {

constexpr int PGS_MAX_TH = 1024;       // threads of the one workgroup: a sequence each
// Up to as many sequences in a workgroup of as many threads (64 sequences: extend 3.5 us,
// with 1024 threads 4.3).
constexpr int PGS_FEW = 256;
constexpr int PGS_HASH = 2048;
// Tokens whose rows the workgroup that takes the pages finds itself; more are left to
// workgroups of their own where T_cap has room for more (us a call, in one kernel and in
// two: 64 sequences, 1024 tokens 5.7 and 7.7, 1536 6.7 and 7.7, 2048 7.7 and 7.6; 4
// sequences, 2048 tokens 5.6 and 6.5).
constexpr int PGS_OWN_TOKENS = 2048;

// Sums over the workgroup, each thread bringing a count below 2^31: the
// inclusive one up to the thread (below 2^31 if the whole is), and the whole.
struct Scan {
    int upto;
    int64_t total;
};
template <int TH>
__device__ __forceinline__ Scan block_scan(int v, int64_t* s_part) {
    const int w = threadIdx.x >> 6;
    const int upto = wave_scan(v);
    // halves of 16 bits: their sums over a wave pass no 32 bits
    const int64_t whole = ((int64_t)wave_sum_int(v >> 16) << 16) + wave_sum_int(v & 0xffff);
    if ((threadIdx.x & 63) == 0) s_part[w] = whole;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) {
        before += i < w ? s_part[i] : 0;
        total += s_part[i];
    }
    return Scan{(int)before + upto, total};
}

// Whether another sequence brought the same slot: an open hash of the slots
// seen.
__device__ __forceinline__ bool seen_before(int* s_hash, int slot) {
    uint32_t at = (uint32_t)slot * 2654435761u >> 21;
    for (;;) {                         // twice as many places as slots: ends
        const int was = atomicCAS(&s_hash[at], -1, slot);
        if (was == -1) return false;
        if (was == slot) return true;
        at = (at + 1) & (PGS_HASH - 1);
    }
}
static_assert(PGS_HASH == 1 << 11 && PGS_HASH >= 2 * PK_MAX_SEQ, "the hash's shift");

// The first sequence whose inclusive sum is above x (which is below the last one's).
__device__ __forceinline__ int find_above(const int* s_upto, int B, int x) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_upto[mid] > x)
            hi = mid;
        else
            lo = mid + 1;
    }
    return lo;
}

__global__ __launch_bounds__(256) void pages_reset_kernel(Pages pg) {
    const int64_t step = (int64_t)gridDim.x * 256, cells = (int64_t)pg.n_slots * pg.max_pages;
    const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = i0; i < cells; i += step) pg.table[i] = -1;
    for (int64_t i = i0; i < pg.n_slots; i += step) pg.held[i] = 0;
    for (int64_t i = i0; i < pg.n_pages; i += step) pg.free_pages[i] = pg.n_pages - 1 - (int)i;
    if (i0 == 0) pg.n_free[0] = pg.n_pages;
}

// The cache row of position pos of a slot, -1 where its page is none.
__device__ __forceinline__ int row_at(const Pages& pg, int page, int in) {
    return (unsigned)page < (unsigned)pg.n_pages ? page * pg.page_size + in : -1;
}

// Two sums over the sequences (tokens, new pages); then a thread per new page and per
// token finds its sequence in them.  Latency: three rounds of loads one after the other
// (descriptors, held, pages: a token's page comes from the table or from the stack that
// the table is filled from, so nothing waits for what was written) in 4 us for 64
// sequences.
template <int TH>
__global__ __launch_bounds__(TH) void pages_extend_kernel(Pages pg, const int32_t* __restrict__ slot,
                                                          const int32_t* __restrict__ pos0,
                                                          const int32_t* __restrict__ n_new, int B, int T_cap,
                                                          int32_t* __restrict__ tok_off, int32_t* __restrict__ tok2seq,
                                                          int32_t* __restrict__ tok_pos, int32_t* __restrict__ tok_row,
                                                          int32_t* __restrict__ last_tok,
                                                          int32_t* __restrict__ status) {
    __shared__ int s_hash[PGS_HASH], s_slot[TH], s_pos0[TH], s_held[TH], s_tok[TH], s_page[TH];
    __shared__ int64_t s_part[2][TH / 64];
    __shared__ int s_err;
    const int b = threadIdx.x;
    const int n_free = pg.n_free[0];
    int sl = 0, p0 = 0, n = 0, held = 0, fresh = 0;
    if (b < B) {
        sl = slot[b];
        p0 = pos0[b];
        n = n_new[b];
    }
    const bool in = sl >= 0 && sl < pg.n_slots;
    if (b < B && in) held = pg.held[sl];
    for (int i = b; i < PGS_HASH; i += TH) s_hash[i] = -1;
    if (b == 0) s_err = 0;
    __syncthreads();
    if (b < B) {
        bool bad = !in || p0 < 0 || n < 0 || n_free < 0 || n_free > pg.n_pages || held < 0 || held > pg.max_pages;
        if (in) bad |= seen_before(s_hash, sl);
        const int64_t rows = (int64_t)p0 + n;
        if (bad)
            atomicOr(&s_err, 1);
        else if (rows > (int64_t)pg.max_pages * pg.page_size)
            atomicOr(&s_err, 2);
        else
            fresh = max(0, (int)(((unsigned)rows + (unsigned)pg.page_size - 1) / (unsigned)pg.page_size) - held);
        n = max(n, 0);
    }
    const Scan tok = block_scan<TH>(n, s_part[0]), page = block_scan<TH>(fresh, s_part[1]);
    s_slot[b] = sl;
    s_pos0[b] = p0;
    s_held[b] = held;
    s_tok[b] = tok.upto;
    s_page[b] = page.upto;
    __syncthreads();
    int err = s_err & 1 ? -1 : s_err ? -2 : 0;
    if (err == 0 && (tok.total > T_cap || page.total > n_free)) err = -2;
    if (b == 0) status[0] = err;
    if (err != 0) return;
    const int T = (int)tok.total, new_pages = (int)page.total;
    if (b < B) {
        tok_off[b] = tok.upto - n;
        if (b == B - 1) tok_off[B] = tok.upto;
        last_tok[b] = n > 0 ? tok.upto - 1 : -1;
        if (fresh > 0) pg.held[sl] = held + fresh;
    }
    if (b == 0) pg.n_free[0] = n_free - new_pages;
    for (int k = threadIdx.x; k < new_pages; k += TH) {
        const int s = find_above(s_page, B, k), first = s > 0 ? s_page[s - 1] : 0;
        pg.table[(int64_t)s_slot[s] * pg.max_pages + s_held[s] + (k - first)] = pg.free_pages[n_free - 1 - k];
    }
    if (T > PGS_OWN_TOKENS) return;
    for (int t = threadIdx.x; t < T; t += TH) {
        const int s = find_above(s_tok, B, t), first = s > 0 ? s_tok[s - 1] : 0;
        const int pos = s_pos0[s] + (t - first), i = (int)((unsigned)pos / (unsigned)pg.page_size), own = i - s_held[s];
        const int pno = own < 0 ? pg.table[(int64_t)s_slot[s] * pg.max_pages + i]
                                : pg.free_pages[n_free - 1 - (s > 0 ? s_page[s - 1] : 0) - own];
        tok2seq[t] = s;
        tok_pos[t] = pos;
        tok_row[t] = row_at(pg, pno, pos - i * pg.page_size);
    }
}

// The same for the tokens of a large batch: its offsets in LDS, a token a thread and round.
constexpr int PGS_TOK_TH = 256, PGS_TOK = 4, PGS_TOK_WGS = 2048;
__global__ __launch_bounds__(PGS_TOK_TH) void pages_tokens_kernel(Pages pg, const int32_t* __restrict__ slot,
                                                                  const int32_t* __restrict__ pos0, int B,
                                                                  const int32_t* __restrict__ tok_off,
                                                                  int32_t* __restrict__ tok2seq,
                                                                  int32_t* __restrict__ tok_pos,
                                                                  int32_t* __restrict__ tok_row,
                                                                  const int32_t* __restrict__ status) {
    __shared__ int s_tok[PK_MAX_SEQ];                  // the sequences' ends
    if (status[0] != 0) return;                        // tok_off is not this call's
    constexpr int PER = PGS_TOK_TH * PGS_TOK;
    const int T = tok_off[B];
    if (T <= PGS_OWN_TOKENS || (int64_t)blockIdx.x * PER >= T) return;
    for (int b = threadIdx.x; b < B; b += PGS_TOK_TH) s_tok[b] = tok_off[b + 1];
    __syncthreads();
    for (int64_t t0 = (int64_t)blockIdx.x * PER; t0 < T; t0 += (int64_t)gridDim.x * PER) {
#pragma unroll
        for (int k = 0; k < PGS_TOK; ++k) {
            const int64_t at = t0 + PGS_TOK_TH * k + threadIdx.x;
            if (at >= T) break;
            const int t = (int)at, s = find_above(s_tok, B, t), first = s > 0 ? s_tok[s - 1] : 0;
            const int pos = pos0[s] + (t - first), i = (int)((unsigned)pos / (unsigned)pg.page_size);
            tok2seq[t] = s;
            tok_pos[t] = pos;
            tok_row[t] = row_at(pg, pg.table[(int64_t)slot[s] * pg.max_pages + i], pos - i * pg.page_size);
        }
    }
}

template <int TH>
__global__ __launch_bounds__(TH) void pages_trim_kernel(Pages pg, const int32_t* __restrict__ slot,
                                                        const int32_t* __restrict__ length, int B,
                                                        int32_t* __restrict__ status) {
    __shared__ int s_hash[PGS_HASH], s_slot[TH], s_keep[TH], s_page[TH];
    __shared__ int64_t s_part[TH / 64];
    __shared__ int s_err;
    const int b = threadIdx.x;
    const int n_free = pg.n_free[0];
    int sl = 0, len = 0, held = 0, keep = 0, back = 0;
    if (b < B) {
        sl = slot[b];
        len = length[b];
    }
    const bool in = sl >= 0 && sl < pg.n_slots;
    if (b < B && in) held = pg.held[sl];
    for (int i = b; i < PGS_HASH; i += TH) s_hash[i] = -1;
    if (b == 0) s_err = 0;
    __syncthreads();
    if (b < B) {
        bool bad = !in || len < 0 || n_free < 0 || n_free > pg.n_pages || held < 0 || held > pg.max_pages;
        if (in) bad |= seen_before(s_hash, sl);
        keep = min(held, (int)(((unsigned)len + (unsigned)pg.page_size - 1) / (unsigned)pg.page_size));
        back = held - keep;
        if (bad) {
            atomicOr(&s_err, 1);
            back = 0;
        }
    }
    const Scan page = block_scan<TH>(back, s_part);
    s_slot[b] = sl;
    s_keep[b] = keep;
    s_page[b] = page.upto;
    __syncthreads();
    int err = s_err ? -1 : 0;
    if (err == 0 && n_free + page.total > pg.n_pages) err = -1;
    const int total = err == 0 ? (int)page.total : 0;
    // Up to four entries in a row a thread and round.  All are looked at before any is given back, the first
    // round's waiting in registers: 3.2 us for 64 sequences, 4.5 for 37 prompts of 930 pages (2.4 and 4.1 unlooked
    // at, when an entry that was no page went back as one).
    const int per = total <= TH ? 1 : 4;
    auto cells_of = [&](int k0, int32_t** cell) {
        int s = find_above(s_page, B, k0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cell[i] = nullptr;
            if (i >= per || k0 + i >= total) continue;
            while (s_page[s] <= k0 + i) ++s;
            const int first = s > 0 ? s_page[s - 1] : 0;
            cell[i] = pg.table + (int64_t)s_slot[s] * pg.max_pages + s_keep[s] + (k0 + i - first);
        }
    };
    int32_t* cell[4] = {};
    int page_no[4] = {};
    bool none = false;
    for (int64_t k0 = per * threadIdx.x; k0 < total; k0 += per * TH) {
        int32_t* at[4];
        int no[4] = {};
        cells_of((int)k0, at);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at[i]) no[i] = *at[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            none |= (unsigned)no[i] >= (unsigned)pg.n_pages;
            if (k0 < per * TH) {
                cell[i] = at[i];
                page_no[i] = no[i];
            }
        }
    }
    if (__syncthreads_or(none)) err = -1;
    if (b == 0) status[0] = err;
    if (err != 0) return;
    if (b < B && back > 0) pg.held[sl] = keep;
    if (b == 0) pg.n_free[0] = n_free + total;
    for (int64_t k0 = per * threadIdx.x; k0 < total; k0 += per * TH) {
        if (k0 >= per * TH) {
            cells_of((int)k0, cell);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (cell[i]) page_no[i] = *cell[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (cell[i]) {
                pg.free_pages[n_free + total - 1 - k0 - i] = page_no[i];
                *cell[i] = -1;
            }
    }
}

// ---------------------------------------------------------------------------
// Rows rounded to the pools' type: 8 elements a thread, so that heads and rows
// of any stride are written 16 (f32: 32) bytes at a time.  Memory bound: 5.9 TB/s for
// 5876 tokens of 8 heads of 128 (12 us; f32 read, f16 written), 2.4 us for 16 tokens.
constexpr int ST_WGS = 65536;
template <class E>
struct Eight {
    E e[8];
};

template <class E>
__global__ __launch_bounds__(256) void kv_store_paged_kernel(slate_hip_paged_kv_t kv, int page_size, int n_rows,
                                                             const float* __restrict__ k, const float* __restrict__ v,
                                                             int64_t ld, const int32_t* __restrict__ tok_row, int T) {
    const int c8 = kv.head_dim / 8;
    for (int t = blockIdx.x; t < T; t += gridDim.x) {
        const int row = tok_row[t];
        if ((unsigned)row >= (unsigned)n_rows) continue;
        const float* src = (blockIdx.y ? v : k) + (int64_t)t * ld;
        const int page = row / page_size;
        E* dst = (E*)(blockIdx.y ? kv.V : kv.K) + page * kv.page_stride + (row - page * page_size) * kv.row_stride;
        for (int c = threadIdx.x; c < kv.n_kv_heads * c8; c += 256) {
            const float4 a = *(const float4*)(src + 8 * c), b = *(const float4*)(src + 8 * c + 4);
            const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            const int h = c / c8;
            Eight<E> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.e[e] = (E)x[e];
            *(Eight<E>*)__builtin_assume_aligned(dst + h * kv.head_stride + 8 * (c - h * c8), 16) = o;
        }
    }
}

int launch_pages_reset(const Pages& pg, hipStream_t s) {
    const int64_t cells = max((int64_t)pg.n_slots * pg.max_pages, (int64_t)pg.n_pages);
    hipLaunchKernelGGL(pages_reset_kernel, dim3((unsigned)min((int64_t)1024, (cells + 255) / 256)), dim3(256), 0, s, pg);
    SH_CHECK_LAUNCH();
    return 0;
}

int launch_pages_extend(const Pages& pg, const int32_t* slot, const int32_t* pos0, const int32_t* n_new, int B,
                        int T_cap, int32_t* tok_off, int32_t* tok2seq, int32_t* tok_pos, int32_t* tok_row,
                        int32_t* last_tok, int32_t* status, hipStream_t s) {
    if (B <= PGS_FEW)
        hipLaunchKernelGGL(pages_extend_kernel<PGS_FEW>, dim3(1), dim3(PGS_FEW), 0, s, pg, slot, pos0, n_new, B, T_cap,
                           tok_off, tok2seq, tok_pos, tok_row, last_tok, status);
    else
        hipLaunchKernelGGL(pages_extend_kernel<PGS_MAX_TH>, dim3(1), dim3(PGS_MAX_TH), 0, s, pg, slot, pos0, n_new, B,
                           T_cap, tok_off, tok2seq, tok_pos, tok_row, last_tok, status);
    constexpr int PER = PGS_TOK_TH * PGS_TOK;
    if (T_cap > PGS_OWN_TOKENS)
        hipLaunchKernelGGL(pages_tokens_kernel, dim3(min(PGS_TOK_WGS, (T_cap - 1) / PER + 1)), dim3(PGS_TOK_TH), 0, s, pg,
                           slot, pos0, B, tok_off, tok2seq, tok_pos, tok_row, status);
    SH_CHECK_LAUNCH();
    return 0;
}

int launch_pages_trim(const Pages& pg, const int32_t* slot, const int32_t* length, int B, int32_t* status,
                      hipStream_t s) {
    if (B <= PGS_FEW)
        hipLaunchKernelGGL(pages_trim_kernel<PGS_FEW>, dim3(1), dim3(PGS_FEW), 0, s, pg, slot, length, B, status);
    else
        hipLaunchKernelGGL(pages_trim_kernel<PGS_MAX_TH>, dim3(1), dim3(PGS_MAX_TH), 0, s, pg, slot, length, B, status);
    SH_CHECK_LAUNCH();
    return 0;
}

int launch_kv_store_paged(const slate_hip_paged_kv_t& kv, const Pages& pg, const float* k, const float* v, int64_t ld,
                          const int32_t* tok_row, int T, hipStream_t s) {
    const dim3 grid(min(T, ST_WGS), 2);
    const int rows = pg.n_pages * pg.page_size;
    if (kv.dtype == KV_F32)
        hipLaunchKernelGGL(kv_store_paged_kernel<float>, grid, dim3(256), 0, s, kv, pg.page_size, rows, k, v, ld,
                           tok_row, T);
    else if (kv.dtype == KV_F16)
        hipLaunchKernelGGL(kv_store_paged_kernel<_Float16>, grid, dim3(256), 0, s, kv, pg.page_size, rows, k, v, ld,
                           tok_row, T);
    else
        hipLaunchKernelGGL(kv_store_paged_kernel<__bf16>, grid, dim3(256), 0, s, kv, pg.page_size, rows, k, v, ld,
                           tok_row, T);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
