// attn_paged.h -- causal attention of new tokens over a K/V cache in pages.
//
// out = sum_k exp(s_k - m) V_k / sum_k exp(s_k - m), s_k = q.K_k / sqrt(hd),
// over the rows 0 .. pos0 + i of the token's slot.
//
//   S^T [keys x 16 rows] = K Q^T,   O^T [hd x 16 rows] += V^T P^T
//
// Few query rows meet many keys, so the bytes of K and V bound it.  A workgroup
// takes a block of 16 RT rows over a range of keys (attn_plan.h), each of its
// four waves every fourth 32 of them.  K and V go from memory straight into the
// registers that the MFMA takes them from, with no LDS and no barrier until the
// range ends; the next keys' loads are under way while a wave works.  That needs
// no transposition between lanes, as the order of a product's terms is free:
//  - K: lane (g, j) = (lane / 16, lane % 16) reads 16 bytes g of each 64 of key j's
//    row, and Q is laid out alike;
//  - S^T leaves the keys 4g + i of row j in lane (g, j), so V's products take
//    lane g's keys from there: its lanes read those keys' rows, CW columns each,
//    whole rows of memory, and columns CW apart share an MFMA.
// f16: Q (scaled by a power of two) and the weights (times 2^11) as two halves, 22
// bits; bf16: as three, 24 bits; f32: f32 MFMAs.  Sums are f32.  A row's running
// maximum moves only when a score passes it by 2^4.
//
// With 8 kv heads of 128 (a 4 GiB copy runs at 4.77 TB/s):
//  - one token of 64 users, 4 query heads, f16, up to 16384 keys: 439 us, 5.95 TB/s;
//  - of 16 users, bf16, up to 4096 keys: 41 us, the joining kernel 4.7 of it and about 3
//    until the first keys are there (plan, table), the rest at 5.9 TB/s;
//  - 3 to 5 tokens of 16 users, f32, up to 8192 keys: 133 us, 4.8 TB/s; the f32 MFMAs are
//    busy for 61 % of that time;
//  - 4 to 8 tokens of 8 users, 8 query heads, bf16, up to 16384 keys: 97 us, 3.75 TB/s;
//    matrix unit 35 %, vector unit 37 %, waves wait in 27 % of their cycles, two a SIMD (64
//    rows a wave, one a SIMD: 120 us).
#pragma once
#include "attn_plan.h"
#include "attn_rows.h"
#include "paged.h"

namespace slate_hip {

// Workgroups: two per CU, one where K and V of a step fill half of the registers.
__host__ __device__ constexpr int paged_wgs(int hd) { return hd > 128 ? 256 : 512; }
constexpr int AP_SLICE = 32;           // keys of a wave within a granule
constexpr int AP_GRAN = 4 * AP_SLICE;  // keys of a granule
// Where slots have room for no more than this many granules no block is cut, which spares
// the joining kernel; calls over larger slots cut where the ranges end, also blocks of short
// sequences (the host knows what a slot can hold, not the lengths).  Decode, bf16, 8 kv heads
// of 128, us cut / not cut: one sequence of 333 keys 10.4 / 9.1, one of 1000 10.9 /
// 10.7, 16 of up to 512 14.3 / 16.2, 32 19.7 / 17.4, 64 27.8 / 24.1, 256 91.0 / 87.4.
constexpr int AP_SHORT = 8;

typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));

__host__ __device__ constexpr int paged_granules(int keys) { return (keys + AP_GRAN - 1) / AP_GRAN; }

template <int ROWS>
struct PagedCount {
    int G, Hkv;
    __device__ __forceinline__ int blocks(const SeqView& s) const { return (s.n * G + ROWS - 1) / ROWS; }
    __device__ __forceinline__ int operator()(const SeqView& s) const {
        return s.n < 1 ? 0 : Hkv * blocks(s) * paged_granules(s.p0 + s.n);
    }
};

// Whether a call's blocks may be cut.
__host__ __device__ constexpr bool paged_cuts(int max_seq) { return paged_granules(max_seq) > AP_SHORT; }

// Where workgroup w's range begins (the place there is for x < plan.total): N w / P,
// or the start of the block there where none is cut.
struct PagedBegin {
    int x;
    Place place;
};
template <int WGS, class PlanT>
__device__ __forceinline__ PagedBegin paged_begin(const PlanT& plan, int w, bool cuts) {
    PagedBegin b{plan.begin(w, WGS), {}};
    if (b.x >= plan.total) return PagedBegin{plan.total, {}};
    b.place = plan.find(b.x);
    if (!cuts) {
        const int in = b.place.at % paged_granules(b.place.seq.p0 + b.place.seq.n);
        b.x -= in;
        b.place.at -= in;
    }
    return b;
}

// Of two halves, `exp` having the exponent's bits: all ones in those of which not all
// of these bits are set.
__device__ __forceinline__ uint32_t finite2(uint32_t u, uint32_t exp) {
    return ((((~u & exp) + 0x7fff7fffu) >> 15) & 0x00010001u) * 0xffffu;
}

// How a type's numbers are multiplied: NP operands stand for one f32.
template <class E>
struct Mul;
template <>
struct Mul<_Float16> {
    static constexpr int NP = 2;
    static constexpr float PEXP = 11;  // weights are scaled by 2^11: at most 2^15 with the slack
    // V's numbers below 2^-16 have products of their own, 2^10 larger: the unit lines up the
    // products of numbers that are not normal as if they were 2^-14 and cuts off what is
    // 2^24 below that (V of 2^-22: outputs 2e-5 off, and 4e-7 so; at 2^-16 the cut is 2^-22
    // of the number).  Each number by itself, so that no other column, and no row that a
    // token does not see, changes its output.  Of V around 1 one step in 20 has such a number:
    // 64 users take 437 us with these products and without, three of 848 rows 12.9 and 11.8.
    static constexpr int LIFT = 10;
    // Of two halves: below LOW_RANKS where they are that small and not 0.
    static __device__ __forceinline__ ushort2v low_rank(uint32_t u) {
        return __builtin_bit_cast(ushort2v, u) * (uint16_t)2 - (uint16_t)1;
    }
    static constexpr uint16_t LOW_RANKS = 0x1ff;
    // all ones in the halves that are not
    static __device__ __forceinline__ uint32_t large(uint32_t u) { return finite2(~u, 0x7f007f00); }
    static __device__ __forceinline__ uint32_t lifted(uint32_t u) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, u) * (_Float16)(1 << LIFT));
    }
    static constexpr uint32_t ONE = 0x3c003c00;
    // all ones in the halves that are finite numbers
    static __device__ __forceinline__ uint32_t finite(uint32_t u) { return finite2(u, 0x7c007c00); }
    static __device__ __forceinline__ void split(const float* x, uint4v* p) {
        half8_t hi, lo;
        halves(x, hi, lo);
        p[0] = __builtin_bit_cast(uint4v, hi);
        p[1] = __builtin_bit_cast(uint4v, lo);
    }
    static __device__ __forceinline__ floatx4 mfma(uint4v a, uint4v b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                      0, 0);
    }
};
template <>
struct Mul<__bf16> {
    static constexpr int NP = 3;
    static constexpr float PEXP = 0;
    static constexpr int LIFT = 0;
    static constexpr uint32_t ONE = 0x3f803f80;
    static __device__ __forceinline__ uint32_t finite(uint32_t u) { return finite2(u, 0x7f807f80); }
    // cut off after 8 bits three times: exact
    static __device__ __forceinline__ void split(const float* x, uint4v* p) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float v[2] = {x[e], x[e + 1]};
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const uint32_t u0 = __float_as_uint(v[0]), u1 = __float_as_uint(v[1]);
                p[k][e / 2] = __builtin_amdgcn_perm(u1, u0, 0x07060302);
                v[0] -= __uint_as_float(u0 & 0xffff0000u);
                v[1] -= __uint_as_float(u1 & 0xffff0000u);
            }
        }
    }
    static __device__ __forceinline__ floatx4 mfma(uint4v a, uint4v b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, a), __builtin_bit_cast(bf8_t, b), c, 0, 0,
                                                       0);
    }
};
template <>
struct Mul<float> {
    static constexpr int NP = 1;
    static constexpr float PEXP = 0;
    static constexpr uint32_t ONE = 0x3f800000;
    static __device__ __forceinline__ uint32_t finite(uint32_t u) {
        return 0u - (((~u & 0x7f800000u) + 0x7fffffffu) >> 31);
    }
    static __device__ __forceinline__ floatx4 mfma(uint4v a, uint4v b, floatx4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
        return c;
    }
};

// A load from global memory (a flat one, which the compiler takes where it does not see
// that, counts as an LDS access too, and waits for Q's would wait for it).
template <class T>
__device__ __forceinline__ T global_load(const char* base, uint32_t off) {
    typedef const __attribute__((address_space(1))) char* Bytes;
    return *(const __attribute__((address_space(1))) T*)((Bytes)(uintptr_t)base + off);
}

template <class E, int HD>
struct PagedGeom {
    static constexpr bool F32 = sizeof(E) == 4;
    static constexpr int KS = F32 ? 16 : 32;           // keys of a step
    static constexpr int NT = KS / 16;                 // 16-key tiles of a step
    static constexpr int EV = 16 / (int)sizeof(E);     // elements of 16 bytes
    static constexpr int CK = HD / (4 * EV);           // 16-byte loads of a key's row per lane
    static constexpr int CW = F32 || HD == 64 ? 4 : 8; // columns of V per lane and load
    static constexpr int HH = HD / (16 * CW);          // such loads of a row
    static constexpr int VK = KS / 4;                  // keys of V per lane
    static constexpr int VD = CW * (int)sizeof(E) / 4; // dwords of such a load
    static constexpr int ND = HD / 16;
    static constexpr int NP = Mul<E>::NP;
};

// RW groups of 4 / RW waves: a group has 16 RT rows and all keys of the range, so
// that a block's K and V come once from memory and RW times from the L2.
// FULL: head_dim is HD (else smaller).  P: pages hold whole tiles of 16 keys, so that a
// tile's page is the same for all lanes; or whole fours, the keys of a lane in S^T; or
// any number of rows (1).
template <class E, int HD, int RT, int RW, bool FULL, int P>
__global__ __launch_bounds__(256, HD > 128 ? 1 : 2) void attn_paged_kernel(PagedAttn a, PagedBatch pb) {
    using Geo = PagedGeom<E, HD>;
    using M = Mul<E>;
    constexpr bool F32 = Geo::F32;
    constexpr int KS = Geo::KS, NT = Geo::NT, EV = Geo::EV, CK = Geo::CK, CW = Geo::CW, HH = Geo::HH, VK = Geo::VK;
    constexpr int VD = Geo::VD, ND = Geo::ND, NP = Geo::NP;
    constexpr bool P16 = P == 16;
    constexpr int KW = 4 / RW, GROUP = 16 * RT, ROWS = RW * GROUP;
    constexpr int SUB = AP_SLICE / KS;                 // steps of a slice
    constexpr bool QLDS = RT > 1 || RW > 1 || HD > 128;        // Q waits in LDS
    constexpr int WGS = paged_wgs(HD);
    constexpr int OS = HD + 4;                         // row stride of a wave's results in LDS (floats)
    // Q while a range is worked on, then the waves' results
    constexpr int Q_BYTES = QLDS ? RW * RT * NP * CK * 64 * 16 : 0, O_BYTES = 4 * GROUP * OS * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[Q_BYTES > O_BYTES ? Q_BYTES : O_BYTES];
    __shared__ float s_m[4][GROUP], s_l[4][GROUP];
    float(*const s_o)[GROUP][OS] = (float(*)[GROUP][OS])smem;
    uint4v(*const s_q)[RT * NP * CK][64] = (uint4v(*)[RT * NP * CK][64])smem;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, j = lane & 15, kw = w % KW, rg = w / KW;
    const int Hkv = a.kv.n_kv_heads, G = a.Hq / Hkv, hd = FULL ? HD : a.kv.head_dim, ps = a.pg.page_size;
    using PlanT = Plan<PagedCount<ROWS>, PagedBatch>;
    const PagedCount<ROWS> count{G, Hkv};
    const PlanT plan(pb, count);
    const bool cuts = paged_cuts(pb.max_seq);
    const PagedBegin begin = paged_begin<WGS>(plan, blockIdx.x, cuts);
    const int x0 = begin.x;
    if (x0 >= plan.total) {
        if (threadIdx.x == 0) entry_of(a.ws, blockIdx.x)->rows = 0;
        return;
    }
    const float scale2 = (1.0f / sqrtf((float)hd)) * LOG2E;
    const int64_t row_b = a.kv.row_stride * (int)sizeof(E);

    struct Piece {
        SeqView seq;
        int h, r0, gran, g0, g1;       // kv head, first row of the block
        const int32_t* table;
        int64_t head_b;                // byte offset of the head
    };
    auto piece_of = [&](const Place& pl) {
        Piece p;
        p.seq = pl.seq;
        p.gran = paged_granules(pl.seq.p0 + pl.seq.n);
        const int nb = count.blocks(pl.seq), b = pl.at / p.gran;
        p.h = b / nb;
        p.r0 = ROWS * (b % nb);
        p.g0 = pl.at % p.gran;
        p.g1 = p.gran;                                 // if the range goes so far
        p.table = a.pg.table + pl.base * a.pg.max_pages;
        p.head_b = p.h * a.kv.head_stride * (int)sizeof(E);
        return p;
    };

    // Pages.  P16: lane l has the page and the row within it of the wave's tile `at` +
    // l; else of the P keys from P l on of a step.
    struct Found {
        int page, row;
    };
    auto look_up = [&](const Piece& p, int key) {
        const int last = p.seq.p0 + p.seq.n - 1, k = min(key, last);
        const int i = (int)((unsigned)k / (unsigned)ps), page = p.table[i];
        int r = k - i * ps;
        r &= ~(P - 1);
        return Found{page, r};                         // (the page is looked at when it is used)
    };
    auto is_page = [&](int page) { return (unsigned)page < (unsigned)a.pg.n_pages; };
    // a wave's slices: every KW-th of a granule
    auto slice_key = [&](const Piece& p, int i) {
        return min(p.g0 + i / RW, p.gran) * AP_GRAN + (kw + KW * (i % RW)) * AP_SLICE;
    };
    auto step_key = [&](const Piece& p, int s) { return slice_key(p, s / SUB) + s % SUB * KS; };
    auto tiles_at = [&](const Piece& p, int at) {
        const int i = at + lane;
        return look_up(p, slice_key(p, i >> 1) + (i & 1) * 16);
    };
    auto keys_at = [&](const Piece& p, int s) { return look_up(p, step_key(p, s) + P * (lane & (KS / P - 1))); };
    // where a step's rows are: byte offsets from the head's start
    struct Where {
        int64_t tile[P16 ? NT : 1];    // P16: of the tiles (the same in all lanes)
        int64_t row;                   // else: of the lane's P keys
        bool good;                     // all of the step's pages are there
        uint64_t there;                // else: which lanes' are
        bool tgood[NT];
    };
    Found near;                        // P16: pages of the 64 tiles at tbase; else of the next step's keys
    int tbase = 0;
    auto where_of = [&](const Piece& p, int s) {
        Where wh;
        if constexpr (P16) {
            wh.good = true;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int i = s * NT + t - tbase;
                const int page = __builtin_amdgcn_readlane(near.page, i), r = __builtin_amdgcn_readlane(near.row, i);
                wh.tgood[t] = is_page(page);
                wh.good &= wh.tgood[t];
                wh.tile[t] = (int64_t)(wh.tgood[t] ? page : 0) * (a.kv.page_stride * (int)sizeof(E)) + r * row_b;
            }
        } else {
            const Found f = near;
            wh.there = __builtin_amdgcn_ballot_w64(is_page(f.page)) | ~((1ull << KS / P) - 1);
            wh.good = wh.there == ~0ull;
            wh.row = (int64_t)(is_page(f.page) ? f.page : 0) * (a.kv.page_stride * (int)sizeof(E)) + f.row * row_b;
        }
        return wh;
    };
    auto from_lane = [&](int64_t v, int l) {
        const uint32_t lo = __shfl((int)(uint32_t)v, l), hi = __shfl((int)((uint64_t)v >> 32), l);
        return (int64_t)((uint64_t)hi << 32 | lo);
    };
    uint4v kr[NT][CK];
    uint32_t vr[VK][HH][VD];
    // the lane's part of the addresses
    const uint32_t k_off = j % P * (uint32_t)row_b + EV * g * (uint32_t)sizeof(E);
    const uint32_t k_last = j % P * (uint32_t)row_b + (hd - EV) * (uint32_t)sizeof(E);
    uint32_t v_off[4], v_last[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t row = (4 * g + i) % P * (uint32_t)row_b;
        v_off[i] = row + CW * j * (uint32_t)sizeof(E);
        v_last[i] = row + (hd - CW) * (uint32_t)sizeof(E);
    }
    uint32_t real = ~0u;                               // 0: loads that nothing waits for, all lanes the same bytes
    auto load_k = [&](const Piece& p, const Where& wh) {
        const char* pool = (const char*)a.kv.K + p.head_b;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const char* base;
            if constexpr (P16)
                base = uniform(pool + wh.tile[t]);
            else
                base = pool + from_lane(wh.row, (16 * t + j) / P);
#pragma unroll
            for (int c = 0; c < CK; ++c) {
                uint32_t off = (k_off & real) + 64 * c;
                if (!FULL) off = min(off, k_last);     // past the row Q is 0
                kr[t][c] = global_load<uint4v>(base, off);
            }
        }
    };
    auto load_v = [&](const Piece& p, const Where& wh) {
        const char* pool = (const char*)a.kv.V + p.head_b;
        const char* base = nullptr;
#pragma unroll
        for (int i = 0; i < VK; ++i) {
            if constexpr (P16) {
                if (i % 4 == 0) base = uniform(pool + wh.tile[i / 4]);
            } else {
                if (i % P == 0) base = pool + from_lane(wh.row, (16 * (i / 4) + 4 * g + i % 4) / P);
            }
#pragma unroll
            for (int hh = 0; hh < HH; ++hh) {
                uint32_t off = (v_off[i % 4] & real) + 16 * CW * hh * (uint32_t)sizeof(E);
                if (!FULL) off = min(off, v_last[i % 4]);      // columns that are not written out
                if constexpr (VD == 4) {
                    const uint4v x = global_load<uint4v>(base, off);
#pragma unroll
                    for (int e = 0; e < 4; ++e) vr[i][hh][e] = x[e];
                } else {
                    const uint2v x = global_load<uint2v>(base, off);
                    vr[i][hh][0] = x[0];
                    vr[i][hh][1] = x[1];
                }
            }
        }
    };

    uint4v qr[QLDS ? 1 : NP][QLDS ? 1 : CK];
    float unq[RT];
    // Q of the block's rows as the B operand, elements as K's loads have them
    auto load_q = [&](const Piece& p) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = p.r0 + GROUP * rg + 16 * rt + j;
            const bool live = r < p.seq.n * G;
            const float* qp =
                a.q + ((int64_t)(p.seq.t0 + (live ? r / G : 0)) * a.Hq + p.h * G + (live ? r % G : 0)) * hd;
            float x[CK][EV], top = 0.f;
#pragma unroll
            for (int c = 0; c < CK; ++c) {
                const int e0 = 4 * EV * c + EV * g;
                const bool in = live && (FULL || e0 < hd);
#pragma unroll
                for (int e = 0; e < EV; e += 4) {
                    const float4u v = *(const float4u*)(qp + (FULL || e0 < hd ? e0 : 0) + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        x[c][e + k] = in ? v[k] * scale2 : 0.f;
                        top = fmaxf(top, fabsf(x[c][e + k]));
                    }
                }
            }
            unq[rt] = 1.0f;
            if constexpr (NP == 2) {                   // to [2^13, 2^14) at the row's largest: lo keeps its bits
                top = cols_max(top);
                const int e2 = top > 0.f ? min(126, 14 - __builtin_amdgcn_frexp_expf(top)) : 0;
                unq[rt] = ldexpf(1.0f, -e2);
#pragma unroll
                for (int c = 0; c < CK; ++c)
#pragma unroll
                    for (int e = 0; e < EV; ++e) x[c][e] = ldexpf(x[c][e], e2);
            }
#pragma unroll
            for (int c = 0; c < CK; ++c) {
                uint4v part[NP];
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[0][e] = __float_as_uint(x[c][e]);
                } else {
                    M::split(x[c], part);
                }
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    if constexpr (QLDS) {
                        if (c % KW == kw) s_q[rg][(rt * NP + k) * CK + c][lane] = part[k];
                    } else {
                        qr[k][c] = part[k];
                    }
                }
            }
        }
    };
    auto q_of = [&](int rt, int k, int c) {
        if constexpr (QLDS)
            return s_q[rg][(rt * NP + k) * CK + c][lane];
        else
            return qr[k][c];
    };

    Piece pc = piece_of(begin.place);
    auto start_piece = [&]() {
        tbase = 0;
        if constexpr (P16) {
            near = tiles_at(pc, 0);
        } else {
            near = keys_at(pc, 0);
        }
        const Where wh = where_of(pc, 0);
        if constexpr (!P16) near = keys_at(pc, 1);
        return wh;
    };
    Where wh = start_piece();
    load_k(pc, wh);
    load_v(pc, wh);
    const int x1 = paged_begin<WGS>(plan, blockIdx.x + 1, cuts).x;
    if (x0 >= x1) {                                    // the block is another workgroup's
        if (threadIdx.x == 0) entry_of(a.ws, blockIdx.x)->rows = 0;
        return;
    }
    pc.g1 = min(pc.gran, pc.g0 + (x1 - x0));
    load_q(pc);
    if (w == 0)
        leave_entry(a.ws, WGS, blockIdx.x, x0, pc.g0, pc.gran, plan,
                    [&](int v) { return paged_begin<WGS>(plan, v, cuts).x; },
                    JoinEntry{pc.seq.t0, min(ROWS, pc.seq.n * G - pc.r0), pc.r0, pc.h, 0, 0});
    if (QLDS) __syncthreads();

    for (int x = x0;;) {
        const SeqView sv = pc.seq;
        const int last = sv.p0 + sv.n - 1, h = pc.h, r0 = pc.r0, rows = min(ROWS, sv.n * G - r0);
        const int rw = r0 + GROUP * rg;                // the group's first row
        const int all_see = sv.p0 + rw / G;            // the last key that all of its rows see
        const int own = min(GROUP, r0 + rows - rw);    // its rows: it may have none
        const int most = sv.p0 + (rw + own - 1) / G;   // the last key that any of them sees
        const bool mixed = most != all_see;
        int lim[RT];                                   // the last key that row j sees
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = rw + 16 * rt + j;
            lim[rt] = r < r0 + rows ? sv.p0 + r / G : -1;
        }
        floatx4 o[RT][ND];                             // column 16 CW hh + CW (4g + i) + c of row j: o[CW hh + c][i]
        float m[RT], l[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.f;
#pragma unroll
            for (int n = 0; n < ND; ++n) o[rt][n] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
        const int xn = x + pc.g1 - pc.g0;
        const bool more = xn < x1, whole = pc.g0 == 0 && pc.g1 == pc.gran;
        // steps that have keys (in the last granule a wave may have none); one at least, for the loads behind it
        int steps = own > 0 ? (pc.g1 - pc.g0) * SUB * RW : 1;
        while (steps > 1 && step_key(pc, steps - 1) > last) --steps;
        for (int s = 0; s < steps; ++s) {
            const int k0 = step_key(pc, s);
            const Where at = wh;
            // scores
            floatx4 sc[RT][NT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int t = 0; t < NT; ++t) sc[rt][t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < CK; ++c)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        const uint4v q = q_of(rt, k, c);
#pragma unroll
                        for (int t = 0; t < NT; ++t) sc[rt][t] = M::mfma(kr[t][c], q, sc[rt][t]);
                    }
            __builtin_amdgcn_sched_barrier(0);
            // the next step's keys, the next piece's or, at the end, some bytes: no load hangs on a
            // branch, so that the compiler can count how many may be under way at a wait
            if (s + 1 < steps) {
                if constexpr (P16) {
                    if ((s + 1) * NT - tbase >= 64) {
                        tbase += 64;
                        near = tiles_at(pc, tbase);
                        SH_WAIT_VMCNT(0);              // here, every 32 steps, rather than where its lanes are read
                    }
                }
                wh = where_of(pc, s + 1);
                if constexpr (!P16) near = keys_at(pc, s + 2);
            } else if (more) {
                pc = piece_of(plan.find(xn));
                pc.g1 = min(pc.gran, pc.g0 + (x1 - xn));
                wh = start_piece();
            } else {
                real = 0;
                if constexpr (!P16) wh.row = 0;
            }
            load_k(pc, wh);
            __builtin_amdgcn_sched_barrier(0);
            // keys that not all rows see; V of those that none sees or that are not there is taken out
            if (k0 + KS - 1 > all_see || !at.good) {
                auto there = [&](int key) {            // a key of the step, counted from k0
                    const bool page = P16 ? at.tgood[NT == 1 ? 0 : key >> 4] : (at.there >> key / P & 1) != 0;
                    return page && k0 + key <= most;
                };
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = 16 * t + 4 * g + i;
                        const bool is = there(key);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            if (!is || k0 + key > lim[rt]) sc[rt][t][i] = -INFINITY;
                        if (!is)
#pragma unroll
                            for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                                for (int d = 0; d < VD; ++d) vr[4 * t + i][hh][d] = 0;
                    }
                // infinities and NaN in V: 0 times them is not 0, so they are taken out, and rows that
                // see them get NaN
                if (mixed) {
                    uint32_t odd = 0;
#pragma unroll
                    for (int i = 0; i < VK; ++i)
#pragma unroll
                        for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                            for (int d = 0; d < VD; ++d) odd |= ~M::finite(vr[i][hh][d]);
                    if (__builtin_amdgcn_ballot_w64(odd != 0)) {
                        uint32_t sees[RT][4];          // 1 where row j sees the lane's key, as P's operand
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (F32)
                                    sees[rt][e] = sc[rt][0][e] != -INFINITY ? M::ONE : 0;
                                else
                                    sees[rt][e] = (sc[rt][e / 2][2 * e % 4] != -INFINITY ? M::ONE & 0xffff : 0) |
                                                  (sc[rt][e / 2][2 * e % 4 + 1] != -INFINITY ? M::ONE & 0xffff0000u : 0);
                            }
#pragma unroll
                        for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                            for (int d = 0; d < VD; ++d) {
                                uint32_t wild[VK];
#pragma unroll
                                for (int i = 0; i < VK; ++i) {
                                    const uint32_t fine = M::finite(vr[i][hh][d]);
                                    wild[i] = ~fine & M::ONE;
                                    vr[i][hh][d] &= fine;
                                }
#pragma unroll
                                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                                    for (int c = 0; c < (F32 ? 1 : 2); ++c) {
                                        floatx4 hit = {0.f, 0.f, 0.f, 0.f};
                                        if constexpr (F32) {
#pragma unroll
                                            for (int i = 0; i < 4; ++i)
                                                hit = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                                    __uint_as_float(wild[i]), __uint_as_float(sees[rt][i]), hit, 0, 0, 0);
                                        } else {
                                            uint4v A;
#pragma unroll
                                            for (int i = 0; i < 4; ++i)
                                                A[i] = __builtin_amdgcn_perm(wild[2 * i + 1], wild[2 * i],
                                                                             c ? 0x07060302 : 0x05040100);
                                            hit = M::mfma(A, uint4v{sees[rt][0], sees[rt][1], sees[rt][2], sees[rt][3]},
                                                          hit);
                                        }
                                        const int n = hh * CW + (F32 ? d : 2 * d + c);
#pragma unroll
                                        for (int i = 0; i < 4; ++i) o[rt][n][i] = hit[i] > 0.f ? NAN : o[rt][n][i];
                                        __builtin_amdgcn_sched_barrier(0);     // few registers at a time
                                    }
                            }
                    }
                }
            }
            // weights: 2^(score - m + PEXP)
            float p[RT][VK];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mx = sc[rt][0][0];
#pragma unroll
                for (int e = 1; e < 4 * NT; ++e) mx = fmaxf(mx, sc[rt][e >> 2][e & 3]);
                mx *= unq[rt];
                if (__builtin_amdgcn_ballot_w64(mx > m[rt] + AR_SLACK)) {
                    const float top = cols_max(mx);
                    if (top > m[rt] + AR_SLACK) {
                        const float f = __builtin_amdgcn_exp2f(m[rt] - top);
                        m[rt] = top;
                        l[rt] *= f;
#pragma unroll
                        for (int n = 0; n < ND; ++n) o[rt][n] *= f;
                    }
                }
                const float by = M::PEXP - (m[rt] == -INFINITY ? 0.f : m[rt]);
#pragma unroll
                for (int e = 0; e < 4 * NT; ++e) {
                    p[rt][e] = __builtin_amdgcn_exp2f(fmaf(sc[rt][e >> 2][e & 3], unq[rt], by));
                    l[rt] += p[rt][e];
                }
            }
            // outputs
            if constexpr (F32) {
#pragma unroll
                for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                    for (int c = 0; c < CW; ++c)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                o[rt][hh * CW + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __uint_as_float(vr[i][hh][c]), p[rt][i], o[rt][hh * CW + c], 0, 0, 0);
            } else {
                uint4v pp[RT][NP];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) M::split(p[rt], pp[rt]);
                if constexpr (M::LIFT > 0) {
                    ushort2v least[HH][VD], all = {0xffff, 0xffff};
#pragma unroll
                    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                        for (int d = 0; d < VD; ++d) {
                            least[hh][d] = M::low_rank(vr[0][hh][d]);
#pragma unroll
                            for (int i = 1; i < VK; ++i)
                                least[hh][d] = __builtin_elementwise_min(least[hh][d], M::low_rank(vr[i][hh][d]));
                            all = __builtin_elementwise_min(all, least[hh][d]);
                        }
                    auto low = [](ushort2v x) {
                        return __builtin_amdgcn_ballot_w64(min(x[0], x[1]) < M::LOW_RANKS) != 0;
                    };
                    if (low(all)) {
#pragma unroll
                        for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                            for (int d = 0; d < VD; ++d) {
                                if (!low(least[hh][d])) continue;
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    uint4v v;
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        const uint32_t two = __builtin_amdgcn_perm(
                                            vr[2 * i + 1][hh][d], vr[2 * i][hh][d], c ? 0x07060302 : 0x05040100);
                                        v[i] = M::lifted(two & ~M::large(two));
                                    }
#pragma unroll
                                    for (int rt = 0; rt < RT; ++rt) {
                                        floatx4& acc = o[rt][hh * CW + 2 * d + c];
                                        acc *= 1 << M::LIFT;
#pragma unroll
                                        for (int k = 0; k < NP; ++k) acc = M::mfma(v, pp[rt][k], acc);
                                        acc *= 1.0f / (1 << M::LIFT);
                                    }
                                }
#pragma unroll
                                for (int i = 0; i < VK; ++i) vr[i][hh][d] &= M::large(vr[i][hh][d]);
                                __builtin_amdgcn_sched_barrier(0);     // few registers at a time
                            }
                    }
                }
#pragma unroll
                for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                    for (int d = 0; d < VD; ++d) {
                        uint4v v0, v1;                 // columns 2d and 2d + 1 of the lane's keys
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            v0[i] = __builtin_amdgcn_perm(vr[2 * i + 1][hh][d], vr[2 * i][hh][d], 0x05040100);
                            v1[i] = __builtin_amdgcn_perm(vr[2 * i + 1][hh][d], vr[2 * i][hh][d], 0x07060302);
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int k = 0; k < NP; ++k) {
                                o[rt][hh * CW + 2 * d] = M::mfma(v0, pp[rt][k], o[rt][hh * CW + 2 * d]);
                                o[rt][hh * CW + 2 * d + 1] = M::mfma(v1, pp[rt][k], o[rt][hh * CW + 2 * d + 1]);
                            }
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v(pc, wh);
            __builtin_amdgcn_sched_barrier(0);
        }

        // the waves' results are joined through LDS
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float sum = cols_sum(l[rt]);
            if (g == 0) {
                s_m[w][16 * rt + j] = m[rt];
                s_l[w][16 * rt + j] = sum;
            }
        }
        if (QLDS) __syncthreads();                     // no wave reads Q any more
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int hh = 0; hh < HH; ++hh)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < CW; c += 4) {
                        floatx4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = o[rt][hh * CW + c + e][i];
                        *(floatx4*)&s_o[w][16 * rt + j][16 * CW * hh + CW * (4 * g + i) + c] = v;
                    }
        __syncthreads();
        float* slot = slot_of(a.ws, WGS, 2 * blockIdx.x + (x == x0 ? 0 : 1), ROWS, HD);
        for (int u = threadIdx.x; u < rows * (HD / 4); u += 256) {
            const int r = u / (HD / 4), c = 4 * (u % (HD / 4)), w0 = r / GROUP * KW, rl = r % GROUP;
            float mt = s_m[w0][rl];
#pragma unroll
            for (int k = 1; k < KW; ++k) mt = fmaxf(mt, s_m[w0 + k][rl]);
            floatx4 sum = {0.f, 0.f, 0.f, 0.f};
            float lt = 0.f;
#pragma unroll
            for (int k = w0; k < w0 + KW; ++k) {
                // a maximum of -infinity with a sum: scores that are NaN, kept; and 0 times NaN or infinity is NaN, so
                // that these are seen whatever weight their part has
                const float f = s_m[k][rl] == -INFINITY ? (s_l[k][rl] == 0.f ? 0.f : 1.f)
                                                        : __builtin_amdgcn_exp2f(s_m[k][rl] - mt);
                lt += f * s_l[k][rl];
                sum += f * *(const floatx4*)&s_o[k][rl][c];
            }
            if (whole) {
                const float inv = lt == 0.f ? 0.f : 1.0f / lt;
                const int row = r0 + r;
                if (FULL || c < hd)
                    *(float4u*)(a.out + ((int64_t)(sv.t0 + row / G) * a.Hq + h * G + row % G) * hd + c) = sum * inv;
            } else {
                *(floatx4*)(slot + r * HD + c) = sum;
                if (c == 0)                            // NaN scores only: nothing else counts beside them
                    *(float2*)(slot + ROWS * HD + 2 * r) = make_float2(mt == -INFINITY && lt != 0.f ? INFINITY : mt, lt);
            }
        }
        if (!more) break;
        __syncthreads();                               // before these rows' places are written again
        load_q(pc);
        if (QLDS) __syncthreads();
        x = xn;
    }
}

// The kernels of a type, each in a file of its own.
template <class E>
void launch_attention_paged_type(const PagedAttn& a, const PagedBatch& pb, hipStream_t s);
template <>
void launch_attention_paged_type<float>(const PagedAttn& a, const PagedBatch& pb, hipStream_t s);
template <>
void launch_attention_paged_type<_Float16>(const PagedAttn& a, const PagedBatch& pb, hipStream_t s);
template <>
void launch_attention_paged_type<__bf16>(const PagedAttn& a, const PagedBatch& pb, hipStream_t s);

// Pages of whole tiles of 16 rows are looked up by the tile, others by four rows or, of odd
// sizes, by the row (decode of 16, bf16, pages of 16 rows: 41, 46 and 54 us; the addresses
// take registers, and the 16-bit kernels of head_dim 128 keep 36 to 152 bytes a lane in
// scratch memory there).
template <class E, int HD, int RT, int RW>
static void launch_paged_rows(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    const dim3 grid(paged_wgs(HD)), th(256);
    if (a.pg.page_size % 4 != 0)
        hipLaunchKernelGGL((attn_paged_kernel<E, HD, RT, RW, false, 1>), grid, th, 0, s, a, pb);
    else if (a.pg.page_size % 16 != 0)
        hipLaunchKernelGGL((attn_paged_kernel<E, HD, RT, RW, false, 4>), grid, th, 0, s, a, pb);
    else if (a.kv.head_dim != HD)
        hipLaunchKernelGGL((attn_paged_kernel<E, HD, RT, RW, false, 16>), grid, th, 0, s, a, pb);
    else
        hipLaunchKernelGGL((attn_paged_kernel<E, HD, RT, RW, true, 16>), grid, th, 0, s, a, pb);
    if (paged_cuts(pb.max_seq))
        launch_attn_join_paged(a.out, a.ws, a.Hq, a.kv.n_kv_heads, a.kv.head_dim, HD, 16 * RT * RW, paged_wgs(HD), s);
}

// Rows of a block, by the query rows that a kv head's sequences may bring (max_new decides
// for the whole call: beside a prompt chunk decode rows lie in its large blocks).  8 kv heads,
// us a call; 16 / 32 / 64 rows in a block:
//  - 4 rows (one token of 4 heads, 16 sequences, bf16 of 128): 41 / 45 / -;
//  - 20 rows (5 tokens of 4 heads, 16 sequences, bf16 of 128): 93 / 84 / 87, of 64: - / 48 / 52;
//  - 64 rows (8 tokens of 8 heads, 8 sequences of up to 16384 keys, of 128): bf16 138 / 120 /
//    101, f32 - / 187 / 194; prompt chunks of 600 tokens: bf16 - / 390 / 276, f32 - / 776 / 766.
// 64 rows share K and V between two groups of waves, which f32's products are too long to
// gain by (16 sequences of 5 tokens of 8 heads: 193 / 211).  head_dim 256 has registers for
// 16 rows a wave; two groups of waves, 32 rows, take 76 us where 16 rows take 86 (64 rows,
// bf16), and 1040 where they take 1397 (chunks).
template <class E>
static void launch_paged_hd(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    constexpr int MOST = sizeof(E) == 4 ? 1 : 2;       // groups of waves
    const int64_t rows = (int64_t)pb.max_new * (a.Hq / a.kv.n_kv_heads);
    if (a.kv.head_dim > 128)
        rows <= 16 ? launch_paged_rows<E, 256, 1, 1>(a, pb, s) : launch_paged_rows<E, 256, 1, 2>(a, pb, s);
    else if (a.kv.head_dim > 64)
        rows <= 16   ? launch_paged_rows<E, 128, 1, 1>(a, pb, s)
        : rows <= 32 ? launch_paged_rows<E, 128, 2, 1>(a, pb, s)
                     : launch_paged_rows<E, 128, 2, MOST>(a, pb, s);
    else
        rows <= 16   ? launch_paged_rows<E, 64, 1, 1>(a, pb, s)
        : rows <= 32 ? launch_paged_rows<E, 64, 2, 1>(a, pb, s)
                     : launch_paged_rows<E, 64, 2, MOST>(a, pb, s);
}

}  // namespace slate_hip
