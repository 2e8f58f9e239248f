// attn_plan.h -- how the packed attention kernels share out their work.
//
// The keys of every (sequence, kv head, block of query rows) are counted in
// granules and laid end to end; workgroup w of P takes the granules
// [N w / P, N (w+1) / P) of that line.  So every workgroup reads the same
// amount to within a granule whatever the lengths are, and only the first
// and the last piece of its range can be parts of a block whose rest lies in
// its neighbours': two slots of partial results per workgroup, whatever the
// batch.  A block that lies inside one range is written straight out.
// Every wave works the plan out by itself from the descriptors, which a lane
// each loads once; N < 2^31: the entries check it for T tokens, and sequences
// behind a fall of tok_off, which could have the same tokens over and over,
// are left out.
#pragma once
#include "lanes.h"
#include "packed.h"

namespace slate_hip {

constexpr float LOG2E = 1.4426950408889634f;

// Inclusive sum over the wave's lanes (DPP: within rows of 16, then across).
__device__ __forceinline__ int wave_scan(int v) {
#define SH_SCAN_STEP(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false)
    SH_SCAN_STEP(0x111, 0xF);          // row_shr:1, 2, 4, 8
    SH_SCAN_STEP(0x112, 0xF);
    SH_SCAN_STEP(0x114, 0xF);
    SH_SCAN_STEP(0x118, 0xF);
    SH_SCAN_STEP(0x142, 0xA);          // row_bcast:15 into rows 1 and 3
    SH_SCAN_STEP(0x143, 0xC);          // row_bcast:31 into rows 2 and 3
#undef SH_SCAN_STEP
    return v;
}

// A value that is the same in all lanes, for the scalar registers.
template <class T>
__device__ __forceinline__ T* uniform(T* p) {
    const uint64_t v = (uint64_t)p;
    return (T*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// A place on the line: granule `at` of the sequence's `own`.
struct Place {
    SeqView seq;
    int64_t base;                      // seq_base
    int at;
};

// Where a sequence's cache is: kv_base.
__device__ __forceinline__ int64_t seq_base(const PackedBatch& pb, int b) { return pb.kv_base[b]; }

// Count(SeqView) -> granules of a sequence (all its heads and blocks).  Batch
// has tok_off and B, seq_view and seq_base.
template <class Count, class Batch = PackedBatch>
class Plan {
  public:
    int total;
    int end;                           // sequences from it on are left out

    __device__ __forceinline__ Plan(const Batch& pb, const Count& count) : pb_(pb), count_(count) {
        end = pb.B;
        first_ = cut_and_load(0);
        total = __builtin_amdgcn_readlane(first_.upto, 63);
        for (int b0 = 64; b0 < end; b0 += 64) total += __builtin_amdgcn_readlane(cut_and_load(b0).upto, 63);
    }
    // The plan's first 64 sequences can wait in LDS instead of in registers.
    struct Lane {
        SeqView seq;
        int64_t base;
        int own, upto;                 // granules of the lane's sequence, and with those of the lanes before it
    };
    __device__ __forceinline__ Plan(const Batch& pb, const Count& count, int total_, int end_, const Lane& first)
        : total(total_), end(end_), pb_(pb), count_(count), first_(first) {}
    __device__ __forceinline__ const Lane& first() const { return first_; }
    // 0 <= x < total
    __device__ __forceinline__ Place find(int x) const {
        Lane s = first_;
        for (int b0 = 0, base = 0;;) {
            const uint64_t past = __builtin_amdgcn_ballot_w64(base + s.upto > x);
            if (past) {
                const int l = __builtin_ctzll(past);
                const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)s.base, l);
                const uint32_t hi = __builtin_amdgcn_readlane((int)((uint64_t)s.base >> 32), l);
                return Place{{__builtin_amdgcn_readlane(s.seq.t0, l), __builtin_amdgcn_readlane(s.seq.n, l),
                              __builtin_amdgcn_readlane(s.seq.p0, l)},
                             (int64_t)((uint64_t)hi << 32 | lo),
                             x - base - __builtin_amdgcn_readlane(s.upto - s.own, l)};
            }
            base += __builtin_amdgcn_readlane(s.upto, 63);
            b0 += 64;
            s = load(b0);
        }
    }
    // First granule of workgroup w of P; with fewer granules than workgroups
    // the first ones get one each.
    __device__ __forceinline__ int begin(int w, int P) const {
        return total < P ? min(w, total) : (int)((uint64_t)(uint32_t)total * (uint32_t)w / (uint32_t)P);
    }

    // The first workgroup whose range begins at x or later.
    __device__ __forceinline__ int first_from(int x, int P) const {
        return total < P ? x : (int)(((uint64_t)(uint32_t)x * (uint32_t)P + (uint32_t)total - 1) / (uint32_t)total);
    }

  private:
    // Sequences b0 .. b0 + 63, all their descriptors in one round of loads.
    struct Read {
        SeqView seq;
        int64_t base;
        bool falls;                    // of tok_off behind the sequence: it ends the plan
    };
    __device__ __forceinline__ Read read(int b0) const {
        const int b = b0 + (int)(threadIdx.x & 63);
        Read r{};
        if (b < pb_.B) r = Read{seq_view(pb_, b), seq_base(pb_, b), pb_.tok_off[b + 1] < pb_.tok_off[b]};
        return r;
    }
    __device__ __forceinline__ Lane lane_of(int b0, const Read& r) const {
        Lane s{r.seq, r.base, 0, 0};
        if (b0 + (int)(threadIdx.x & 63) < end) s.own = count_(r.seq);
        s.upto = wave_scan(s.own);
        return s;
    }
    __device__ __forceinline__ Lane load(int b0) const { return lane_of(b0, read(b0)); }
    __device__ __forceinline__ Lane cut_and_load(int b0) {
        const Read r = read(b0);
        const uint64_t falls = __builtin_amdgcn_ballot_w64(r.falls);
        if (falls) end = min(end, b0 + __builtin_ctzll(falls));
        return lane_of(b0, r);
    }
    const Batch& pb_;
    const Count count_;
    Lane first_;
};

// What the join kernel does about the boundary before a workgroup, left in
// the workspace by that workgroup: the block that is first cut there.
struct JoinEntry {
    int t0, rows;                      // first token of the sequence, query rows of the block (0: nothing to join)
    int r0, h;                         // first row of the block, kv head
    int pieces;                        // this many neighbours hold a part each, from the workgroup before on
    int slot0;                         // the slot of the first part
};

// Workspace of P workgroups: a JoinEntry each, then two slots each of `rows` rows of
// hd outputs and a pair (m, l) per row.  Outputs and l are relative to 2^m.
__host__ __device__ constexpr int64_t slot_floats(int rows, int hd) { return (int64_t)rows * (hd + 2); }
__device__ __forceinline__ float* slot_of(void* ws, int P, int i, int rows, int hd) {
    return (float*)((char*)ws + 32 * P) + i * slot_floats(rows, hd);
}
__device__ __forceinline__ JoinEntry* entry_of(void* ws, int w) { return (JoinEntry*)((char*)ws + 32 * w); }
inline int64_t plan_bytes(int P, int rows, int hd) {
    return 32 * P + 2 * P * slot_floats(rows, hd) * (int64_t)sizeof(float);
}
// hd 32, 64 or 128.
void launch_attn_join(float* out, void* ws, int Hq, int Hkv, int hd, int slot_rows, int P, hipStream_t s);
// The same for slots of `slot_hd` (64, 128, 256) columns of which the first hd are
// real, and rows that may have seen no key (their outputs are zeros).
void launch_attn_join_paged(float* out, void* ws, int Hq, int Hkv, int hd, int slot_hd, int slot_rows, int P,
                            hipStream_t s);

// The entry of workgroup w, whose range begins at x0 in granule `in` of a
// block of `gran`; begin(w) are the ranges' beginnings.  Called by a whole
// wave (the searches are the wave's).
template <class PlanT, class Begin>
__device__ __forceinline__ void leave_entry(void* ws, int P, int w, int x0, int in, int gran, const PlanT& plan,
                                            const Begin& begin, JoinEntry e) {
    const int start = x0 - in;
    const int from = in > 0 ? begin(w - 1) : 0;
    e.pieces = in > 0 && from <= start ? min(P, plan.first_from(start + gran, P)) - (w - 1) : 0;
    if (e.pieces == 0) e.rows = 0;
    e.slot0 = 2 * (w - 1) + (from != start);
    if ((threadIdx.x & 63) == 0) *entry_of(ws, w) = e;
}

}  // namespace slate_hip
