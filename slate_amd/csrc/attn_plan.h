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
    int64_t base;                      // kv_base
    int at;
};

// Count(SeqView) -> granules of a sequence (all its heads and blocks).
template <class Count>
class Plan {
  public:
    int total;
    int end;                           // sequences from it on are left out

    __device__ __forceinline__ Plan(const PackedBatch& pb, const Count& count) : pb_(pb), count_(count) {
        end = pb.B;
        cut(0);
        first_ = load(0);
        total = __builtin_amdgcn_readlane(first_.upto, 63);
        for (int b0 = 64; b0 < end; b0 += 64) {
            cut(b0);
            total += __builtin_amdgcn_readlane(load(b0).upto, 63);
        }
    }
    // The plan's first 64 sequences can wait in LDS instead of in registers.
    struct Lane {
        SeqView seq;
        int64_t base;
        int own, upto;                 // granules of the lane's sequence, and with those of the lanes before it
    };
    __device__ __forceinline__ Plan(const PackedBatch& pb, const Count& count, int total_, int end_, const Lane& first)
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
    __device__ __forceinline__ void cut(int b0) {
        const int b = b0 + (int)(threadIdx.x & 63);
        const uint64_t falls = __builtin_amdgcn_ballot_w64(b < end && pb_.tok_off[b + 1] < pb_.tok_off[b]);
        if (falls) end = b0 + __builtin_ctzll(falls);
    }
    __device__ __forceinline__ Lane load(int b0) const {
        const int b = b0 + (int)(threadIdx.x & 63);
        Lane s{};
        if (b < end) {
            s.seq = seq_view(pb_, b);
            s.base = pb_.kv_base[b];
            s.own = count_(s.seq);
        }
        s.upto = wave_scan(s.own);
        return s;
    }
    const PackedBatch& pb_;
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
