// attn_plan.h -- how the packed attention kernels share out their work.
//
// The keys of every (sequence, kv head, block of query rows) are counted in
// granules and laid end to end; workgroup w of P takes the granules
// [N w / P, N (w+1) / P) of that line.  So every workgroup reads the same
// amount to within a granule whatever the lengths are, and at most the first
// and the last piece of its range are parts of a block whose rest lies in a
// neighbour's: two slots of partial results per workgroup, whatever the
// batch.  A block that lies inside one range is written straight out.
// Every wave works the plan out by itself from the descriptors.
#pragma once
#include "packed.h"

namespace slate_hip {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}
__device__ __forceinline__ int64_t read_lane64(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), lane);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// A value that is the same in all lanes, for the scalar registers.
template <class T>
__device__ __forceinline__ T* uniform(T* p) {
    const uint64_t v = (uint64_t)p;
    return (T*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// A place on the line: granule `at` of sequence b's `count`.
struct Place {
    int b;
    int64_t at;
};

// Count(SeqView) -> granules of a sequence (all its heads and blocks).
template <class Count>
struct Plan {
    const PackedBatch& pb;
    const Count count;
    int64_t own, upto;                 // the lane's sequence (of the first 64), and with those before it
    int64_t total;

    __device__ __forceinline__ Plan(const PackedBatch& pb_, const Count& c) : pb(pb_), count(c) {
        load(0);
        total = read_lane64(upto, 63);
        for (int b0 = 64; b0 < pb.B; b0 += 64) total += read_lane64(wave_scan(of(b0)), 63);
    }
    __device__ __forceinline__ int64_t of(int b0) const {
        const int b = b0 + (int)(threadIdx.x & 63);
        return b < pb.B ? count(seq_view(pb, b)) : 0;
    }
    __device__ __forceinline__ void load(int b0) {
        own = of(b0);
        upto = wave_scan(own);
    }
    // 0 <= x < total
    __device__ __forceinline__ Place find(int64_t x) const {
        int64_t c = own, u = upto, base = 0;
        for (int b0 = 0;;) {
            const uint64_t past = __builtin_amdgcn_ballot_w64(base + u > x);
            if (past) {
                const int l = __builtin_ctzll(past);
                return Place{b0 + l, x - base - (read_lane64(u, l) - read_lane64(c, l))};
            }
            base += read_lane64(u, 63);
            b0 += 64;
            c = of(b0);
            u = wave_scan(c);
        }
    }
    __device__ __forceinline__ int64_t begin(int64_t w, int64_t P) const { return total * w / P; }
};

}  // namespace slate_hip
