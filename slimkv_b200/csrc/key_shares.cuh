// Equal shares of a batch's key tiles, cut on the device from its lengths.
//
// A unit is one key tile of one segment (sequence, KV head, row group);
// the units of all segments in a row are cut into one equal share per CTA, and
// the part of a segment inside a share is a piece.  In front of its tiles a
// segment has kPieceUnits units without work: what a further piece costs a CTA
// (every CTA has one), so that shares with several short pieces take no longer
// than those within one segment.  Plan names the work:
//   static constexpr int kPieceUnits;
//   int batch, kv_heads, ctas;
//   Seq sequence(int b) const;     // with int tiles, groups: a sequence's key
//                                  // tiles and row groups (0: nothing to do)
#pragma once

#include "common.cuh"

namespace slimkv {

// Callers make sure that a call has fewer than 2^31 units.
template <class Plan, class Seq>
__device__ __forceinline__ uint32_t segment_units(const Plan&, const Seq& s) {
    return s.tiles > 0 ? uint32_t(s.tiles + Plan::kPieceUnits) : 0u;
}
template <class Plan>
__device__ __forceinline__ uint32_t units_of(const Plan& P, int b) {
    const auto s = P.sequence(b);
    return uint32_t(P.kv_heads) * uint32_t(s.groups) * segment_units(P, s);
}
// CTAs with a share: every share holds at least one unit.
__device__ __forceinline__ uint32_t share_count(uint32_t total, int ctas) { return min(total, uint32_t(ctas)); }
// floor(total cta / ctas) in 32 bits.
__device__ __forceinline__ uint32_t share_begin(uint32_t total, uint32_t cta, uint32_t ctas) {
    const uint32_t q = total / ctas;
    return q * cta + (total - q * ctas) * cta / ctas;
}
// The CTA whose share holds unit u: an estimate, put right.
__device__ __forceinline__ uint32_t share_of(uint32_t total, uint32_t u, uint32_t ctas) {
    uint32_t c = min(uint32_t(float(u) * float(ctas) / float(total)), ctas - 1);
    while (share_begin(total, c, ctas) > u) --c;
    while (c + 1 < ctas && share_begin(total, c + 1, ctas) <= u) ++c;
    return c;
}

// Units of all sequences, and of those before sequence `upto`, by one warp.
template <class Plan>
__device__ __forceinline__ void sum_units(const Plan& P, int upto, uint32_t& total, uint32_t& before) {
    total = before = 0;
    for (int b = threadIdx.x & 31; b < P.batch; b += 32) {
        const uint32_t u = units_of(P, b);
        total += u;
        if (b < upto) before += u;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    before = __reduce_add_sync(0xffffffffu, before);
}

// Where a CTA's share begins, in shared memory.
struct Share {
    uint32_t total;             // units of all sequences
    uint32_t first_u;           // units before sequence first_b
    int first_b;
    int ctas;                   // CTAs with a share
};

// Fills `share`, by one warp (the caller synchronises before reading it).
template <class Plan>
__device__ __forceinline__ void find_share(const Plan& P, Share* share) {
    const int lane = threadIdx.x & 31;
    uint32_t total = 0, first = 0;              // units of the first 32 sequences stay in registers
    for (int b = lane; b < P.batch; b += 32) {
        const uint32_t u = units_of(P, b);
        if (b == lane) first = u;
        total += u;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    const uint32_t ctas = share_count(total, P.ctas);
    if (lane == 0) { share->total = total; share->ctas = int(ctas); }
    if (blockIdx.x >= ctas) return;
    const uint32_t u0 = share_begin(total, blockIdx.x, ctas);
    uint32_t base = 0;
    for (int b0 = 0; b0 < P.batch && base <= u0; b0 += 32) {
        const uint32_t own = b0 == 0 ? first : b0 + lane < P.batch ? units_of(P, b0 + lane) : 0;
        uint32_t incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const uint32_t ex = base + incl - own;
        if (own && u0 >= ex && u0 < ex + own) {
            share->first_b = b0 + lane;
            share->first_u = ex;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// A CTA's pieces in order (CTAs with a share only; there may be none).
template <class Plan>
struct Walk {
    int left;                   // units of the share still to come
    int at;                     // units of the segment that are done
    int b, g, group;            // the piece's segment
    decltype(((const Plan*)nullptr)->sequence(0)) s;
    int t0, t1;                 // its key tiles
    int piece;                  // pieces begun before this one
    __device__ __forceinline__ void start(const Plan& P, const Share* share) {
        const uint32_t u = share_begin(share->total, blockIdx.x, share->ctas);
        left = int(share_begin(share->total, blockIdx.x + 1, share->ctas) - u);
        piece = -1;
        b = share->first_b;
        s = P.sequence(b);
        const uint32_t off = u - share->first_u, units = segment_units(P, s), seg = off / units;
        g = int(seg / uint32_t(s.groups));
        group = int(seg) - g * s.groups;
        at = int(off - seg * units);
    }
    // Moves to the next piece; false when the share is done.
    __device__ __forceinline__ bool next(const Plan& P) {
        for (; left > 0;) {
            if (at >= s.tiles + Plan::kPieceUnits) {
                at = 0;
                if (++group >= s.groups) {
                    group = 0;
                    if (++g >= P.kv_heads) {
                        g = 0;
                        do s = P.sequence(++b);
                        while ((s.groups == 0 || s.tiles == 0) && b + 1 < P.batch);
                    }
                }
            }
            t0 = max(at - Plan::kPieceUnits, 0);
            const int step = min(s.tiles + Plan::kPieceUnits - at, left);
            at += step;
            left -= step;
            t1 = at - Plan::kPieceUnits;
            if (t1 > t0) {
                ++piece;
                return true;
            }
        }
        return false;
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == s.tiles; }
};

}  // namespace slimkv
