// Equal shares of a batch's key tiles, cut on the device from its lengths.
//
// A unit is one 128-key tile of one segment (sequence, KV head, row group);
// the units of all segments in a row are cut into one equal share per CTA, and
// the part of a segment inside a share is a piece.  Plan names the work:
//   int batch, kv_heads, ctas;
//   Seq sequence(int b) const;     // with int tiles, groups: a sequence's key
//                                  // tiles and row groups (0: nothing to do)
#pragma once

#include "common.cuh"

namespace slimkv {

template <class Plan>
__device__ __forceinline__ long long units_of(const Plan& P, int b) {
    const auto s = P.sequence(b);
    return (long long)P.kv_heads * s.groups * s.tiles;
}
// CTAs with a share: every share holds at least one unit.
__device__ __forceinline__ int share_count(long long total, int ctas) { return int(min(total, (long long)ctas)); }
__device__ __forceinline__ long long share_begin(long long total, int cta, int ctas) { return total * cta / ctas; }
// The CTA whose share holds unit u.
__device__ __forceinline__ int share_of(long long total, long long u, int ctas) { return int(((u + 1) * ctas - 1) / total); }

// Units of all sequences, and of those before sequence `upto`, over the block
// (`scan`: two words per warp).
template <int kThreads, class Plan>
__device__ __forceinline__ void sum_units(const Plan& P, int upto, long long& total, long long& before, long long* scan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long all = 0, head = 0;
    for (int b = tid; b < P.batch; b += kThreads) {
        const long long u = units_of(P, b);
        all += u;
        if (b < upto) head += u;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
        head += __shfl_xor_sync(0xffffffffu, head, o);
    }
    if (lane == 0) { scan[2 * warp] = all; scan[2 * warp + 1] = head; }
    __syncthreads();
    total = before = 0;
    for (int w = 0; w < kThreads / 32; ++w) { total += scan[2 * w]; before += scan[2 * w + 1]; }
    __syncthreads();
}

// Where a CTA's share begins, in shared memory.
struct Share {
    long long total;            // units of all sequences
    long long first_u;          // units before sequence first_b
    int first_b;
    int ctas;                   // CTAs with a share
    long long scan[40];         // two words for each of up to 20 warps
};

// Fills `share` (all threads; the caller synchronises before reading it).
template <int kThreads, class Plan>
__device__ __forceinline__ void find_share(const Plan& P, Share* share) {
    const int lane = threadIdx.x & 31;
    long long total, before;
    sum_units<kThreads>(P, 0, total, before, share->scan);
    const int ctas = share_count(total, P.ctas);
    if (threadIdx.x == 0) { share->total = total; share->ctas = ctas; }
    if (threadIdx.x >= 32 || int(blockIdx.x) >= ctas) return;
    const long long u0 = share_begin(total, blockIdx.x, ctas);
    long long base = 0;
    for (int b0 = 0; b0 < P.batch && base <= u0; b0 += 32) {
        const long long own = b0 + lane < P.batch ? units_of(P, b0 + lane) : 0;
        long long incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const long long ex = base + incl - own;
        if (own && u0 >= ex && u0 < ex + own) {
            share->first_b = b0 + lane;
            share->first_u = ex;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
}

// A CTA's pieces in order (CTAs with a share only).
template <class Plan>
struct Walk {
    int left;                   // units of the share still to come
    int b, g, group;            // the piece's segment
    decltype(((const Plan*)nullptr)->sequence(0)) s;
    int t0, t1;                 // its key tiles
    int piece;                  // pieces begun before this one
    __device__ __forceinline__ void start(const Plan& P, const Share* share) {
        const long long u = share_begin(share->total, blockIdx.x, share->ctas);
        left = int(share_begin(share->total, blockIdx.x + 1, share->ctas) - u);
        piece = -1;
        b = share->first_b;
        s = P.sequence(b);
        const long long off = u - share->first_u;
        const int seg = int(off / s.tiles);
        g = seg / s.groups;
        group = seg - g * s.groups;
        t1 = int(off - (long long)seg * s.tiles);       // as if a piece had ended here
    }
    // Moves to the next piece; false when the share is done.
    __device__ __forceinline__ bool next(const Plan& P) {
        if (left == 0) return false;
        if (t1 >= s.tiles) {
            t1 = 0;
            if (++group >= s.groups) {
                group = 0;
                if (++g >= P.kv_heads) {
                    g = 0;
                    do s = P.sequence(++b);
                    while ((s.groups == 0 || s.tiles == 0) && b + 1 < P.batch);
                }
            }
        }
        t0 = t1;
        t1 = min(s.tiles, t0 + left);
        left -= t1 - t0;
        ++piece;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == s.tiles; }
};

}  // namespace slimkv
