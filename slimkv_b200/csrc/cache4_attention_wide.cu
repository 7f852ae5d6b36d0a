// Attention over a 4-bit cache for more than 16 query rows to a KV head and more
// than 192 dims: the heads of a token over the latents (C ABI
// slimkv_cache4_attention).
//
// A warp of cache4_attention.cu has registers for 16 rows of 320 dims, so 32 rows
// would turn every code into an operand twice.  Here tcgen05 has the products, keys
// on its M side, the rows on N:
//   S^T [128 keys x N rows] = K . Q^T,    O^T [128 dims x N rows] (up to 3) += V^T . P^T.
// The codes become 16-bit operands once for 32 rows.  A K row belongs to one
// thread, which writes it to tensor memory (the A operand of S); V^T needs its keys
// side by side and goes through shared memory, which 320 dims leave room for one
// tile of.  A thread's lane is a key in S^T too, so its scores and its share of
// each row's sum are its own; a row's maximum is kept until a score passes it by
// 2^8, so only then do threads exchange maxima.
//
// Bound: a tile's steps, which follow one another through one V tile and (320 dims)
// one P tile, and what surrounds them.  16 sequences of 8k latents of 320 dims, 32 rows
// (7 tiles to a CTA), in a graph 37 us: by time stamps of each CTA the first tile's K
// is ready after 6.0 us, a tile takes 2.7, from the last P to the rows written it takes
// 4.9, the last CTA ends after 34.0, and the merge comes behind.  (K's codes in eight
// warps of their own: the same.  Sixteen warps for all codes: 43.  64 rows to a pass:
// 156 against 170 us for 256 rows, slower for 32 to 96.)
//
// Warps: 0 and 3 load the 4-bit K and V rows (TMA; 3 finds the CTA's share), 1
// issues the products, 2 owns tensor memory, 4-11 turn K's codes into operands and
// have the softmax (4-7 every other group of 32 dims and the first half of the
// rows, 8-11 the others), 12-19 turn V's codes into operands.  K of a tile is made
// ready before the softmax of the tile before it, which hides S.  Every wait is
// bounded; after one that ran out a warp still meets the others at every barrier
// of threads, but arrives at no mbarrier any more: a ring slot that is called empty
// while its copy is under way would get another copy, on a barrier whose phase has
// had its one arrival, and the CTA could end with copies under way.
#include <algorithm>
#include <type_traits>

#include "cache4_attention.cuh"

namespace slimkv {
namespace {

using namespace attention4;

constexpr int kKeys = kWideKeys;
constexpr int kHalfKeys = kKeys / 2;             // keys of a ring slot, and of half a V tile
constexpr int kSoftWarps = 8, kValueWarps = 8;
constexpr int kThreads = 32 * (4 + kSoftWarps + kValueWarps);
constexpr uint32_t kChunk = kKeys * 128;         // [128 keys x 64] 16-bit elements
constexpr uint32_t kTileArea = 223 * 1024;

// Shared memory: V tile | P tiles | Q | ring of 4-bit K rows | ring of 4-bit V rows.
template <int G, int N>
struct Layout {
    static_assert(G % 2 == 0, "whole chunks");
    static constexpr int kChunks = G / 2;                        // 64-dim chunks of a row
    static constexpr uint32_t kV = uint32_t(kChunks) * kChunk, kP = kChunk, kQ = uint32_t(kChunks) * N * 128;
    static constexpr uint32_t kSlot = kHalfKeys * uint32_t(row4_bytes(kGroupDims * G));
    static constexpr int kPBufs = kV + 2 * kP + kQ + 8 * kSlot <= kTileArea ? 2 : 1;
    static constexpr uint32_t kOffP = kV, kOffQ = kOffP + kPBufs * kP, kOffRing = kOffQ + kQ;
    static constexpr int kRing = (kTileArea - kOffRing) / (2 * kSlot) < 6 ? int((kTileArea - kOffRing) / (2 * kSlot)) : 6;
    static_assert(kRing >= 3, "a tile and a half under way");
    // Tensor memory: O^T blocks of 128 dims, two S^T, K.
    static constexpr int kBlocks = (kChunks + 1) / 2;
    static constexpr int kColS = kBlocks * N, kColK = kColS + 2 * N;
    static constexpr int kKBufs = 2;
    static_assert(kColK + 16 * G * kKBufs <= 512, "tensor memory");
    // A K slot is half a tile and belongs to the warps of its keys.  Of an odd ring they skip every
    // other phase of a slot's barrier; that one is over, since the other half's warps have been through
    // its tile, kKBufs or more tiles back, when kempty lets them go on.
    static_assert(kRing % 2 == 0 || kRing > 2 * kKBufs, "phases of the K slots");
};

template <int N>
struct Bars {
    uint64_t kraw_full[6], kraw_empty[6], vraw_full[6], vraw_empty[6];
    // pempty: P . V of the tile in the buffer is over, so O has it.  One for each buffer: a softmax warp
    // waits for every phase of it in order, before the tile that starts the next, and so never takes
    // the phase before last, which has the same parity, for the one that it waits for.
    uint64_t kfull[2], kempty[2], sfull[2], sempty[2], pfull[2], pempty[2];
    uint64_t vfull[2], vempty[2];                // half V tiles
    uint64_t qfull, oempty, final_mma;
    // (Not at a multiple of 16 bytes, where its loads become one: 16 x 8k latents took 38.7 us then, 37.3 so.)
    Share share;
    uint32_t tmem_base;
    int abort;
    int bad_values[4];                           // 1 + a piece whose nodes' values hold NaN, by piece % 4
    alignas(16) float top[N], shift[N], alpha[N], inv[N];
    int64_t out_at[N];                           // of each row
    float column[kSoftWarps][N / 2];             // a warp's maxima, then sums, of its columns
};
template <int G, int N>
constexpr uint32_t kSmemBytes = 1024 + kTileArea + uint32_t(sizeof(Bars<N>));

// A from tensor memory (two 16-bit K elements to a column), B from shared memory.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Whether x holds for any of the 128 threads of the barrier.
__device__ __forceinline__ bool any_of_128(int id, bool x) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"(uint32_t(x)), "r"(id)
        : "memory");
    return any != 0;
}
// Floats as integers of the same order (NaN: as -inf), and back.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(fmaxf(x, -INFINITY));
    return i ^ (i >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ (i >> 31 & 0x7fffffff)); }

template <int G, int N, bool kHalf>
__global__ void __launch_bounds__(kThreads, 1)
cache4_wide_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Job J) {
    using P = Pair<kHalf>;
    using L = Layout<G, N>;
    using Work = Plan<N / 8, kKeys>;
    constexpr int NC = N / 2;                    // columns (rows of the segment) of a softmax thread
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    auto* bs = reinterpret_cast<Bars<N>*>(smem + kTileArea);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t slot_k = uint32_t(kHalfKeys * J.k_pitch), slot_v = uint32_t(kHalfKeys * J.v_pitch);
    uint8_t* const ring_k = smem + L::kOffRing;
    uint8_t* const ring_v = ring_k + L::kRing * L::kSlot;

    if (tid < L::kRing) {
        mbar_init(&bs->kraw_full[tid], 1); mbar_init(&bs->kraw_empty[tid], kSoftWarps / 2);         // (a slot is two lane quarters)
        mbar_init(&bs->vraw_full[tid], 1); mbar_init(&bs->vraw_empty[tid], kValueWarps);
    } else if (tid >= 8 && tid < 10) {
        const int i = tid - 8;
        mbar_init(&bs->kfull[i], kSoftWarps); mbar_init(&bs->kempty[i], 1);
        mbar_init(&bs->sfull[i], 1); mbar_init(&bs->sempty[i], kSoftWarps);
        mbar_init(&bs->pfull[i], kSoftWarps); mbar_init(&bs->pempty[i], 1);
        mbar_init(&bs->vfull[i], kValueWarps); mbar_init(&bs->vempty[i], 1);
        bs->bad_values[i] = bs->bad_values[2 + i] = 0;
    } else if (tid == 10) {
        mbar_init(&bs->qfull, kSoftWarps);
        mbar_init(&bs->oempty, kSoftWarps);
        mbar_init(&bs->final_mma, 1);
        bs->abort = 0;
    }
    if (tid < 32) fence_barrier_init();
    if (tid == 32) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    if (warp == 2) {
        tmem_alloc(&bs->tmem_base, 512);
        tmem_relinquish();
    }
    grid_launch_dependents();
    const Work plan(J);
    if (warp == 3) find_share(plan, &bs->share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // All 512 tensor memory columns are this CTA's: addresses begin at column 0.
    const uint32_t sbase = smem_u32(smem);
    const bool any = int(blockIdx.x) < bs->share.ctas;

    if (any && (warp == 0 || warp == 3)) {
        // ---- 4-bit rows: warp 0 K, warp 3 V, 64 keys to a slot ----
        const bool keys = warp == 0;
        uint64_t* full = keys ? bs->kraw_full : bs->vraw_full;
        uint64_t* empty = keys ? bs->kraw_empty : bs->vraw_empty;
        const CUtensorMap* map = keys ? &kmap : &vmap;
        uint8_t* ring = keys ? ring_k : ring_v;
        const int pitch = keys ? J.k_pitch : J.v_pitch, boxes = kHalfKeys / J.box;
        const uint32_t bytes = keys ? slot_k : slot_v;
        int slot = 0;
        uint32_t lap = 0;
        bool ok = true;
        Walk<Work> w;
        w.start(plan, &bs->share);
        while (ok && w.next(plan)) {
            for (int half = 2 * w.t0; half < 2 * w.t1 && ok; ++half) {
                // Boxes past the last used row repeat that row's (they are masked).
                int row = half * kHalfKeys + lane * J.box, page = J.shared_cache ? 0 : w.b;
                if (J.paged && lane < boxes) {
                    const int n = min(row, (w.s.end - 1) & -J.box), i = int(J.page_div.div(uint32_t(n)));
                    page = __ldg(J.cache.table + w.b * J.cache.table_stride + i);
                    row = n - i * J.cache.rows;
                    if (page < 0 || page >= J.cache.num_pages) {
                        report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
                        page = min(max(page, 0), J.cache.num_pages - 1);
                    }
                }
                if (lap && !(ok = warp_wait(&empty[slot], (lap - 1) & 1, bs, J))) break;
                if (lane == 0) mbar_expect_tx(&full[slot], bytes);
                __syncwarp();
                if (lane < boxes) tma_load_4d(ring + slot * L::kSlot + lane * J.box * pitch, map, &full[slot], 0, w.g, row, page);
                if (++slot == L::kRing) { slot = 0; ++lap; }
            }
        }
    } else if (any && warp == 1) {
        // ---- products: the warp stays converged, its branches go by votes, and one elected
        // thread has the instructions, so that their operands are uniform registers ----
        // fp16: both operand formats (bits [7,10) and [10,13)) are 0.
        constexpr uint32_t kType = kHalf ? (1u << 7) | (1u << 10) : 0u;
        const uint32_t idesc_s = umma_idesc_bf16(128, N, 0, 0) & ~kType, idesc_o = umma_idesc_bf16(128, N, 1, 1) & ~kType;
        const uint64_t q_desc = umma_desc_sw128(sbase + L::kOffQ, 16, 1024);
        const uint64_t v_desc = umma_desc_sw128(sbase, kChunk, 1024), p_desc = umma_desc_sw128(sbase + L::kOffP, kChunk, 1024);
        bool ok = true;
        uint32_t i = 0;                          // tiles whose S has been issued
        uint32_t o = 0;                          // tiles whose P . V has been
        uint32_t piece = 0;
        auto issue_o = [&](bool first) {
            const uint32_t pb = o % L::kPBufs;
            ok = ok && wait_bar(&bs->pfull[pb], (o / L::kPBufs) & 1, bs, J);
            if (first && piece > 0) ok = ok && wait_bar(&bs->oempty, (piece - 1) & 1, bs, J);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ok = ok && wait_bar(&bs->vfull[h], o & 1, bs, J);
                if (!all_lanes(ok)) return;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int b = 0; b < L::kBlocks; ++b)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_bf16(uint32_t(b * N), v_desc + ((2 * b * kChunk + h * (kChunk / 2) + k * 2048) >> 4),
                                      p_desc + ((pb * L::kP + h * (kChunk / 2) + k * 2048) >> 4), idesc_o, !first || h || k);
                    umma_commit(&bs->vempty[h]);
                    if (h) umma_commit(&bs->pempty[pb]);
                }
                __syncwarp();
            }
            ++o;
        };
        Walk<Work> w;
        w.start(plan, &bs->share);
        while (all_lanes(ok && w.next(plan))) {
            ok = ok && wait_bar(&bs->qfull, piece & 1, bs, J);
            for (int tile = w.t0; all_lanes(ok && tile < w.t1); ++tile, ++i) {
                const uint32_t kb = i % L::kKBufs, sb = i & 1;
                ok = ok && wait_bar(&bs->kfull[kb], (i / L::kKBufs) & 1, bs, J);
                if (i >= 2) ok = ok && wait_bar(&bs->sempty[sb], (i / 2 - 1) & 1, bs, J);
                if (!all_lanes(ok)) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 2 * G; ++k)
                        umma_ts(uint32_t(L::kColS) + sb * N, uint32_t(L::kColK) + kb * 16 * G + 8 * k, q_desc + (((k / 4) * N * 128 + (k % 4) * 32) >> 4),
                                idesc_s, k != 0);
                    umma_commit(&bs->sfull[sb]);
                    umma_commit(&bs->kempty[kb]);
                }
                __syncwarp();
                if (tile > w.t0) issue_o(tile - 1 == w.t0);
            }
            if (all_lanes(ok)) issue_o(w.t1 - 1 == w.t0);
            ++piece;
        }
        if (elect_one()) umma_commit(&bs->final_mma);
        __syncwarp();
    } else if (any && warp >= 4 && warp < 4 + kSoftWarps) {
        // ---- K operands and the softmax: a thread has key 32 quarter + lane of each tile, and of it every
        // other group of 32 dims and half of the rows ----
        const int a = (warp - 4) >> 2, quarter = warp & 3, cb = a * NC, gt = tid & 127;
        const uint32_t lane_addr = uint32_t(32 * quarter) << 16;
        const int key = 32 * quarter + lane;
        const typename P::Constants constants;
        // Whether row r sees a node of the piece whose values of group grp are NaN: V's operands have
        // zeros for them.
        auto sees_nan = [&](const Walk<Work>& w, int r, int grp) {
            const int t = int(J.group_div.div(uint32_t(r)));
            if (t >= w.s.nodes) return false;
            for (int m = max(w.s.len, w.t0 * kKeys); m < min(w.s.end, w.t1 * kKeys); ++m) {
                const int node = m - w.s.len;
                if (!(J.mask ? __ldg(J.mask + w.b * J.mask_stride + int64_t(t) * J.words + (node >> 5)) >> (node & 31) & 1 : node <= t)) continue;
                int64_t page = J.shared_cache ? 0 : w.b;
                int row = m;
                if (J.paged) cache_row(J.cache, w.b, m, page, row);
                const uint8_t* at = J.v + page * J.cache.v_stride[0] + row * J.cache.v_stride[1] + w.g * J.cache.v_stride[2] + 16 * J.vg + 4 * grp;
                if (!P::finite(*reinterpret_cast<const uint32_t*>(at))) return true;
            }
            return false;
        };
        bool ok = true;
        uint32_t i = 0;                          // tiles whose K has been made ready
        uint32_t o = 0;                          // tiles whose softmax is done
        uint32_t piece = 0;
        Walk<Work> w;
        w.start(plan, &bs->share);
        while (w.next(plan)) {
            const int row0 = w.group * N;
            // ---- the piece's Q, 16 bytes to a lane at a time, all of them under way at once ----
            {
                constexpr int kUnits = N * 8 * L::kChunks / (32 * kSoftWarps);
                uint4 q[kUnits];
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
                    const int u = tid - 128 + k * 32 * kSoftWarps, r = u / (8 * L::kChunks), d = 8 * (u % (8 * L::kChunks));
                    q[k] = make_uint4(0, 0, 0, 0);
                    if (row0 + r < J.rows && d < J.kg * kGroupDims) {
                        const int node = int(J.group_div.div(uint32_t(row0 + r))), h = w.g * J.group + row0 + r - node * J.group;
                        q[k] = __ldg(reinterpret_cast<const uint4*>(J.q + w.b * J.q_sb + node * J.q_st + h * J.q_sh + d));
                    }
                }
#pragma unroll
                for (int k = 0; k < kUnits; ++k) {
                    const int u = tid - 128 + k * 32 * kSoftWarps, r = u / (8 * L::kChunks), x = u % (8 * L::kChunks);
                    *reinterpret_cast<uint4*>(smem + L::kOffQ + (x >> 3) * (N * 128) + r * 128 + (((x ^ r) & 7) << 4)) = q[k];
                }
            }
            fence_async_shared();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&bs->qfull);
            if (gt < NC) {
                bs->top[cb + gt] = -INFINITY;
                bs->shift[cb + gt] = 3e38f;
            }
            named_bar(1 + a, 128);
            float sum[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) sum[c] = 0.f;

            auto keys_of = [&] {
                const uint32_t kb = i % L::kKBufs, use = 2 * i + uint32_t(quarter >> 1), slot = use % L::kRing;
                if (i >= uint32_t(L::kKBufs)) ok = ok && warp_wait(&bs->kempty[kb], (i / L::kKBufs - 1) & 1, bs, J);
                ok = ok && warp_wait(&bs->kraw_full[slot], (use / L::kRing) & 1, bs, J);
                if (ok) {
                    tc_fence_after();
                    const uint8_t* row = ring_k + slot * L::kSlot + (key & (kHalfKeys - 1)) * J.k_pitch;
#pragma unroll
                    for (int g2 = 0; g2 < G / 2; ++g2) {
                        const int grp = 2 * g2 + a;
                        float x[16];
                        uint32_t word[4] = {0, 0, 0, 0}, pair = 0;      // (dims behind the row: zeros)
                        if (grp < J.kg) {
                            load_words<4>(row + 16 * grp, word);
                            pair = load_word(row + 16 * J.kg + 4 * grp);
                        }
                        const auto sc = P::as(low_twice(pair)), lo = P::as(high_twice(pair));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            x[4 * k] = __uint_as_float(P::template values<0>(constants, word[k], sc, lo));
                            x[4 * k + 1] = __uint_as_float(P::template values<1>(constants, word[k], sc, lo));
                            x[4 * k + 2] = __uint_as_float(P::template values<2>(constants, word[k], sc, lo));
                            x[4 * k + 3] = __uint_as_float(P::template values<3>(constants, word[k], sc, lo));
                        }
                        tmem_st16(lane_addr + uint32_t(L::kColK) + kb * 16 * G + 16 * grp, x);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (ok && lane == 0) {
                    mbar_arrive(&bs->kraw_empty[slot]);
                    mbar_arrive(&bs->kfull[kb]);
                }
                ++i;
            };
            auto soften = [&](int tile) {
                const uint32_t sb = o & 1, pb = o % L::kPBufs;
                const int n = tile * kKeys + key;
                ok = ok && warp_wait(&bs->sfull[sb], (o / 2) & 1, bs, J);
                tc_fence_after();
                float s[NC];
                tmem_ld_cols<NC>(lane_addr + uint32_t(L::kColS) + sb * N + cb, s);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&bs->sempty[sb]);
                if ((tile + 1) * kKeys > w.s.len) {
                    // Which rows see the key: all the context, a node's those that have it among their ancestors.
                    const int node = n - w.s.len;
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        bool seen = n < w.s.end;
                        if (seen && node >= 0) {
                            const int t = int(J.group_div.div(uint32_t(row0 + cb + c)));
                            if (t >= w.s.nodes) seen = false;
                            else if (J.mask) seen = __ldg(J.mask + w.b * J.mask_stride + int64_t(t) * J.words + (node >> 5)) >> (node & 31) & 1;
                            else seen = node <= t;
                        }
                        if (!seen) s[c] = -INFINITY;
                    }
                }
                // A score far above its row's maximum calls for another.
                bool grown = false;
#pragma unroll
                for (int c = 0; c < NC; c += 4) {
                    const float4 shift = *reinterpret_cast<const float4*>(&bs->shift[cb + c]);
                    constexpr float kMost = kLazyLog2 + kDownLog2<kHalf>;
                    grown |= fmaf(s[c], J.scale_log2, shift.x) > kMost || fmaf(s[c + 1], J.scale_log2, shift.y) > kMost ||
                             fmaf(s[c + 2], J.scale_log2, shift.z) > kMost || fmaf(s[c + 3], J.scale_log2, shift.w) > kMost;
                }
                if (any_of_128(1 + a, ok && grown)) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const int m = __reduce_max_sync(0xffffffffu, ordered(s[c]));
                        if (lane == c) bs->column[warp - 4][c] = from_ordered(m);
                    }
                    named_bar(1 + a, 128);
                    if (gt < NC) {
                        float mx = bs->column[4 * a][gt];
#pragma unroll
                        for (int k = 1; k < 4; ++k) mx = fmaxf(mx, bs->column[4 * a + k][gt]);
                        const float old = bs->top[cb + gt], m = fmaxf(old, mx * J.scale_log2 - kDownLog2<kHalf>);
                        bs->alpha[cb + gt] = old == m ? 1.f : sfu_exp2(old - m);        // (both may be -inf)
                        bs->top[cb + gt] = m;
                        bs->shift[cb + gt] = -fmaxf(m, -3e38f);         // (-inf: nothing seen yet)
                    }
                    named_bar(1 + a, 128);
#pragma unroll
                    for (int c = 0; c < NC; ++c) sum[c] *= bs->alpha[cb + c];
                    if (tile > w.t0) {
                        ok = ok && warp_wait(&bs->pempty[(o - 1) % L::kPBufs], ((o - 1) / L::kPBufs) & 1, bs, J);
                        if (ok) {
                            tc_fence_after();
#pragma unroll 1
                            for (int b = 0; b < L::kBlocks; ++b) {
                                const uint32_t at = lane_addr + uint32_t(b * N + cb);
#pragma unroll
                                for (int c0 = 0; c0 < NC; c0 += 16) {
                                    float v[16];
                                    tmem_ld16(at + c0, v);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int c = 0; c < 16; ++c) v[c] *= bs->alpha[cb + c0 + c];
                                    tmem_st16(at + c0, v);
                                }
                            }
                            tmem_wait_st();
                            tc_fence_before();
                        }
                    }
                }
                if (o >= uint32_t(L::kPBufs)) ok = ok && warp_wait(&bs->pempty[pb], (o / L::kPBufs - 1) & 1, bs, J);
                if (ok) {
                    uint8_t* row = smem + L::kOffP + pb * L::kP + key * 128;
#pragma unroll
                    for (int c = 0; c < NC; c += 8) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const float4 shift = *reinterpret_cast<const float4*>(&bs->shift[cb + c + e]);
                            const float p0 = sfu_exp2(fmaf(s[c + e], J.scale_log2, shift.x)), p1 = sfu_exp2(fmaf(s[c + e + 1], J.scale_log2, shift.y));
                            const float p2 = sfu_exp2(fmaf(s[c + e + 2], J.scale_log2, shift.z)), p3 = sfu_exp2(fmaf(s[c + e + 3], J.scale_log2, shift.w));
                            sum[c + e] += p0; sum[c + e + 1] += p1; sum[c + e + 2] += p2; sum[c + e + 3] += p3;
                            y[e / 2] = pack2<kHalf>(p0, p1);
                            y[e / 2 + 1] = pack2<kHalf>(p2, p3);
                        }
                        *reinterpret_cast<uint4*>(row + ((((cb + c) / 8) ^ (key & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                    fence_async_shared();
                }
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&bs->pfull[pb]);
                ++o;
            };
            for (int tile = w.t0; tile < w.t1; ++tile) {
                keys_of();
                if (tile > w.t0) soften(tile - 1);
            }
            soften(w.t1 - 1);

            // ---- the piece's rows ----
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float x = sum[c];
#pragma unroll
                for (int k = 16; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
                if (lane == c) bs->column[warp - 4][c] = x;
            }
            named_bar(1 + a, 128);
            if (gt < NC) {
                const float l = (bs->column[4 * a][gt] + bs->column[4 * a + 1][gt]) + (bs->column[4 * a + 2][gt] + bs->column[4 * a + 3][gt]);
                const int r = row0 + cb + gt, node = int(J.group_div.div(uint32_t(r))), h = w.g * J.group + r - node * J.group;
                bs->inv[cb + gt] = l != 0.f && node < w.s.nodes ? 1.f / l : 0.f;         // (a NaN sum stays)
                bs->out_at[cb + gt] = w.b * J.o_sb + node * J.o_st + h * J.o_sh;
                if (ok && r < J.rows) {
                    const float lse2 = l == 0.f || node >= w.s.nodes ? -INFINITY : bs->top[cb + gt] + log2f(l);
                    if (w.whole()) J.lse[(int64_t(w.b) * J.nodes + node) * J.heads + h] = lse2 * kLn2;
                    else J.part_lse[int64_t(2 * blockIdx.x + (w.piece > 0)) * N + cb + gt] = lse2;
                }
            }
            named_bar(1 + a, 128);
            ok = ok && warp_wait(&bs->pempty[(o - 1) % L::kPBufs], ((o - 1) / L::kPBufs) & 1, bs, J);
            if (ok) {
                tc_fence_after();
                const bool bad = *const_cast<volatile int*>(&bs->bad_values[piece & 3]) == int(piece) + 1, whole = w.whole();
                const int dims = J.vg * kGroupDims, cols = min(NC, J.rows - row0 - cb);
#pragma unroll 1
                for (int b = 0; b < L::kBlocks; ++b) {
                    const int d = 128 * b + key;
                    float* part = J.part_o + (int64_t(2 * blockIdx.x + (w.piece > 0)) * N + cb) * dims + d;
#pragma unroll 1
                    for (int c0 = 0; c0 < NC; c0 += 16) {
                        float v[16];
                        tmem_ld16(lane_addr + uint32_t(b * N + cb + c0), v);
                        tmem_wait_ld();
                        if (d >= dims) continue;        // (the whole warp)
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            const float f = bs->inv[cb + c0 + c];
                            v[c] = f == 0.f ? 0.f : v[c] * f;       // (a row of no node may hold NaN)
                        }
                        if (bad) {
#pragma unroll 1
                            for (int c = 0; c < 16; ++c)
                                if (c0 + c < cols && sees_nan(w, row0 + cb + c0 + c, d / kGroupDims)) {
#pragma unroll
                                    for (int e = 0; e < 16; ++e)
                                        if (e == c) v[e] = NAN;
                                }
                        }
                        if (whole) {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (c0 + c < cols) J.out[bs->out_at[cb + c0 + c] + d] = uint16_t(pack2<kHalf>(v[c], 0.f));
                        } else {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (c0 + c < cols) part[(c0 + c) * dims] = v[c];
                        }
                    }
                }
                tc_fence_before();
            }
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&bs->oempty);
            ++piece;
        }
    } else if (any && warp >= 4 + kSoftWarps) {
        // ---- V operands: a warp has 32 of a half's keys, a lane to a key, and every fourth group of 32 dims ----
        const int vw = warp - (4 + kSoftWarps), key = 32 * (vw & 1) + lane, first = vw >> 1;
        const typename P::Constants constants;
        const uint8_t* const from = ring_v + key * J.v_pitch + 16 * first;
        const int pair_at = 16 * J.vg + 4 * first - 16 * first;
        uint8_t* const to = smem + (first >> 1) * kChunk + key * 128;
        int unit[4];                             // of the group's words in the swizzled row (groups four apart: the same in other chunks)
#pragma unroll
        for (int e = 0; e < 4; ++e) unit[e] = ((4 * (first & 1) + e) ^ (key & 7)) << 4;
        bool ok = true;
        uint32_t i = 0;                          // half tiles done
        uint32_t piece = 0;
        Walk<Work> w;
        w.start(plan, &bs->share);
        while (w.next(plan)) {
            for (int half = 2 * w.t0; half < 2 * w.t1; ++half, ++i) {
                const uint32_t slot = i % L::kRing, buf = i & 1;
                if (i >= 2) ok = ok && warp_wait(&bs->vempty[buf], (i / 2 - 1) & 1, bs, J);
                ok = ok && warp_wait(&bs->vraw_full[slot], (i / L::kRing) & 1, bs, J);
                if (ok) {
                    const uint8_t* row = from + slot * L::kSlot;
                    uint8_t* tile = to + buf * (kChunk / 2);
                    const bool context = (half + 1) * kHalfKeys <= w.s.len;
                    const int n = half * kHalfKeys + key;
                    bool bad = false;
#pragma unroll
                    for (int j = 0; j < (G + 3) / 4; ++j) {
                        if (first + 4 * j >= J.vg) break;
                        uint32_t word[4], pair = load_word(row + pair_at + 16 * j);
                        load_words<4>(row + 64 * j, word);
                        if (!context) {
                            // Keys that nobody sees count as zero (their P is 0, and 0 x NaN is not 0),
                            // a node's NaN too: the epilogue gives it to the rows that see it.
                            if (n >= w.s.end) pair = 0;
                            else if (n >= w.s.len && !P::finite(pair)) { pair = 0; bad = true; }
                        }
                        const auto sc = P::as(low_twice(pair)), lo = P::as(high_twice(pair));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<uint4*>(tile + 2 * j * kChunk + unit[e]) =
                                make_uint4(P::template values<0>(constants, word[e], sc, lo), P::template values<1>(constants, word[e], sc, lo),
                                           P::template values<2>(constants, word[e], sc, lo), P::template values<3>(constants, word[e], sc, lo));
                    }
                    // (V is one tile ahead of the products at most, so four pieces' flags are more than enough.)
                    if (bad) *const_cast<volatile int*>(&bs->bad_values[piece & 3]) = int(piece) + 1;
                    fence_async_shared();
                }
                __syncwarp();
                if (ok && lane == 0) {
                    mbar_arrive(&bs->vraw_empty[slot]);
                    mbar_arrive(&bs->vfull[buf]);
                }
            }
            ++piece;
        }
    }
    __syncthreads();
    if (any) {
        // Nothing of this CTA is in flight when its tensor memory goes: the products, and after a
        // wait that ran out the copies that nobody waited for.
        if (tid == 64) mbar_wait(&bs->final_mma, 0, 2000000000ull);
        if (bs->abort && tid == 0)
            for (int s = 0; s < L::kRing; ++s) {
                mbar_wait(&bs->kraw_full[s], 0, 100000000ull);
                mbar_wait(&bs->kraw_full[s], 1, 100000000ull);
                mbar_wait(&bs->vraw_full[s], 0, 100000000ull);
                mbar_wait(&bs->vraw_full[s], 1, 100000000ull);
            }
    }
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(bs->tmem_base, 512);
    }
}

template <int G, int N, bool kHalf>
int launch(const CUtensorMap& km, const CUtensorMap& vm, const Job& J, cudaStream_t stream) {
    auto kernel = cache4_wide_kernel<G, N, kHalf>;
    static_assert(kSmemBytes<G, N> <= 232448, "shared memory budget");
    static bool configured[64] = {};
    const int dev = device_info().device;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes<G, N>)) != cudaSuccess)
            return fail(SLIMKV_ERR_CUDA, "cudaFuncSetAttribute (4-bit attention) failed");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    kernel<<<J.ctas, kThreads, kSmemBytes<G, N>, stream>>>(km, vm, J);
    return launch_combine<N / 8, kKeys, kHalf>(J, stream);
}

}  // namespace

namespace attention4 {

int launch_wide(const CUtensorMap& km, const CUtensorMap& vm, const Job& J, bool half, cudaStream_t stream) {
    if (std::max(J.kg, J.vg) <= 8) return half ? launch<8, kWideRows, true>(km, vm, J, stream) : launch<8, kWideRows, false>(km, vm, J, stream);
    return half ? launch<10, kWideRows, true>(km, vm, J, stream) : launch<10, kWideRows, false>(km, vm, J, stream);
}

}  // namespace attention4
}  // namespace slimkv
