// Attention over a 4-bit cache, split over the keys (C ABI
// slimkv_cache4_attention).
//
// For every query row (node t, head h) over the keys n that the node sees
//   s_n = scale q . k_n,   lse = log sum_n e^{s_n},   out = sum_n e^{s_n - lse} v_n,
// k_n and v_n being the 16-bit rows that the codes stand for (cache4.cuh).
//
// A decode step has few query rows to a KV head and must read 0.625 bytes a
// value, so what counts is how few instructions a value costs between its load
// and the tensor core.  Codes never go back to shared memory: a warp takes 16
// keys, turns their codes into MMA operands in its registers, and has the keys
// (for V: the dims) on the 16 side of mma.sync.m16n8k16 and 8 query rows on the
// other:
//   S [16 keys x 8 rows] += K [16 x 16 dims] . Q^T,   O^T [16 dims x 8 rows] += V^T [16 x 16 keys] . P^T
// Any order of the dims serves as the products' inner (outer) index as long as
// both sides have the same one, so each lane reads whole words of one group:
// one (scale, low) pair serves up to 32 values.  The softmax keeps a row's
// maximum until a score passes it by 2^8, so a vote replaces the reduction over
// keys; P goes from the layout of S to that of the second product by two
// transpositions of 8 x 8 blocks in registers.
//
// Work: equal shares of all segments' tiles of 64 or 128 keys (key_shares.cuh), a
// segment being the keys of one (sequence, KV head, 8 or 16 query rows); in a CTA's
// piece of a segment each of its four warps takes a quarter of every tile, with
// its own ring of TMA loads and its own running softmax, and the warps meet only
// at the piece's end.  Pieces that are not a whole segment leave normalised
// partial rows, which a dependent launch merges.  Lengths are read on the device.
//
// Bound: instructions and their latency (61 % of the cycles issue, the logic unit
// is busy for 50 %).  A word of bf16 codes (8 values) takes 15 of them, 7 of the
// logic unit and 8 on pairs of 16-bit values, and either kind issues every other
// cycle; once started the CTAs go through the keys at 5.7 TB/s together.  Around that,
// by time stamps of each, the first keys come after 6.0 us and the CTAs end between 30
// and 44 (38 in the mean).  Measured in a graph (bf16, 32 / 8 heads of 128 dims): 16
// sequences of 8k rows, one token 47 us = 3.6 TB/s (the same rows in 16 bits: 107 us),
// four nodes 64, one sequence of 131072 rows in 16-row pages 51 or 56 (two GPUs), one
// token over 517 rows 8.5.  What that took, for the first:
// 67.5 us; constant row lengths, plain shared-memory loads 61; and + or of the
// codes in one instruction 55; 32 keys to a warp's step 49; masks only in a
// sequence's last steps 47.  More CTAs than fit (each pays the start): 54 to 63; five
// of 16 keys a step on an SM instead of four of 32: 56; contiguous copies in place of
// the TMA's boxes: 48.
#include <algorithm>
#include <type_traits>

#include "cache4_attention.cuh"

namespace slimkv {
namespace {

using namespace attention4;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

// ---------------------------------------------------------------- layout --
// The words of a V row that lane row g takes: of every eight groups one, then
// half, a quarter; of a last single group lanes 0 to 3 one each.
template <int G>
struct ValueWords {
    static constexpr int kOcts = G / 8, kQuad = G / 4 % 2, kPair = G / 2 % 2, kOne = G % 2;
    static constexpr int kWords = 4 * kOcts + 2 * kQuad + kPair + kOne;
    __device__ __forceinline__ static constexpr int dim(int i, int g) {
        return i < 4 * kOcts               ? 256 * (i / 4) + 32 * g + 8 * (i % 4)
               : i < 4 * kOcts + 2 * kQuad ? 256 * kOcts + 16 * g + 8 * (i - 4 * kOcts)
               : kPair && i == 4 * kOcts + 2 * kQuad ? 256 * kOcts + 128 * kQuad + 8 * g
                                           : 256 * kOcts + 128 * kQuad + 64 * kPair + 8 * g;
    }
};

template <int G, int NT>
struct Shape {
    static constexpr int kWordsV = ValueWords<G>::kWords;
    // Blocks of 16 keys in a warp's step: two where their scores have room in registers.
    static constexpr int kHalves = NT * G > 10 ? 1 : 2;
    static constexpr int kSlab = 16 * kHalves, kKeys = kSlab * kWarps;
    // Slabs of a warp's ring: what leaves shared memory to kBlocks blocks.
    static constexpr int kStages = G <= 6 ? 64 / kSlab : kHalves == 2 ? 2 : 3;
    // Q operands in registers where there is room for them, else in shared memory.
    static constexpr bool kQShared = NT * G > 10;
    static constexpr int kBlocks = G <= 4 ? (NT == 1 ? 4 : 3) : G <= 6 && NT == 1 ? 3 : 2;
    // What the four warps' O takes when they are added up (over the rings).
    static constexpr uint32_t kMerge = uint32_t(kWordsV) * 2 * NT * kWarps * 32 * 32;
    static constexpr uint32_t kQBytes = kQShared ? uint32_t(NT) * G * 512 : 0;
    static constexpr uint32_t kRing = uint32_t(kWarps) * kStages * kSlab * 2 * row4_bytes(kGroupDims * G) + 512;
    static_assert(kBlocks * ((kRing > kMerge ? kRing : kMerge) + kQBytes + 2048) <= 228 * 1024, "shared memory of the blocks of an SM");
};

// A CTA's part of a segment.
struct Piece {
    int more;                   // 0: there is none
    int b, g, group;
    int t0, t1;                 // its key tiles
    Seq s;
    int slot;                   // of its partial rows, -1: a whole segment
};
template <class Work, int kRows, int kStages>
struct Bars {
    uint64_t full[kWarps][kStages];
    int abort;
    Share share;
    Walk<Work> walk;            // thread 0's
    Piece piece[2];             // this one and the next
    float top[kWarps][kRows], sum[kWarps][kRows];
};
template <int G, int NT>
uint32_t smem_bytes(int k_pitch, int v_pitch) {
    const uint32_t ring = uint32_t(kWarps * Shape<G, NT>::kStages * Shape<G, NT>::kSlab) * uint32_t(k_pitch + v_pitch) + 512;    // 512: words behind a short row
    return std::max(ring, Shape<G, NT>::kMerge) + Shape<G, NT>::kQBytes + uint32_t(sizeof(Bars<Plan<NT, Shape<G, NT>::kKeys>, 8 * NT, Shape<G, NT>::kStages>));
}

// ----------------------------------------------------------------- kernel --
template <int G, int NT, bool kHalf, bool kExact>
__global__ void __launch_bounds__(kThreads, Shape<G, NT>::kBlocks)
cache4_attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Job J) {
    using P = Pair<kHalf>;
    using VW = ValueWords<G>;
    using S = Shape<G, NT>;
    constexpr int kRows = 8 * NT, kWordsV = VW::kWords, kHalves = S::kHalves, kSlab = S::kSlab, kKeys = S::kKeys, kStages = S::kStages;
    using Work = Plan<NT, kKeys>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 127) {                  // (TMA writes at multiples of 128 bytes)
        report(J.status, SLIMKV_DEVICE_MISALIGNED);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const RowShape<G, kExact> kshape{J.kg}, vshape{J.vg};
    const uint32_t k_pitch = uint32_t(kshape.pitch()), v_pitch = uint32_t(vshape.pitch());
    const uint32_t k_bytes = kSlab * k_pitch, stage_bytes = k_bytes + kSlab * v_pitch;
    const uint32_t area = max(uint32_t(kWarps * kStages) * stage_bytes + 512u, S::kMerge);
    uint8_t* ring = smem + uint32_t(warp * kStages) * stage_bytes;
    uint4* q_shared = reinterpret_cast<uint4*>(smem + area);
    auto* bs = reinterpret_cast<Bars<Work, kRows, kStages>*>(smem + area + S::kQBytes);

    if (tid < kWarps * kStages) mbar_init(&bs->full[tid / kStages][tid % kStages], 1);
    if (tid == 0) bs->abort = 0;
    if (tid < 32) fence_barrier_init();
    if (tid == 32) {
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    grid_launch_dependents();
    const Work plan(J);
    // One thread goes through the share's pieces; the others find each in shared memory.
    auto next_piece = [&](Piece& p) {
        Walk<Work>& w = bs->walk;
        p.more = w.next(plan);
        p.b = w.b; p.g = w.g; p.group = w.group;
        p.t0 = w.t0; p.t1 = w.t1;
        p.s = w.s;
        p.slot = w.whole() ? -1 : 2 * int(blockIdx.x) + (w.piece > 0);
    };
    if (warp == 0) {
        find_share(plan, &bs->share);
        __syncwarp();
        if (lane == 0 && int(blockIdx.x) < bs->share.ctas) {
            bs->walk.start(plan, &bs->share);
            next_piece(bs->piece[0]);
        }
    }
    __syncthreads();
    if (int(blockIdx.x) >= bs->share.ctas) return;

    const int boxes = kSlab / J.box, box_shift = 31 - __clz(boxes);
    const typename P::Constants constants;
    const float unscale = 1.f / J.scale_log2;
    int stage = 0;                               // of the next slab to be used
    uint32_t lap = 0;
    uint32_t pending = 0;                        // stages with a load under way
    bool ok = true;
    for (int turn = 0;; turn ^= 1) {
        const Piece w = bs->piece[turn];
        if (!w.more) break;
        // The piece's slabs of this warp, a quarter of each tile; the last may lie behind the keys.
        const int first_key = w.t0 * kKeys + warp * kSlab;
        const int slabs = max(0, min(w.t1 - w.t0, (w.s.end - first_key + kKeys - 1) / kKeys));
        // Where box lane % boxes of slab `first` + lane / boxes lies: its page (dense: its sequence)
        // and row.  Boxes past the last used row repeat that row's (they are masked).
        auto locate = [&](int first, int& row) {
            const int slab = first + (lane >> box_shift);
            row = first_key + slab * kKeys + (lane & (boxes - 1)) * J.box;
            if (!J.paged) return J.shared_cache ? 0 : w.b;
            int page = 0;
            if (slab < min(slabs, first + kStages)) {
                const int n = min(row, (w.s.end - 1) & -J.box), i = int(J.page_div.div(uint32_t(n)));
                page = __ldg(J.cache.table + w.b * J.cache.table_stride + i);
                row = n - i * J.cache.rows;
                if (page < 0 || page >= J.cache.num_pages) {
                    report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
                    page = min(max(page, 0), J.cache.num_pages - 1);
                }
            }
            return page;
        };
        // Loads a slab that the lanes from `from` on have located.
        auto issue = [&](int st, int page, int row, int from) {
            uint64_t* bar = &bs->full[warp][st];
            uint8_t* at = ring + uint32_t(st) * stage_bytes;
            // One elected thread has the copies: their operands are uniform registers.
            for (int box = 0; box < boxes; ++box) {
                const int p = __shfl_sync(0xffffffffu, page, from + box), r = __shfl_sync(0xffffffffu, row, from + box);
                if (elect_one()) {
                    if (box == 0) mbar_expect_tx(bar, stage_bytes);
                    tma_load_4d(at + uint32_t(box * J.box) * k_pitch, &kmap, bar, 0, w.g, r, p);
                    tma_load_4d(at + k_bytes + uint32_t(box * J.box) * v_pitch, &vmap, bar, 0, w.g, r, p);
                }
            }
            pending |= 1u << st;
        };
        if (ok) {
            int row;
            const int page = locate(0, row);
            for (int s = 0, st = stage; s < min(slabs, kStages); ++s) {
                issue(st, page, row, s << box_shift);
                if (++st == kStages) st = 0;
            }
        }

        // ---- Q: row g of each row tile, the dims of lane column t ----
        const int row0 = w.group * kRows;
        uint4 qf[S::kQShared ? 1 : NT * G];
        auto load_q = [&](int n, int i) {
            const int r = row0 + 8 * n + g, d = KeyWords<G>::dim(i, t);
            if (r >= J.rows || !kshape.has(d)) return make_uint4(0, 0, 0, 0);
            const int node = int(J.group_div.div(uint32_t(r))), h = w.g * J.group + r - node * J.group;
            return __ldg(reinterpret_cast<const uint4*>(J.q + w.b * J.q_sb + node * J.q_st + h * J.q_sh + d));
        };
        if constexpr (S::kQShared) {
            for (int i = warp; i < NT * G; i += kWarps) q_shared[i * 32 + lane] = load_q(i / G, i % G);
            __syncthreads();
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < G; ++i) qf[n * G + i] = load_q(n, i);
        }
        float o[4 * kWordsV][NT][4];
#pragma unroll
        for (int m = 0; m < 4 * kWordsV; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][n][e] = 0.f;
        // Of the rows 2t and 2t + 1 of each row tile: the maximum that P is taken from (log2), the
        // score (unscaled) that calls for another one, the sum.
        float top[NT][2], limit[NT][2], sum[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n][0] = top[n][1] = limit[n][0] = limit[n][1] = -INFINITY;
            sum[n][0] = sum[n][1] = 0.f;
        }

        for (int i = 0; i < slabs && ok; ++i) {
            const int key0 = first_key + i * kKeys;
            int next_row;
            const int next_page = locate(i + kStages, next_row);
            if (!(ok = warp_wait(&bs->full[warp][stage], lap, bs, J))) break;
            pending &= ~(1u << stage);
            // Slabs of context that every row sees whole, all but a sequence's last ones, do without masks.
            auto step = [&](auto all) {
            constexpr bool whole_slab = decltype(all)::value;
            const uint8_t *ks = ring + uint32_t(stage) * stage_bytes, *vs = ks + k_bytes;

            // ---- S ----
            float s[kHalves][NT][4];
#pragma unroll
            for (int b = 0; b < kHalves; ++b) {
#pragma unroll
                for (int n = 0; n < NT; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.f;
                key_products<G, NT, kHalf>(s[b], ks + uint32_t(16 * b + g) * k_pitch, kshape, t, constants, [&](int n, int i) {
                    if constexpr (S::kQShared) return q_shared[(n * G + i) * 32 + lane];
                    else return qf[n * G + i];
                });
            }

            // ---- what the rows see of the slab's keys (16 b + g and 16 b + g + 8 here) ----
            auto seen_of = [&](int r) {
                const int node = int(J.group_div.div(uint32_t(r)));
                if (node >= w.s.nodes) return 0u;
                if (J.context_only) return low_bits(w.s.end - key0);
                const int32_t* words = J.mask ? J.mask + w.b * J.mask_stride + int64_t(node) * J.words : nullptr;
                return seen_keys(words, J.words, node, w.s.end - w.s.len, key0 - w.s.len);
            };
            if constexpr (!whole_slab) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t seen = seen_of(row0 + 8 * n + 2 * t + e) >> g;
#pragma unroll
                        for (int b = 0; b < kHalves; ++b) {
                            if (!(seen >> (16 * b) & 1u)) s[b][n][e] = -INFINITY;
                            if (!(seen >> (16 * b) & 256u)) s[b][n][2 + e] = -INFINITY;
                        }
                    }
            }

            // ---- softmax ----
            bool grown = false;
#pragma unroll
            for (int b = 0; b < kHalves; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) grown |= s[b][n][e] > limit[n][e & 1];
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float alpha[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[0][n][e], s[0][n][2 + e]);
                        if constexpr (kHalves == 2) mx = fmaxf(mx, fmaxf(s[1][n][e], s[1][n][2 + e]));
#pragma unroll
                        for (int k = 4; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
                        const float m = fmaxf(top[n][e], mx * J.scale_log2 - kDownLog2<kHalf>);
                        alpha[e] = top[n][e] == m ? 1.f : sfu_exp2(top[n][e] - m);      // (both may be -inf)
                        top[n][e] = m;
                        limit[n][e] = (m + (kLazyLog2 + kDownLog2<kHalf>)) * unscale;
                        sum[n][e] *= alpha[e];
                    }
#pragma unroll
                    for (int m = 0; m < 4 * kWordsV; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[m][n][e] *= alpha[e & 1];
                }
            }
            uint32_t pf[kHalves][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float shift[2] = {-fmaxf(top[n][0], -3e38f), -fmaxf(top[n][1], -3e38f)};      // (-inf: nothing seen yet)
#pragma unroll
                for (int b = 0; b < kHalves; ++b) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = sfu_exp2(fmaf(s[b][n][e], J.scale_log2, shift[e & 1]));
                    sum[n][0] += p[0] + p[2];
                    sum[n][1] += p[1] + p[3];
                    pf[b][n][0] = transpose8x8(pack2<kHalf>(p[0], p[1]));
                    pf[b][n][1] = transpose8x8(pack2<kHalf>(p[2], p[3]));
                }
            }

            // ---- O: the keys 2t, 2t + 1, 2t + 8, 2t + 9 of a half and the dims of lane row g.  A key that
            // nobody sees counts as zero (its P is 0, and 0 x NaN is not 0); so does a group of a
            // node's row that is NaN, which the rows that see it get afterwards. ----
            const uint32_t live = low_bits(w.s.end - key0);
            const bool nodes_here = !whole_slab && !J.context_only;
            auto pair_of = [&](int key, int grp) { return load_word(vs + uint32_t(key) * v_pitch + vshape.pair_at(kGroupDims * grp)); };
            bool bad = false;
            if (nodes_here) {
                for (int k = lane; k < kSlab * J.vg; k += 32)
                    if (live >> (k / J.vg) & 1) bad |= !P::finite(pair_of(k / J.vg, k % J.vg));
                bad = __any_sync(0xffffffffu, bad);
            }
#pragma unroll
            for (int b = 0; b < kHalves; ++b) {
                const uint8_t* v0 = vs + uint32_t(16 * b + 2 * t) * v_pitch;
                auto value_words = [&](auto width, auto first) {
                    constexpr int W = decltype(width)::value, i0 = decltype(first)::value;
                    const int d0 = VW::dim(i0, g);
                    uint32_t a[4][W], p[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint8_t* row = v0 + uint32_t((k & 1) + 8 * (k >> 1)) * v_pitch;
                        load_words<W>(row + d0 / 2, a[k]);
                        p[k] = load_word(row + vshape.pair_at(d0));
                        if (!vshape.has(d0) || (G % 2 && d0 >= kGroupDims * G)) p[k] = 0;
                    }
                    if constexpr (!whole_slab) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (!(live >> (16 * b + 2 * t + (k & 1) + 8 * (k >> 1)) & 1) || (nodes_here && !P::finite(p[k]))) p[k] = 0;
                    }
                    const auto sc0 = P::as(low_halves(p[0], p[1])), lo0 = P::as(high_halves(p[0], p[1]));
                    const auto sc1 = P::as(low_halves(p[2], p[3])), lo1 = P::as(high_halves(p[2], p[3]));
#pragma unroll
                    for (int k = 0; k < W; ++k) {
                        // The codes of the even and of the odd dims, a key in each half.
                        const uint32_t x0 = low_halves(a[0][k], a[1][k]), y0 = high_halves(a[0][k], a[1][k]);
                        const uint32_t x1 = low_halves(a[2][k], a[3][k]), y1 = high_halves(a[2][k], a[3][k]);
                        auto pair = [&](auto which) {
                            constexpr int j = decltype(which)::value;
                            const uint32_t x[4] = {P::template values<j>(constants, x0, sc0, lo0), P::template values<j>(constants, y0, sc0, lo0),
                                                   P::template values<j>(constants, x1, sc1, lo1), P::template values<j>(constants, y1, sc1, lo1)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma<kHalf>(o[4 * (i0 + k) + j][n], x, pf[b][n][0], pf[b][n][1]);
                        };
                        pair(std::integral_constant<int, 0>());
                        pair(std::integral_constant<int, 1>());
                        pair(std::integral_constant<int, 2>());
                        pair(std::integral_constant<int, 3>());
                    }
                };
                using std::integral_constant;
                if constexpr (VW::kOcts > 0) value_words(integral_constant<int, 4>(), integral_constant<int, 0>());
                if constexpr (VW::kQuad != 0) value_words(integral_constant<int, 2>(), integral_constant<int, 4 * VW::kOcts>());
                if constexpr (VW::kPair != 0) value_words(integral_constant<int, 1>(), integral_constant<int, 4 * VW::kOcts + 2 * VW::kQuad>());
                if constexpr (VW::kOne != 0)
                    value_words(integral_constant<int, 1>(), integral_constant<int, 4 * VW::kOcts + 2 * VW::kQuad + VW::kPair>());
            }
            if (bad) {
#pragma unroll 1
                for (int k = 0; k < kSlab * J.vg; ++k) {
                    const int key = k / J.vg, grp = k % J.vg;
                    if (!(live >> key & 1) || P::finite(pair_of(key, grp))) continue;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (seen_of(row0 + 8 * n + 2 * t + e) >> key & 1) {
#pragma unroll
                                for (int m = 0; m < 4 * kWordsV; ++m)
                                    if (VW::dim(m / 4, g) / kGroupDims == grp) o[m][n][e] = o[m][n][2 + e] = NAN;
                            }
                }
            }
            };
            if (key0 + kSlab <= w.s.len) step(std::true_type());
            else step(std::false_type());
            __syncwarp();
            if (i + kStages < slabs) issue(stage, next_page, next_row, 0);
            if (++stage == kStages) { stage = 0; lap ^= 1; }
        }

        // ---- the piece's end: the warps' O to a common maximum, added up ----
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) sum[n][e] += __shfl_xor_sync(0xffffffffu, sum[n][e], k);
                if (g == 0) {
                    bs->top[warp][8 * n + 2 * t + e] = top[n][e];
                    bs->sum[warp][8 * n + 2 * t + e] = sum[n][e];
                }
            }
        __syncthreads();                         // (every slab has been used: the rings are free)
        auto row_total = [&](int r, float& m) {
            m = -INFINITY;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) m = fmaxf(m, bs->top[k][r]);
            float l = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float x = bs->top[k][r];
                l += x == -INFINITY ? bs->sum[k][r] : bs->sum[k][r] * sfu_exp2(x - m);    // (a NaN sum stays)
            }
            return l;
        };
        float4* merge = reinterpret_cast<float4*>(smem);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float m;
                const float l = row_total(8 * n + 2 * t + e, m);
                // (a NaN sum stays)
                const float f = l == 0.f ? 0.f : (top[n][e] == -INFINITY ? 0.f : sfu_exp2(top[n][e] - m)) * __fdividef(1.f, l);
#pragma unroll
                for (int k = 0; k < kWordsV; ++k)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        merge[((((k * NT + n) * 2 + e) * 2 + half) * kWarps + warp) * 32 + lane] =
                            make_float4(o[4 * k + 2 * half][n][e] * f, o[4 * k + 2 * half][n][2 + e] * f,
                                        o[4 * k + 2 * half + 1][n][e] * f, o[4 * k + 2 * half + 1][n][2 + e] * f);
            }
        if (tid == 0) next_piece(bs->piece[turn ^ 1]);
        __syncthreads();
        const bool whole = w.slot < 0;
        const int slot = w.slot;
        if (ok) {
            for (int u = warp; u < kWordsV * NT * 2; u += kWarps) {
                const int k = u / (2 * NT), n = u / 2 % NT, e = u & 1, r = row0 + 8 * n + 2 * t + e;
                int d = 0;
#pragma unroll
                for (int i = 0; i < kWordsV; ++i)
                    if (i == k) d = VW::dim(i, g);
                float4 x[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    x[half] = merge[((u * 2 + half) * kWarps) * 32 + lane];
#pragma unroll
                    for (int v = 1; v < kWarps; ++v) {
                        const float4 y = merge[((u * 2 + half) * kWarps + v) * 32 + lane];
                        x[half].x += y.x; x[half].y += y.y; x[half].z += y.z; x[half].w += y.w;
                    }
                }
                if (r >= J.rows || d >= vshape.groups() * kGroupDims) continue;
                const int node = int(J.group_div.div(uint32_t(r))), h = w.g * J.group + r - node * J.group;
                if (whole) {
                    uint4 y = make_uint4(0, 0, 0, 0);
                    if (node < w.s.nodes)
                        y = make_uint4(pack2<kHalf>(x[0].x, x[0].y), pack2<kHalf>(x[0].z, x[0].w), pack2<kHalf>(x[1].x, x[1].y),
                                       pack2<kHalf>(x[1].z, x[1].w));
                    *reinterpret_cast<uint4*>(J.out + w.b * J.o_sb + node * J.o_st + h * J.o_sh + d) = y;
                } else {
                    float4* part = reinterpret_cast<float4*>(J.part_o + (int64_t(slot) * kRows + r - row0) * (J.vg * kGroupDims) + d);
                    part[0] = x[0];
                    part[1] = x[1];
                }
            }
            if (tid < kRows && row0 + tid < J.rows) {
                float m;
                const float l = row_total(tid, m);
                const int r = row0 + tid, node = r / J.group, h = w.g * J.group + r - node * J.group;
                const float lse2 = l == 0.f || node >= w.s.nodes ? -INFINITY : m + log2f(l);
                if (whole) J.lse[(int64_t(w.b) * J.nodes + node) * J.heads + h] = lse2 * kLn2;
                else J.part_lse[int64_t(slot) * kRows + tid] = lse2;
            }
        }
        fence_async_shared();                    // the merge's stores before the next piece's copies
        __syncthreads();
    }
    // After a wait that ran out copies may still be under way.
    if (bs->abort && lane == 0)
        for (int s = 0; s < kStages; ++s)
            if (pending >> s & 1) {
                mbar_wait(&bs->full[warp][s], 0, 100000000ull);
                mbar_wait(&bs->full[warp][s], 1, 100000000ull);
            }
}

// ------------------------------------------------------------------- host --
// The wide kernel or this file's.  In a graph, 8 sequences of one KV head, wide against not:
// 32 rows over 8192 keys of 320 dims 27.1 and 32.2 us, 128 rows 56.9 and 76.2, of 256 dims 24.3 and
// 26.8, 52.4 and 63.6, 32 rows of 224 dims 24.3 and 26.3, of 192 dims 27.0 and 23.4, 128 rows 62.3
// and 56.2, 20 rows of 128 dims (8 KV heads) 83.4 and 63.2.  Short caches lose by the rule: 600 keys,
// 32 rows of 256 dims 15.4 and 13.4, of 320 16.0 and 14.7, 128 rows 22.3 and 21.9.
bool is_wide(const slimkv_tree_attention_args* a) {
    return a->nodes * (a->heads / a->kv_heads) > 16 && std::max(a->dim_qk, a->dim_v) > 192;
}
// Query rows that a pass over the keys serves.
int rows_of(const slimkv_tree_attention_args* a) {
    return is_wide(a) ? kWideRows : a->nodes * (a->heads / a->kv_heads) > 8 ? 16 : 8;
}
// Instantiated row lengths in groups of 32 dims (1, 7 and 9 take the next).
int groups_of(const slimkv_tree_attention_args* a) {
    const int g = (std::max(a->dim_qk, a->dim_v) + kGroupDims - 1) / kGroupDims;
    return g == 1 ? 2 : g == 7 ? 8 : g == 9 ? 10 : g;
}

int check_attention4(const slimkv_tree_attention_args* a) {
    if (!a) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->batch < 1 || a->batch > 4096 || a->nodes < 1 || a->nodes > 1024 || a->heads < 1 || a->kv_heads < 1 ||
        a->heads % a->kv_heads)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "4-bit attention: batch in 1..4096, nodes in 1..1024, heads a multiple of kv_heads");
    if (a->heads / a->kv_heads > 128)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "4-bit attention: at most 128 query heads per KV head");
    for (int dim : {a->dim_qk, a->dim_v})
        if (dim < kGroupDims || dim > kMaxDims4 || dim % kGroupDims)
            return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "4-bit attention: dims must be multiples of 32 up to 320");
    if (a->type != SLIMKV_BF16 && a->type != SLIMKV_FP16)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "4-bit attention: bf16 or fp16 tensors");
    return SLIMKV_OK;
}

// Calls f(G, NT) with the constants of a call's kernel.
template <class F>
auto with_shape(const slimkv_tree_attention_args* a, F f) {
    using std::integral_constant;
    auto rows = [&](auto g) { return rows_of(a) > 8 ? f(g, integral_constant<int, 2>()) : f(g, integral_constant<int, 1>()); };
    switch (groups_of(a)) {
        case 2: return rows(integral_constant<int, 2>());
        case 3: return rows(integral_constant<int, 3>());
        case 4: return rows(integral_constant<int, 4>());
        case 5: return rows(integral_constant<int, 5>());
        case 6: return rows(integral_constant<int, 6>());
        case 8: return rows(integral_constant<int, 8>());
        default: return rows(integral_constant<int, 10>());
    }
}

void carve(Carver& c, const slimkv_tree_attention_args* a, Job& J) {
    J.row_tile = rows_of(a);
    J.ctas = device_info().sm_count;
    if (!is_wide(a)) J.ctas *= with_shape(a, [](auto g, auto nt) { return Shape<decltype(g)::value, decltype(nt)::value>::kBlocks; });
    const size_t rows = size_t(2) * J.ctas * J.row_tile;
    J.part_o = c.take<float>(rows * a->dim_v);
    J.part_lse = c.take<float>(rows);
}

template <int G, int NT, bool kHalf, bool kExact>
int launch(const CUtensorMap& km, const CUtensorMap& vm, const Job& J, cudaStream_t stream) {
    auto kernel = cache4_attention_kernel<G, NT, kHalf, kExact>;
    const uint32_t bytes = smem_bytes<G, NT>(J.k_pitch, J.v_pitch);
    static bool configured[64] = {};
    const int dev = device_info().device;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(smem_bytes<G, NT>(row4_bytes(G * kGroupDims), row4_bytes(G * kGroupDims)))) != cudaSuccess)
            return fail(SLIMKV_ERR_CUDA, "cudaFuncSetAttribute (4-bit attention) failed");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    kernel<<<J.ctas, kThreads, bytes, stream>>>(km, vm, J);
    return launch_combine<NT, Shape<G, NT>::kKeys, kHalf>(J, stream);
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_cache4_attention_workspace_size(const slimkv_tree_attention_args* a) {
    if (check_attention4(a) != SLIMKV_OK) return 0;
    Job J{};
    Carver c(nullptr, 0);
    carve(c, a, J);
    return c.used;
}

extern "C" int slimkv_cache4_attention(const slimkv_tree_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_attention4(a)) return rc;
    if (!a->q || !a->lengths || !a->out || !a->lse) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "4-bit attention: null pointer");
    if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "4-bit attention: scale must be positive");
    const int k_pitch = row4_bytes(a->dim_qk), v_pitch = row4_bytes(a->dim_v);
    if (int rc = check_cache(a->cache, a->batch, k_pitch, v_pitch, 1, true, "4-bit attention")) return rc;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8 || a->out_stride[i] % 8)
            return fail(SLIMKV_ERR_ALIGNMENT, "4-bit attention: strides must be multiples of 8 elements");
    if (!aligned16(a->q) || !aligned16(a->out)) return fail(SLIMKV_ERR_ALIGNMENT, "4-bit attention: 16-byte aligned tensors");
    const slimkv_cache& cache = a->cache;
    const bool paged = cache.table != nullptr;
    if (paged && cache.rows % 8) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "4-bit attention: pages of a multiple of 8 rows");
    Job J{};
    Carver c(workspace, workspace_bytes);
    carve(c, a, J);
    if (!workspace || !c.fits() || !aligned16(workspace))
        return fail(SLIMKV_ERR_WORKSPACE, "4-bit attention: %zu bytes of 16-byte aligned workspace needed", c.used);
    // A box of TMA rows stays inside a page.
    const bool wide = is_wide(a);
    const int slab = wide ? kWideBox : with_shape(a, [](auto g, auto nt) { return Shape<decltype(g)::value, decltype(nt)::value>::kSlab; });
    const int tile = wide ? kWideKeys : slab * kWarps;
    J.box = paged ? std::min(slab, cache.rows & -cache.rows) : slab;
    J.shared_cache = !paged && cache.k_stride[0] == 0 && cache.v_stride[0] == 0;
    if (a->batch > 1 && !paged && !J.shared_cache && (cache.k_stride[0] == 0 || cache.v_stride[0] == 0))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "4-bit attention: K and V are both shared by the batch or neither");
    const uint64_t planes = paged ? uint64_t(cache.num_pages) : J.shared_cache ? 1 : uint64_t(a->batch);
    // One tensor map {row, heads, rows, planes}; a dimension of one (or shared) entry takes any valid stride.
    auto encode = [&](CUtensorMap* m, const void* base, int pitch, const int64_t* st) {
        return encode_map_words_4d(m, base, pitch / 4, a->kv_heads, cache.rows, planes, a->kv_heads > 1 ? st[2] : pitch,
                                   cache.rows > 1 ? st[1] : pitch, planes > 1 ? st[0] : pitch, J.box);
    };
    CUtensorMap km, vm;
    int rc;
    if ((rc = encode(&km, cache.k, k_pitch, cache.k_stride)) || (rc = encode(&vm, cache.v, v_pitch, cache.v_stride))) return rc;
    J.batch = a->batch;
    J.nodes = a->nodes;
    J.heads = a->heads;
    J.kv_heads = a->kv_heads;
    J.group = a->heads / a->kv_heads;
    J.group_div = FastDiv(uint32_t(J.group));
    J.page_div = FastDiv(uint32_t(cache.rows));
    J.rows = a->nodes * J.group;
    J.row_groups = (J.rows + J.row_tile - 1) / J.row_tile;
    J.kg = a->dim_qk / kGroupDims;
    J.vg = a->dim_v / kGroupDims;
    J.k_pitch = k_pitch;
    J.v_pitch = v_pitch;
    J.context_only = a->context_only;
    J.paged = paged;
    J.v = static_cast<const uint8_t*>(cache.v);
    J.cache = cache_view(cache);
    J.capacity = cache_capacity(J.cache);
    if (J.capacity > 0x7fffffffLL - 4096 ||
        double(J.batch) * J.kv_heads * J.row_groups * double(J.capacity / tile + 1 + Plan<4, kWideKeys>::kPieceUnits) >= 2147483648.0)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "4-bit attention: too many rows in one call");
    J.lengths = a->lengths;
    J.nodes_len = a->nodes_len;
    J.mask = a->context_only ? nullptr : a->mask;
    J.mask_stride = a->mask_stride;
    J.words = (a->nodes + 31) / 32;
    J.scale_log2 = a->scale * kLog2e;
    J.q = static_cast<const uint16_t*>(a->q);
    J.q_sb = a->q_stride[0]; J.q_st = a->q_stride[1]; J.q_sh = a->q_stride[2];
    J.out = static_cast<uint16_t*>(a->out);
    J.o_sb = a->out_stride[0]; J.o_st = a->out_stride[1]; J.o_sh = a->out_stride[2];
    J.lse = a->lse;
    J.status = status_word();
    J.wait_ns = a->wait_limit_ns ? a->wait_limit_ns : 2000000000ull;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool half = a->type == SLIMKV_FP16;
    if (wide) return launch_wide(km, vm, J, half, st);
    return with_shape(a, [&](auto g, auto nt) {
        constexpr int G = decltype(g)::value, NT = decltype(nt)::value;
        if (J.kg == G && J.vg == G) return half ? launch<G, NT, true, true>(km, vm, J, st) : launch<G, NT, false, true>(km, vm, J, st);
        return half ? launch<G, NT, true, false>(km, vm, J, st) : launch<G, NT, false, false>(km, vm, J, st);
    });
}
