// Attention of a tree of drafted tokens over a cache, split over the keys
// (C ABI slimkv_tree_attention).
//
// For every query row (node t, head h) over the keys n that the node sees
//   s_n = scale q . k_n,   lse = log sum_n e^{s_n},   out = sum_n e^{s_n - lse} v_n.
// The G = heads / kv_heads query heads of a KV head share its keys, so the
// rows of a KV head are (node, head of the group) pairs: 128 of them (whole
// nodes) fill one M = 128 tile of the tensor core, and a 64-key tile of K and V
// serves one or two such row tiles:
//   S [128 rows x 64 keys] = Q . K^T,   O [128 rows x dim_v] += P . V
// with tcgen05 (fp32 accumulators in TMEM; P = 2^(s - m) written back to TMEM
// in the inputs' 16-bit type as the A operand of the second product, which
// costs about what rounding the output costs (1.25 to 1.4 times the error of a
// rounded fp32 result in all); the row sums stay in fp32 before that rounding,
// so lse keeps fp32 accuracy).
//
// Work: a unit is one 64-key tile of one (sequence, KV head, group of NQ row
// tiles) segment: the context rows, then the nodes' own rows, of which each
// row sees what its ancestor words say.  The units of all
// segments in a row are cut into one equal share per CTA; a share's part of a
// segment is a piece.  A piece that holds a whole segment writes the output;
// the others (at most two per CTA: its first and its last) leave normalised
// fp32 partial rows and their log-sum-exps, which combine_kernel merges.
// Lengths are read on the device; nothing on the host depends on them.
//
// Bound: with few rows per KV head HBM (each K / V row read once); with 128
// rows or more the tensor cores and the exponentials; with few tiles to a CTA
// its start, the ends of its pieces and the merge.  Measured (bf16, 8 KV heads
// of 128 dims, with the merge, in a graph): 2 x 8 nodes over 131,000 rows
// 192 us = 5.6 TB/s, 16 x 16 over 8k 111 us = 4.9 TB/s, 16 x 64 nodes (256 rows
// a KV head) over 8k 167 us = 820 TFLOP/s, one token over 517 rows 13 us.
// (In calls back to back the last of the three large ones draws the board's
// 1000 W and runs at 1.65 GHz, 200 to 206 us.)
//
// Why 64 keys: S and P of a tile fit 64 tensor-memory columns, so two to four
// tiles are under way for each row tile next to O (320 + 3 x 64, or 2 x (128 +
// 2 x 64) columns): the S of tile n + 1 is there when the softmax of tile n
// ends, and the softmax never waits for a product.  (With 128-key tiles and one
// S per row tile, softmax and products took turns: 4,870 cycles for two row
// tiles and 128 keys, 2,700 of them the softmax.)
//
// One CTA per SM, warps: 0 = Q and K loads (TMA), 3 = V loads, 1 and 2 = MMA
// issue (2 owns the TMEM), the others from 4 on = softmax.  Every wait is bounded.
#include <algorithm>
#include <type_traits>

#include "bounded_wait.cuh"
#include "cache_view.cuh"
#include "host_utils.h"
#include "key_shares.cuh"

namespace slimkv {
namespace {

constexpr int kRows = 128;
constexpr int kKeys = 64;                        // keys of a tile
constexpr uint32_t kQChunk = 128 * 128;          // [128 rows x 64] 16-bit elements
constexpr uint32_t kChunk = kKeys * 128;         // [64 keys x 64]
constexpr int kMaxRing = 12;
constexpr int kMaxChunks = 5;                    // dims <= 320
constexpr float kLazyLog2 = 8.f;                 // O is rescaled when a row's maximum grows by more than 2^8
// P = 2^(s - m) with m this far below the row's maximum.  Of fp16's exponents P then uses those
// up to 2^15 (with the 2^8 above), and what it loses below its smallest number is 2^-32 of the
// largest probability for each key (2^-25 with m at the maximum, up to 0.4 % of the weight of
// 131,000 keys behind one dominant one); bf16 has fp32's exponents.
template <bool kHalf>
constexpr float kDownLog2 = kHalf ? 7.f : 0.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;

// Threads that share a row's softmax: two with one row tile, where the row's
// latency counts; one with two row tiles, which keep the units busy by turns.
template <int NQ>
constexpr int kHalvesOf = NQ == 1 ? 2 : 1;
template <int NQ>
constexpr int kSoftmaxThreads = 128 * NQ * kHalvesOf<NQ>;
// Whether the kernel leaves a block of the merge room next to it, so that this
// one is there and has done its planning when the last piece ends (one token
// over 517 rows 14.5 -> 13.6 us, 16 sequences of 8k 113.5 -> 110.7).  Rows of
// more than 256 dims need the shared memory for their rings (latents 34.4 ->
// 38.4), two row tiles their threads' registers.
template <int NQ, int C>
constexpr bool kEarlyMerge = NQ == 1 && C <= 4;
// Q and the rings.
template <int NQ, int C>
constexpr uint32_t kTileArea = (kEarlyMerge<NQ, C> ? 216 : 224) * 1024;

struct Bars {
    uint64_t kfull[kMaxRing], kempty[kMaxRing], vfull[kMaxRing], vempty[kMaxRing], vfixed[kMaxRing];
    uint64_t qfull, qempty;
    // [row tile][S/P buffer]
    uint64_t sfull[2][4], pfull[2][4], odone[2][4], oempty[2], final_mma;
    uint32_t tmem_base;
    int abort;
    int bad_values[4];           // 1 + a piece whose node values hold infinities or NaN, by piece % 4
    float exchange[kRows];       // between a row's two threads
    Share share;
};
template <int NQ, int C>
constexpr uint32_t kSmemBytes = 1024 + kTileArea<NQ, C> + uint32_t(sizeof(Bars));
static_assert(kSmemBytes<2, 2> <= 232448, "shared memory budget");

struct Job {
    int batch, nodes, heads, kv_heads, group;
    int tpt, tile_rows;         // nodes of a row tile and its rows (tpt * group <= 128)
    int row_groups;             // groups of NQ row tiles
    int dim_v;
    int context_only, paged, shared_cache;
    int box;                    // rows of one TMA box
    CacheView cache;
    int64_t capacity;
    const int32_t *lengths, *nodes_len, *mask;
    int64_t mask_stride;
    int words;
    float scale_log2;
    const void* v;
    void* out;
    int64_t o_sb, o_st, o_sh;
    float* lse;
    float* part_o;              // [2 ctas][dim_v / 4][NQ * tile_rows][4]
    float* part_lse;            // [2 ctas][NQ * tile_rows]
    int ctas;
    unsigned int* status;
    uint64_t wait_ns;
};

// ------------------------------------------------------------- schedule --
// What one sequence asks for: its keys are the cache rows [0, end), the context
// and then the nodes' own rows.
struct Seq {
    int len, nodes, end;
    int tiles;                  // key tiles
    int groups;                 // groups of row tiles with live rows
    // Keys of a tile that any row sees, and whether some of them are nodes.
    __device__ __forceinline__ int hi(int tile) const { return min(kKeys, end - tile * kKeys); }
    __device__ __forceinline__ bool has_nodes(int tile) const { return (tile + 1) * kKeys > len && end > len; }
};
template <int NQ>
struct Plan {
    // A piece's end and the next one's first products take 3 to 5 us, a tile 1.  (None: 36.6 us
    // for the ragged pages, 71 for 64 short sequences; two: 31.7 and 56.7; three: 31.2 and 55.8; six: 32.1 and 55.9.)
    static constexpr int kPieceUnits = 3;
    const Job& J;
    int batch, kv_heads, ctas;
    __device__ __forceinline__ explicit Plan(const Job& j) : J(j), batch(j.batch), kv_heads(j.kv_heads), ctas(j.ctas) {}
    __device__ __forceinline__ Seq sequence(int b) const {
        Seq s;
        s.nodes = J.nodes_len ? min(max(__ldg(J.nodes_len + b), 0), J.nodes) : J.nodes;
        // A sequence that its cache cannot hold is cut to what fits (and reported).
        const int64_t own = J.context_only ? 0 : min(int64_t(s.nodes), J.capacity);
        s.len = int(min(int64_t(max(__ldg(J.lengths + b), 0)), J.capacity - own));
        s.end = s.len + int(own);
        s.tiles = (s.end + kKeys - 1) / kKeys;
        s.groups = (s.nodes + NQ * J.tpt - 1) / (NQ * J.tpt);
        return s;
    }
};

// ------------------------------------------------------------------ types --
template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kHalf) {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        return pack_bf16x2(lo, hi);
    }
}
template <bool kHalf>
__device__ __forceinline__ float value_at(const void* p, int64_t i) {
    if constexpr (kHalf) return __half2float(static_cast<const __half*>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// Instruction descriptor of kind::f16: the bf16 one with both operand formats
// (bits [7,10) and [10,13)) 0 for fp16.
template <bool kHalf>
__device__ __forceinline__ constexpr uint32_t idesc(int m, int n, int a_mn, int b_mn) {
    return umma_idesc_bf16(m, n, a_mn, b_mn) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
}
// A from tensor memory (two 16-bit K elements per column), B from shared memory.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc_, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc_), "r"(accumulate)
        : "memory");
}

// Whether `x` holds for any of the 256 softmax threads of a row tile (their
// barrier `id`).
__device__ __forceinline__ bool any_of_row_tile(int id, bool x) {
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 256, p;\n selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(any)
        : "r"(uint32_t(x)), "r"(id)
        : "memory");
    return any != 0;
}

// Tensor memory columns: O of each row tile, then its S buffers, as many as
// fit; a tile's P goes over its S, which is in registers by then.
template <int NQ, int C>
struct Columns {
    static constexpr int kO = NQ == 1 ? 64 * C : 128;
    static constexpr int kBufs = NQ == 2 ? 2 : (512 - kO) / kKeys < 4 ? (512 - kO) / kKeys : 4;
    __device__ static constexpr uint32_t o(int q) { return uint32_t(q * kO); }
    __device__ static constexpr uint32_t s(int q, int buf) { return uint32_t(NQ * kO + (kBufs * q + buf) * kKeys); }
    static_assert(NQ * (kO + kBufs * kKeys) <= 512 && kBufs >= 2, "tensor memory");
};

__device__ __forceinline__ uint32_t mask_word(const int32_t* row, int words, int w) {
    return w >= 0 && w < words ? uint32_t(__ldg(row + w)) : 0u;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// Which of the 32 keys from node `first` on (below 0: context) node t sees:
// the context, and the nodes of its words (without words: up to itself).
__device__ __forceinline__ uint32_t seen_keys(const int32_t* row, int words, int t, int nodes, int first) {
    const uint32_t context = low_bits(-first);
    uint32_t bits;
    if (row) {
        const int w = first >> 5;               // floor
        bits = __funnelshift_r(mask_word(row, words, w), mask_word(row, words, w + 1), first & 31);
    } else {
        bits = low_bits(t + 1 - first);
    }
    return context | (bits & low_bits(nodes - first));
}

// The box of a key tile that this lane loads: its page (dense: its sequence)
// and row.  Boxes past the last used row repeat that row's (they are masked).
template <class W>
__device__ __forceinline__ int box_of(const Job& J, const W& w, int tile, int lane, int& row) {
    row = tile * kKeys + lane * J.box;
    if (!J.paged) return J.shared_cache ? 0 : w.b;
    int64_t page = 0;
    if (lane < kKeys / J.box) {
        const int last = tile * kKeys + w.s.hi(tile) - 1;
        if (!cache_row(J.cache, w.b, min(row, last / J.box * J.box), page, row)) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    return int(page);
}
// Whether a V tile holds rows that nobody sees, or the nodes' own.
__device__ __forceinline__ bool needs_fix(const Seq& s, int tile) { return s.has_nodes(tile) || s.hi(tile) < kKeys; }

// Row r of a V chunk in shared memory (every kStep-th 16 bytes): zeroed when nobody sees it (its P is 0,
// and 0 x NaN is not 0); of a node's row, infinities and NaN become 0 (the
// epilogue adds them to the rows that see them).  True when there were any.
template <bool kHalf, int kStep>
__device__ __forceinline__ bool fix_values(uint8_t* chunk, int r, int u0, bool seen, bool node) {
    constexpr uint32_t kExp = kHalf ? 0x7c00u : 0x7f80u;
    if (seen && !node) return false;
    bool bad = false;
#pragma unroll 1
    for (int u = u0; u < 8; u += kStep) {
        uint4* at = reinterpret_cast<uint4*>(chunk + r * 128) + ((u ^ r) & 7);
        uint4 v = make_uint4(0, 0, 0, 0);
        bool write = !seen;
        if (seen) {
            v = *at;
            uint32_t* x = &v.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if ((x[e] & kExp) == kExp) { x[e] &= 0xffff0000u; write = true; }
                if ((x[e] >> 16 & kExp) == kExp) { x[e] &= 0xffffu; write = true; }
            }
            bad |= write;
        }
        if (write) *at = v;
    }
    return bad;
}

// Ring geometry for rows of C 64-column chunks (shorter ones are filled up with
// zeros).  A V slot is a whole row, a K slot too up to 128 dims, and one chunk
// above, where whole rows would leave no second tile.  All of it constant: with
// loops of run-time length the MMA operands are no uniform registers, and the
// wide rows' MMAs took 100 cycles each.
template <int NQ, int C>
struct Rings {
    static constexpr int kFree = int((kTileArea<NQ, C> - uint32_t(NQ * C) * kQChunk) / kChunk);
    static constexpr int kGroup = C > 2 ? 1 : C;             // chunks of a K slot
    static constexpr int kPer = C / kGroup;                  // K slots of a tile
    static constexpr int kV = kFree / 2 / C < 2 ? 2 : kFree / 2 / C < kMaxRing ? kFree / 2 / C : kMaxRing;
    static constexpr int kK = (kFree - kV * C) / kGroup < kMaxRing ? (kFree - kV * C) / kGroup : kMaxRing;
    static_assert(kK >= kPer + 1 && kV >= 2, "two tiles under way");
};

// ----------------------------------------------------------------- kernel --
template <int NQ, int C, bool kHalf>
__global__ void __launch_bounds__(kEarlyMerge<NQ, C> ? 512 : 128 + kSoftmaxThreads<NQ>, 1)     // (512: 128 registers a thread)
tree_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Job J) {
    constexpr int kThreads = 128 + kSoftmaxThreads<NQ>;
    constexpr int kHalves = kHalvesOf<NQ>, kWarps = 4 * kHalves, kCols = kKeys / kHalves;
    using Col = Columns<NQ, C>;
    using R = Rings<NQ, C>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* bs = reinterpret_cast<Bars*>(smem + kTileArea<NQ, C>);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Layout: Q (NQ x C chunks) | K ring | V ring.
    const uint32_t off_k = uint32_t(NQ * C) * kQChunk;
    const uint32_t off_v = off_k + uint32_t(R::kK * R::kGroup) * kChunk;

    if (tid < kMaxRing) {
        mbar_init(&bs->kfull[tid], 1); mbar_init(&bs->kempty[tid], NQ);
        mbar_init(&bs->vfull[tid], 1); mbar_init(&bs->vempty[tid], NQ); mbar_init(&bs->vfixed[tid], kWarps);
    } else if (tid < kMaxRing + 8) {
        const int q = (tid - kMaxRing) & 1, s = (tid - kMaxRing) >> 1;
        mbar_init(&bs->sfull[q][s], 1);
        mbar_init(&bs->pfull[q][s], kWarps);
        mbar_init(&bs->odone[q][s], 1);
        if (s == 0) mbar_init(&bs->oempty[q], kWarps);
    } else if (tid == kMaxRing + 8) {
        mbar_init(&bs->qfull, 1);
        mbar_init(&bs->qempty, NQ);
        mbar_init(&bs->final_mma, 2);
        bs->abort = 0;
        for (int& x : bs->bad_values) x = 0;
    }
    if (tid < 32) fence_barrier_init();
    if (tid == 32) {
        tma_prefetch_desc(&qmap);
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    if (warp == 2) {
        tmem_alloc(&bs->tmem_base, 512);
        tmem_relinquish();
    }
    if (kEarlyMerge<NQ, C>) grid_launch_dependents();
    const Plan<NQ> plan(J);
    if (warp == 3) find_share(plan, &bs->share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // All 512 tensor memory columns are this CTA's: addresses begin at column 0.
    const uint32_t sbase = smem_u32(smem);
    const bool any = int(blockIdx.x) < bs->share.ctas;

    if (any && (warp == 0 || warp == 3)) {
        // ---- loads: warp 0 each piece's Q and the K chunks, warp 3 the V chunks ----
        const bool keys = warp == 0;
        const int per = keys ? R::kGroup : C, ring = keys ? R::kK : R::kV;
        uint64_t* full = keys ? bs->kfull : bs->vfull;
        uint64_t* empty = keys ? bs->kempty : bs->vempty;
        const CUtensorMap* map = keys ? &kmap : &vmap;
        uint8_t* dst = smem + (keys ? off_k : off_v);
        const int boxes = kKeys / J.box;
        int slot = 0;
        uint32_t lap = 0;
        bool ok = true;
        Walk<Plan<NQ>> w;
        w.start(plan, &bs->share);
        while (ok && w.next(plan)) {
            if (keys) {
                if (w.piece > 0 && !(ok = warp_wait(&bs->qempty, (w.piece - 1) & 1, bs, J))) break;
                if (lane == 0) {
                    mbar_expect_tx(&bs->qfull, uint32_t(NQ * C) * uint32_t(J.tile_rows) * 128u);
                    for (int q = 0; q < NQ; ++q)
                        for (int c = 0; c < C; ++c)
                            tma_load_4d(smem + (q * C + c) * kQChunk, &qmap, &bs->qfull, c * 64, w.g * J.group,
                                        (w.group * NQ + q) * J.tpt, w.b);
                }
                __syncwarp();
            }
            for (int tile = w.t0; tile < w.t1 && ok; ++tile) {
                int row;
                const int page = box_of(J, w, tile, lane, row);
                for (int c = 0; c < C; c += per) {
                    if (lap && !(ok = warp_wait(&empty[slot], (lap - 1) & 1, bs, J))) break;
                    if (lane == 0) mbar_expect_tx(&full[slot], uint32_t(per) * kChunk);
                    __syncwarp();
                    if (lane < boxes)
                        for (int k = 0; k < per; ++k)
                            tma_load_4d(dst + (slot * per + k) * kChunk + lane * J.box * 128, map, &full[slot], (c + k) * 64, w.g, row, page);
                    if (++slot == ring) { slot = 0; ++lap; }
                }
            }
        }
    } else if (any && warp <= 2) {
        // ---- MMA issue by two warps: with one row tile, warp 1 the S and warp 2 the P.V;
        // with two, warp 1 + q both products of row tile q, S two tiles ahead.  The tensor
        // core queues only a few MMAs, so what a warp does between them is time lost unless
        // another warp's MMAs fill it (two row tiles, 128 keys: 8,100 cycles with one warp,
        // 4,600 with two; 320 dims, 64 keys: 3,450 and 1,900).  A warp stays converged, its
        // branches go by votes, and one elected thread has the instructions alone, so that
        // operands are uniform registers. ----
        constexpr int kBufs = Col::kBufs;
        const int q = NQ == 2 ? warp - 1 : 0;
        const uint32_t idesc_s = idesc<kHalf>(128, kKeys, 0, 0);
        const uint32_t idesc_o = idesc<kHalf>(128, 64 * (C < 4 ? C : 4), 0, 1), idesc_o1 = idesc<kHalf>(128, 64, 0, 1);
        // Matrix descriptors (K-major Q and K; MN-major V): the low word moves with the address.
        constexpr uint64_t kQStep = kQChunk >> 4, kStep = kChunk >> 4;
        const uint64_t q_desc = umma_desc_sw128(sbase, 16, 1024) + uint32_t(q * C) * kQStep;
        const uint64_t k_desc = umma_desc_sw128(sbase + off_k, 16, 1024), v_desc = umma_desc_sw128(sbase + off_v, kChunk, 1024);
        bool ok = true;                          // of this lane; votes at the branches
        // S of the share's tiles in order.
        struct {
            int slot, tile;
            uint32_t lap, buf, round, q_lap;     // round: of the S buffers
            bool more;
        } f{};
        Walk<Plan<NQ>> ws;
        auto begin_s = [&] {
            ws.start(plan, &bs->share);
            f.more = all_lanes(ws.next(plan));
            f.tile = ws.t0;
        };
        auto issue_s = [&] {
            if (all_lanes(f.tile == ws.t0)) {
                ok = ok && wait_bar(&bs->qfull, f.q_lap, bs, J);
                f.q_lap ^= 1;
            }
            // The buffer's last P has been read (two row tiles: this warp issued that P.V before).
            if (NQ == 1 && f.round) ok = ok && wait_bar(&bs->odone[0][f.buf], (f.round - 1) & 1, bs, J);
#pragma unroll
            for (int c = 0, slot = f.slot, lap = f.lap; c < C; c += R::kGroup) {
                ok = ok && wait_bar(&bs->kfull[slot], lap, bs, J);
                if (++slot == R::kK) { slot = 0; lap ^= 1; }
            }
            const bool last = all_lanes(f.tile == ws.t1 - 1);
            if (!all_lanes(ok)) return;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t d = Col::s(q, f.buf);
#pragma unroll
                for (int c = 0, slot = f.slot; c < C; c += R::kGroup) {
#pragma unroll
                    for (int k = 0; k < R::kGroup; ++k) {
                        const uint64_t a = q_desc + uint32_t(c + k) * kQStep, b = k_desc + uint32_t(slot * R::kGroup + k) * kStep;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) umma_bf16(d, a + 2 * kk, b + 2 * kk, idesc_s, (c | k | kk) != 0);
                    }
                    umma_commit(&bs->kempty[slot]);
                    if (++slot == R::kK) slot = 0;
                }
                umma_commit(&bs->sfull[q][f.buf]);
                if (last) umma_commit(&bs->qempty);
            }
            __syncwarp();
            f.slot += R::kPer;
            if (f.slot >= R::kK) { f.slot -= R::kK; f.lap ^= 1; }
            if (++f.buf == kBufs) { f.buf = 0; ++f.round; }
            ++f.tile;
            if (last) {
                f.more = all_lanes(ws.next(plan));
                f.tile = ws.t0;
            }
        };
        if (NQ == 2 || warp == 1) begin_s();
        if (NQ == 1 && warp == 1) {
            while (all_lanes(ok && f.more)) issue_s();
        } else {
            if constexpr (NQ == 2) {
                if (f.more) issue_s();
                if (f.more) issue_s();
            }
            int slot = 0;
            uint32_t lap = 0, buf = 0, round = 0, o_lap = 0, fixes = 0;     // fixes: each slot's parity of vfixed
            bool again = false;                  // a piece came before
            Walk<Plan<NQ>> wp;
            wp.start(plan, &bs->share);
            while (all_lanes(ok && wp.next(plan))) {
                int tile = wp.t0;
                bool first = true;
                do {
                    if (first && again) {        // the previous piece has left its O
                        ok = ok && wait_bar(&bs->oempty[q], o_lap, bs, J);
                        o_lap ^= 1;
                    }
                    ok = ok && wait_bar(&bs->vfull[slot], lap, bs, J);
                    // Row tile 0 looks after the V rows (fix_values), row tile 1 waits for it.
                    if (NQ == 2 && q == 1 && all_lanes(needs_fix(wp.s, tile))) {
                        ok = ok && wait_bar(&bs->vfixed[slot], fixes >> slot & 1, bs, J);
                        fixes ^= 1u << slot;
                    }
                    ok = ok && wait_bar(&bs->pfull[q][buf], round & 1, bs, J);
                    if (!all_lanes(ok)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t a = Col::s(q, buf);
                        const uint64_t b = v_desc + uint32_t(slot * C) * kStep;
                        // The row's chunks lie side by side: up to four are one MMA of N = 256.
#pragma unroll
                        for (int ks = 0; ks < kKeys / 16; ++ks) {
                            umma_ts(Col::o(q), a + 8u * ks, b + 128 * ks, idesc_o, (!first || ks > 0) ? 1u : 0u);
                            if constexpr (C == 5)
                                umma_ts(Col::o(q) + 256u, a + 8u * ks, b + 4 * kStep + 128 * ks, idesc_o1, (!first || ks > 0) ? 1u : 0u);
                        }
                        umma_commit(&bs->vempty[slot]);
                        umma_commit(&bs->odone[q][buf]);
                    }
                    __syncwarp();
                    if (++slot == R::kV) { slot = 0; lap ^= 1; }
                    if (++buf == kBufs) { buf = 0; ++round; }
                    first = false;
                    ++tile;
                    if (NQ == 2 && f.more) issue_s();
                } while (all_lanes(ok && tile < wp.t1));
                again = true;
            }
        }
        if (elect_one()) umma_commit(&bs->final_mma);
        __syncwarp();
    } else if (any && warp >= 4) {
        // ---- softmax and epilogue of row tile qt: kHalves threads for a row (TMEM lane), each
        // with kCols of a tile's keys.  Two threads share the row's running maximum: a barrier
        // of the row tile's threads asks whether any row outgrew it by 2^8, and only then do
        // they exchange maxima.  After a wait that ran out every thread still meets at every
        // barrier, without work. ----
        const int qt = (warp - 4) / kWarps, half = kHalves == 2 ? (warp >> 2) & 1 : 0, quarter = warp & 3;
        const int r = 32 * quarter + lane;
        const uint32_t lane_addr = uint32_t(32 * quarter) << 16;
        const uint32_t o_base = lane_addr + Col::o(qt);
        const int jh = r % J.group;
        // All threads of a row get op over their x.
        auto over_row = [&](float x, auto op) {
            if constexpr (kHalves == 1) return x;
            float* at = &bs->exchange[r];
            if (half) *at = x;
            named_bar(1 + qt, 256);
            if (!half) *at = x = op(x, *at);
            named_bar(1 + qt, 256);
            return half ? *at : x;
        };
        constexpr int kBufs = Col::kBufs;
        bool ok = true;
        int i = 0;                                              // tiles done
        Walk<Plan<NQ>> w;
        w.start(plan, &bs->share);
        while (w.next(plan)) {
            const int t = (w.group * NQ + qt) * J.tpt + r / J.group;
            const bool live = r < J.tile_rows && t < w.s.nodes;
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int32_t* words = J.mask ? J.mask + w.b * J.mask_stride + int64_t(min(t, J.nodes - 1)) * J.words : nullptr;
            float m_run = -INFINITY, l_run = 0.f;               // the exponent m taken out, and the sum of P
            for (int tile = w.t0; tile < w.t1; ++tile, ++i) {
                const bool masked = needs_fix(w.s, tile);
                uint32_t seen[kCols / 32];                      // which of its keys the row sees
                if (masked) {
#pragma unroll
                    for (int c = 0; c < kCols / 32; ++c) {
                        const int k = kCols * half + 32 * c;
                        seen[c] = w.s.has_nodes(tile) ? seen_keys(words, J.words, t, w.s.end - w.s.len, tile * kKeys + k - w.s.len)
                                                      : low_bits(w.s.hi(tile) - k);
                    }
                }
                const int buf = i % kBufs;
                ok = ok && warp_wait(&bs->sfull[qt][buf], (i / kBufs) & 1, bs, J);
                tc_fence_after();
                const uint32_t s_addr = lane_addr + Col::s(qt, buf);
                float v[kCols];
                float mx = -INFINITY;
                if (warp_live) {
#pragma unroll
                    for (int c = 0; c < kCols; c += 32) tmem_ld32(s_addr + uint32_t(kCols * half + c), v + c);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < kCols; ++e)
                            if (!(seen[e / 32] >> (e % 32) & 1)) v[e] = -INFINITY;
                    }
                    float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int e = 4; e < kCols - 4; e += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) m4[k] = fmaxf(fmaxf(m4[k], v[e + k]), v[e + 4 + k]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) m4[k] = fmaxf(m4[k], v[kCols - 4 + k]);
                    mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                }
                mx *= J.scale_log2;                             // scale > 0
                // Two threads of a row: all have read this tile's S when they pass here, so P may
                // go over it.
                const bool more = live && mx > m_run + (kLazyLog2 + kDownLog2<kHalf>);
                const bool grown = kHalves == 2 ? any_of_row_tile(1 + qt, more) : __any_sync(0xffffffffu, more);
                const bool fix = qt == 0 && masked;
                // (A ring of more V slots than S buffers: the slot's last tile is over, S(i) came after it.)
                if (((grown && tile > w.t0) || (fix && R::kV <= kBufs)) && i > 0) {
                    ok = ok && warp_wait(&bs->odone[qt][(i - 1) % kBufs], ((i - 1) / kBufs) & 1, bs, J);
                    tc_fence_after();
                }
                if (grown) {
                    mx = over_row(mx, [](float a, float b) { return fmaxf(a, b); });
                    float alpha = 1.f;
                    if (mx > m_run + (kLazyLog2 + kDownLog2<kHalf>)) {
                        const float m = mx - kDownLog2<kHalf>;
                        alpha = m_run == -INFINITY ? 1.f : exp2f(m_run - m);
                        m_run = m;
                        l_run *= alpha;
                    }
                    if (ok && tile > w.t0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                        for (int c = half; c < 4 * C; c += kHalves) {
                            float o[16];
                            tmem_ld16(o_base + 16u * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] *= alpha;
                            tmem_st16(o_base + 16u * c, o);
                        }
                        tmem_wait_st();
                    }
                }
                if (warp_live) {
                    const float shift = m_run == -INFINITY ? 0.f : m_run;
                    // Plain scalar arithmetic: packed pairs of fp32 (f32x2) took twice the time next
                    // to the exponentials, 1,138 against 497 cycles for 64 keys of a warp.
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < kCols; c += 32) {
                        float packed[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float p0 = sfu_exp2(fmaf(v[c + 2 * k], J.scale_log2, -shift));
                            const float p1 = sfu_exp2(fmaf(v[c + 2 * k + 1], J.scale_log2, -shift));
                            sum[2 * k & 3] += p0;
                            sum[(2 * k + 1) & 3] += p1;
                            packed[k] = __uint_as_float(pack2<kHalf>(p0, p1));
                        }
                        tmem_st16(s_addr + uint32_t(kCols * half + c) / 2, packed);
                    }
                    l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_wait_st();
                }
                if (fix && ok) {
                    // The slot's tile before this one is over, so this is the next that lands there.
                    const int slot = i % R::kV;
                    bool bad = false;
                    ok = warp_wait(&bs->vfull[slot], (i / R::kV) & 1, bs, J);
                    for (int c = 0; c < C && ok; ++c)
                        bad |= fix_values<kHalf, 2 * kHalves>(smem + off_v + uint32_t(slot * C + c) * kChunk, r & 63, 2 * half + (r >> 6),
                                                              (r & 63) < w.s.hi(tile), tile * kKeys + (r & 63) >= w.s.len);
                    // (Row tile 0 is up to three pieces ahead of row tile 1: a Q goes when both have
                    // issued its products, and a row tile issues S up to two tiles ahead.)
                    if (bad) *const_cast<volatile int*>(&bs->bad_values[w.piece & 3]) = w.piece + 1;
                    fence_async_shared();
                    if constexpr (NQ == 2) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bs->vfixed[slot]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bs->pfull[qt][buf]);
            }
            // ---- the piece's rows: the sums of all threads of a row, then each its columns ----
            l_run = over_row(l_run, [](float a, float b) { return a + b; });
            ok = ok && warp_wait(&bs->odone[qt][(i - 1) % kBufs], ((i - 1) / kBufs) & 1, bs, J);
            if (!ok) continue;
            tc_fence_after();
            const bool whole = w.whole();
            const bool bad = *const_cast<volatile int*>(&bs->bad_values[w.piece & 3]) == w.piece + 1;
            const float inv = l_run != 0.f ? 1.f / l_run : 0.f;      // a NaN sum stays NaN
            const float lse2 = l_run != 0.f ? m_run + log2f(l_run) : -INFINITY;
            const int h = w.g * J.group + jh;
            const int rows = NQ * J.tile_rows, slot = 2 * blockIdx.x + (w.piece > 0), row = qt * J.tile_rows + r;
            float4* part = reinterpret_cast<float4*>(J.part_o) + int64_t(slot) * (J.dim_v / 4) * rows + row;
#pragma unroll 1
            for (int c = half; c < 4 * C; c += kHalves) {
                float o[16];
                if (warp_live) {
                    tmem_ld16(o_base + 16u * c, o);
                    tmem_wait_ld();
                }
                if (live) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= inv;
                    if (bad) {
                        // Infinities and NaN of the nodes' values, for the rows that see them.
                        for (int n0 = 0; n0 < w.s.nodes; n0 += 32) {
                            uint32_t bits = seen_keys(words, J.words, t, w.s.nodes, n0);
                            for (; bits; bits &= bits - 1) {
                                int at = w.s.len + n0 + __ffs(int(bits)) - 1;
                                if (at < w.t0 * kKeys || at >= w.t1 * kKeys) continue;
                                int64_t page = J.shared_cache ? 0 : w.b;
                                if (J.paged) cache_row(J.cache, w.b, at, page, at);
                                const int64_t base = page * J.cache.v_stride[0] + at * J.cache.v_stride[1] + w.g * J.cache.v_stride[2];
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const int d = 16 * c + e;
                                    if (d < J.dim_v) {
                                        const float x = value_at<kHalf>(J.v, base + d);
                                        if (!isfinite(x)) o[e] += x;
                                    }
                                }
                            }
                        }
                    }
                    if (whole) {
                        uint16_t* dst = static_cast<uint16_t*>(J.out) + w.b * J.o_sb + t * J.o_st + h * J.o_sh;
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int d = 16 * c + 8 * u;
                            if (d < J.dim_v)
                                *reinterpret_cast<uint4*>(dst + d) =
                                    make_uint4(pack2<kHalf>(o[8 * u], o[8 * u + 1]), pack2<kHalf>(o[8 * u + 2], o[8 * u + 3]),
                                               pack2<kHalf>(o[8 * u + 4], o[8 * u + 5]), pack2<kHalf>(o[8 * u + 6], o[8 * u + 7]));
                        }
                    } else {
                        // [slot][4 dims][row]: the rows of a warp side by side.
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (16 * c + 4 * u < J.dim_v)
                                part[int64_t(4 * c + u) * rows] = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                    }
                }
                __syncwarp();
            }
            if (live && half == 0) {
                if (whole) J.lse[(int64_t(w.b) * J.nodes + t) * J.heads + h] = lse2 * kLn2;
                else J.part_lse[slot * rows + row] = lse2;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bs->oempty[qt]);
        }
    }
    __syncthreads();
    if (!kEarlyMerge<NQ, C>) grid_launch_dependents();
    if (any) {
        // Nothing of this CTA is in flight when its tensor memory goes: the
        // MMAs (they follow every copy that was waited for), and after a wait
        // that ran out the copies that were not.
        if (tid == 64) mbar_wait(&bs->final_mma, 0, 2000000000ull);
        if (bs->abort && tid == 0) {
            for (int s = 0; s < R::kK; ++s) {
                mbar_wait(&bs->kfull[s], 0, 100000000ull);
                mbar_wait(&bs->kfull[s], 1, 100000000ull);
            }
            for (int s = 0; s < R::kV; ++s) {
                mbar_wait(&bs->vfull[s], 0, 100000000ull);
                mbar_wait(&bs->vfull[s], 1, 100000000ull);
            }
            mbar_wait(&bs->qfull, 0, 100000000ull);
            mbar_wait(&bs->qfull, 1, 100000000ull);
        }
    }
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(bs->tmem_base, 512);
    }
}

constexpr int kCombineThreads = 256;

// Merges the pieces of a segment's rows, and writes the rows that see nothing.
// A (sequence, KV head, row group) has gridDim.y blocks, which take its parts
// of 32 rows (a lane each) and 64 dims (8 to a warp) by turns, four pieces'
// loads under way at a time.  Segments have two or three pieces when there are
// many, tens when there are few: fewer dims to a warp cost the first case
// instructions, more the second latency; and many blocks to a segment cost many
// short segments more than the merge.  Alone, caches cold: 10.7 us for 8 segments
// of 128 rows x 320 dims in 19 pieces each (24 MB), 17 us for 128 segments of 256
// rows x 128 dims, 7.5 us for 64 segments of 65 rows, 7 us for one token.
template <int NQ, bool kHalf>
__global__ void __launch_bounds__(kCombineThreads, 4) combine_kernel(const __grid_constant__ Job J) {
    __shared__ int range[3];                // first and last CTA of the segment's pieces, slot of the first
    __shared__ uint2 tile[32][17];          // the merged rows, 4 dims to an entry (17: no bank twice)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int at = blockIdx.x;
    const int group = at % J.row_groups;
    at /= J.row_groups;
    const int g = at % J.kv_heads, b = at / J.kv_heads;
    const Plan<NQ> plan(J);
    const Seq s = plan.sequence(b);
    const bool some = group < s.groups && s.tiles > 0;
    if (some && warp == 0) {
        uint32_t total, before;
        sum_units(plan, b, total, before);
        if (lane == 0) {
            const uint32_t units = segment_units(plan, s), u0 = before + uint32_t(g * s.groups + group) * units;
            const uint32_t ctas = share_count(total, J.ctas), c0 = share_of(total, u0 + Plan<NQ>::kPieceUnits, ctas);
            range[0] = int(c0);
            range[1] = int(share_of(total, u0 + units - 1, ctas));
            range[2] = 2 * int(c0) + (share_begin(total, c0, ctas) < u0 ? 1 : 0);   // a piece of another segment before it
        }
    }
    if (threadIdx.x == 32 && g == 0 && group == 0 && blockIdx.y == 0) {
        const int len = __ldg(J.lengths + b), nodes = J.nodes_len ? __ldg(J.nodes_len + b) : J.nodes;
        if (len != s.len || nodes != s.nodes || (!J.context_only && s.end != s.len + s.nodes)) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    __syncthreads();
    const int c0 = some ? range[0] : 0, c1 = some ? range[1] : 0, slot0 = some ? range[2] : 0;
    grid_dependency_wait();                 // every block: what follows this grid counts on the one before it too
    // A segment in one piece whose rows are all live is written already.
    if (some && c0 == c1 && min((group + 1) * NQ * J.tpt, J.nodes) <= s.nodes) return;
    const int rows = NQ * J.tile_rows, first_node = group * NQ * J.tpt;
    const int used = min(rows, (J.nodes - first_node) * J.group);       // the group's rows that are nodes
    const int dim_parts = (J.dim_v + 63) / 64, parts = (used + 31) / 32 * dim_parts;
    const bool split = c0 != c1;
    auto slot_of = [&](int c) { return int64_t(c == c0 ? slot0 : 2 * c); };
    auto node_of = [&](int row) { return first_node + row / J.group; };
    auto head_of = [&](int row) { return g * J.group + row % J.group; };
    // Whether a row is this kernel's to write.
    auto mine = [&](int row) { return row < used && (split || !some || node_of(row) >= s.nodes); };
    for (int part = blockIdx.y; part < parts; part += gridDim.y) {
        const int r0 = part / dim_parts * 32, r = r0 + lane, dim0 = part % dim_parts * 64, d0 = dim0 + 8 * warp;
        const bool live = some && mine(r) && node_of(r) < s.nodes && d0 < J.dim_v;
        // In one pass, the largest exponent so far taken out: a piece's lse and rows are one latency.
        float m = -INFINITY, sum = 0.f, shift = 0.f;
        float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        if (live) {
            constexpr int kAhead = 4;
            const float4* part = reinterpret_cast<const float4*>(J.part_o) + int64_t(d0 / 4) * rows + r;
            const int64_t step = int64_t(J.dim_v / 4) * rows;
            for (int c = c0; c <= c1; c += kAhead) {
                float w[kAhead];
                float4 x[kAhead][2];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    w[k] = -INFINITY;
                    if (c + k > c1) continue;
                    const int64_t slot = slot_of(c + k);
                    w[k] = J.part_lse[slot * rows + r];
                    x[k][0] = part[slot * step];
                    x[k][1] = part[slot * step + rows];
                }
                const float before = shift;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) m = fmaxf(m, w[k]);
                shift = m == -INFINITY ? 0.f : m;
                const float old = sum != 0.f ? sfu_exp2(before - shift) : 0.f;
                sum *= old;
#pragma unroll
                for (int u = 0; u < 2; ++u) { acc[u].x *= old; acc[u].y *= old; acc[u].z *= old; acc[u].w *= old; }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const float f = sfu_exp2(w[k] - shift);
                    sum += f;
                    if (f == 0.f) continue;             // (an empty piece's rows are not read into the sum)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        acc[u].x = fmaf(f, x[k][u].x, acc[u].x); acc[u].y = fmaf(f, x[k][u].y, acc[u].y);
                        acc[u].z = fmaf(f, x[k][u].z, acc[u].z); acc[u].w = fmaf(f, x[k][u].w, acc[u].w);
                    }
                }
            }
        }
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            tile[lane][2 * warp + u] = make_uint2(pack2<kHalf>(acc[u].x * inv, acc[u].y * inv), pack2<kHalf>(acc[u].z * inv, acc[u].w * inv));
        if (d0 == 0 && mine(r))
            J.lse[(int64_t(b) * J.nodes + node_of(r)) * J.heads + head_of(r)] = sum != 0.f ? (shift + log2f(sum)) * kLn2 : -INFINITY;
        __syncthreads();
        // Out by rows: 16 lanes hold 64 dims, 128 bytes, of a row.
        const int u = threadIdx.x & 15, d = dim0 + 4 * u;
#pragma unroll
        for (int k = threadIdx.x >> 4; k < 32; k += kCombineThreads / 16)
            if (mine(r0 + k) && d < J.dim_v) {
                uint16_t* dst = static_cast<uint16_t*>(J.out) + b * J.o_sb + node_of(r0 + k) * J.o_st + head_of(r0 + k) * J.o_sh + d;
                *reinterpret_cast<uint2*>(dst) = tile[k][u];
            }
        __syncthreads();                        // the next part's rows go into the same tile
    }
}

// ------------------------------------------------------------------- host --
int row_tiles_per_cta(const slimkv_tree_attention_args* a) {
    // Two row tiles share each K / V tile where their O and S fit tensor memory
    // and there are rows for both.
    const int tpt = kRows / (a->heads / a->kv_heads);
    return a->dim_qk <= 128 && a->dim_v <= 128 && a->nodes > tpt ? 2 : 1;
}

int check_tree(const slimkv_tree_attention_args* a) {
    if (!a) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->batch < 1 || a->batch > 4096 || a->nodes < 1 || a->nodes > 1024 || a->heads < 1 || a->kv_heads < 1 ||
        a->heads % a->kv_heads)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree attention: batch in 1..4096, nodes in 1..1024, heads a multiple of kv_heads");
    if (a->heads / a->kv_heads > kRows)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "tree attention: at most 128 query heads per KV head");
    if (a->dim_qk < 8 || a->dim_qk > 64 * kMaxChunks || a->dim_qk % 8 || a->dim_v < 8 || a->dim_v > 64 * kMaxChunks || a->dim_v % 8)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "tree attention: dims must be multiples of 8 up to 320");
    if (a->type != SLIMKV_BF16 && a->type != SLIMKV_FP16)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree attention: bf16 or fp16 tensors");
    return SLIMKV_OK;
}

void carve(Carver& c, const slimkv_tree_attention_args* a, Job& J) {
    J.group = a->heads / a->kv_heads;
    J.tpt = kRows / J.group;
    J.tile_rows = J.tpt * J.group;
    J.ctas = device_info().sm_count;
    const size_t rows = size_t(2) * J.ctas * row_tiles_per_cta(a) * J.tile_rows;
    J.part_o = c.take<float>(rows * a->dim_v);
    J.part_lse = c.take<float>(rows);
}

template <int NQ, int C, bool kHalf>
int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const Job& J, cudaStream_t stream) {
    auto kernel = tree_attention_kernel<NQ, C, kHalf>;
    static bool configured[64] = {};
    const int dev = device_info().device;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes<NQ, C>)) != cudaSuccess)
            return fail(SLIMKV_ERR_CUDA, "cudaFuncSetAttribute (tree attention) failed");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    kernel<<<J.ctas, 128 + kSoftmaxThreads<NQ>, kSmemBytes<NQ, C>, stream>>>(qm, km, vm, J);
    cudaLaunchConfig_t cfg{};
    const int segments = J.batch * J.kv_heads * J.row_groups;
    const int parts = (std::min(NQ * J.tile_rows, J.nodes * J.group) + 31) / 32 * ((J.dim_v + 63) / 64);
    cfg.gridDim = dim3(segments, std::max(1, std::min(parts, 8 * J.ctas / segments)));
    cfg.blockDim = dim3(kCombineThreads);
    cfg.stream = stream;
    cudaLaunchAttribute dependent{};
    dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &dependent;
    cfg.numAttrs = 1;
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, combine_kernel<NQ, kHalf>, J);
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "tree attention launch failed: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_tree_attention_workspace_size(const slimkv_tree_attention_args* a) {
    if (check_tree(a) != SLIMKV_OK) return 0;
    Job J{};
    Carver c(nullptr, 0);
    carve(c, a, J);
    return c.used;
}

extern "C" int slimkv_tree_attention(const slimkv_tree_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_tree(a)) return rc;
    if (!a->q || !a->lengths || !a->out || !a->lse) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree attention: null pointer");
    if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree attention: scale must be positive");
    if (int rc = check_cache(a->cache, a->batch, a->dim_qk, a->dim_v, 2, true, "tree attention")) return rc;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8 || a->q_stride[i] < 0 || a->out_stride[i] % 8)
            return fail(SLIMKV_ERR_ALIGNMENT, "tree attention: strides must be multiples of 8 elements");
    if (!aligned16(a->q) || !aligned16(a->out)) return fail(SLIMKV_ERR_ALIGNMENT, "tree attention: 16-byte aligned tensors");
    const slimkv_cache& cache = a->cache;
    const bool paged = cache.table != nullptr;
    if (paged && cache.rows % 8) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "tree attention: pages of a multiple of 8 rows");
    Job J{};
    Carver c(workspace, workspace_bytes);
    carve(c, a, J);
    if (!workspace || !c.fits() || !aligned16(workspace))
        return fail(SLIMKV_ERR_WORKSPACE, "tree attention: %zu bytes of 16-byte aligned workspace needed", c.used);
    const int nq = row_tiles_per_cta(a);
    // A box of TMA rows stays inside a page: the largest power of two (up to a
    // key tile) that divides the page.
    J.box = paged ? std::min(kKeys, cache.rows & -cache.rows) : kKeys;
    const uint64_t planes = paged ? uint64_t(cache.num_pages) : uint64_t(a->batch);
    // One tensor map {dim, heads, rows, planes}; a dimension of one (or shared)
    // entry takes any valid stride.
    auto encode = [&](CUtensorMap* m, const void* base, int dim, const int64_t* st, bool shared) {
        const uint64_t row = uint64_t(st[1]) * 2, plane = uint64_t(st[0]) * 2, head = uint64_t(st[2]) * 2;
        const uint64_t any = uint64_t(dim) * 2;
        return encode_map_4d(m, base, dim, a->kv_heads, cache.rows, shared ? 1 : planes, a->kv_heads > 1 ? head : any,
                             cache.rows > 1 ? row : any, planes > 1 && !shared ? plane : any, J.box);
    };
    J.shared_cache = !paged && cache.k_stride[0] == 0 && cache.v_stride[0] == 0;
    if (a->batch > 1 && !paged && !J.shared_cache && (cache.k_stride[0] == 0 || cache.v_stride[0] == 0))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree attention: K and V are both shared by the batch or neither");
    CUtensorMap qm, km, vm;
    int rc;
    if ((rc = encode_map_4d_box(&qm, a->q, a->dim_qk, a->heads, a->nodes, a->batch, uint64_t(a->heads > 1 ? a->q_stride[2] : a->dim_qk) * 2,
                                uint64_t(a->nodes > 1 ? a->q_stride[1] : a->dim_qk) * 2, uint64_t(a->batch > 1 ? a->q_stride[0] : a->dim_qk) * 2,
                                J.group, J.tpt)) ||
        (rc = encode(&km, cache.k, a->dim_qk, cache.k_stride, J.shared_cache)) ||
        (rc = encode(&vm, cache.v, a->dim_v, cache.v_stride, J.shared_cache)))
        return rc;
    J.batch = a->batch;
    J.nodes = a->nodes;
    J.heads = a->heads;
    J.kv_heads = a->kv_heads;
    J.row_groups = (a->nodes + nq * J.tpt - 1) / (nq * J.tpt);
    J.dim_v = a->dim_v;
    J.context_only = a->context_only;
    J.paged = paged;
    J.cache = cache_view(cache);
    J.capacity = cache_capacity(J.cache);
    if (double(J.batch) * J.kv_heads * J.row_groups * double(J.capacity / kKeys + 1 + Plan<1>::kPieceUnits) >= 2147483648.0)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "tree attention: too many rows in one call");
    J.lengths = a->lengths;
    J.nodes_len = a->nodes_len;
    J.mask = a->context_only ? nullptr : a->mask;
    J.mask_stride = a->mask_stride;
    J.words = (a->nodes + 31) / 32;
    J.scale_log2 = a->scale * kLog2e;
    J.v = cache.v;
    J.out = a->out;
    J.o_sb = a->out_stride[0]; J.o_st = a->out_stride[1]; J.o_sh = a->out_stride[2];
    J.lse = a->lse;
    J.status = status_word();
    J.wait_ns = a->wait_limit_ns ? a->wait_limit_ns : 2000000000ull;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool half = a->type == SLIMKV_FP16;
    auto run = [&](auto rows, auto chunks) {
        return half ? launch<decltype(rows)::value, decltype(chunks)::value, true>(qm, km, vm, J, st)
                    : launch<decltype(rows)::value, decltype(chunks)::value, false>(qm, km, vm, J, st);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    switch ((std::max(a->dim_qk, a->dim_v) + 63) / 64) {
        case 1: return nq == 2 ? run(two, one) : run(one, one);
        case 2: return nq == 2 ? run(two, two) : run(one, two);
        case 3: return run(one, integral_constant<int, 3>());
        case 4: return run(one, integral_constant<int, 4>());
        default: return run(one, integral_constant<int, 5>());
    }
}
