// Attention of a tree of drafted tokens over a cache, split over the keys
// (C ABI slimkv_tree_attention).
//
// For every query row (node t, head h) over the keys n that the node sees
//   s_n = scale q . k_n,   lse = log sum_n e^{s_n},   out = sum_n e^{s_n - lse} v_n.
// The G = heads / kv_heads query heads of a KV head share its keys, so the
// rows of a KV head are (node, head of the group) pairs: 128 of them (whole
// nodes) fill one M = 128 tile of the tensor core, and a 128-key tile of K and
// V serves them all:
//   S [128 rows x 128 keys] = Q . K^T,   O [128 rows x dim_v] += P . V
// with tcgen05 (fp32 accumulators in TMEM; P = 2^(s - m) written back to TMEM
// in the inputs' 16-bit type as the A operand of the second product, which
// costs about what rounding the output costs; the row sums stay in fp32
// before that rounding, so lse keeps fp32 accuracy).
//
// Work: a unit is one 128-key tile of one (sequence, KV head, group of NQ row
// tiles) segment: the context rows, then the nodes' own rows, of which each
// row sees what its ancestor words say.  The units of all
// segments in a row are cut into one equal share per CTA; a share's part of a
// segment is a piece.  A piece that holds a whole segment writes the output;
// the others (at most two per CTA: its first and its last) leave normalised
// fp32 partial rows and their log-sum-exps, which combine_kernel merges.
// Lengths are read on the device; nothing on the host depends on them.
//
// Bound: with few rows per KV head HBM (each K / V row read once); with 128
// rows or more the tensor cores and the exponentials.
//
// One CTA per SM, warps: 0 = Q and K loads (TMA), 3 = V loads, 1 = MMA issue
// (one thread), 2 = TMEM owner, 4-7 (and 8-11) = softmax of row tile 0 (1), a
// thread per row.  Every wait is bounded.
#include <algorithm>

#include "cache_view.cuh"
#include "host_utils.h"
#include "key_shares.cuh"

namespace slimkv {
namespace {

constexpr int kRows = 128;
constexpr int kKeys = 128;
constexpr uint32_t kChunk = 128 * 128;           // [128 x 64] 16-bit elements
constexpr uint32_t kTileArea = 224 * 1024;
constexpr int kMaxRing = 8;
constexpr int kMaxChunks = 5;                    // dims <= 320
constexpr float kLazyLog2 = 8.f;                 // O is rescaled when a row's maximum grows by more than 2^8
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;

struct Bars {
    uint64_t kfull[kMaxRing], kempty[kMaxRing];                 // per 64-column chunk
    uint64_t vfull[kMaxRing], vempty[kMaxRing];                 // per tile
    uint64_t qfull, qempty;
    // [row tile][buffer]
    uint64_t sfull[2][2], sempty[2][2], pfull[2][2], odone[2][2], oempty[2], final_mma;
    uint32_t tmem_base;
    int abort;
    int bad_values[2];           // 1 + a piece whose node values hold infinities or NaN
    Share share;
};
constexpr uint32_t kSmemBytes = 1024 + kTileArea + uint32_t(sizeof(Bars));
static_assert(kSmemBytes <= 232448, "shared memory budget");

struct Job {
    int batch, nodes, heads, kv_heads, group;
    int tpt, tile_rows;         // nodes of a row tile and its rows (tpt * group <= 128)
    int row_groups;             // groups of NQ row tiles
    int kc, vc, dim_v;          // 64-column chunks of a K / V row
    int kring;                  // K chunks in shared memory
    int vstages;                // V tiles in shared memory
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

// A wait that is over costs one test; one that is not looks for an abort of
// another warp and for its limit.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Bars* bs, const Job& J) {
    if (mbar_test(bar, parity)) return true;
    for (uint64_t waited = 0; waited < J.wait_ns;) {
        const uint64_t step = min(J.wait_ns - waited, uint64_t(100000));
        if (mbar_wait(bar, parity, step)) return true;
        if (*const_cast<volatile int*>(&bs->abort)) return false;
        waited += step;
    }
    bs->abort = 1;
    report(J.status, SLIMKV_DEVICE_TIMEOUT);
    return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, Bars* bs, const Job& J) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, bs, J));
}

// Tensor memory columns.  One row tile, dims <= 128: O, two S, two P.  One row
// tile, wider: O (up to 320), S, P.  Two row tiles: O and S of each, P in its
// S (a tile's scores are in registers before its P is written, and the next
// S is issued behind the P.V that reads that P).
template <int NQ, bool kWide>
struct Columns {
    static constexpr int kBufs = NQ == 1 && !kWide ? 2 : 1;
    __device__ static constexpr uint32_t o(int q) { return uint32_t(q * 128); }
    __device__ static constexpr uint32_t s(int q, int buf) { return NQ == 2 ? 256u + 128u * q : kWide ? 320u : 128u + 128u * buf; }
    __device__ static constexpr uint32_t p(int q, int buf) { return NQ == 2 ? s(q, 0) : kWide ? 448u : 384u + 64u * buf; }
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

// Row r of a V tile in shared memory: zeroed when nobody sees it (its P is 0,
// and 0 x NaN is not 0); of a node's row, infinities and NaN become 0 (the
// epilogue adds them to the rows that see them).  True when there were any.
template <bool kHalf>
__device__ __forceinline__ bool fix_values(uint8_t* tile, int chunks, int r, bool seen, bool node) {
    constexpr uint32_t kExp = kHalf ? 0x7c00u : 0x7f80u;
    if (seen && !node) return false;
    bool bad = false;
#pragma unroll 1
    for (int j = 0; j < chunks * 8; ++j) {
        uint4* at = reinterpret_cast<uint4*>(tile + (j >> 3) * kChunk + r * 128) + ((j ^ r) & 7);
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

// ----------------------------------------------------------------- kernel --
template <int NQ, bool kWide, bool kHalf>
__global__ void __launch_bounds__(128 + 128 * NQ, 1)
tree_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Job J) {
    constexpr int kThreads = 128 + 128 * NQ;
    using Col = Columns<NQ, kWide>;
    constexpr int kBufs = Col::kBufs;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* bs = reinterpret_cast<Bars*>(smem + kTileArea);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Layout: Q (NQ x kc chunks) | K ring | V ring.
    const uint32_t off_k = uint32_t(NQ * J.kc) * kChunk;
    const uint32_t off_v = off_k + uint32_t(J.kring) * kChunk;

    if (tid == 0) {
        for (int s = 0; s < kMaxRing; ++s) {
            mbar_init(&bs->kfull[s], 1); mbar_init(&bs->kempty[s], 1);
            mbar_init(&bs->vfull[s], 1); mbar_init(&bs->vempty[s], 1);
        }
        mbar_init(&bs->qfull, 1);
        mbar_init(&bs->qempty, 1);
        for (int q = 0; q < 2; ++q) {
            mbar_init(&bs->oempty[q], 4);
            for (int s = 0; s < 2; ++s) {
                mbar_init(&bs->sfull[q][s], 1);
                mbar_init(&bs->sempty[q][s], 4);
                mbar_init(&bs->pfull[q][s], 4);
                mbar_init(&bs->odone[q][s], 1);
            }
        }
        mbar_init(&bs->final_mma, 1);
        bs->abort = 0;
        bs->bad_values[0] = bs->bad_values[1] = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        tmem_alloc(&bs->tmem_base, 512);
        tmem_relinquish();
    }
    const Plan<NQ> plan(J);
    find_share<kThreads>(plan, &bs->share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = bs->tmem_base;
    const uint32_t sbase = smem_u32(smem);
    const bool any = int(blockIdx.x) < bs->share.ctas;

    if (any && warp == 0) {
        // ---- each piece's Q, and the K chunks ----
        const int boxes = kKeys / J.box;
        int slot = 0;
        uint32_t lap = 0;
        bool ok = true;
        Walk<Plan<NQ>> w;
        w.start(plan, &bs->share);
        while (ok && w.next(plan)) {
            if (w.piece > 0 && !(ok = warp_wait(&bs->qempty, (w.piece - 1) & 1, bs, J))) break;
            if (lane == 0) {
                mbar_expect_tx(&bs->qfull, uint32_t(NQ * J.kc) * uint32_t(J.tile_rows) * 128u);
                for (int q = 0; q < NQ; ++q)
                    for (int c = 0; c < J.kc; ++c)
                        tma_load_4d(smem + (q * J.kc + c) * kChunk, &qmap, &bs->qfull, c * 64, w.g * J.group,
                                    (w.group * NQ + q) * J.tpt, w.b);
            }
            __syncwarp();
            for (int tile = w.t0; tile < w.t1 && ok; ++tile) {
                int row;
                const int page = box_of(J, w, tile, lane, row);
                for (int c = 0; c < J.kc; ++c) {
                    if (lap && !(ok = warp_wait(&bs->kempty[slot], (lap - 1) & 1, bs, J))) break;
                    if (lane == 0) mbar_expect_tx(&bs->kfull[slot], kChunk);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_4d(smem + off_k + slot * kChunk + lane * J.box * 128, &kmap, &bs->kfull[slot], c * 64, w.g, row, page);
                    if (++slot == J.kring) { slot = 0; ++lap; }
                }
            }
        }
    } else if (any && warp == 3) {
        // ---- the V tiles ----
        const int boxes = kKeys / J.box;
        int stage = 0;
        uint32_t lap = 0;
        bool ok = true;
        Walk<Plan<NQ>> w;
        w.start(plan, &bs->share);
        while (ok && w.next(plan)) {
            for (int tile = w.t0; tile < w.t1; ++tile) {
                int row;
                const int page = box_of(J, w, tile, lane, row);
                if (lap && !(ok = warp_wait(&bs->vempty[stage], (lap - 1) & 1, bs, J))) break;
                if (lane == 0) mbar_expect_tx(&bs->vfull[stage], uint32_t(J.vc) * kChunk);
                __syncwarp();
                if (lane < boxes)
                    for (int c = 0; c < J.vc; ++c)
                        tma_load_4d(smem + off_v + (stage * J.vc + c) * kChunk + lane * J.box * 128, &vmap, &bs->vfull[stage], c * 64,
                                    w.g, row, page);
                if (++stage == J.vstages) { stage = 0; ++lap; }
            }
        }
    } else if (any && warp == 1) {
        if (elect_one()) {
            // ---- MMA issue: S runs one tile ahead of P.V ----
            const uint32_t idesc_s = idesc<kHalf>(128, kKeys, 0, 0);
            // Matrix descriptors (K-major Q and K; MN-major V): the low word moves with the address.
            const uint64_t q_desc = umma_desc_sw128(sbase, 16, 1024), k_desc = umma_desc_sw128(sbase + off_k, 16, 1024);
            const uint64_t v_desc = umma_desc_sw128(sbase + off_v, kChunk, 1024);
            constexpr uint64_t kChunkStep = kChunk >> 4;
            int kslot = 0, stage = 0, s_tile, p_tile = 0, s_count = 0;
            uint32_t klap = 0, vlap = 0;
            bool ok = true;
            Walk<Plan<NQ>> ws, wp;
            ws.start(plan, &bs->share);
            wp = ws;
            bool s_more = ws.next(plan);
            s_tile = ws.t0;
            // The K chunks of a tile are awaited for its first row tile and released by its last.
            auto issue_s = [&](int q) {
                const int buf = kBufs == 2 ? s_count & 1 : 0;
                if (q == 0) {
                    if (s_tile == ws.t0) ok = wait_bar(&bs->qfull, ws.piece & 1, bs, J);
                    if (NQ == 1 && ok && s_count >= kBufs) ok = wait_bar(&bs->sempty[0][buf], ((s_count / kBufs) - 1) & 1, bs, J);
                    if (!ok) return;
                    tc_fence_after();
                }
                const uint32_t d = tbase + Col::s(q, buf);
                for (int c = 0; c < J.kc; ++c) {
                    int slot = kslot + c;
                    uint32_t lap = klap;
                    while (slot >= J.kring) { slot -= J.kring; ++lap; }
                    if (q == 0 && !(ok = wait_bar(&bs->kfull[slot], lap & 1, bs, J))) return;
                    const uint64_t a = q_desc + uint32_t(q * J.kc + c) * kChunkStep, b = k_desc + uint32_t(slot) * kChunkStep;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) umma_bf16(d, a + 2 * kk, b + 2 * kk, idesc_s, (c | kk) != 0);
                    if (q == NQ - 1) umma_commit(&bs->kempty[slot]);
                }
                umma_commit(&bs->sfull[q][buf]);
                if (q == NQ - 1) {
                    if (s_tile == ws.t1 - 1) umma_commit(&bs->qempty);
                    kslot += J.kc;
                    while (kslot >= J.kring) { kslot -= J.kring; ++klap; }
                    ++s_count;
                    if (++s_tile == ws.t1) {
                        s_more = ws.next(plan);
                        s_tile = ws.t0;
                    }
                }
            };
            for (int q = 0; q < NQ && ok; ++q) issue_s(q);
            for (int i = 0; ok; ++i) {
                if (i == 0 || p_tile == wp.t1) {
                    if (!wp.next(plan)) break;
                    p_tile = wp.t0;
                }
                if (NQ == 1 && s_more) issue_s(0);
                const bool first = p_tile == wp.t0;
                const bool s_next = s_more;      // NQ == 2: the S tile issued behind this tile's P.V
                // Every row tile's previous piece has left its O.
                for (int q = 0; q < NQ && ok && first && wp.piece > 0; ++q) ok = wait_bar(&bs->oempty[q], (wp.piece - 1) & 1, bs, J);
                if (ok) ok = wait_bar(&bs->vfull[stage], vlap & 1, bs, J);
                const uint64_t vb = v_desc + uint32_t(stage * J.vc) * kChunkStep;
                for (int q = 0; q < NQ && ok; ++q) {
                    if (!(ok = wait_bar(&bs->pfull[q][i & 1], (i >> 1) & 1, bs, J))) break;
                    tc_fence_after();
                    const uint32_t a = tbase + Col::p(q, kBufs == 2 ? i & 1 : 0);
                    // A V tile's chunks lie side by side: up to four are one MMA of N = 256.
                    for (int c = 0; c < J.vc; c += 4) {
                        const uint32_t d = tbase + Col::o(q) + 64u * c, id = idesc<kHalf>(128, 64 * min(4, J.vc - c), 0, 1);
                        const uint64_t b = vb + uint32_t(c) * kChunkStep;
#pragma unroll
                        for (int ks = 0; ks < kKeys / 16; ++ks)
                            umma_ts(d, a + 8u * ks, b + 128 * ks, id, (!first || ks > 0) ? 1u : 0u);
                    }
                    if (q == NQ - 1) umma_commit(&bs->vempty[stage]);
                    umma_commit(&bs->odone[q][i & 1]);
                    if (NQ == 2 && s_next) issue_s(q);
                }
                if (++stage == J.vstages) { stage = 0; ++vlap; }
                ++p_tile;
            }
            umma_commit(&bs->final_mma);
        }
        __syncwarp();
    } else if (any && warp >= 4) {
        // ---- softmax and epilogue of row tile qt: thread <-> row (TMEM lane) ----
        const int qt = (warp - 4) >> 2, quarter = warp & 3;
        const int r = 32 * quarter + lane;
        const uint32_t lane_addr = uint32_t(32 * quarter) << 16;
        const uint32_t o_base = tbase + lane_addr + Col::o(qt);
        const int jh = r % J.group;
        bool failed = false;
        int i = 0, stage = 0;                                   // tiles done, V stage
        uint32_t vlap = 0;
        Walk<Plan<NQ>> w;
        w.start(plan, &bs->share);
        while (!failed && w.next(plan)) {
            const int t = (w.group * NQ + qt) * J.tpt + r / J.group;
            const bool live = r < J.tile_rows && t < w.s.nodes;
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int32_t* words = J.mask ? J.mask + w.b * J.mask_stride + int64_t(min(t, J.nodes - 1)) * J.words : nullptr;
            float m_run = -INFINITY, l_run = 0.f;
            for (int tile = w.t0; tile < w.t1; ++tile, ++i) {
                const int sb = kBufs == 2 ? i & 1 : 0;
                const bool masked = needs_fix(w.s, tile);
                // Which keys the row sees, 32 to a word.
                uint32_t seen[kKeys / 32];
                if (masked) {
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c)
                        seen[c] = w.s.has_nodes(tile) ? seen_keys(words, J.words, t, w.s.end - w.s.len, tile * kKeys + 32 * c - w.s.len)
                                                      : low_bits(w.s.hi(tile) - 32 * c);
                }
                if (!warp_wait(&bs->sfull[qt][sb], (i / kBufs) & 1, bs, J)) { failed = true; break; }
                tc_fence_after();
                const uint32_t s_addr = tbase + lane_addr + Col::s(qt, sb);
                const uint32_t p_addr = tbase + lane_addr + Col::p(qt, sb);
                // kStep scores at a time, twice over them: the row maximum, then the probabilities
                // (loops, not one straight run: the code of a tile has to come through the
                // instruction cache once per launch).  Wide rows have one S buffer and hold all
                // of a tile's scores, so that the next S may start.
                constexpr int kStep = kWide ? kKeys : 64;
                float v[kStep];
                auto load = [&](int c) {
#pragma unroll
                    for (int e = 0; e < kStep; e += 32) tmem_ld32(s_addr + uint32_t(c + e), v + e);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < kStep; e += 32) {
                            const uint32_t bits = kWide ? seen[e / 32] : e == 0 ? (c ? seen[2] : seen[0]) : (c ? seen[3] : seen[1]);
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (!(bits >> k & 1)) v[e + k] = -INFINITY;
                        }
                    }
                };
                float mx = -INFINITY;
                if (warp_live) {
#pragma unroll 1
                    for (int c = 0; c < kKeys; c += kStep) {
                        load(c);
                        float m2 = -INFINITY;
#pragma unroll
                        for (int e = 0; e < kStep; e += 2) { mx = fmaxf(mx, v[e]); m2 = fmaxf(m2, v[e + 1]); }
                        mx = fmaxf(mx, m2);
                    }
                }
                if constexpr (kWide) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bs->sempty[0][sb]);
                }
                mx *= J.scale_log2;                             // scale > 0
                float alpha = 1.f;
                if (mx > m_run + kLazyLog2 || m_run == -INFINITY) {
                    alpha = mx == -INFINITY || m_run == -INFINITY ? 1.f : exp2f(m_run - mx);
                    m_run = fmaxf(m_run, mx);
                    l_run *= alpha;
                }
                // P(i) takes the buffer of P(i - kBufs); a rescale of O needs P.V(i - 1) done.
                const bool rescale = tile > w.t0 && __any_sync(0xffffffffu, alpha != 1.f);
                const bool fix = qt == 0 && masked;
                const int back = rescale || fix ? 1 : kBufs;
                if (i >= back) {
                    if (!warp_wait(&bs->odone[qt][(i - back) & 1], ((i - back) >> 1) & 1, bs, J)) { failed = true; break; }
                    tc_fence_after();
                }
                if (rescale) {
#pragma unroll 1
                    for (int c = 0; c < 2 * J.vc; ++c) {
                        float o[32];
                        tmem_ld32(o_base + 32u * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= alpha;
                        tmem_st32(o_base + 32u * c, o);
                    }
                    tmem_wait_st();
                }
                if (warp_live) {
                    const float shift = m_run == -INFINITY ? 0.f : m_run;
                    float sum = 0.f, sum2 = 0.f;
#pragma unroll 1
                    for (int c = 0; c < kKeys; c += kStep) {
                        if constexpr (!kWide) load(c);
#pragma unroll
                        for (int e = 0; e < kStep; e += 32) {
                            float packed[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const float p0 = sfu_exp2(fmaf(v[e + 2 * k], J.scale_log2, -shift));
                                const float p1 = sfu_exp2(fmaf(v[e + 2 * k + 1], J.scale_log2, -shift));
                                sum += p0;
                                sum2 += p1;
                                packed[k] = __uint_as_float(pack2<kHalf>(p0, p1));
                            }
                            tmem_st16(p_addr + uint32_t(c + e) / 2, packed);
                        }
                    }
                    l_run += sum + sum2;
                    tmem_wait_st();
                }
                if constexpr (NQ == 1 && !kWide) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bs->sempty[0][sb]);
                }
                if (fix) {
                    // P.V(i - 1) is done, so this tile is the next that lands in its stage.
                    if (!warp_wait(&bs->vfull[stage], vlap & 1, bs, J)) { failed = true; break; }
                    const bool bad = fix_values<kHalf>(smem + off_v + uint32_t(stage * J.vc) * kChunk, J.vc, r, r < w.s.hi(tile),
                                                       tile * kKeys + r >= w.s.len);
                    if (bad) *const_cast<volatile int*>(&bs->bad_values[w.piece & 1]) = w.piece + 1;
                    fence_async_shared();
                }
                if (++stage == J.vstages) { stage = 0; ++vlap; }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bs->pfull[qt][i & 1]);
            }
            if (failed) break;
            // ---- the piece's rows ----
            if (!warp_wait(&bs->odone[qt][(i - 1) & 1], ((i - 1) >> 1) & 1, bs, J)) { failed = true; break; }
            tc_fence_after();
            const bool whole = w.whole();
            const bool bad = *const_cast<volatile int*>(&bs->bad_values[w.piece & 1]) == w.piece + 1;
            const float inv = l_run != 0.f ? 1.f / l_run : 0.f;      // a NaN sum stays NaN
            const float lse2 = l_run != 0.f ? m_run + log2f(l_run) : -INFINITY;
            const int h = w.g * J.group + jh;
            const int rows = NQ * J.tile_rows, slot = 2 * blockIdx.x + (w.piece > 0), row = qt * J.tile_rows + r;
            float4* part = reinterpret_cast<float4*>(J.part_o) + int64_t(slot) * (J.dim_v / 4) * rows + row;
#pragma unroll 1
            for (int c = 0; c < 2 * J.vc; ++c) {
                float o[32];
                if (warp_live) {
                    tmem_ld32(o_base + 32u * c, o);
                    tmem_wait_ld();
                }
                if (live) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] *= inv;
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
                                for (int e = 0; e < 32; ++e) {
                                    const int d = 32 * c + e;
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
                        for (int u = 0; u < 4; ++u) {
                            const int d = 32 * c + 8 * u;
                            if (d < J.dim_v)
                                *reinterpret_cast<uint4*>(dst + d) =
                                    make_uint4(pack2<kHalf>(o[8 * u], o[8 * u + 1]), pack2<kHalf>(o[8 * u + 2], o[8 * u + 3]),
                                               pack2<kHalf>(o[8 * u + 4], o[8 * u + 5]), pack2<kHalf>(o[8 * u + 6], o[8 * u + 7]));
                        }
                    } else {
                        // [slot][4 dims][row]: the rows of a warp side by side.
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            if (32 * c + 4 * u < J.dim_v)
                                part[int64_t(8 * c + u) * rows] = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                    }
                }
                __syncwarp();
            }
            if (live) {
                if (whole) J.lse[(int64_t(w.b) * J.nodes + t) * J.heads + h] = lse2 * kLn2;
                else J.part_lse[slot * rows + row] = lse2;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bs->oempty[qt]);
        }
    }
    __syncthreads();
    grid_launch_dependents();
    if (any) {
        // Nothing of this CTA is in flight when its tensor memory goes: the
        // MMAs (they follow every copy that was waited for), and after a wait
        // that ran out the copies that were not.
        if (tid == 64) mbar_wait(&bs->final_mma, 0, 2000000000ull);
        if (bs->abort && tid == 0) {
            for (int s = 0; s < J.kring; ++s) {
                mbar_wait(&bs->kfull[s], 0, 100000000ull);
                mbar_wait(&bs->kfull[s], 1, 100000000ull);
            }
            for (int s = 0; s < J.vstages; ++s) {
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
        tmem_dealloc(tbase, 512);
    }
}

// Merges the pieces of a segment's rows, and writes the rows that see nothing:
// 32 rows (a lane each) and 64 dims (16 to a warp) of a (sequence, KV head,
// row group) per block.
template <int NQ, bool kHalf>
__global__ void __launch_bounds__(128) combine_kernel(const __grid_constant__ Job J) {
    __shared__ long long scan[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int at = blockIdx.x;
    const int group = at % J.row_groups;
    at /= J.row_groups;
    const int g = at % J.kv_heads, b = at / J.kv_heads;
    const Plan<NQ> plan(J);
    long long total, before;
    sum_units<128>(plan, b, total, before, scan);
    const Seq s = plan.sequence(b);
    int c0 = 0, c1 = 0, slot0 = 0;
    const bool some = group < s.groups && s.tiles > 0;
    if (some) {
        const long long u0 = before + ((long long)g * s.groups + group) * s.tiles;
        const int ctas = share_count(total, J.ctas);
        c0 = share_of(total, u0, ctas);
        c1 = share_of(total, u0 + s.tiles - 1, ctas);
        slot0 = 2 * c0 + (share_begin(total, c0, ctas) != u0 ? 1 : 0);
    }
    if (threadIdx.x == 0 && g == 0 && group == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
        const int len = __ldg(J.lengths + b), nodes = J.nodes_len ? __ldg(J.nodes_len + b) : J.nodes;
        if (len != s.len || nodes != s.nodes || (!J.context_only && s.end != s.len + s.nodes)) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    const int rows = NQ * J.tile_rows, r = blockIdx.y * 32 + lane, d0 = blockIdx.z * 64 + 16 * warp;
    const int t = group * NQ * J.tpt + r / J.group, h = g * J.group + r % J.group;
    const bool live = some && t < s.nodes;
    grid_dependency_wait();
    if (r >= rows || t >= J.nodes || d0 >= J.dim_v || (live && c0 == c1)) return;
    auto slot_of = [&](int c) { return int64_t(c == c0 ? slot0 : 2 * c); };
    float m = -INFINITY, sum = 0.f, shift = 0.f;
    float4 acc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) m = fmaxf(m, J.part_lse[slot_of(c) * rows + r]);
        shift = m == -INFINITY ? 0.f : m;
#pragma unroll 2
        for (int c = c0; c <= c1; ++c) {
            const int64_t slot = slot_of(c);
            const float w = exp2f(J.part_lse[slot * rows + r] - shift);
            const float4* part = reinterpret_cast<const float4*>(J.part_o) + (slot * (J.dim_v / 4) + d0 / 4) * rows + r;
            float4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = d0 + 4 * u < J.dim_v ? part[int64_t(u) * rows] : make_float4(0.f, 0.f, 0.f, 0.f);
            sum += w;
            if (w != 0.f)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    acc[u].x = fmaf(w, x[u].x, acc[u].x); acc[u].y = fmaf(w, x[u].y, acc[u].y);
                    acc[u].z = fmaf(w, x[u].z, acc[u].z); acc[u].w = fmaf(w, x[u].w, acc[u].w);
                }
        }
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    uint16_t* dst = static_cast<uint16_t*>(J.out) + b * J.o_sb + t * J.o_st + h * J.o_sh + d0;
#pragma unroll
    for (int u = 0; u < 4; u += 2)
        if (d0 + 4 * u < J.dim_v)
            *reinterpret_cast<uint4*>(dst + 4 * u) =
                make_uint4(pack2<kHalf>(acc[u].x * inv, acc[u].y * inv), pack2<kHalf>(acc[u].z * inv, acc[u].w * inv),
                           pack2<kHalf>(acc[u + 1].x * inv, acc[u + 1].y * inv), pack2<kHalf>(acc[u + 1].z * inv, acc[u + 1].w * inv));
    if (d0 == 0) J.lse[(int64_t(b) * J.nodes + t) * J.heads + h] = sum != 0.f ? (shift + log2f(sum)) * kLn2 : -INFINITY;
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

template <int NQ, bool kWide, bool kHalf>
int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const Job& J, cudaStream_t stream) {
    auto kernel = tree_attention_kernel<NQ, kWide, kHalf>;
    static bool configured[64] = {};
    const int dev = device_info().device;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes)) != cudaSuccess)
            return fail(SLIMKV_ERR_CUDA, "cudaFuncSetAttribute (tree attention) failed");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    kernel<<<J.ctas, 128 + 128 * NQ, kSmemBytes, stream>>>(qm, km, vm, J);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(J.batch * J.kv_heads * J.row_groups, (NQ * J.tile_rows + 31) / 32, (J.dim_v + 63) / 64);
    cfg.blockDim = dim3(128);
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
    if (int64_t(J.batch) * J.kv_heads * J.row_groups > 0x7fffffffLL)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "tree attention: too many rows in one call");
    J.kc = (a->dim_qk + 63) / 64;
    J.vc = (a->dim_v + 63) / 64;
    J.dim_v = a->dim_v;
    const int slots = int(kTileArea / kChunk) - nq * J.kc;
    J.vstages = std::max(1, slots / 2 / J.vc);
    J.kring = std::min(kMaxRing, slots - J.vstages * J.vc);
    J.context_only = a->context_only;
    J.paged = paged;
    J.cache = cache_view(cache);
    J.capacity = cache_capacity(J.cache);
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
    const bool wide = J.kc > 2 || J.vc > 2, half = a->type == SLIMKV_FP16;
    if (nq == 2) return half ? launch<2, false, true>(qm, km, vm, J, st) : launch<2, false, false>(qm, km, vm, J, st);
    if (wide) return half ? launch<1, true, true>(qm, km, vm, J, st) : launch<1, true, false>(qm, km, vm, J, st);
    return half ? launch<1, false, true>(qm, km, vm, J, st) : launch<1, false, false>(qm, km, vm, J, st);
}
