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
// tiles) segment: the context rows, then (a tile of their own) the nodes' own
// rows, where each row sees what its ancestor words say.  The units of all
// segments in a row are cut into one equal share per CTA; a share's part of a
// segment is a piece.  A piece that holds a whole segment writes the output;
// the others (at most two per CTA: its first and its last) leave normalised
// fp32 partial rows and their log-sum-exps, which combine_kernel merges.
// Lengths are read on the device; nothing on the host depends on them.
//
// Bound: with few rows per KV head HBM (each K / V row read once); with 128
// rows or more the tensor cores and the exponentials.
//
// One CTA per SM, warps: 0 = Q and K loads (TMA), 3 = V loads, 1 = MMA issue,
// 2 = TMEM owner, 4-7 (and 8-11) = softmax of row tile 0 (1), a thread per
// row.  Every wait is bounded.
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
constexpr int kCombineRows = 16;

struct Bars {
    uint64_t kfull[kMaxRing], kempty[kMaxRing], vfull[kMaxRing], vempty[kMaxRing];
    uint64_t qfull, qempty;
    // [row tile][buffer]
    uint64_t sfull[2][2], sempty[2][2], pfull[2][2], odone[2][2], oempty[2], final_mma;
    uint32_t tmem_base;
    int abort;
    int bad_values;          // 1 + the piece whose node values hold infinities or NaN
    Share share;
};
constexpr uint32_t kSmemBytes = 1024 + kTileArea + uint32_t(sizeof(Bars));
static_assert(kSmemBytes <= 232448, "shared memory budget");

struct Job {
    int batch, nodes, heads, kv_heads, group;
    int tpt, tile_rows;         // nodes of a row tile and its rows (tpt * group <= 128)
    int row_groups;             // groups of NQ row tiles
    int kc, vc, dim_v;          // 64-column chunks of a K / V row
    int kring, vring;
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
    float* part_o;              // [2 ctas][NQ * tile_rows][dim_v]
    float* part_lse;            // [2 ctas][NQ * tile_rows]
    int ctas;
    unsigned int* status;
    uint64_t wait_ns;
};

// ------------------------------------------------------------- schedule --
// What one sequence asks for.
struct Seq {
    int len, nodes;             // context rows, nodes
    int ctx_tiles, tiles;       // key tiles of the context, and with the nodes' own rows
    int tree_row;               // cache row at which the first node tile starts
    int groups;                 // groups of row tiles with live rows
    // First cache row of a key tile and its keys [lo, hi) that any row sees.
    __device__ __forceinline__ int row0(int tile) const {
        return tile < ctx_tiles ? tile * kKeys : tree_row + (tile - ctx_tiles) * kKeys;
    }
    __device__ __forceinline__ int lo(int tile) const { return tile < ctx_tiles ? 0 : min(max(len - row0(tile), 0), kKeys); }
    __device__ __forceinline__ int hi(int tile) const { return min(kKeys, (tile < ctx_tiles ? len : len + nodes) - row0(tile)); }
};
template <int NQ>
struct Plan {
    const Job& J;
    int batch, kv_heads, ctas;
    __device__ __forceinline__ explicit Plan(const Job& j) : J(j), batch(j.batch), kv_heads(j.kv_heads), ctas(j.ctas) {}
    __device__ __forceinline__ Seq sequence(int b) const {
        Seq s;
        const int nodes = J.nodes_len ? min(max(__ldg(J.nodes_len + b), 0), J.nodes) : J.nodes;
        const int64_t room = J.capacity - (J.context_only ? 0 : nodes);
        s.len = int(min(int64_t(max(__ldg(J.lengths + b), 0)), max(room, int64_t(0))));
        s.nodes = nodes;
        s.ctx_tiles = (s.len + kKeys - 1) / kKeys;
        s.tree_row = s.len;
        int tree = 0;
        if (!J.context_only && nodes > 0 && room >= 0) {
            if (J.paged) s.tree_row = s.len / J.box * J.box;     // boxes do not cross pages
            tree = (s.len - s.tree_row + nodes + kKeys - 1) / kKeys;
        }
        s.tiles = s.ctx_tiles + tree;
        s.groups = (nodes + NQ * J.tpt - 1) / (NQ * J.tpt);
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

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Bars* bs, const Job& J) {
    if (*const_cast<volatile int*>(&bs->abort)) return false;
    if (mbar_wait(bar, parity, J.wait_ns)) return true;
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

// Which of 32 nodes from `first` (may be negative) node t sees.
__device__ __forceinline__ uint32_t mask_word(const int32_t* row, int words, int w) {
    return w >= 0 && w < words ? uint32_t(__ldg(row + w)) : 0u;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen_nodes(const int32_t* row, int words, int t, int nodes, int first) {
    uint32_t bits;
    if (row) {
        const int w = first >> 5;               // floor
        bits = __funnelshift_r(mask_word(row, words, w), mask_word(row, words, w + 1), first & 31);
    } else {
        bits = low_bits(t + 1 - first);
    }
    return bits & low_bits(nodes - first) & ~low_bits(-first);
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
        bs->bad_values = 0;
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

    if (any && (warp == 0 || warp == 3)) {
        // ---- producers: warp 0 each piece's Q and K chunks, warp 3 the V chunks ----
        const bool keys = warp == 0;
        const int chunks = keys ? J.kc : J.vc, ring = keys ? J.kring : J.vring;
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
                if (w.piece > 0) ok = warp_wait(&bs->qempty, (w.piece - 1) & 1, bs, J);
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(&bs->qfull, uint32_t(NQ * J.kc) * uint32_t(J.tile_rows) * 128u);
                    for (int q = 0; q < NQ; ++q)
                        for (int c = 0; c < J.kc; ++c)
                            tma_load_4d(smem + (q * J.kc + c) * kChunk, &qmap, &bs->qfull, c * 64, w.g * J.group,
                                        (w.group * NQ + q) * J.tpt, w.b);
                }
                __syncwarp();
            }
            for (int tile = w.t0; tile < w.t1 && ok; ++tile) {
                // This lane's box: rows past the last used one repeat its box (they are masked).
                int64_t page = J.shared_cache ? 0 : w.b;
                int row = w.s.row0(tile) + lane * J.box;
                if (J.paged && lane < boxes) {
                    const int last = w.s.row0(tile) + w.s.hi(tile) - 1;
                    if (!cache_row(J.cache, w.b, min(row, last / J.box * J.box), page, row) && keys)
                        report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
                }
                for (int c = 0; c < chunks; ++c) {
                    if (lap && !(ok = warp_wait(&empty[slot], (lap - 1) & 1, bs, J))) break;
                    if (lane == 0) mbar_expect_tx(&full[slot], kChunk);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_4d(dst + slot * kChunk + lane * J.box * 128, map, &full[slot], c * 64, w.g, row, int(page));
                    if (++slot == ring) { slot = 0; ++lap; }
                }
            }
        }
    } else if (any && warp == 1) {
        // ---- MMA issuer ----
        const bool leader = lane == 0;
        const uint32_t idesc_s = idesc<kHalf>(128, kKeys, 0, 0);
        const uint32_t idesc_o = idesc<kHalf>(128, 64, 0, 1);
        int kslot = 0, vslot = 0;
        uint32_t klap = 0, vlap = 0;
        bool ok = true;
        Walk<Plan<NQ>> ws, wp;                     // S runs one tile ahead of P.V
        ws.start(plan, &bs->share);
        wp.start(plan, &bs->share);
        int s_tile = 0, p_tile = 0;          // next tile of the piece each is in
        int s_count = 0;                     // S tiles begun before
        bool s_more = ws.next(plan);
        s_tile = ws.t0;
        // The K chunks of S tile `s_count` are awaited by its first row tile and released by its last.
        auto issue_s = [&](int q) {
            if (q == 0) {
                if (s_tile == ws.t0) ok = warp_wait(&bs->qfull, ws.piece & 1, bs, J);
                const int sb = s_count % kBufs;
                if (NQ == 1 && ok && s_count >= kBufs) ok = warp_wait(&bs->sempty[0][sb], ((s_count / kBufs) - 1) & 1, bs, J);
                if (!ok) return;
            }
            tc_fence_after();
            for (int c = 0; c < J.kc && ok; ++c) {
                int slot = kslot + c;
                uint32_t lap = klap;
                while (slot >= J.kring) { slot -= J.kring; ++lap; }
                if (q == 0) {
                    ok = warp_wait(&bs->kfull[slot], lap & 1, bs, J);
                    if (!ok) return;
                    tc_fence_after();
                }
                if (leader) {
                    const uint32_t ka = sbase + off_k + slot * kChunk;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_bf16(tbase + Col::s(q, s_count % kBufs),
                                  umma_desc_sw128(sbase + (q * J.kc + c) * kChunk + kk * 32, 16, 1024),
                                  umma_desc_sw128(ka + kk * 32, 16, 1024), idesc_s, (c | kk) != 0);
                    if (q == NQ - 1) umma_commit(&bs->kempty[slot]);
                }
                __syncwarp();
            }
            if (leader) umma_commit(&bs->sfull[q][s_count % kBufs]);
            if (q == NQ - 1) {
                if (leader && s_tile == ws.t1 - 1) umma_commit(&bs->qempty);
                kslot += J.kc;
                while (kslot >= J.kring) { kslot -= J.kring; ++klap; }
                ++s_count;
                if (++s_tile == ws.t1) {
                    s_more = ws.next(plan);
                    s_tile = ws.t0;
                }
            }
            __syncwarp();
        };
        for (int q = 0; q < NQ && ok; ++q) issue_s(q);
        for (int i = 0; ok; ++i) {
            if (i == 0 || p_tile == wp.t1) {
                if (!wp.next(plan)) break;
                p_tile = wp.t0;
            }
            if (NQ == 1 && s_more) issue_s(0);
            const bool first = p_tile == wp.t0;
            const int lo = wp.s.lo(p_tile), hi = wp.s.hi(p_tile);
            const bool own_rows = p_tile >= wp.s.ctx_tiles;
            const bool s_next = s_more;      // NQ == 2: the S tile issued behind this tile's P.V
            // Every row tile's previous piece has left its O (and bad_values).
            for (int q = 0; q < NQ && ok && first && wp.piece > 0; ++q) ok = warp_wait(&bs->oempty[q], (wp.piece - 1) & 1, bs, J);
            for (int q = 0; q < NQ && ok; ++q) {
                ok = warp_wait(&bs->pfull[q][i & 1], (i >> 1) & 1, bs, J);
                if (!ok) break;
                tc_fence_after();
                for (int c = 0; c < J.vc && ok; ++c) {
                    int slot = vslot + c;
                    uint32_t lap = vlap;
                    while (slot >= J.vring) { slot -= J.vring; ++lap; }
                    if (q == 0) {
                        ok = warp_wait(&bs->vfull[slot], lap & 1, bs, J);
                        if (!ok) break;
                        if (lo > 0 || hi < kKeys || own_rows) {
                            // Rows nobody sees are zeroed (their P is 0, and 0 x NaN is not), and so are
                            // infinities and NaN among the nodes' values: the epilogue adds those to the
                            // rows that see them.
                            uint4* rows = reinterpret_cast<uint4*>(smem + off_v + slot * kChunk);
                            bool bad = false;
                            for (int j = lane; j < kKeys * 8; j += 32) {
                                const int r = j >> 3;
                                if (r < lo || r >= hi) {
                                    rows[j] = make_uint4(0, 0, 0, 0);
                                } else if (own_rows) {
                                    constexpr uint32_t kExp = kHalf ? 0x7c00u : 0x7f80u;
                                    uint4 v = rows[j];
                                    uint32_t* x = &v.x;
                                    bool hit = false;
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        if ((x[e] & kExp) == kExp) { x[e] &= 0xffff0000u; hit = true; }
                                        if ((x[e] >> 16 & kExp) == kExp) { x[e] &= 0xffffu; hit = true; }
                                    }
                                    if (hit) { rows[j] = v; bad = true; }
                                }
                            }
                            if (__any_sync(0xffffffffu, bad) && leader)
                                *const_cast<volatile int*>(&bs->bad_values) = wp.piece + 1;
                            __threadfence_block();
                            fence_async_shared();
                            __syncwarp();
                        }
                        tc_fence_after();
                    }
                    if (leader) {
                        const uint32_t va = sbase + off_v + slot * kChunk;
#pragma unroll
                        for (int ks = 0; ks < kKeys / 16; ++ks)
                            umma_ts(tbase + Col::o(q) + 64u * c, tbase + Col::p(q, i % kBufs) + 8u * ks,
                                    umma_desc_sw128(va + ks * 2048, kChunk, 1024), idesc_o, (!first || ks > 0) ? 1u : 0u);
                        if (q == NQ - 1) umma_commit(&bs->vempty[slot]);
                    }
                    __syncwarp();
                }
                if (ok && leader) umma_commit(&bs->odone[q][i & 1]);
                __syncwarp();
                if (NQ == 2 && ok && s_next) issue_s(q);
            }
            vslot += J.vc;
            while (vslot >= J.vring) { vslot -= J.vring; ++vlap; }
            ++p_tile;
        }
        if (leader) umma_commit(&bs->final_mma);
    } else if (any && warp >= 4) {
        // ---- softmax and epilogue of row tile qt: thread <-> row (TMEM lane) ----
        const int qt = (warp - 4) >> 2, quarter = warp & 3;
        const int r = 32 * quarter + lane;
        const uint32_t lane_addr = uint32_t(32 * quarter) << 16;
        const uint32_t o_base = tbase + lane_addr + Col::o(qt);
        const int jh = r % J.group;
        bool failed = false;
        int i = 0;                                              // tiles done
        Walk<Plan<NQ>> w;
        w.start(plan, &bs->share);
        while (!failed && w.next(plan)) {
            const int t = (w.group * NQ + qt) * J.tpt + r / J.group;
            const bool live = r < J.tile_rows && t < w.s.nodes;
            const bool warp_live = __any_sync(0xffffffffu, live);
            const int32_t* words = J.mask ? J.mask + w.b * J.mask_stride + int64_t(min(t, J.nodes - 1)) * J.words : nullptr;
            float m_run = -INFINITY, l_run = 0.f;
            for (int tile = w.t0; tile < w.t1; ++tile, ++i) {
                const int sb = i % kBufs;
                if (!warp_wait(&bs->sfull[qt][sb], (i / kBufs) & 1, bs, J)) { failed = true; break; }
                tc_fence_after();
                const uint32_t s_addr = tbase + lane_addr + Col::s(qt, sb);
                const uint32_t p_addr = tbase + lane_addr + Col::p(qt, sb);
                const int row0 = w.s.row0(tile), hi = w.s.hi(tile);
                const bool own_rows = tile >= w.s.ctx_tiles;
                auto seen = [&](int c) -> uint32_t {            // of the keys 32c .. 32c + 31
                    return own_rows ? seen_nodes(words, J.words, t, w.s.nodes, row0 + 32 * c - w.s.len) : low_bits(hi - 32 * c);
                };
                const bool masked = own_rows || hi < kKeys;
                float v[NQ == 1 ? kKeys : 32];
                float mx = -INFINITY;
                if (warp_live) {
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        float* x = NQ == 1 ? v + 32 * c : v;
                        tmem_ld32(s_addr + 32u * c, x);
                        if (NQ != 1 || c == kKeys / 32 - 1) tmem_wait_ld();
                        if constexpr (NQ != 1) {
                            if (masked) {
                                const uint32_t bits = seen(c);
#pragma unroll
                                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, bits >> e & 1 ? x[e] : -INFINITY);
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e) mx = fmaxf(mx, x[e]);
                            }
                        }
                    }
                }
                if constexpr (NQ == 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bs->sempty[0][sb]);
                    if (warp_live) {
                        if (masked) {
#pragma unroll
                            for (int c = 0; c < kKeys / 32; ++c) {
                                const uint32_t bits = seen(c);
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (!(bits >> e & 1)) v[(NQ == 1 ? 32 * c : 0) + e] = -INFINITY;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < (NQ == 1 ? kKeys : 32); ++e) mx = fmaxf(mx, v[e]);
                    }
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
                const int back = rescale ? 1 : kBufs;
                if (i >= back) {
                    if (!warp_wait(&bs->odone[qt][(i - back) & 1], ((i - back) >> 1) & 1, bs, J)) { failed = true; break; }
                    tc_fence_after();
                }
                if (rescale) {
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
                    float sum = 0.f;
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        float* x = NQ == 1 ? v + 32 * c : v;
                        if constexpr (NQ != 1) {
                            tmem_ld32(s_addr + 32u * c, x);
                            tmem_wait_ld();
                            if (masked) {
                                const uint32_t bits = seen(c);
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (!(bits >> e & 1)) x[e] = -INFINITY;
                            }
                        }
                        float packed[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float p0 = sfu_exp2(fmaf(x[2 * e], J.scale_log2, -shift));
                            const float p1 = sfu_exp2(fmaf(x[2 * e + 1], J.scale_log2, -shift));
                            sum += p0 + p1;
                            packed[e] = __uint_as_float(pack2<kHalf>(p0, p1));
                        }
                        tmem_st16(p_addr + 16u * c, packed);
                    }
                    l_run += sum;
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bs->pfull[qt][i & 1]);
            }
            if (failed) break;
            // ---- the piece's rows ----
            if (!warp_wait(&bs->odone[qt][(i - 1) & 1], ((i - 1) >> 1) & 1, bs, J)) { failed = true; break; }
            tc_fence_after();
            const bool whole = w.whole();
            const bool bad = *const_cast<volatile int*>(&bs->bad_values) == w.piece + 1;
            const float inv = l_run != 0.f ? 1.f / l_run : 0.f;      // a NaN sum stays NaN
            const float lse2 = l_run != 0.f ? m_run + log2f(l_run) : -INFINITY;
            const int h = w.g * J.group + jh;
            const int64_t slot_row = int64_t(2 * blockIdx.x + (w.piece > 0)) * (NQ * J.tile_rows) + qt * J.tile_rows + r;
            for (int c = 0; c < 2 * J.vc; ++c) {
                float o[32];
                if (warp_live) {
                    tmem_ld32(o_base + 32u * c, o);
                    tmem_wait_ld();
                }
                if (live) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] *= inv;
                    if (bad && w.t1 > w.s.ctx_tiles) {
                        // Infinities and NaN of the nodes' values, for the rows that see them.
                        for (int n0 = 0; n0 < w.s.nodes; n0 += 32) {
                            uint32_t bits = seen_nodes(words, J.words, t, w.s.nodes, n0);
                            for (; bits; bits &= bits - 1) {
                                const int row = w.s.len + n0 + __ffs(int(bits)) - 1;
                                if (row < w.s.row0(max(w.t0, w.s.ctx_tiles)) || row >= w.s.row0(w.t1 - 1) + kKeys) continue;
                                int64_t page = J.shared_cache ? 0 : w.b;
                                int at = row;
                                if (J.paged) cache_row(J.cache, w.b, row, page, at);
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
                        float* dst = J.part_o + slot_row * J.dim_v;
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            const int d = 32 * c + 4 * u;
                            if (d < J.dim_v) *reinterpret_cast<float4*>(dst + d) = make_float4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
                        }
                    }
                }
                __syncwarp();
            }
            if (live) {
                if (whole) J.lse[(int64_t(w.b) * J.nodes + t) * J.heads + h] = lse2 * kLn2;
                else J.part_lse[slot_row] = lse2;
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
            for (int s = 0; s < J.vring; ++s) {
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
// kCombineRows rows of a (sequence, KV head, row group) per block, a warp per
// row at a time.
template <int NQ, bool kHalf>
__global__ void __launch_bounds__(128) combine_kernel(const __grid_constant__ Job J) {
    __shared__ long long scan[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = blockIdx.x;
    const int group = s % J.row_groups;
    s /= J.row_groups;
    const int g = s % J.kv_heads, b = s / J.kv_heads;
    const Plan<NQ> plan(J);
    long long total, before;
    sum_units<128>(plan, b, total, before, scan);
    const Seq q = plan.sequence(b);
    int c0 = 0, c1 = 0, slot0 = 0;
    const bool some = group < q.groups && q.tiles > 0;
    if (some) {
        const long long u0 = before + ((long long)g * q.groups + group) * q.tiles;
        const int ctas = share_count(total, J.ctas);
        c0 = share_of(total, u0, ctas);
        c1 = share_of(total, u0 + q.tiles - 1, ctas);
        slot0 = 2 * c0 + (share_begin(total, c0, ctas) != u0 ? 1 : 0);
    }
    if (threadIdx.x == 0 && g == 0 && group == 0 && blockIdx.y == 0) {
        const int len = __ldg(J.lengths + b), nodes = J.nodes_len ? __ldg(J.nodes_len + b) : J.nodes;
        if (len != q.len || nodes != q.nodes) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    grid_dependency_wait();
    const int rows = NQ * J.tile_rows;
    for (int k = warp; k < kCombineRows; k += 4) {
        const int r = blockIdx.y * kCombineRows + k;
        if (r >= rows) break;
        const int t = group * NQ * J.tpt + r / J.group, h = g * J.group + r % J.group;
        if (t >= J.nodes) break;
        const bool live = some && t < q.nodes;
        if (live && c0 == c1) continue;
        uint16_t* dst = static_cast<uint16_t*>(J.out) + b * J.o_sb + t * J.o_st + h * J.o_sh;
        float* lse = J.lse + (int64_t(b) * J.nodes + t) * J.heads + h;
        if (!live) {
            for (int d = 8 * lane; d < J.dim_v; d += 256) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
            if (lane == 0) *lse = -INFINITY;
            continue;
        }
        auto row_of = [&](int c) { return int64_t(c == c0 ? slot0 : 2 * c) * rows + r; };
        float m = -INFINITY;
        for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, J.part_lse[row_of(c)]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float shift = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
        for (int c = c0 + lane; c <= c1; c += 32) sum += exp2f(J.part_lse[row_of(c)] - shift);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        if (lane == 0) *lse = sum != 0.f ? (shift + log2f(sum)) * kLn2 : -INFINITY;
        for (int d = 4 * lane; d < J.dim_v; d += 128) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = c0; c <= c1; ++c) {
                const int64_t row = row_of(c);
                const float w = exp2f(J.part_lse[row] - shift);
                if (w == 0.f) continue;
                const float4 x = *reinterpret_cast<const float4*>(J.part_o + row * J.dim_v + d);
                acc.x = fmaf(w, x.x, acc.x); acc.y = fmaf(w, x.y, acc.y);
                acc.z = fmaf(w, x.z, acc.z); acc.w = fmaf(w, x.w, acc.w);
            }
            *reinterpret_cast<uint2*>(dst + d) = make_uint2(pack2<kHalf>(acc.x * inv, acc.y * inv), pack2<kHalf>(acc.z * inv, acc.w * inv));
        }
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
    cfg.gridDim = dim3(J.batch * J.kv_heads * J.row_groups, (NQ * J.tile_rows + kCombineRows - 1) / kCombineRows);
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
    J.kring = std::min(kMaxRing, slots / 2);
    J.vring = std::min(kMaxRing, slots - J.kring);
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
