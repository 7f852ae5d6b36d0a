// Attention weight of each key (C ABI slimkv_key_mass).
//
// For the accepted rows of a step (i < count, each one query per head) and a
// key n of KV head g
//   mass[n] = decay mass[n] + sum_i sum_{h of g} exp(scale q_ih . k_n - lse_ih).
// The log-sum-exps are known, so nothing runs along the keys: keys fill the
// M = 128 side of the tensor core and the rows its N side,
//   S^T [128 keys x rows] = K . Q^T   (tcgen05, fp32 in TMEM),
// a thread owns one key (its TMEM lane) and adds the exponentials of its
// columns in registers (fp32).  No value of another thread is needed, so the
// sum's order is fixed and the update is in place without atomics.
//
// Work: the 128-key tiles of all (sequence, KV head) segments in equal shares,
// one CTA per SM (key_shares.cuh).  More rows than one block of columns (256)
// are taken block by block over the piece's tiles.
// Bound: HBM (each K row read once) with few rows, the products and the
// exponentials with many.  Measured: 16 sequences of 8k latents (320 dims, 1 to 8
// accepted rows of 32 heads) 29 us = 3.0 TB/s; the 256 rows' Q leaves 64 KB for
// the K ring, less than one tile of 80 KB, so loads and products take turns.
// (Two warps to a tile's keys, or shares that count a tile's columns, gained 1
// us here and cost short calls as much.)  One token over 1028 rows 6 us.
//
// Warps: 0 = K loads (TMA), 1 = MMA issue, 2 = TMEM owner, 4-11 = Q rows
// gathered into shared memory, then the sums, 4-7 of a CTA's even tiles and
// 8-11 of its odd ones.  Every wait is bounded.
#include <algorithm>

#include "bounded_wait.cuh"
#include "cache_view.cuh"
#include "host_utils.h"
#include "key_shares.cuh"

namespace slimkv {
namespace {

constexpr int kKeys = 128;
constexpr int kMaxCols = 256;
constexpr uint32_t kChunk = 128 * 128;
constexpr uint32_t kTileArea = 224 * 1024;
constexpr int kMaxRing = 12;
constexpr int kThreads = 384;
constexpr float kLog2e = 1.4426950408889634f;

struct Bars {
    uint64_t kfull[kMaxRing], kempty[kMaxRing];
    uint64_t qfull, sfull[2], sempty[2], final_mma;
    uint32_t tmem_base;
    int abort;
    Share share;
    alignas(16) float lse[kMaxCols];    // lse log2(e) of the block's rows, +inf: gives nothing
};
constexpr uint32_t kSmemBytes = 1024 + kTileArea + uint32_t(sizeof(Bars));
static_assert(kSmemBytes <= 232448, "shared memory budget");

struct Job {
    int batch, nodes, heads, kv_heads, group, ctas;
    int dim, kring, cols;       // ring slots (64-column chunks of 128 keys), columns of a row block
    int context_only, paged, shared_cache, box;
    CacheView cache;
    int64_t capacity;           // rows a sequence may hold (cache and mass)
    const uint16_t* q;
    int64_t q_sb, q_st, q_sh;
    const int32_t *lengths, *rows, *counts;
    const float* lse;
    float* mass;
    int64_t m_sb, m_sh;
    float scale_log2, decay;
    unsigned int* status;
    uint64_t wait_ns;
};

struct Seq {
    int len, count, end;        // old rows, accepted rows, keys with a mass
    int tiles, groups;
};
struct Plan {
    // (None: 33.9 us for 64 sequences of 100..900 rows; one: 28.3; two: 26.3.)
    static constexpr int kPieceUnits = 2;
    const Job& J;
    int batch, kv_heads, ctas;
    __device__ __forceinline__ explicit Plan(const Job& j) : J(j), batch(j.batch), kv_heads(j.kv_heads), ctas(j.ctas) {}
    __device__ __forceinline__ Seq sequence(int b) const {
        Seq s;
        s.count = J.counts ? min(max(__ldg(J.counts + b), 0), J.nodes) : J.nodes;
        const int64_t room = max(J.capacity - (J.context_only ? 0 : s.count), int64_t(0));
        s.len = int(min(int64_t(max(__ldg(J.lengths + b), 0)), room));
        s.end = int(min(int64_t(s.len) + (J.context_only ? 0 : s.count), J.capacity));
        s.tiles = (s.end + kKeys - 1) / kKeys;
        s.groups = 1;
        return s;
    }
};

// 16 bytes global -> shared, or zeros.
__device__ __forceinline__ void copy16(void* dst, const void* src, bool some) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(some ? 16 : 0) : "memory");
}

// kc: 64-column chunks of a K row.
template <int kc, bool kHalf>
__global__ void __launch_bounds__(kThreads, 1)
key_mass_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ Job J) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* bs = reinterpret_cast<Bars*>(smem + kTileArea);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Layout: Q (kc chunks of cols x 64) | K ring.
    const uint32_t q_chunk = uint32_t(J.cols) * 128u;
    const uint32_t off_k = (uint32_t(kc) * q_chunk + 1023u) & ~1023u;

    if (tid == 0) {
        for (int s = 0; s < kMaxRing; ++s) { mbar_init(&bs->kfull[s], 1); mbar_init(&bs->kempty[s], 1); }
        mbar_init(&bs->qfull, 8);
        for (int s = 0; s < 2; ++s) { mbar_init(&bs->sfull[s], 1); mbar_init(&bs->sempty[s], 4); }
        mbar_init(&bs->final_mma, 1);
        bs->abort = 0;
        fence_barrier_init();
    }
    if (tid == 32) tma_prefetch_desc(&kmap);
    if (warp == 2) {
        tmem_alloc(&bs->tmem_base, 512);
        tmem_relinquish();
    }
    const Plan plan(J);
    if (warp == 3) find_share(plan, &bs->share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // All 512 tensor memory columns are this CTA's: addresses begin at column 0.
    const uint32_t sbase = smem_u32(smem);
    const bool any = int(blockIdx.x) < bs->share.ctas;
    auto blocks_of = [&](const Seq& s) { return max(1, (s.count * J.group + J.cols - 1) / J.cols); };
    auto cols_of = [&](const Seq& s, int block) { return min(J.cols, s.count * J.group - block * J.cols); };

    if (any && warp == 0) {
        // ---- K chunks, every row block over the piece's tiles ----
        const int boxes = kKeys / J.box;
        int slot = 0;
        uint32_t lap = 0;
        bool ok = true;
        Walk<Plan> w;
        w.start(plan, &bs->share);
        while (ok && w.next(plan)) {
            const int blocks = blocks_of(w.s);
            for (int block = 0; block < blocks && ok; ++block)
                for (int tile = w.t0; tile < w.t1 && ok; ++tile) {
                    int64_t page = J.shared_cache ? 0 : w.b;
                    int row = tile * kKeys + lane * J.box;
                    if (J.paged && lane < boxes) {
                        const int last = min(tile * kKeys + kKeys, w.s.end) - 1;
                        if (!cache_row(J.cache, w.b, min(row, last / J.box * J.box), page, row))
                            report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
                    }
                    for (int c = 0; c < kc; ++c) {
                        if (lap && !(ok = warp_wait(&bs->kempty[slot], (lap - 1) & 1, bs, J))) break;
                        if (lane == 0) mbar_expect_tx(&bs->kfull[slot], kChunk);
                        __syncwarp();
                        if (lane < boxes)
                            tma_load_4d(smem + off_k + slot * kChunk + lane * J.box * 128, &kmap, &bs->kfull[slot], c * 64, w.g,
                                        row, int(page));
                        if (++slot == J.kring) { slot = 0; ++lap; }
                    }
                }
        }
    } else if (any && warp == 1) {
        // ---- MMA issue: the warp stays converged and one elected thread has the
        // instructions, so that their operands are uniform registers ----
        const uint64_t q_desc = umma_desc_sw128(sbase, 16, 1024), k_desc = umma_desc_sw128(sbase + off_k, 16, 1024);
        const uint32_t q_step = q_chunk >> 4;
        int slot = 0;
        uint32_t lap = 0, buf = 0, s_lap = 0, q_lap = 0;
        bool again = false, ok = true;                      // again: both S buffers have been used
        Walk<Plan> w;
        w.start(plan, &bs->share);
        while (all_lanes(ok && w.next(plan))) {
            const int blocks = blocks_of(w.s);
            for (int block = 0; all_lanes(ok && block < blocks); ++block) {
                const int n = max(16, (cols_of(w.s, block) + 15) & ~15);
                // fp16: both operand formats (bits [7,10) and [10,13)) are 0.
                const uint32_t idesc = umma_idesc_bf16(128, n, 0, 0) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
                ok = ok && wait_bar(&bs->qfull, q_lap, bs, J);
                q_lap ^= 1;
                for (int tile = w.t0; all_lanes(ok && tile < w.t1); ++tile) {
                    if (again) ok = ok && wait_bar(&bs->sempty[buf], s_lap ^ 1, bs, J);
#pragma unroll
                    for (int c = 0; c < kc; ++c) {
                        ok = ok && wait_bar(&bs->kfull[slot], lap, bs, J);
                        if (!all_lanes(ok)) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t a = k_desc + uint32_t(slot) * (kChunk >> 4), b = q_desc + uint32_t(c) * q_step;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) umma_bf16(buf * kMaxCols, a + 2 * kk, b + 2 * kk, idesc, (c | kk) != 0);
                            umma_commit(&bs->kempty[slot]);
                            if (c == kc - 1) umma_commit(&bs->sfull[buf]);
                        }
                        __syncwarp();
                        if (++slot == J.kring) { slot = 0; lap ^= 1; }
                    }
                    if (buf) { s_lap ^= 1; again = true; }
                    buf ^= 1;
                }
            }
        }
        if (elect_one()) umma_commit(&bs->final_mma);
        __syncwarp();
    } else if (any && warp >= 4) {
        // ---- Q rows into shared memory, then a key per thread ----
        const int quarter = warp & 3, turn = (warp >> 2) - 1;
        const uint32_t lane_addr = uint32_t(32 * quarter) << 16;
        int i = 0;                                          // tiles begun before
        bool ok = true;
        Walk<Plan> w;
        w.start(plan, &bs->share);
        // After a wait that ran out the eight warps still meet at every barrier, without work.
        while (w.next(plan)) {
            const int blocks = blocks_of(w.s);
            float* mass = J.mass + w.b * J.m_sb + w.g * J.m_sh;
            for (int block = 0; block < blocks; ++block) {
                // The products of the block before are done: each S was awaited by its warps.
                named_bar(1, 256);
                const int cols = cols_of(w.s, block), padded = max(16, (cols + 15) & ~15);
                // Warp w takes the columns w, w + 8, ...: first a lane for each (row and
                // log-sum-exp, one latency for all), then all lanes for one after the other, 16
                // bytes a lane; zeros past the block's rows.
                {
                    const int col = warp - 4 + 8 * lane, at = block * J.cols + col, row = at / J.group;
                    int r = row;
                    if (J.rows && col < cols) r = __ldg(J.rows + int64_t(w.b) * J.nodes + row);
                    const bool some = col < cols && r >= 0 && r < J.nodes;
                    const int h = w.g * J.group + at - row * J.group;
                    float off = INFINITY;
                    if (some) {
                        off = __ldg(J.lse + (int64_t(w.b) * J.nodes + r) * J.heads + h) * kLog2e;
                    } else if (col < cols) {
                        report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
                    }
                    if (col < padded) bs->lse[col] = off;
                    const int64_t mine = some ? w.b * J.q_sb + r * J.q_st + h * J.q_sh : -1;
#pragma unroll 4
                    for (int l = 0; l < 32; ++l) {
                        const int64_t from = __shfl_sync(0xffffffffu, mine, l);
                        const int c = warp - 4 + 8 * l;
                        if (c >= padded) break;
#pragma unroll
                        for (int u0 = 0; u0 < kc * 8; u0 += 32) {
                            const int u = u0 + lane;
                            const bool live = from >= 0 && u * 8 < J.dim;
                            if (u < kc * 8)
                                copy16(smem + (u >> 3) * q_chunk + c * 128 + (((u & 7) ^ (c & 7)) << 4), J.q + (live ? from + u * 8 : 0), live);
                        }
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_shared();
                named_bar(1, 256);
                if (lane == 0) mbar_arrive(&bs->qfull);
                for (int tile = w.t0; tile < w.t1; ++tile, ++i) {
                    if ((i & 1) != turn || !ok) continue;
                    const int n = tile * kKeys + 32 * quarter + lane;
                    const bool live = n < w.s.end;
                    const float old = !live ? 0.f : block ? mass[n] : n < w.s.len ? J.decay * mass[n] : 0.f;
                    if (!(ok = warp_wait(&bs->sfull[turn], (i >> 1) & 1, bs, J))) continue;
                    tc_fence_after();
                    // The columns of rows that see key n: all for an old key, those of its own
                    // row and the rows behind it for an accepted one.
                    const int first = n < w.s.len ? 0 : (n - w.s.len) * J.group - block * J.cols;
                    const bool whole = __all_sync(0xffffffffu, first <= 0);
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                    for (int c = 0; c < cols; c += 32) {
                        float v[32];
                        tmem_ld32(lane_addr + uint32_t(turn * kMaxCols + c), v);
                        tmem_wait_ld();
                        if (whole && c + 32 <= cols) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 off = *reinterpret_cast<const float4*>(&bs->lse[c + e]);
                                acc[0] += sfu_exp2(fmaf(v[e], J.scale_log2, -off.x));
                                acc[1] += sfu_exp2(fmaf(v[e + 1], J.scale_log2, -off.y));
                                acc[2] += sfu_exp2(fmaf(v[e + 2], J.scale_log2, -off.z));
                                acc[3] += sfu_exp2(fmaf(v[e + 3], J.scale_log2, -off.w));
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float p = sfu_exp2(fmaf(v[e], J.scale_log2, -bs->lse[c + e]));
                                acc[e & 3] += c + e >= first && c + e < cols ? p : 0.f;
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bs->sempty[turn]);
                    if (live) mass[n] = old + ((acc[0] + acc[1]) + (acc[2] + acc[3]));
                }
            }
        }
    }
    __syncthreads();
    if (any) {
        if (tid == 64) mbar_wait(&bs->final_mma, 0, 2000000000ull);
        if (bs->abort && tid == 0)
            for (int s = 0; s < J.kring; ++s) {
                mbar_wait(&bs->kfull[s], 0, 100000000ull);
                mbar_wait(&bs->kfull[s], 1, 100000000ull);
            }
    }
    if (blockIdx.x == 0)
        for (int b = tid; b < J.batch; b += kThreads) {
            const Seq s = plan.sequence(b);
            if (s.len != __ldg(J.lengths + b) || (J.counts && s.count != __ldg(J.counts + b))) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
        }
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(bs->tmem_base, 512);
    }
}

template <int kc, bool kHalf>
int launch(const CUtensorMap& km, const Job& J, cudaStream_t stream) {
    auto kernel = key_mass_kernel<kc, kHalf>;
    static bool configured[64] = {};
    const int dev = device_info().device;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes)) != cudaSuccess)
            return fail(SLIMKV_ERR_CUDA, "cudaFuncSetAttribute (key mass) failed");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    kernel<<<J.ctas, kThreads, kSmemBytes, stream>>>(km, J);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "key mass launch failed: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_key_mass(const slimkv_key_mass_args* a, void* stream) {
    if (!a || !a->q || !a->lengths || !a->lse || !a->mass) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "key mass: null pointer");
    if (a->batch < 1 || a->batch > 4096 || a->nodes < 1 || a->nodes > 1024 || a->heads < 1 || a->kv_heads < 1 ||
        a->heads % a->kv_heads || a->mass_rows < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "key mass: batch in 1..4096, nodes in 1..1024, heads a multiple of kv_heads, mass rows");
    if (a->heads / a->kv_heads > 128) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "key mass: at most 128 query heads per KV head");
    if (a->dim < 8 || a->dim > 320 || a->dim % 8) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "key mass: dims must be multiples of 8 up to 320");
    if (a->type != SLIMKV_BF16 && a->type != SLIMKV_FP16) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "key mass: bf16 or fp16 tensors");
    if (!(a->scale > -INFINITY && a->scale < INFINITY) || !(a->decay > -INFINITY && a->decay < INFINITY))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "key mass: finite scale and decay");
    if (int rc = check_cache(a->cache, a->batch, a->dim, a->dim, 2, false, "key mass")) return rc;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8) return fail(SLIMKV_ERR_ALIGNMENT, "key mass: strides must be multiples of 8 elements");
    if (!aligned16(a->q)) return fail(SLIMKV_ERR_ALIGNMENT, "key mass: 16-byte aligned tensors");
    const slimkv_cache& cache = a->cache;
    const bool paged = cache.table != nullptr;
    if (paged && cache.rows % 8) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "key mass: pages of a multiple of 8 rows");
    Job J{};
    J.box = paged ? std::min(kKeys, cache.rows & -cache.rows) : kKeys;
    J.shared_cache = !paged && cache.k_stride[0] == 0;
    const uint64_t planes = paged ? uint64_t(cache.num_pages) : J.shared_cache ? 1 : uint64_t(a->batch), any = uint64_t(a->dim) * 2;
    CUtensorMap km;
    if (int rc = encode_map_4d(&km, cache.k, a->dim, a->kv_heads, cache.rows, planes,
                               a->kv_heads > 1 ? uint64_t(cache.k_stride[2]) * 2 : any,
                               cache.rows > 1 ? uint64_t(cache.k_stride[1]) * 2 : any,
                               planes > 1 ? uint64_t(cache.k_stride[0]) * 2 : any, J.box))
        return rc;
    J.batch = a->batch;
    J.nodes = a->nodes;
    J.heads = a->heads;
    J.kv_heads = a->kv_heads;
    J.group = a->heads / a->kv_heads;
    J.ctas = device_info().sm_count;
    J.dim = a->dim;
    const int kc = (a->dim + 63) / 64;
    J.cols = std::min(kMaxCols, (a->nodes * J.group + 15) / 16 * 16);
    J.kring = std::min<int>(kMaxRing, (kTileArea - ((uint32_t(kc) * J.cols * 128u + 1023u) & ~1023u)) / kChunk);
    J.context_only = a->context_only;
    J.paged = paged;
    J.cache = cache_view(cache);
    J.capacity = std::min<int64_t>(cache_capacity(J.cache), a->mass_rows);
    if (double(J.batch) * J.kv_heads * double(J.capacity / kKeys + 1 + Plan::kPieceUnits) >= 2147483648.0)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "key mass: too many rows in one call");
    J.q = static_cast<const uint16_t*>(a->q);
    J.q_sb = a->q_stride[0]; J.q_st = a->q_stride[1]; J.q_sh = a->q_stride[2];
    J.lengths = a->lengths;
    J.rows = a->rows;
    J.counts = a->counts;
    J.lse = a->lse;
    J.mass = a->mass;
    J.m_sb = a->mass_stride[0]; J.m_sh = a->mass_stride[1];
    J.scale_log2 = a->scale * kLog2e;
    J.decay = a->decay;
    J.status = status_word();
    J.wait_ns = a->wait_limit_ns ? a->wait_limit_ns : 2000000000ull;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool half = a->type == SLIMKV_FP16;
    switch (kc) {
        case 1: return half ? launch<1, true>(km, J, st) : launch<1, false>(km, J, st);
        case 2: return half ? launch<2, true>(km, J, st) : launch<2, false>(km, J, st);
        case 3: return half ? launch<3, true>(km, J, st) : launch<3, false>(km, J, st);
        case 4: return half ? launch<4, true>(km, J, st) : launch<4, false>(km, J, st);
        default: return half ? launch<5, true>(km, J, st) : launch<5, false>(km, J, st);
    }
}
