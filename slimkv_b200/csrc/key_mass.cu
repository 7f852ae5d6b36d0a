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
// Bound: HBM (each K row read once) up to about 170 rows of 128, then the
// exponentials.
//
// Warps: 0 = K loads (TMA), 1 = MMA issue, 2 = TMEM owner, 4-7 = Q rows
// gathered into shared memory, then the sums.  Every wait is bounded.
#include <algorithm>

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
constexpr int kThreads = 256;
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
    int dim, kc, kring, cols;   // 64-column chunks of a K row, ring slots, columns of a row block
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
// 16 bytes global -> shared, or zeros.
__device__ __forceinline__ void copy16(void* dst, const void* src, bool some) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(some ? 16 : 0) : "memory");
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads, 1)
key_mass_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ Job J) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* bs = reinterpret_cast<Bars*>(smem + kTileArea);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Layout: Q (kc chunks of cols x 64) | K ring.
    const uint32_t q_chunk = uint32_t(J.cols) * 128u;
    const uint32_t off_k = (uint32_t(J.kc) * q_chunk + 1023u) & ~1023u;

    if (tid == 0) {
        for (int s = 0; s < kMaxRing; ++s) { mbar_init(&bs->kfull[s], 1); mbar_init(&bs->kempty[s], 1); }
        mbar_init(&bs->qfull, 4);
        for (int s = 0; s < 2; ++s) { mbar_init(&bs->sfull[s], 1); mbar_init(&bs->sempty[s], 4); }
        mbar_init(&bs->final_mma, 1);
        bs->abort = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        tmem_alloc(&bs->tmem_base, 512);
        tmem_relinquish();
    }
    const Plan plan(J);
    find_share<kThreads>(plan, &bs->share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = bs->tmem_base;
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
                    for (int c = 0; c < J.kc; ++c) {
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
        // ---- MMA issuer ----
        const bool leader = lane == 0;
        int slot = 0, i = 0, q_blocks = 0;
        uint32_t lap = 0;
        bool ok = true;
        Walk<Plan> w;
        w.start(plan, &bs->share);
        while (ok && w.next(plan)) {
            const int blocks = blocks_of(w.s);
            for (int block = 0; block < blocks && ok; ++block, ++q_blocks) {
                const int n = max(16, (cols_of(w.s, block) + 15) & ~15);
                // fp16: both operand formats (bits [7,10) and [10,13)) are 0.
                const uint32_t idesc = umma_idesc_bf16(128, n, 0, 0) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
                ok = warp_wait(&bs->qfull, q_blocks & 1, bs, J);
                for (int tile = w.t0; tile < w.t1 && ok; ++tile, ++i) {
                    const int sb = i & 1;
                    if (i >= 2) ok = warp_wait(&bs->sempty[sb], ((i >> 1) - 1) & 1, bs, J);
                    for (int c = 0; c < J.kc && ok; ++c) {
                        ok = warp_wait(&bs->kfull[slot], lap & 1, bs, J);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            const uint32_t ka = sbase + off_k + slot * kChunk, qa = sbase + c * q_chunk;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                umma_bf16(tbase + sb * kMaxCols, umma_desc_sw128(ka + kk * 32, 16, 1024),
                                          umma_desc_sw128(qa + kk * 32, 16, 1024), idesc, (c | kk) != 0);
                            umma_commit(&bs->kempty[slot]);
                        }
                        __syncwarp();
                        if (++slot == J.kring) { slot = 0; ++lap; }
                    }
                    if (ok && leader) umma_commit(&bs->sfull[sb]);
                    __syncwarp();
                }
            }
        }
        if (leader) umma_commit(&bs->final_mma);
    } else if (any && warp >= 4) {
        // ---- Q rows into shared memory, then a key per thread ----
        const int quarter = warp & 3, st = tid - 128;
        const uint32_t lane_addr = uint32_t(32 * quarter) << 16;
        int i = 0;
        bool failed = false;
        Walk<Plan> w;
        w.start(plan, &bs->share);
        // After a wait that ran out the four warps still meet at every barrier, without work.
        while (w.next(plan)) {
            const int blocks = blocks_of(w.s);
            float* mass = J.mass + w.b * J.m_sb + w.g * J.m_sh;
            for (int block = 0; block < blocks; ++block) {
                // The products of the block before are done (their S was awaited by every thread of the four warps).
                named_bar(1, 128);
                const int cols = cols_of(w.s, block), padded = max(16, (cols + 15) & ~15);
                const int units = J.kc * 8;
                for (int k = st; k < padded * units; k += 128) {
                    const int col = k / units, u = k - col * units;
                    const int at = block * J.cols + col, row = at / J.group;
                    int r = row;
                    if (J.rows && col < cols) r = __ldg(J.rows + int64_t(w.b) * J.nodes + row);
                    const bool some = col < cols && r >= 0 && r < J.nodes && u * 8 < J.dim;
                    const uint16_t* src = some ? J.q + w.b * J.q_sb + r * J.q_st + (w.g * J.group + at % J.group) * J.q_sh + u * 8 : J.q;
                    copy16(smem + (u >> 3) * q_chunk + col * 128 + (((u & 7) ^ (col & 7)) << 4), src, some);
                }
                for (int col = st; col < padded; col += 128) {
                    const int at = block * J.cols + col, row = at / J.group;
                    float off = INFINITY;
                    if (col < cols) {
                        const int r = J.rows ? __ldg(J.rows + int64_t(w.b) * J.nodes + row) : row;
                        if (r >= 0 && r < J.nodes) {
                            const float x = __ldg(J.lse + (int64_t(w.b) * J.nodes + r) * J.heads + w.g * J.group + at % J.group);
                            if (x != -INFINITY) off = x * kLog2e;
                        } else {
                            report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
                        }
                    }
                    bs->lse[col] = off;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_shared();
                named_bar(1, 128);
                if (lane == 0) mbar_arrive(&bs->qfull);
                for (int tile = w.t0; tile < w.t1 && !failed; ++tile, ++i) {
                    const int sb = i & 1;
                    const int n = tile * kKeys + 32 * quarter + lane;
                    const bool live = n < w.s.end;
                    const float old = !live ? 0.f : block ? mass[n] : n < w.s.len ? J.decay * mass[n] : 0.f;
                    if (!warp_wait(&bs->sfull[sb], (i >> 1) & 1, bs, J)) { failed = true; break; }
                    tc_fence_after();
                    // The columns of rows that see key n: all for an old key, those of its own
                    // row and the rows behind it for an accepted one.
                    const int first = n < w.s.len ? 0 : (n - w.s.len) * J.group - block * J.cols;
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    for (int c = 0; c < cols; c += 32) {
                        float v[32];
                        tmem_ld32(tbase + lane_addr + uint32_t(sb * kMaxCols + c), v);
                        tmem_wait_ld();
                        const bool full = __all_sync(0xffffffffu, first <= c) && c + 32 <= cols;
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 off = *reinterpret_cast<const float4*>(&bs->lse[c + e]);
                            float p0 = sfu_exp2(fmaf(v[e], J.scale_log2, -off.x)), p1 = sfu_exp2(fmaf(v[e + 1], J.scale_log2, -off.y));
                            float p2 = sfu_exp2(fmaf(v[e + 2], J.scale_log2, -off.z)), p3 = sfu_exp2(fmaf(v[e + 3], J.scale_log2, -off.w));
                            if (!full) {
                                const int k = c + e;
                                p0 = k >= first && k < cols ? p0 : 0.f;
                                p1 = k + 1 >= first && k + 1 < cols ? p1 : 0.f;
                                p2 = k + 2 >= first && k + 2 < cols ? p2 : 0.f;
                                p3 = k + 3 >= first && k + 3 < cols ? p3 : 0.f;
                            }
                            acc[0] += p0; acc[1] += p1; acc[2] += p2; acc[3] += p3;
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bs->sempty[sb]);
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
        tmem_dealloc(tbase, 512);
    }
}

template <bool kHalf>
int launch(const CUtensorMap& km, const Job& J, cudaStream_t stream) {
    auto kernel = key_mass_kernel<kHalf>;
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
    J.kc = (a->dim + 63) / 64;
    J.cols = std::min(kMaxCols, (a->nodes * J.group + 15) / 16 * 16);
    J.kring = std::min<int>(kMaxRing, (kTileArea - ((uint32_t(J.kc) * J.cols * 128u + 1023u) & ~1023u)) / kChunk);
    J.context_only = a->context_only;
    J.paged = paged;
    J.cache = cache_view(cache);
    J.capacity = std::min<int64_t>(cache_capacity(J.cache), a->mass_rows);
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
    return a->type == SLIMKV_FP16 ? launch<true>(km, J, st) : launch<false>(km, J, st);
}
