// Attention weight of each key of a 4-bit cache (C ABI slimkv_cache4_key_mass).
//
// For the accepted rows of a step (i < count, each one query per head) and a
// key n of KV head g
//   mass[n] = decay mass[n] + sum_i sum_{h of g} exp(scale q_ih . k_n - lse_ih).
// As in the attention over these rows a warp takes 16 keys and turns their codes
// into operands in its registers, once for up to 64 query rows, whose operands
// lie in shared memory; a key's sum over rows ends in two shuffles of one warp,
// so its order is fixed and the update is in place without atomics.
//
// Work: the 64-key tiles of all (sequence, KV head) segments in equal shares
// (key_shares.cuh), a quarter of each tile to a warp with its own ring of TMA
// loads.  More than 64 rows are taken block by block over the piece's tiles.
// Bound: instructions and their latency (57 % of the cycles issue, at a third of
// HBM's rate).  Measured in a graph (bf16): 1 to 5 accepted rows of 32 heads for 16
// sequences of 8k keys (8 KV heads of 128 dims) 48 us = 1.9 TB/s, one row over 1028
// keys 6 us.  Against the 16-bit keys' kernel (tcgen05), every row accepted: 5
// rows of that shape 54 us and 53; 8 rows (256 queries of a KV head) over 16 x 8k
// latents of 320 dims 137 us and 31: it saves memory, and time only for few rows.
#include <algorithm>
#include <type_traits>

#include "bounded_wait.cuh"
#include "cache4.cuh"
#include "cache_view.cuh"
#include "host_utils.h"
#include "key_shares.cuh"

namespace slimkv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlab = 16;                        // keys of a warp's step
constexpr int kKeys = kSlab * kWarps;            // keys of a tile
constexpr int kTiles = 8;                        // row tiles (8 rows) of a block
constexpr int kBlockRows = 8 * kTiles;
constexpr int kMaxRows = 2048;                   // that a key tile's weight counts
constexpr float kLog2e = 1.4426950408889634f;
template <int G>
constexpr int kStages = G <= 6 ? 6 : 3;
template <int G>
constexpr int kBlocks = G <= 4 ? 4 : G <= 6 ? 3 : 2;

struct Job {
    int batch, nodes, heads, kv_heads, group, ctas;
    int kg, k_pitch;
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
    int weight;                 // units of a key tile
    int tiles, groups;          // units of the keys
};
struct Plan {
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
        // A key tile counts as one unit for every four row tiles.  (16 sequences of 32 to 256 rows over
        // 8k latents: 111 us without weights, 104 with one more for each row tile, which costs 1 to 5
        // rows of 4 heads 2 us of 47: their time is not the products'.)
        s.weight = (min(s.count * J.group, kMaxRows) + 8 * 4 - 1) / (8 * 4) + (s.count == 0);
        s.tiles = (s.end + kKeys - 1) / kKeys * s.weight;
        s.groups = 1;
        return s;
    }
};

template <int G>
struct Bars {
    uint64_t full[kWarps][kStages<G>];
    int abort;
    Share share;
    alignas(8) float lse[kBlockRows];   // lse log2(e) of the block's rows, +inf: gives nothing
};
template <int G>
uint32_t smem_bytes(int k_pitch) {
    return uint32_t(kWarps * kStages<G> * kSlab * k_pitch) + 512 + uint32_t(kTiles) * G * 512 + uint32_t(sizeof(Bars<G>));
}

template <int G, bool kHalf, bool kExact>
__global__ void __launch_bounds__(kThreads, kBlocks<G>)
cache4_mass_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ Job J) {
    constexpr int kRing = kStages<G>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 127) {                  // (TMA writes at multiples of 128 bytes)
        report(J.status, SLIMKV_DEVICE_MISALIGNED);
        return;
    }
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const RowShape<G, kExact> shape{J.kg};
    const uint32_t pitch = uint32_t(shape.pitch()), stage_bytes = kSlab * pitch, area = uint32_t(kWarps * kRing) * stage_bytes + 512u;
    uint8_t* ring = smem + uint32_t(warp * kRing) * stage_bytes;
    uint4* q_shared = reinterpret_cast<uint4*>(smem + area);
    Bars<G>* bs = reinterpret_cast<Bars<G>*>(smem + area + uint32_t(kTiles) * G * 512u);

    if (tid < kWarps * kRing) mbar_init(&bs->full[tid / kRing][tid % kRing], 1);
    if (tid == 0) bs->abort = 0;
    if (tid < 32) fence_barrier_init();
    if (tid == 32) tma_prefetch_desc(&kmap);
    const Plan plan(J);
    if (warp == 0) find_share(plan, &bs->share);
    if (blockIdx.x == 0)
        for (int b = tid; b < J.batch; b += kThreads) {
            const Seq s = plan.sequence(b);
            if (s.len != __ldg(J.lengths + b) || (J.counts && s.count != __ldg(J.counts + b))) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
        }
    __syncthreads();
    if (int(blockIdx.x) >= bs->share.ctas) return;

    const typename Pair<kHalf>::Constants constants;
    const int boxes = kSlab / J.box;
    int stage = 0;                               // of the next slab to be used
    uint32_t lap = 0;
    uint32_t pending = 0;                        // stages with a load under way
    bool ok = true;
    Walk<Plan> w;
    w.start(plan, &bs->share);
    while (w.next(plan)) {
        // The key tiles whose first unit is in the piece.
        const int k0 = (w.t0 + w.s.weight - 1) / w.s.weight, k1 = (w.t1 + w.s.weight - 1) / w.s.weight;
        if (k0 == k1) continue;                  // (all warps)
        const int first_key = k0 * kKeys + warp * kSlab;
        const int slabs = max(0, min(k1 - k0, (w.s.end - first_key + kKeys - 1) / kKeys));
        auto locate = [&](int slab, int& row) {
            row = first_key + slab * kKeys + lane * J.box;
            if (!J.paged) return J.shared_cache ? 0 : w.b;
            int64_t page = 0;
            if (lane < boxes && slab < slabs) {
                if (!cache_row(J.cache, w.b, min(row, (w.s.end - 1) & -J.box), page, row)) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
            }
            return int(page);
        };
        auto issue = [&](int st, int page, int row) {
            uint64_t* bar = &bs->full[warp][st];
            // One elected thread has the copies: their operands are uniform registers.
            for (int box = 0; box < boxes; ++box) {
                const int p = __shfl_sync(0xffffffffu, page, box), r = __shfl_sync(0xffffffffu, row, box);
                if (elect_one()) {
                    if (box == 0) mbar_expect_tx(bar, stage_bytes);
                    tma_load_4d(ring + uint32_t(st) * stage_bytes + uint32_t(box * J.box) * pitch, &kmap, bar, 0, w.g, r, p);
                }
            }
            pending |= 1u << st;
        };
        float* mass = J.mass + w.b * J.m_sb + w.g * J.m_sh;
        const int rows = w.s.count * J.group;
        // (No rows: one block of none, for the decay.)
        for (int row0 = 0; row0 == 0 || row0 < rows; row0 += kBlockRows) {
            if (ok) {
                int page[kRing], row[kRing];
#pragma unroll
                for (int s = 0; s < kRing; ++s) page[s] = locate(s, row[s]);
#pragma unroll
                for (int s = 0; s < kRing; ++s)
                    if (s < slabs) issue((stage + s) % kRing, page[s], row[s]);
            }
            // ---- the block's Q operands and log-sum-exps ----
            __syncthreads();                     // (those of the block before have been used)
            const int tiles = min(kTiles, (rows - row0 + 7) / 8);
            auto source = [&](int r, bool& some, int& node, int& h) {
                const int i = r / J.group;
                h = w.g * J.group + r - i * J.group;
                node = r >= rows ? -1 : J.rows ? __ldg(J.rows + int64_t(w.b) * J.nodes + i) : i;
                some = node >= 0 && node < J.nodes;
            };
            for (int i = warp; i < tiles * G; i += kWarps) {
                const int d = KeyWords<G>::dim(i % G, t);
                bool some;
                int node, h;
                source(row0 + i / G * 8 + g, some, node, h);
                uint4 x = make_uint4(0, 0, 0, 0);
                if (some && shape.has(d))
                    x = __ldg(reinterpret_cast<const uint4*>(J.q + w.b * J.q_sb + node * J.q_st + h * J.q_sh + d));
                q_shared[i * 32 + lane] = x;
            }
            if (tid < kBlockRows) {
                bool some;
                int node, h;
                source(row0 + tid, some, node, h);
                bs->lse[tid] = some ? __ldg(J.lse + (int64_t(w.b) * J.nodes + node) * J.heads + h) * kLog2e : INFINITY;
                if (!some && row0 + tid < rows) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
            }
            __syncthreads();

            // Lane column 0 has the key g of a slab, column 1 the key g + 8; their old masses are on
            // their way a slab ahead (16 sequences of 8k keys took 55.5 us without, 48 with it).
            auto old_mass = [&](int i) {
                const int n = first_key + i * kKeys + g + 8 * t;
                if (t > 1 || i >= slabs || n >= w.s.end) return 0.f;
                return row0 || n < w.s.len ? mass[n] : 0.f;
            };
            float next_old = old_mass(0);
            for (int i = 0; i < slabs && ok; ++i) {
                const int key0 = first_key + i * kKeys;
                int next_row;
                const int next_page = locate(i + kRing, next_row);
                const int n = key0 + g + 8 * t;
                const bool live = t < 2 && n < w.s.end;
                const float old = row0 ? next_old : J.decay * next_old;
                next_old = old_mass(i + 1);
                if (!(ok = warp_wait(&bs->full[warp][stage], lap, bs, J))) break;
                pending &= ~(1u << stage);
                const uint8_t* k0 = ring + uint32_t(stage) * stage_bytes + uint32_t(g) * pitch;
                // First of the block's rows that see the keys g and g + 8: all see an old key, an
                // accepted one its own row and those behind it.
                const int first0 = key0 + g < w.s.len ? 0 : (key0 + g - w.s.len) * J.group - row0;
                const int first1 = key0 + g + 8 < w.s.len ? 0 : (key0 + g + 8 - w.s.len) * J.group - row0;
                float acc0 = 0.f, acc1 = 0.f;
                auto run = [&](auto count) {
                    constexpr int NT = decltype(count)::value;
                    float s[NT][4];
#pragma unroll
                    for (int m = 0; m < NT; ++m) s[m][0] = s[m][1] = s[m][2] = s[m][3] = 0.f;
                    key_products<G, NT, kHalf>(s, k0, shape, t, constants, [&](int m, int j) { return q_shared[(m * G + j) * 32 + lane]; });
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        const int r = 8 * m + 2 * t;
                        const float2 off = *reinterpret_cast<const float2*>(&bs->lse[r]);
                        const float p0 = sfu_exp2(fmaf(s[m][0], J.scale_log2, -off.x)), p1 = sfu_exp2(fmaf(s[m][1], J.scale_log2, -off.y));
                        const float p2 = sfu_exp2(fmaf(s[m][2], J.scale_log2, -off.x)), p3 = sfu_exp2(fmaf(s[m][3], J.scale_log2, -off.y));
                        acc0 += (r >= first0 && row0 + r < rows ? p0 : 0.f) + (r + 1 >= first0 && row0 + r + 1 < rows ? p1 : 0.f);
                        acc1 += (r >= first1 && row0 + r < rows ? p2 : 0.f) + (r + 1 >= first1 && row0 + r + 1 < rows ? p3 : 0.f);
                    }
                };
                if (tiles == 1) run(std::integral_constant<int, 1>());
                else if (tiles == 2) run(std::integral_constant<int, 2>());
                else if (tiles == 3) run(std::integral_constant<int, 3>());
                else if (tiles == 4) run(std::integral_constant<int, 4>());
                else if (tiles <= 6) run(std::integral_constant<int, 6>());
                else if (tiles > 0) run(std::integral_constant<int, kTiles>());
#pragma unroll
                for (int k = 1; k < 4; k <<= 1) {
                    acc0 += __shfl_xor_sync(0xffffffffu, acc0, k);
                    acc1 += __shfl_xor_sync(0xffffffffu, acc1, k);
                }
                if (live) mass[n] = old + (t ? acc1 : acc0);
                __syncwarp();
                if (i + kRing < slabs) issue(stage, next_page, next_row);
                if (++stage == kRing) { stage = 0; lap ^= 1; }
            }
        }
    }
    // After a wait that ran out copies may still be under way.
    if (bs->abort && lane == 0)
        for (int s = 0; s < kRing; ++s)
            if (pending >> s & 1) {
                mbar_wait(&bs->full[warp][s], 0, 100000000ull);
                mbar_wait(&bs->full[warp][s], 1, 100000000ull);
            }
}

template <int G, bool kHalf, bool kExact>
int launch(const CUtensorMap& km, const Job& J, cudaStream_t stream) {
    auto kernel = cache4_mass_kernel<G, kHalf, kExact>;
    static bool configured[64] = {};
    const int dev = device_info().device;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_bytes<G>(row4_bytes(G * kGroupDims)))) != cudaSuccess)
            return fail(SLIMKV_ERR_CUDA, "cudaFuncSetAttribute (4-bit key mass) failed");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    kernel<<<J.ctas, kThreads, smem_bytes<G>(J.k_pitch), stream>>>(km, J);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "4-bit key mass launch failed: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_cache4_key_mass(const slimkv_key_mass_args* a, void* stream) {
    const char* what = "4-bit key mass";
    if (!a || !a->q || !a->lengths || !a->lse || !a->mass) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (a->batch < 1 || a->batch > 4096 || a->nodes < 1 || a->nodes > 1024 || a->heads < 1 || a->kv_heads < 1 ||
        a->heads % a->kv_heads || a->mass_rows < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: batch in 1..4096, nodes in 1..1024, heads a multiple of kv_heads, mass rows", what);
    if (a->heads / a->kv_heads > 128) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: at most 128 query heads per KV head", what);
    if (a->dim < kGroupDims || a->dim > kMaxDims4 || a->dim % kGroupDims)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: dims must be multiples of 32 up to 320", what);
    if (a->type != SLIMKV_BF16 && a->type != SLIMKV_FP16) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: bf16 or fp16 tensors", what);
    if (!(a->scale > -INFINITY && a->scale < INFINITY) || !(a->decay > -INFINITY && a->decay < INFINITY))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: finite scale and decay", what);
    const int k_pitch = row4_bytes(a->dim);
    if (int rc = check_cache(a->cache, a->batch, k_pitch, k_pitch, 1, false, what)) return rc;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8) return fail(SLIMKV_ERR_ALIGNMENT, "%s: strides must be multiples of 8 elements", what);
    if (!aligned16(a->q)) return fail(SLIMKV_ERR_ALIGNMENT, "%s: 16-byte aligned tensors", what);
    const slimkv_cache& cache = a->cache;
    const bool paged = cache.table != nullptr;
    if (paged && cache.rows % 8) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: pages of a multiple of 8 rows", what);
    Job J{};
    J.box = paged && cache.rows % kSlab ? 8 : kSlab;
    J.shared_cache = !paged && cache.k_stride[0] == 0;
    const uint64_t planes = paged ? uint64_t(cache.num_pages) : J.shared_cache ? 1 : uint64_t(a->batch);
    CUtensorMap km;
    if (int rc = encode_map_words_4d(&km, cache.k, k_pitch / 4, a->kv_heads, cache.rows, planes, a->kv_heads > 1 ? cache.k_stride[2] : k_pitch,
                                     cache.rows > 1 ? cache.k_stride[1] : k_pitch, planes > 1 ? cache.k_stride[0] : k_pitch, J.box))
        return rc;
    J.batch = a->batch;
    J.nodes = a->nodes;
    J.heads = a->heads;
    J.kv_heads = a->kv_heads;
    J.group = a->heads / a->kv_heads;
    J.kg = a->dim / kGroupDims;
    J.k_pitch = k_pitch;
    J.context_only = a->context_only;
    J.paged = paged;
    J.cache = cache_view(cache);
    J.capacity = std::min<int64_t>(cache_capacity(J.cache), a->mass_rows);
    if (J.capacity > 0x7fffffffLL - 4096 ||
        double(J.batch) * J.kv_heads * (double(J.capacity / kKeys + 1) * (kMaxRows / 32 + 1) + Plan::kPieceUnits) >= 2147483648.0)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: too many rows in one call", what);
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
    auto run = [&](auto groups) {
        constexpr int G = decltype(groups)::value;
        J.ctas = device_info().sm_count * kBlocks<G>;
        if (J.kg == G) return half ? launch<G, true, true>(km, J, st) : launch<G, false, true>(km, J, st);
        return half ? launch<G, true, false>(km, J, st) : launch<G, false, false>(km, J, st);
    };
    using std::integral_constant;
    switch (J.kg) {
        case 1: case 2: return run(integral_constant<int, 2>());
        case 3: return run(integral_constant<int, 3>());
        case 4: return run(integral_constant<int, 4>());
        case 5: return run(integral_constant<int, 5>());
        case 6: return run(integral_constant<int, 6>());
        case 7: case 8: return run(integral_constant<int, 8>());
        default: return run(integral_constant<int, 10>());
    }
}
