// Eviction of cache rows by accumulated attention weight (C ABI slimkv_evict).
//
// Each (sequence, KV head) segment keeps its first `sinks` rows, its last
// `recent` rows and the rows of the largest mass up to `keep`, in order.  Two
// launches:
//   evict_select_kernel  one cluster of CTAs per segment: the keep-th largest
//     of its masses (order-preserving 32-bit keys, radix selection with four
//     8-bit digits, whose counts the CTAs add up over distributed shared
//     memory), how many rows equal to it still fit, and for every run of kRun
//     rows how many rows above it and equal to it come before the run;
//   evict_gather_kernel  one block per run, a dependent launch: which of its
//     rows stay and where they go, then their K, V, mass and position moved, 16
//     bytes a lane, eight of them under way at a time.
// Bound: HBM, the masses once (later readings come from L2) and each kept row
// read and written.
#include <algorithm>

#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

constexpr int kRun = 128;                 // rows of one gather block
constexpr int kGatherThreads = 256;
constexpr int kMaxCluster = 8;
constexpr int kSelectThreads = 1024;
constexpr int kBins = 256, kKeys = 4;      // digit values; keys of a thread in registers
constexpr int kTile = kKeys * kSelectThreads, kChunks = kTile / 32;   // rows of a CTA's tile, 32 to a chunk
constexpr uint32_t kAlways = 0xffffffffu; // key of a protected row

struct EvictArgs {
    int batch, kv_heads, k_units, v_units;    // 16-byte units of a K / V row
    const uint8_t *k, *v;
    uint8_t *out_k, *out_v;
    CacheView in, out;                        // strides in bytes
    const int32_t* lengths;
    const float* mass;
    int64_t mass_stride[2];
    const int32_t* positions;
    int64_t positions_stride[2];
    float* out_mass;
    int64_t out_mass_stride[2];
    int32_t* out_positions;
    int64_t out_positions_stride[2];
    int rows;                                 // rows a segment can hold
    int keep, sinks, recent, runs;
    int32_t* new_lengths;
    unsigned int* status;
    // Workspace, one entry per segment: the threshold key, the rows equal to
    // it that stay, and [runs] pairs of counts before each run.
    uint32_t* threshold;
    uint32_t* ties;
    uint2* before;
};

// Order-preserving key of row n's mass; kAlways for a protected row.  A NaN
// ranks above every number, the two zeros are equal.
__device__ __forceinline__ uint32_t key_of(float x, int n, int len, int sinks, int recent) {
    if (n < sinks || n >= len - recent) return kAlways;
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? kAlways - 1 : (u >> 31 ? ~u : u | 0x80000000u);
}

__device__ __forceinline__ int segment_length(const EvictArgs& a, int b) {
    return min(max(__ldg(a.lengths + b), 0), a.rows);
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[4][kBins];       // one per digit: no pass clears what another still reads
    __shared__ uint32_t warp_sum[8];
    __shared__ uint32_t pick[2];              // the chosen digit, rows above it
    __shared__ uint32_t counts[2];            // this CTA's rows above and equal to the threshold
    __shared__ uint2 chunk[kChunks];
    const uint32_t ranks = cluster_size(), rank = cluster_rank();
    const int segment = blockIdx.x / ranks, g = segment % a.kv_heads, b = segment / a.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int len = segment_length(a, b);
    const float* mass = a.mass + b * a.mass_stride[0] + g * a.mass_stride[1];
    if (g == 0 && rank == 0 && tid == 0) {
        const int given = __ldg(a.lengths + b);
        a.new_lengths[b] = min(len, a.keep);
        if (given != len) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    grid_launch_dependents();
    // This CTA's rows: whole runs, in tiles of kTile; key j of a thread is row
    // 32 (32 j + warp) + lane of the tile.
    const int runs_each = (a.runs + int(ranks) - 1) / int(ranks);
    const int run0 = min(int(rank) * runs_each, a.runs), run1 = min(run0 + runs_each, a.runs);
    const int n0 = min(run0 * kRun, len), n1 = min(run1 * kRun, len);
    const int tiles = (n1 - n0 + kTile - 1) / kTile;
    uint32_t keys[kKeys];
    auto load = [&](int tile) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int n = n0 + tile * kTile + 32 * (32 * j + warp) + lane;
            keys[j] = n < n1 ? key_of(__ldg(mass + n), n, len, a.sinks, a.recent) : 0u;   // 0: below every row's key
        }
    };
    for (int i = tid; i < 4 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
    if (tiles == 1) load(0);
    uint32_t prefix = 0, want = uint32_t(min(a.keep, len));
    const bool all = len <= a.keep;
    if (!all) {
        __syncthreads();
        // `want` of the rows that match `prefix` so far are still to be found.
#pragma unroll 1
        for (int pass = 0; pass < 4; ++pass) {
            const int shift = 24 - 8 * pass;
            for (int tile = 0; tile < tiles; ++tile) {
                if (tiles > 1) load(tile);
#pragma unroll
                for (int j = 0; j < kKeys; ++j) {
                    // Masses share few exponents: lanes with the same digit count once.
                    const bool in = keys[j] && (pass == 0 || (keys[j] ^ prefix) >> (shift + 8) == 0);
                    const uint32_t digit = in ? keys[j] >> shift & 255 : 256u;
                    const unsigned same = __match_any_sync(0xffffffffu, digit);
                    if (in && lane == __ffs(int(same)) - 1) atomicAdd(&hist[pass][digit], uint32_t(__popc(same)));
                }
            }
            __syncthreads();
            if (ranks > 1) cluster_sync();
            // Thread t < 256 has bin 255 - t, of all CTAs: rows above it, from the top.
            uint32_t c = 0, above = 0;
            if (tid < kBins) {
                const uint32_t* bin = &hist[pass][kBins - 1 - tid];
                if (ranks == 1) {
                    c = *bin;
                } else {
                    uint32_t of[kMaxCluster];
#pragma unroll
                    for (uint32_t r = 0; r < kMaxCluster; ++r) of[r] = r < ranks ? cluster_load(bin, r) : 0u;
#pragma unroll
                    for (uint32_t r = 0; r < kMaxCluster; ++r) c += of[r];
                }
                above = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, above, o);
                    if (lane >= o) above += up;
                }
                if (lane == 31) warp_sum[warp] = above;
            }
            __syncthreads();
            if (tid < kBins) {
                above -= c;
                for (int w = 0; w < warp; ++w) above += warp_sum[w];
                if (above < want && above + c >= want) {
                    pick[0] = uint32_t(kBins - 1 - tid);
                    pick[1] = above;
                }
            }
            __syncthreads();
            prefix |= pick[0] << shift;
            want -= pick[1];
        }
    }
    if (rank == 0 && tid == 0) {
        a.threshold[segment] = prefix;        // all: 0, below every row's key
        a.ties[segment] = all ? 0u : want;
    }
    // Rows above and equal to the threshold before each run, first within the CTA.
    uint2* before = a.before + int64_t(segment) * a.runs;
    uint32_t base_gt = 0, base_tie = 0;
    for (int tile = 0; tile < tiles; ++tile) {
        if (tiles > 1) load(tile);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const uint32_t gt = __popc(__ballot_sync(0xffffffffu, keys[j] > prefix));
            const uint32_t tie = __popc(__ballot_sync(0xffffffffu, keys[j] && keys[j] == prefix));
            if (lane == 0) chunk[32 * j + warp] = make_uint2(gt, tie);
        }
        __syncthreads();
        // Every warp scans the tile's chunks, four to a lane.
        uint2 own[4], sum = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            own[i] = chunk[4 * lane + i];
            sum.x += own[i].x;
            sum.y += own[i].y;
        }
        uint2 incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t gu = __shfl_up_sync(0xffffffffu, incl.x, o), tu = __shfl_up_sync(0xffffffffu, incl.y, o);
            if (lane >= o) { incl.x += gu; incl.y += tu; }
        }
        const int run = run0 + tile * (kTile / kRun) + lane;      // (a run is four chunks)
        if (warp == 0 && run < run1) before[run] = make_uint2(base_gt + incl.x - sum.x, base_tie + incl.y - sum.y);
        base_gt += __shfl_sync(0xffffffffu, incl.x, 31);
        base_tie += __shfl_sync(0xffffffffu, incl.y, 31);
    }
    // Runs of this CTA past its rows (all of them in a segment shorter than the budget).
    for (int run = run0 + tiles * (kTile / kRun) + tid; run < run1; run += kSelectThreads) before[run] = make_uint2(base_gt, base_tie);
    if (ranks == 1) return;
    // Then what the CTAs before this one hold.
    if (tid == 0) { counts[0] = base_gt; counts[1] = base_tie; }
    __syncthreads();
    cluster_sync();
    uint32_t add_gt = 0, add_tie = 0;
    for (uint32_t r = 0; r < rank; ++r) {
        add_gt += cluster_load(&counts[0], r);
        add_tie += cluster_load(&counts[1], r);
    }
    for (int r = run0 + tid; r < run1; r += kSelectThreads) {
        uint2 x = before[r];
        x.x += add_gt;
        x.y += add_tie;
        before[r] = x;
    }
    cluster_sync();                           // no CTA leaves while another reads its counts
}
static_assert(kRun == 128 && kChunks == 128, "a run is four chunks, a tile 32 runs");

__global__ void __launch_bounds__(kGatherThreads) evict_gather_kernel(EvictArgs a) {
    __shared__ int64_t from[2][kRun], to[2][kRun];      // byte offsets of the kept rows: K, V (-1: no such page)
    __shared__ uint32_t warp_tie[kRun / 32], warp_keep[kRun / 32];
    const int run = blockIdx.x, g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int segment = b * a.kv_heads + g;
    const int len = segment_length(a, b);
    const int kept = min(len, a.keep);
    const int n0 = run * kRun, n = n0 + tid;
    const unsigned below = (1u << lane) - 1u;
    float x = 0.f;
    if (tid < kRun && n < len) x = __ldg(a.mass + b * a.mass_stride[0] + g * a.mass_stride[1] + n);
    grid_dependency_wait();
    const uint32_t threshold = a.threshold[segment], ties = a.ties[segment];
    const uint2 before = a.before[int64_t(segment) * a.runs + run];
    // Which rows stay: those above the threshold and the first `ties` equal to it.
    const uint32_t key = key_of(x, n, len, a.sinks, a.recent);
    const bool own = tid < kRun && n < len;
    const bool gt = own && key > threshold, tie = own && key == threshold;
    const unsigned tie_lanes = __ballot_sync(0xffffffffu, tie);
    if (lane == 0 && warp < kRun / 32) warp_tie[warp] = __popc(tie_lanes);
    __syncthreads();
    uint32_t at = before.y + __popc(tie_lanes & below);
    for (int w = 0; w < min(warp, kRun / 32); ++w) at += warp_tie[w];
    const bool stays = gt || (tie && at < ties);
    const unsigned keep_lanes = __ballot_sync(0xffffffffu, stays);
    if (lane == 0 && warp < kRun / 32) warp_keep[warp] = __popc(keep_lanes);
    __syncthreads();
    int local = __popc(keep_lanes & below), total = 0;
#pragma unroll
    for (int w = 0; w < kRun / 32; ++w) {
        if (w < warp) local += warp_keep[w];
        total += warp_keep[w];
    }
    const int first = int(before.x + min(before.y, ties));
    bool bad = false;
    if (stays) {
        const int d = first + local;
        int64_t ip, op;
        int ir, orow;
        const bool in = cache_row(a.in, b, n, ip, ir), out = cache_row(a.out, b, d, op, orow);
        bad = !in || !out;
        from[0][local] = bad ? -1 : ip * a.in.k_stride[0] + ir * a.in.k_stride[1] + g * a.in.k_stride[2];
        from[1][local] = bad ? -1 : ip * a.in.v_stride[0] + ir * a.in.v_stride[1] + g * a.in.v_stride[2];
        to[0][local] = op * a.out.k_stride[0] + orow * a.out.k_stride[1] + g * a.out.k_stride[2];
        to[1][local] = op * a.out.v_stride[0] + orow * a.out.v_stride[1] + g * a.out.v_stride[2];
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = x;
        if (a.out_positions)
            a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] =
                __ldg(a.positions + b * a.positions_stride[0] + g * a.positions_stride[1] + n);
    }
    __syncthreads();
    // The kept rows: pieces of 32 lanes x 16 bytes of a row's K and V, kPieces of a warp
    // under way at a time; then the zeroed rows [kept, keep) of this run.
    constexpr int kWarps = kGatherThreads / 32, kPieces = 8;
    const int units = a.k_units + a.v_units, per_row = (units + 31) / 32, pieces = total * per_row;
    // p / per_row by multiplication: exact while p per_row < 2^20 (p < 128 per_row, per_row <= 64).
    const uint32_t inverse = (1u << 20) / uint32_t(per_row) + 1u;
    const bool small = per_row <= 64;
    for (int p0 = warp; p0 < pieces; p0 += kWarps * kPieces) {
        uint4 w[kPieces];
        uint4* dst[kPieces];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int p = p0 + k * kWarps;
            dst[k] = nullptr;
            if (p >= pieces) continue;
            const int r = small ? int(uint32_t(p) * inverse >> 20) : p / per_row;
            int u = (p - r * per_row) * 32 + lane;
            if (u >= units) continue;
            const int is_v = u >= a.k_units;
            if (is_v) u -= a.k_units;
            const int64_t i = from[is_v][r];
            if (i < 0) continue;
            dst[k] = reinterpret_cast<uint4*>((is_v ? a.out_v : a.out_k) + to[is_v][r]) + u;
            w[k] = __ldcs(reinterpret_cast<const uint4*>((is_v ? a.v : a.k) + i) + u);
        }
#pragma unroll
        for (int k = 0; k < kPieces; ++k)
            if (dst[k]) __stcs(dst[k], w[k]);
    }
    const int z0 = max(n0, kept), z1 = min(n0 + kRun, a.keep);
    for (int d = z0 + tid; d < z1; d += kGatherThreads) {
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = 0.f;
        if (a.out_positions) a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] = 0;
    }
    for (int d = z0 + warp; d < z1; d += kWarps) {
        int64_t page;
        int row;
        if (!cache_row(a.out, b, d, page, row)) { bad = true; continue; }
        uint4* ok = reinterpret_cast<uint4*>(a.out_k + page * a.out.k_stride[0] + row * a.out.k_stride[1] + g * a.out.k_stride[2]);
        uint4* ov = reinterpret_cast<uint4*>(a.out_v + page * a.out.v_stride[0] + row * a.out.v_stride[1] + g * a.out.v_stride[2]);
        for (int u = lane; u < a.k_units; u += 32) ok[u] = make_uint4(0, 0, 0, 0);
        for (int u = lane; u < a.v_units; u += 32) ov[u] = make_uint4(0, 0, 0, 0);
    }
    if (bad) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
}

int evict_rows(const slimkv_evict_args* a) {
    return int(std::min<int64_t>(cache_capacity(cache_view(a->in)), a->mass_rows));
}

int check_evict(const slimkv_evict_args* a) {
    if (!a) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->batch < 1 || a->batch > 65535 || a->kv_heads < 1 || int64_t(a->batch) * a->kv_heads > (1 << 24) || a->kv_heads > 65535 || a->mass_rows < 1 || a->in.rows < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: batch and heads in 1..65535 (2^24 segments), mass and cache need rows");
    if (a->keep < 1 || a->sinks < 0 || a->recent < 0 || int64_t(a->sinks) + a->recent > a->keep)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: keep >= 1 and sinks + recent <= keep");
    if (a->in.table && (a->in.table_pages < 1 || int64_t(a->in.rows) * a->in.table_pages > 0x7fffffffLL))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: block tables need pages and fewer than 2^31 rows");
    return SLIMKV_OK;
}

int evict_runs(const slimkv_evict_args* a) { return int((std::max<int64_t>(evict_rows(a), a->keep) + kRun - 1) / kRun); }

void carve(Carver& c, const slimkv_evict_args* a, EvictArgs& k) {
    const size_t segments = size_t(a->batch) * a->kv_heads;
    k.threshold = c.take<uint32_t>(segments);
    k.ties = c.take<uint32_t>(segments);
    k.before = c.take<uint2>(segments * k.runs);
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_evict_workspace_size(const slimkv_evict_args* a) {
    if (check_evict(a) != SLIMKV_OK) return 0;
    EvictArgs k{};
    k.runs = evict_runs(a);
    Carver c(nullptr, 0);
    carve(c, a, k);
    return c.used;
}

extern "C" int slimkv_evict(const slimkv_evict_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_evict(a)) return rc;
    if (!a->lengths || !a->mass || !a->new_lengths || !a->positions != !a->out_positions)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: null pointer, or positions without their output");
    const int e = a->elem_bytes;
    if (e != 1 && e != 2 && e != 4) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: elements of 1, 2 or 4 bytes");
    if (int rc = check_cache(a->in, a->batch, a->dim_qk, a->dim_v, e, true, "evict")) return rc;
    if (int rc = check_cache(a->out, a->batch, a->dim_qk, a->dim_v, e, true, "evict (output)")) return rc;
    if (cache_capacity(cache_view(a->out)) < a->keep)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: the output cache holds fewer than %d rows", a->keep);
    if (a->in.k == a->out.k || a->in.v == a->out.v || static_cast<const void*>(a->mass) == a->out_mass ||
        (a->positions && a->positions == a->out_positions))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: the output must not be the input");
    EvictArgs k{};
    k.batch = a->batch;
    k.kv_heads = a->kv_heads;
    k.k_units = a->dim_qk * e / 16;
    k.v_units = a->dim_v * e / 16;
    k.k = static_cast<const uint8_t*>(a->in.k);
    k.v = static_cast<const uint8_t*>(a->in.v);
    k.out_k = static_cast<uint8_t*>(const_cast<void*>(a->out.k));
    k.out_v = static_cast<uint8_t*>(const_cast<void*>(a->out.v));
    k.in = cache_view(a->in);
    k.out = cache_view(a->out);
    for (CacheView* v : {&k.in, &k.out})
        for (int i = 0; i < 3; ++i) { v->k_stride[i] *= e; v->v_stride[i] *= e; }
    k.lengths = a->lengths;
    k.mass = a->mass;
    k.positions = a->positions;
    k.out_mass = a->out_mass;
    k.out_positions = a->out_positions;
    for (int i = 0; i < 2; ++i) {
        k.mass_stride[i] = a->mass_stride[i];
        k.positions_stride[i] = a->positions_stride[i];
        k.out_mass_stride[i] = a->out_mass_stride[i];
        k.out_positions_stride[i] = a->out_positions_stride[i];
    }
    k.rows = evict_rows(a);
    k.keep = a->keep;
    k.sinks = a->sinks;
    k.recent = a->recent;
    k.runs = evict_runs(a);
    k.new_lengths = a->new_lengths;
    k.status = status_word();
    Carver c(workspace, workspace_bytes);
    carve(c, a, k);
    if (!workspace || !c.fits() || reinterpret_cast<uintptr_t>(workspace) % 8)
        return fail(SLIMKV_ERR_WORKSPACE, "evict: workspace of %zu bytes needed", c.used);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // CTAs of a cluster as many (up to 8) as keep their keys in registers.
    int ranks = 1;
    while (ranks < kMaxCluster && int64_t(k.rows) > int64_t(ranks) * kTile) ranks *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(a->kv_heads) * unsigned(a->batch) * unsigned(ranks));
    cfg.blockDim = dim3(kSelectThreads);
    cfg.stream = st;
    cudaLaunchAttribute cluster{}, dependent{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = unsigned(ranks);
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    cudaError_t err = cudaLaunchKernelEx(&cfg, evict_select_kernel, k);
    dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(k.runs, a->kv_heads, a->batch);
    cfg.blockDim = dim3(kGatherThreads);
    cfg.attrs = &dependent;
    if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, evict_gather_kernel, k);
    return err == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "evict launch failed: %s", cudaGetErrorString(err));
}
