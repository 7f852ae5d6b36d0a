// Eviction of cache rows by accumulated attention weight (C ABI slimkv_evict).
//
// Each (sequence, KV head) segment keeps its first `sinks` rows, its last
// `recent` rows and the rows of the largest mass up to `keep`, in order.  Two
// launches:
//   evict_select_kernel  one cluster of CTAs per segment: the keep-th largest
//     of its masses (order-preserving 32-bit keys, radix selection with digits
//     of 11, 11 and 10 bits, whose counts the CTAs add up over distributed
//     shared memory), how many rows equal to it still fit, and for every run
//     of kRun rows how many rows above it and equal to it come before the run;
//   evict_gather_kernel  one block per run, a dependent launch: which of its
//     rows stay and where they go, then their K, V, mass and position moved, a
//     warp to a row, 16 bytes a lane.
// Bound: HBM, the masses once (later readings come from L2) and each kept row
// read and written.
#include <algorithm>

#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

constexpr int kRun = 128;                 // rows of one gather block
constexpr int kGatherThreads = 256;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kSelectThreads = 1024;
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
    __shared__ uint32_t hist[3][kBins];       // one per digit: no pass clears what another still reads
    __shared__ uint32_t warp_sum[32];
    __shared__ uint32_t pick[2];              // the chosen digit, rows above it
    __shared__ uint32_t counts[2];            // this CTA's rows above and equal to the threshold
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
    // This CTA's rows: whole runs.
    const int runs_each = (a.runs + int(ranks) - 1) / int(ranks);
    const int run0 = min(int(rank) * runs_each, a.runs), run1 = min(run0 + runs_each, a.runs);
    const int n0 = min(run0 * kRun, len), n1 = min(run1 * kRun, len);
    uint32_t prefix = 0, want = uint32_t(min(a.keep, len));
    const bool all = len <= a.keep;
    if (!all) {
        for (int i = tid; i < 3 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
        __syncthreads();
        // `want` of the rows that match `prefix` so far are still to be found.
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above_bits = pass == 0 ? 32 : shift + 11 - (pass == 2);
            const uint32_t bins = pass == 2 ? 1024u : 2048u;
            for (int n = n0 + tid; n < n1; n += kSelectThreads) {
                const uint32_t key = key_of(__ldg(mass + n), n, len, a.sinks, a.recent);
                if (pass == 0 || (key >> above_bits) == (prefix >> above_bits)) atomicAdd(&hist[pass][key >> shift & (bins - 1)], 1u);
            }
            __syncthreads();
            cluster_sync();
            // Bins of all CTAs from the top: thread t has bins 2047 - 2t and 2046 - 2t.
            uint32_t c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t* bin = &hist[pass][kBins - 1 - 2 * tid - i];
                c[i] = 0;
                for (uint32_t r = 0; r < ranks; ++r) c[i] += cluster_load(bin, r);
            }
            const uint32_t sum = c[0] + c[1];
            uint32_t above = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, above, o);
                if (lane >= o) above += up;
            }
            if (lane == 31) warp_sum[warp] = above;
            __syncthreads();
            uint32_t before = warp_sum[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += up;
            }
            before = __shfl_sync(0xffffffffu, before, warp ? warp - 1 : 0);
            above += (warp ? before : 0u) - sum;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (above < want && above + c[i] >= want) {
                    pick[0] = uint32_t(kBins - 1 - 2 * tid - i);
                    pick[1] = above;
                }
                above += c[i];
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
    // Rows above and equal to the threshold before each run: a warp takes a run
    // at a time, 32 of them are scanned together, first within the CTA.
    uint2* before = a.before + int64_t(segment) * a.runs;
    uint32_t* gt_of = hist[0];                // (every CTA of the cluster is past pass 0)
    uint32_t* tie_of = hist[0] + 32;
    uint32_t base_gt = 0, base_tie = 0;
    for (int r0 = run0; r0 < run1; r0 += 32) {
        uint32_t gt = 0, tie = 0;
        if (r0 + warp < run1) {
            for (int i = 0; i < kRun; i += 32) {
                const int n = (r0 + warp) * kRun + i + lane;
                const uint32_t key = n < len ? key_of(__ldg(mass + n), n, len, a.sinks, a.recent) : 0u;
                gt += __popc(__ballot_sync(0xffffffffu, n < len && key > prefix));
                tie += __popc(__ballot_sync(0xffffffffu, n < len && key == prefix));
            }
        }
        __syncthreads();
        if (lane == 0) { gt_of[warp] = gt; tie_of[warp] = tie; }
        __syncthreads();
        uint32_t g_in = gt_of[lane], t_in = tie_of[lane];
        const uint32_t g_own = g_in, t_own = t_in;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t gu = __shfl_up_sync(0xffffffffu, g_in, o), tu = __shfl_up_sync(0xffffffffu, t_in, o);
            if (lane >= o) { g_in += gu; t_in += tu; }
        }
        if (warp == 0 && r0 + lane < run1) before[r0 + lane] = make_uint2(base_gt + g_in - g_own, base_tie + t_in - t_own);
        base_gt += __shfl_sync(0xffffffffu, g_in, 31);
        base_tie += __shfl_sync(0xffffffffu, t_in, 31);
    }
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

__global__ void __launch_bounds__(kGatherThreads) evict_gather_kernel(EvictArgs a) {
    __shared__ uint8_t src[kRun];
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
    if (stays) {
        src[local] = uint8_t(tid);
        const int d = first + local;
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = x;
        if (a.out_positions)
            a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] =
                __ldg(a.positions + b * a.positions_stride[0] + g * a.positions_stride[1] + n);
    }
    __syncthreads();
    // The kept rows, kRows of a warp at a time so that their loads overlap; then the zeroed
    // rows [kept, keep) of this run.
    constexpr int kWarps = kGatherThreads / 32, kRows = 4;
    bool bad = false;
    auto row_of = [&](const CacheView& c, int m, const int64_t* st) -> int64_t {
        int64_t page;
        int row;
        if (!cache_row(c, b, m, page, row)) { bad = true; return -1; }
        return page * st[0] + row * st[1] + g * st[2];
    };
    auto move = [&](const uint8_t* from, uint8_t* to, const int64_t* in, const int64_t* out, int units) {
        for (int r0 = warp; r0 < total; r0 += kWarps * kRows) {
            const uint4* p[kRows];
            uint4* q[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int r = r0 + k * kWarps;
                p[k] = nullptr;
                if (r < total) {
                    const int64_t i = row_of(a.in, n0 + src[r], in), o = row_of(a.out, first + r, out);
                    if (i >= 0 && o >= 0) {
                        p[k] = reinterpret_cast<const uint4*>(from + i);
                        q[k] = reinterpret_cast<uint4*>(to + o);
                    }
                }
            }
            for (int u = lane; u < units; u += 32) {
                uint4 w[kRows];
#pragma unroll
                for (int k = 0; k < kRows; ++k)
                    if (p[k]) w[k] = __ldcs(p[k] + u);
#pragma unroll
                for (int k = 0; k < kRows; ++k)
                    if (p[k]) __stcs(q[k] + u, w[k]);
            }
        }
    };
    move(a.k, a.out_k, a.in.k_stride, a.out.k_stride, a.k_units);
    move(a.v, a.out_v, a.in.v_stride, a.out.v_stride, a.v_units);
    const int z0 = max(n0, kept), z1 = min(n0 + kRun, a.keep);
    for (int d = z0 + tid; d < z1; d += kGatherThreads) {
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = 0.f;
        if (a.out_positions) a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] = 0;
    }
    for (int d = z0 + warp; d < z1; d += kWarps) {
        const int64_t ok = row_of(a.out, d, a.out.k_stride), ov = row_of(a.out, d, a.out.v_stride);
        if (ok < 0 || ov < 0) continue;
        for (int u = lane; u < a.k_units; u += 32) reinterpret_cast<uint4*>(a.out_k + ok)[u] = make_uint4(0, 0, 0, 0);
        for (int u = lane; u < a.v_units; u += 32) reinterpret_cast<uint4*>(a.out_v + ov)[u] = make_uint4(0, 0, 0, 0);
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
    // A CTA of a cluster takes at least four rows a thread: up to 8 CTAs (32768 rows and more).
    int ranks = 1;
    while (ranks < kMaxCluster && int64_t(k.rows) > int64_t(ranks) * 4 * kSelectThreads) ranks *= 2;
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
