// Eviction of cache rows by accumulated attention weight (C ABI slimkv_evict).
//
// Each (sequence, KV head) segment keeps its first `sinks` rows, its last
// `recent` rows and the rows of the largest mass up to `keep`, in order.  Two
// launches:
//   evict_select_kernel  the keep-th largest of the segment's masses (as
//     order-preserving 32-bit keys), how many rows equal to it still fit, and
//     for every run of kRun rows how many rows above it and equal to it come
//     before the run;
//   evict_gather_kernel  one block per run: which of its rows stay and where
//     they go, then their K, V, mass and position moved as 16-byte units.
// Bound: HBM, the masses once (their second reading comes from L2) and each
// kept row read and written.
#include <algorithm>

#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

constexpr int kRun = 256;                 // rows of one gather block
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
    __shared__ uint32_t hist[256];
    __shared__ uint32_t pick[2];              // the chosen digit, rows above it
    __shared__ uint32_t warp_gt[32], warp_tie[32];
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int segment = b * a.kv_heads + g;
    const int len = segment_length(a, b);
    const float* mass = a.mass + b * a.mass_stride[0] + g * a.mass_stride[1];
    if (g == 0 && tid == 0) {
        const int given = __ldg(a.lengths + b);
        a.new_lengths[b] = min(len, a.keep);
        if (given != len) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    uint32_t prefix = 0, want = uint32_t(min(a.keep, len));
    const bool all = len <= a.keep;
    if (!all) {
        // Radix selection, 8 bits a pass: `want` of the rows that match
        // `prefix` so far are still to be found.
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int n = tid; n < len; n += kSelectThreads) {
                const uint32_t key = key_of(__ldg(mass + n), n, len, a.sinks, a.recent);
                if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[key >> shift & 255], 1u);
            }
            __syncthreads();
            if (warp == 0) {
                // Lane l holds digits 255 - 8l .. 248 - 8l: counts from above.
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) { c[i] = hist[255 - 8 * lane - i]; sum += c[i]; }
                uint32_t above = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, above, o);
                    if (lane >= o) above += up;
                }
                above -= sum;
                if (above < want && above + sum >= want) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (above < want && above + c[i] >= want) {
                            pick[0] = uint32_t(255 - 8 * lane - i);
                            pick[1] = above;
                        }
                        above += c[i];
                    }
                }
            }
            __syncthreads();
            prefix |= pick[0] << shift;
            want -= pick[1];
            __syncthreads();
        }
    }
    if (tid == 0) {
        a.threshold[segment] = prefix;        // all: 0, below every row's key
        a.ties[segment] = all ? 0u : want;
    }
    // Rows above and equal to the threshold before each run: warp w takes the
    // runs w, w + 32, ... of a block of 32 runs, then the block scans them.
    uint2* before = a.before + int64_t(segment) * a.runs;
    uint32_t base_gt = 0, base_tie = 0;
    for (int r0 = 0; r0 < a.runs; r0 += 32) {
        uint32_t gt = 0, tie = 0;
        const int n0 = (r0 + warp) * kRun;
        if (r0 + warp < a.runs) {
            for (int i = 0; i < kRun; i += 32) {
                const int n = n0 + i + lane;
                const uint32_t key = n < len ? key_of(__ldg(mass + n), n, len, a.sinks, a.recent) : 0u;
                gt += __popc(__ballot_sync(0xffffffffu, n < len && key > prefix));
                tie += __popc(__ballot_sync(0xffffffffu, n < len && key == prefix));
            }
        }
        if (lane == 0) { warp_gt[warp] = gt; warp_tie[warp] = tie; }
        __syncthreads();
        uint32_t g_in = warp_gt[lane], t_in = warp_tie[lane];
        const uint32_t g_own = g_in, t_own = t_in;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t gu = __shfl_up_sync(0xffffffffu, g_in, o), tu = __shfl_up_sync(0xffffffffu, t_in, o);
            if (lane >= o) { g_in += gu; t_in += tu; }
        }
        if (warp == 0 && r0 + lane < a.runs) before[r0 + lane] = make_uint2(base_gt + g_in - g_own, base_tie + t_in - t_own);
        base_gt += __shfl_sync(0xffffffffu, g_in, 31);
        base_tie += __shfl_sync(0xffffffffu, t_in, 31);
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kRun) evict_gather_kernel(EvictArgs a) {
    __shared__ int16_t src[kRun];
    __shared__ uint32_t warp_tie[kRun / 32], warp_keep[kRun / 32];
    const int run = blockIdx.x, g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int segment = b * a.kv_heads + g;
    const int len = segment_length(a, b);
    const int kept = min(len, a.keep);
    const int n0 = run * kRun, n = n0 + tid;
    const unsigned below = (1u << lane) - 1u;
    const uint32_t threshold = a.threshold[segment], ties = a.ties[segment];
    const uint2 before = a.before[int64_t(segment) * a.runs + run];
    // Which rows stay: those above the threshold and the first `ties` equal to it.
    float x = 0.f;
    bool gt = false, tie = false;
    if (n < len) {
        x = __ldg(a.mass + b * a.mass_stride[0] + g * a.mass_stride[1] + n);
        const uint32_t key = key_of(x, n, len, a.sinks, a.recent);
        gt = key > threshold;
        tie = key == threshold;
    }
    const unsigned tie_lanes = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) warp_tie[warp] = __popc(tie_lanes);
    __syncthreads();
    uint32_t rank = before.y + __popc(tie_lanes & below);
    for (int w = 0; w < warp; ++w) rank += warp_tie[w];
    const bool stays = gt || (tie && rank < ties);
    const unsigned keep_lanes = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) warp_keep[warp] = __popc(keep_lanes);
    __syncthreads();
    int local = __popc(keep_lanes & below), total = 0;
#pragma unroll
    for (int w = 0; w < kRun / 32; ++w) {
        if (w < warp) local += warp_keep[w];
        total += warp_keep[w];
    }
    const int first = int(before.x + min(before.y, ties));
    if (stays) {
        src[local] = int16_t(tid);
        const int d = first + local;
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = x;
        if (a.out_positions)
            a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] =
                __ldg(a.positions + b * a.positions_stride[0] + g * a.positions_stride[1] + n);
    }
    __syncthreads();
    // The kept rows, then the zeroed rows [kept, keep) of this run, 16 bytes a thread.
    const int units = a.k_units + a.v_units;
    bool bad = false;
    for (int i = tid; i < total * units; i += kRun) {
        const int r = i / units, u = i - r * units;
        const bool is_v = u >= a.k_units;
        int64_t ip, op;
        int ir, orow;
        bad |= !cache_row(a.in, b, n0 + src[r], ip, ir);
        if (!cache_row(a.out, b, first + r, op, orow)) { bad = true; continue; }
        if (!is_v) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.k + ip * a.in.k_stride[0] + ir * a.in.k_stride[1] + g * a.in.k_stride[2]) + u);
            *(reinterpret_cast<uint4*>(a.out_k + op * a.out.k_stride[0] + orow * a.out.k_stride[1] + g * a.out.k_stride[2]) + u) = w;
        } else {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.v + ip * a.in.v_stride[0] + ir * a.in.v_stride[1] + g * a.in.v_stride[2]) + (u - a.k_units));
            *(reinterpret_cast<uint4*>(a.out_v + op * a.out.v_stride[0] + orow * a.out.v_stride[1] + g * a.out.v_stride[2]) + (u - a.k_units)) = w;
        }
    }
    const int z0 = max(n0, kept), z1 = min(n0 + kRun, a.keep);
    for (int d = z0 + tid; d < z1; d += kRun) {
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = 0.f;
        if (a.out_positions) a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] = 0;
    }
    for (int i = tid; i < max(z1 - z0, 0) * units; i += kRun) {
        const int r = i / units, u = i - r * units;
        int64_t op;
        int orow;
        if (!cache_row(a.out, b, z0 + r, op, orow)) { bad = true; continue; }
        uint8_t* dst = u < a.k_units
                           ? a.out_k + op * a.out.k_stride[0] + orow * a.out.k_stride[1] + g * a.out.k_stride[2] + int64_t(u) * 16
                           : a.out_v + op * a.out.v_stride[0] + orow * a.out.v_stride[1] + g * a.out.v_stride[2] + int64_t(u - a.k_units) * 16;
        *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
    }
    if (bad) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
}

int evict_rows(const slimkv_evict_args* a) {
    return int(std::min<int64_t>(cache_capacity(cache_view(a->in)), a->mass_rows));
}

int check_evict(const slimkv_evict_args* a) {
    if (!a) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->batch < 1 || a->batch > 65535 || a->kv_heads < 1 || a->kv_heads > 65535 || a->mass_rows < 1 || a->in.rows < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: batch and heads in 1..65535, mass and cache need rows");
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
    evict_select_kernel<<<dim3(a->kv_heads, a->batch), kSelectThreads, 0, st>>>(k);
    evict_gather_kernel<<<dim3(k.runs, a->kv_heads, a->batch), kRun, 0, st>>>(k);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "evict launch failed: %s", cudaGetErrorString(err));
}
