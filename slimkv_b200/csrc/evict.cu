// Eviction of cache rows by accumulated attention weight (C ABI slimkv_evict).
//
// Each (sequence, KV head) segment keeps its first `sinks` rows, its last
// `recent` rows and the rows of the largest mass up to `keep`, in order.  Two
// launches:
//   evict_select_kernel  one cluster of CTAs per segment: the keep-th largest
//     of its masses (order-preserving 32-bit keys, radix selection with four
//     8-bit digits, whose counts the CTAs add up over distributed shared memory;
//     the same counts say what the CTAs before this one keep), then the kept
//     rows in order, into a list;
//   evict_gather_kernel  a dependent launch, one block per 32 rows of the output:
//     K, V, mass and position of the listed rows moved, 16 bytes a lane.
// Bound: HBM, the masses once (later readings come from L2) and each kept row
// read and written.  Measured: 16 segments of 32k latents cut to 8k (336 MB
// moved) 74 us in a graph, the selection 20 and the gather 52 alone (6.5 TB/s);
// two sequences of 1.2k rows cut to 1028, 12.3 us.
#include <algorithm>

#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

constexpr int kRows = 32;                 // output rows of one gather block
constexpr int kGatherThreads = 256;
constexpr int kMaxCluster = 8;
constexpr int kSelectThreads = 1024;
// Four digits of 8 bits: with three of 11, 11 and 10 each CTA of a cluster of 8 reads
// 128 KB of the others' counts for a digit, and 16 segments of 32k rows took 42 us.
constexpr int kPasses = 4, kBins = 256;
constexpr int kKeys = 4;                  // keys of a thread in registers
constexpr int kTile = kKeys * kSelectThreads, kChunks = kTile / 32;   // rows of a CTA's tile, 32 to a chunk
static_assert(kChunks == 128, "four chunks to a lane");
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
    int keep, sinks, recent;
    int32_t* new_lengths;
    unsigned int* status;
    int32_t* kept;                            // workspace: each segment's kept rows, list_rows to a segment
    int list_rows;
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

// (Two CTAs on an SM: a cluster stays in one part of the chip, where 16 clusters of 8
// else came one after the other, 31 us against 23.)
__global__ void __launch_bounds__(kSelectThreads, 2) evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[kPasses][kBins];      // one per digit: no pass clears what another still reads
    __shared__ uint32_t warp_sum[kBins / 32];
    __shared__ uint32_t pick[3];              // the chosen digit, rows above it, rows with it
    __shared__ uint32_t earlier[2];           // rows above and equal to the threshold of the CTAs before this one
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
    // This CTA's rows, in tiles of kTile; key j of a thread is row 32 (32 j + warp) + lane of the tile.
    const int each = ((len + int(ranks) - 1) / int(ranks) + 31) / 32 * 32;      // whole lines, at most a tile's where one does
    const int n0 = min(int(rank) * each, len), n1 = min(n0 + each, len);
    const int tiles = (n1 - n0 + kTile - 1) / kTile;
    uint32_t keys[kKeys];
    auto load = [&](int tile) {
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int n = n0 + tile * kTile + 32 * (32 * j + warp) + lane;
            keys[j] = n < n1 ? key_of(__ldg(mass + n), n, len, a.sinks, a.recent) : 0u;   // 0: below every row's key
        }
    };
    for (int i = tid; i < kPasses * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
    if (tid < 2) earlier[tid] = 0;
    if (tiles == 1) load(0);
    // Nothing to choose: every key is above threshold 0.
    const bool all = len <= a.keep;
    uint32_t prefix = 0, want = uint32_t(min(a.keep, len));
    uint32_t base_gt = all ? uint32_t(n0) : 0, base_tie = 0;
    if (!all) {
        uint32_t gt = 0, tie = 0;             // of the CTAs before this one, in this thread's bins
        __syncthreads();
        // `want` of the rows that match `prefix` so far are still to be found.
#pragma unroll 1
        for (int pass = 0; pass < kPasses; ++pass) {
            const int shift = 24 - 8 * pass;
            for (int tile = 0; tile < tiles; ++tile) {
                if (tiles > 1) load(tile);
#pragma unroll
                for (int j = 0; j < kKeys; ++j) {
                    // Masses share few exponents: lanes with the same digit count once.
                    const bool in = keys[j] && (pass == 0 || (keys[j] ^ prefix) >> (shift + 8) == 0);
                    const uint32_t digit = in ? keys[j] >> shift & (kBins - 1) : uint32_t(kBins);
                    const unsigned same = __match_any_sync(0xffffffffu, digit);
                    if (in && lane == __ffs(int(same)) - 1) atomicAdd(&hist[pass][digit], uint32_t(__popc(same)));
                }
            }
            __syncthreads();
            if (ranks > 1) cluster_sync();
            // Thread t < 256 has bin 255 - t, of all CTAs: rows above it, from the top.
            const uint32_t bin = uint32_t(kBins - 1 - tid);
            uint32_t c = 0, less = 0, above = 0;
            if (tid < kBins) {
                if (ranks == 1) {
                    c = hist[pass][bin];
                } else {
                    uint32_t of[kMaxCluster];
#pragma unroll
                    for (uint32_t r = 0; r < kMaxCluster; ++r) of[r] = r < ranks ? cluster_load(&hist[pass][bin], r) : 0u;
#pragma unroll
                    for (uint32_t r = 0; r < kMaxCluster; ++r) {
                        c += of[r];
                        if (r < rank) less += of[r];
                    }
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
                above += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0u) - c;
                if (above < want && above + c >= want) {
                    pick[0] = bin;
                    pick[1] = above;
                    pick[2] = c;
                }
            }
            __syncthreads();
            const uint32_t digit = pick[0];
            prefix |= digit << shift;
            want -= pick[1];
            // When all rows with these digits stay, the rest of their digits does not matter
            // (most often known after three of them).
            const bool done = pick[2] == want;
            if (tid < kBins) {
                if (bin > digit || (done && bin == digit)) gt += less;
                else if (pass == kPasses - 1 && bin == digit) tie = less;
            }
            if (done) {
                prefix -= 1;                  // every key from the prefix on is above the threshold (no key begins with 0, 0)
                want = 0;
                break;
            }
        }
        if (ranks > 1) {
            cluster_arrive();                 // this CTA has read the others' counts
            gt = __reduce_add_sync(0xffffffffu, gt);
            if (lane == 0 && gt) atomicAdd(&earlier[0], gt);
            if (tie) atomicAdd(&earlier[1], tie);
            __syncthreads();
            base_gt = earlier[0];
            base_tie = earlier[1];
        }
    }
    // The kept rows in order: those above the threshold and the first `want` equal to it.
    const uint32_t ties = all ? 0u : want;
    int32_t* list = a.kept + int64_t(segment) * a.list_rows;
    for (int tile = 0; tile < tiles; ++tile) {
        if (tiles > 1) load(tile);
        __syncthreads();
        unsigned gt[kKeys], tie[kKeys];       // lanes
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            gt[j] = __ballot_sync(0xffffffffu, keys[j] > prefix);
            tie[j] = __ballot_sync(0xffffffffu, keys[j] && keys[j] == prefix);
            if (lane == 0) chunk[32 * j + warp] = make_uint2(__popc(gt[j]), __popc(tie[j]));
        }
        __syncthreads();
        // Every warp scans the tile's chunks, four to a lane; its own chunk 32 j + warp is number
        // warp % 4 of lane 8 j + warp / 4.
        uint2 sum = make_uint2(0, 0), at = make_uint2(0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i == warp % 4) at = sum;
            const uint2 x = chunk[4 * lane + i];
            sum.x += x.x;
            sum.y += x.y;
        }
        uint2 incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t gu = __shfl_up_sync(0xffffffffu, incl.x, o), tu = __shfl_up_sync(0xffffffffu, incl.y, o);
            if (lane >= o) { incl.x += gu; incl.y += tu; }
        }
        at.x += incl.x - sum.x;
        at.y += incl.y - sum.y;
        const unsigned below = (1u << lane) - 1u;
#pragma unroll
        for (int j = 0; j < kKeys; ++j) {
            const int from = 8 * j + warp / 4;
            const uint32_t g0 = base_gt + __shfl_sync(0xffffffffu, at.x, from) + __popc(gt[j] & below);
            const uint32_t t0 = base_tie + __shfl_sync(0xffffffffu, at.y, from) + __popc(tie[j] & below);
            const bool above = gt[j] >> lane & 1, equal = tie[j] >> lane & 1;
            if (above || (equal && t0 < ties)) list[g0 + min(t0, ties)] = n0 + tile * kTile + 32 * (32 * j + warp) + lane;
        }
        base_gt += __shfl_sync(0xffffffffu, incl.x, 31);
        base_tie += __shfl_sync(0xffffffffu, incl.y, 31);
    }
    if (ranks > 1 && !all) cluster_wait();    // no CTA leaves while another reads its counts
}

__global__ void __launch_bounds__(kGatherThreads) evict_gather_kernel(EvictArgs a) {
    // Byte offsets of the rows: K, V (from -1: zeros, to -1: nothing).  A row of a page outside
    // the pool is read from the page that cache_row puts in its place, never written there.
    __shared__ int64_t from[2][kRows], to[2][kRows];
    const int d0 = blockIdx.x * kRows, g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int kept = min(segment_length(a, b), a.keep), rows = min(kRows, a.keep - d0);
    const int d = d0 + tid;
    float mass = 0.f;
    int position = 0;
    grid_dependency_wait();
    if (tid < rows) {
        const bool some = d < kept;
        const int n = some ? a.kept[int64_t(b * a.kv_heads + g) * a.list_rows + d] : 0;
        int64_t ip = 0, op;
        int ir = 0, orow;
        const bool in = !some || cache_row(a.in, b, n, ip, ir), out = cache_row(a.out, b, d, op, orow);
        from[0][tid] = some ? ip * a.in.k_stride[0] + ir * a.in.k_stride[1] + g * a.in.k_stride[2] : -1;
        from[1][tid] = some ? ip * a.in.v_stride[0] + ir * a.in.v_stride[1] + g * a.in.v_stride[2] : -1;
        to[0][tid] = out ? op * a.out.k_stride[0] + orow * a.out.k_stride[1] + g * a.out.k_stride[2] : -1;
        to[1][tid] = out ? op * a.out.v_stride[0] + orow * a.out.v_stride[1] + g * a.out.v_stride[2] : -1;
        if (!in || !out) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
        // On their way while the rows move.
        if (some && a.out_mass) mass = __ldg(a.mass + b * a.mass_stride[0] + g * a.mass_stride[1] + n);
        if (some && a.out_positions) position = __ldg(a.positions + b * a.positions_stride[0] + g * a.positions_stride[1] + n);
    }
    __syncthreads();
    // 16-byte units of the rows' K and V, kUnits of a thread under way at a time.  In a graph, 3 / 4 /
    // 5 / 8 of them: 16 x 32k rows of 320 dims 75.6 / 74.7 / 73.8 / 74.2 us, 16 x 8 heads of 8k rows of
    // 128 dims 112 / 106 / 106 / 116, 4 x 4 heads of 40k rows of 64 dims 63 / 66 / 66 / 72, 8 x 50k rows of
    // 160 dims 76.6 / 80.7 / 75.0 / 78.4 (best where they divide the 32 rows' units), 1.2k rows 12.4 with all.
    constexpr int kUnits = 5;
    const int units = a.k_units + a.v_units, total = rows * units;
    // p / units by multiplication: exact while p units < 2^20 (p < kRows units, units <= 181).
    const uint32_t inverse = (1u << 20) / uint32_t(units) + 1u;
    const bool small = units <= 181;
    for (int p0 = tid; p0 < total; p0 += kGatherThreads * kUnits) {
        uint4 w[kUnits];
        uint4* dst[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int p = p0 + k * kGatherThreads;
            dst[k] = nullptr;
            if (p >= total) continue;
            const int r = small ? int(uint32_t(p) * inverse >> 20) : p / units;
            int u = p - r * units;
            const int is_v = u >= a.k_units;
            if (is_v) u -= a.k_units;
            const int64_t i = from[is_v][r], o = to[is_v][r];
            if (o >= 0) dst[k] = reinterpret_cast<uint4*>((is_v ? a.out_v : a.out_k) + o) + u;
            w[k] = make_uint4(0, 0, 0, 0);
            if (i >= 0 && o >= 0) w[k] = __ldcs(reinterpret_cast<const uint4*>((is_v ? a.v : a.k) + i) + u);
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k)
            if (dst[k]) __stcs(dst[k], w[k]);
    }
    if (tid < rows) {
        if (a.out_mass) a.out_mass[b * a.out_mass_stride[0] + g * a.out_mass_stride[1] + d] = mass;
        if (a.out_positions) a.out_positions[b * a.out_positions_stride[0] + g * a.out_positions_stride[1] + d] = position;
    }
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

// Rows are read while others are written, so no output row may lie over an input row (`rows` to a segment).
bool output_shares_input(const slimkv_evict_args* a, int rows) {
    const int e = a->elem_bytes;
    slimkv_cache in = a->in, out = a->out;
    if (!in.table) in.rows = rows;
    if (!out.table) out.rows = a->keep;
    auto part = [&](const slimkv_cache& c, bool is_v) {
        return cache_rows(is_v ? c.v : c.k, is_v ? c.v_stride : c.k_stride, int64_t(is_v ? a->dim_v : a->dim_qk) * e, e, c, a->batch, a->kv_heads);
    };
    auto plane = [&](const void* at, const int64_t* strides, int n) {
        return Rows{at, int64_t(n) * 4, {1, 1, a->batch, a->kv_heads}, {0, 0, strides[0] * 4, strides[1] * 4}};
    };
    for (bool o : {false, true})
        for (bool i : {false, true})
            if (share_rows(part(out, o), part(in, i))) return true;
    return (a->out_mass && share_rows(plane(a->out_mass, a->out_mass_stride, a->keep), plane(a->mass, a->mass_stride, rows))) ||
           (a->positions && share_rows(plane(a->out_positions, a->out_positions_stride, a->keep), plane(a->positions, a->positions_stride, rows)));
}

void carve(Carver& c, const slimkv_evict_args* a, EvictArgs& k) {
    k.list_rows = std::min(evict_rows(a), a->keep);
    k.kept = c.take<int32_t>(size_t(a->batch) * a->kv_heads * k.list_rows);
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_evict_workspace_size(const slimkv_evict_args* a) {
    if (check_evict(a) != SLIMKV_OK) return 0;
    EvictArgs k{};
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
    k.new_lengths = a->new_lengths;
    k.status = status_word();
    Carver c(workspace, workspace_bytes);
    carve(c, a, k);
    if (!workspace || !c.fits() || reinterpret_cast<uintptr_t>(workspace) % 8)
        return fail(SLIMKV_ERR_WORKSPACE, "evict: workspace of %zu bytes needed", c.used);
    // A block would read a length that another has written.
    const size_t lengths_bytes = size_t(a->batch) * sizeof(int32_t);
    if (share_bytes(a->lengths, lengths_bytes, a->new_lengths, lengths_bytes))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: new_lengths must not be lengths");
    const int64_t *ks = a->out.k_stride, *vs = a->out.v_stride;
    if (!a->out.table && ((a->batch > 1 && (ks[0] == 0 || vs[0] == 0)) || (a->keep > 1 && (ks[1] == 0 || vs[1] == 0)) ||
                          (a->kv_heads > 1 && (ks[2] == 0 || vs[2] == 0))))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: each output row needs its own place (no stride of 0)");
    if (output_shares_input(a, k.rows))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "evict: the output must not overlap the input");
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
    cfg.gridDim = dim3((a->keep - 1) / kRows + 1, a->kv_heads, a->batch);
    cfg.blockDim = dim3(kGatherThreads);
    cfg.attrs = &dependent;
    if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, evict_gather_kernel, k);
    return err == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "evict launch failed: %s", cudaGetErrorString(err));
}
