// The steps around the attention of a drafted tree (C ABI slimkv_tree_masks,
// slimkv_tree_accept, slimkv_tree_commit): the ancestor words of a tree, its
// greedy acceptance, and the move of the accepted rows next to the context.
#include <algorithm>
#include <cstdlib>

#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

// ------------------------------------------------------------ tree masks --
// One thread per node: walk up the parents (each below its child, so the walk
// ends) and set their bits in the node's own row of words.
__global__ void tree_masks_kernel(const int32_t* parents, int nodes, int words, int32_t* masks) {
    const int t = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
    if (t >= nodes) return;
    const int32_t* par = parents + int64_t(b) * nodes;
    int32_t* row = masks + (int64_t(b) * nodes + t) * words;
    int at = t;
    for (int w = words - 1; w >= 0; --w) {          // ancestors descend: one word after the other
        uint32_t bits = 0;
        while (at >= 32 * w && at >= 0) {
            bits |= 1u << (at & 31);
            const int p = __ldg(par + at);
            at = p < at ? p : -1;
        }
        row[w] = int32_t(bits);
    }
}

// ---------------------------------------------------------------- argmax --
// The largest logit of a row as one 64-bit number: its order-preserving bits
// (NaN above everything, the two zeros equal) over the complement of its
// index, so that a maximum of them takes the lowest index of equal values.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : (u >> 31 ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// What the threads of a block exchange in scan_row.
template <int kThreads>
struct ScanScratch {
    uint32_t keys[kThreads / 32];
    uint32_t index;
};

// The best of elements [lo, hi) of a row, over the threads of a block (0: no
// elements).  A thread keeps its largest value and the vector that holds it
// (its elements come in ascending order, so an equal one is not wanted); only
// the thread with the block's largest looks for the element.
template <typename T, int kThreads>
__device__ __forceinline__ uint64_t scan_row(const T* row, int lo, int hi, ScanScratch<kThreads>* scratch) {
    constexpr int kN = 16 / int(sizeof(T));
    const int lead = int(((16 - (reinterpret_cast<uintptr_t>(row + lo) & 15)) & 15) / sizeof(T));
    const int body = min(lo + lead, hi);
    const int vectors = (hi - body) / kN, tail = body + vectors * kN;
    float top = 0.f;
    bool some = false;
    uint32_t at = 0;
    alignas(16) T best[kN];
    auto better = [&](float m) { return !some || m > top || (m != m && top == top); };
    auto one = [&](int i) {
        const T x = row[i];
        if (!better(to_float(x))) return;
        some = true;
        top = to_float(x);
        at = uint32_t(i);
#pragma unroll
        for (int e = 0; e < kN; ++e) best[e] = x;
    };
    if (threadIdx.x == 0) scratch->index = 0xffffffffu;
    for (int i = lo + int(threadIdx.x); i < body; i += kThreads) one(i);
    const uint4* v = reinterpret_cast<const uint4*>(row + body);
    for (int i = threadIdx.x; i < vectors; i += 4 * kThreads) {
        uint4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * kThreads < vectors) w[k] = __ldg(v + i + k * kThreads);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k * kThreads >= vectors) continue;
            const T* x = reinterpret_cast<const T*>(&w[k]);
            float m = to_float(x[0]);
#pragma unroll
            for (int e = 1; e < kN; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(to_float(x[e])));
            if (better(m)) {
                some = true;
                top = m;
                at = uint32_t(body + (i + k * kThreads) * kN);
                *reinterpret_cast<uint4*>(best) = w[k];
            }
        }
    }
    for (int i = tail + int(threadIdx.x); i < hi; i += kThreads) one(i);
    const uint32_t key = some ? key_of(top) : 0u, of_warp = __reduce_max_sync(0xffffffffu, key);
    if ((threadIdx.x & 31) == 0) scratch->keys[threadIdx.x >> 5] = of_warp;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const uint32_t largest = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? scratch->keys[lane] : 0u);
    if (some && key == largest) {
        uint32_t first = 0;
#pragma unroll
        for (int e = kN - 1; e >= 0; --e)
            if (key_of(to_float(best[e])) == largest) first = uint32_t(e);
        atomicMin(&scratch->index, at + first);
    }
    __syncthreads();
    return uint64_t(largest) << 32 | uint32_t(~scratch->index);
}

// (96 bytes: with 104 a launch cost the host 0.3 us more, the Python call 0.9.)
struct AcceptArgs {
    int nodes, vocab, splits;
    int max_steps;              // nodes after which the walk with its argmaxes stops (all: never)
    const void* logits;
    int64_t stride_batch, stride_node;
    const int64_t* tokens;
    const int32_t* parents;
    const int32_t* nodes_len;
    int32_t* path;
    int32_t* count;
    int64_t* next;
    uint64_t* best;             // [batch][nodes][splits]; before it what resume_of says
    __device__ __forceinline__ bool stops() const { return max_steps < nodes; }
    // Where a walk that stops would go on: its next node (-1: it is over) and the steps taken.
    __device__ __forceinline__ int2& resume_of(int b) const { return reinterpret_cast<int2*>(best)[-1 - b]; }
};

constexpr int kScanThreads = 256;

// Every node's argmax, its vocabulary split over gridDim.x blocks; after a walk
// that stopped, of the nodes from its last on (children come after their parents).
template <typename T>
__global__ void __launch_bounds__(kScanThreads) accept_scan_kernel(AcceptArgs a) {
    __shared__ ScanScratch<kScanThreads> scratch;
    const int t = blockIdx.y, b = blockIdx.z;
    grid_launch_dependents();               // the walk over the argmaxes, which waits for this grid
    if (a.stops()) {
        grid_dependency_wait();
        const int from = a.resume_of(b).x;
        if (from < 0 || t < from) return;
    }
    if (a.nodes_len && t >= __ldg(a.nodes_len + b)) return;
    const T* row = static_cast<const T*>(a.logits) + b * a.stride_batch + t * a.stride_node;
    const int lo = int(int64_t(a.vocab) * blockIdx.x / a.splits), hi = int(int64_t(a.vocab) * (blockIdx.x + 1) / a.splits);
    const uint64_t best = scan_row<T, kScanThreads>(row, lo, hi, &scratch);
    if (threadIdx.x == 0) a.best[(int64_t(b) * a.nodes + t) * a.splits + blockIdx.x] = best;
}

// The walk over every node's argmax, in shared memory: a block per sequence
// gathers the nodes, its first warp walks.
constexpr int kWalkThreads = 128, kMaxNodes = 1024;

__global__ void __launch_bounds__(kWalkThreads) accept_walk_kernel(AcceptArgs a) {
    __shared__ int32_t parents[kMaxNodes], tokens[kMaxNodes], best[kMaxNodes];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const int n = a.nodes_len ? min(max(__ldg(a.nodes_len + b), 0), a.nodes) : a.nodes;
    for (int i = tid; i < n; i += kWalkThreads) {
        parents[i] = __ldg(a.parents + int64_t(b) * a.nodes + i);
        // A token outside the vocabulary matches nothing.
        const int64_t token = __ldg(a.tokens + int64_t(b) * a.nodes + i);
        tokens[i] = token >= 0 && token < a.vocab ? int(token) : -1;
    }
    grid_dependency_wait();
    const int2 start = a.stops() ? a.resume_of(b) : make_int2(n > 0 ? 0 : -1, 0);
    if (a.stops() && start.x < 0) return;               // the walk before has written everything
    for (int i = max(start.x, 0) + tid; i < n; i += kWalkThreads) {
        uint64_t top = 0;
        for (int k = 0; k < a.splits; ++k) top = max_u64(top, a.best[(int64_t(b) * a.nodes + i) * a.splits + k]);
        best[i] = int(~uint32_t(top));
    }
    __syncthreads();
    if (tid >= 32) return;
    int32_t* path = a.path + int64_t(b) * a.nodes;
    int cur = start.x, len = start.y, next = -1;
    while (cur >= 0) {
        if (lane == 0) path[len] = cur;
        ++len;
        next = best[cur];
        int child = -1;
        for (int c0 = cur + 1; c0 < n && child < 0; c0 += 32) {
            const int c = c0 + lane;
            const unsigned hit = __ballot_sync(0xffffffffu, c < n && parents[c] == cur && tokens[c] == next);
            if (hit) child = c0 + __ffs(int(hit)) - 1;
        }
        cur = child;
    }
    for (int i = len + lane; i < a.nodes; i += 32) path[i] = -1;
    if (lane == 0) {
        a.count[b] = len;
        a.next[b] = next;
    }
}

// The walk with each node's argmax taken when the walk gets there: a cluster of
// CTAs per sequence, each scanning its part of the vocabulary, their results
// exchanged over distributed shared memory.  Reads the logits of the accepted
// path alone; a step is one pass over V / 8 logits and one cluster barrier.  After
// max_steps nodes it leaves the rest to the two kernels above.
constexpr int kPathCtas = 8, kPathThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kPathThreads) accept_path_kernel(AcceptArgs a) {
    __shared__ int64_t tokens[kMaxNodes];
    __shared__ int32_t parents[kMaxNodes];
    __shared__ ScanScratch<kPathThreads> scratch;
    __shared__ uint64_t of_rank[2][kPathCtas];          // by the step's parity
    __shared__ int child[2];
    const uint32_t rank = cluster_rank();
    cluster_arrive();                                   // the others run, before anything is stored to them
    const int b = blockIdx.x / kPathCtas, tid = threadIdx.x;
    const int n = a.nodes_len ? min(max(__ldg(a.nodes_len + b), 0), a.nodes) : a.nodes;
    for (int i = tid; i < n; i += kPathThreads) {
        tokens[i] = __ldg(a.tokens + int64_t(b) * a.nodes + i);
        parents[i] = __ldg(a.parents + int64_t(b) * a.nodes + i);
    }
    if (tid < 2) child[tid] = kMaxNodes;
    const int lo = int(int64_t(a.vocab) * rank / kPathCtas), hi = int(int64_t(a.vocab) * (rank + 1) / kPathCtas);
    int32_t* path = a.path + int64_t(b) * a.nodes;
    int cur = n > 0 ? 0 : -1, len = 0;
    int64_t next = -1;
    cluster_wait();
    if (a.stops()) grid_launch_dependents();
    while (cur >= 0 && len < a.max_steps) {
        const int parity = len & 1;
        if (rank == 0 && tid == 0) path[len] = cur;
        ++len;
        __syncthreads();
        const uint64_t best = scan_row<T, kPathThreads>(
            static_cast<const T*>(a.logits) + b * a.stride_batch + cur * a.stride_node, lo, hi, &scratch);
        if (tid < kPathCtas) cluster_store(&of_rank[parity][rank], tid, best);
        cluster_sync();
        uint64_t all = of_rank[parity][0];
#pragma unroll
        for (int r = 1; r < kPathCtas; ++r) all = max_u64(all, of_rank[parity][r]);
        next = int64_t(uint32_t(~uint32_t(all)));
        for (int c = cur + 1 + tid; c < n; c += kPathThreads)
            if (parents[c] == cur && tokens[c] == next) atomicMin(&child[parity], c);
        if (tid == 0) child[parity ^ 1] = kMaxNodes;    // of the step before: read by all before the cluster barrier
        __syncthreads();
        cur = child[parity] < kMaxNodes ? child[parity] : -1;
    }
    if (rank == 0 && tid == 0 && a.stops()) a.resume_of(b) = make_int2(cur, len);
    if (rank == 0 && cur < 0) {
        for (int i = len + tid; i < a.nodes; i += kPathThreads) path[i] = -1;
        if (tid == 0) {
            a.count[b] = len;
            a.next[b] = next;
        }
    }
    cluster_sync();                                     // no CTA leaves while another may still store to it
}

// Scanning every node reads all the logits, the walk with its argmaxes takes 2.3
// us a step (bf16, in a graph, logits up to L2's size read again from there, as
// after the product that wrote them).  Scan / walk with so many nodes accepted:
//   1 x 64 of 128256 (16 MB)     10.1 / 17.9 (7)    20.1 / 142 (all 64)
//   16 x 8 of 128256 (33 MB)     11.4 / 22.8 (all 8)
//   64 x 16 of 32000 (66 MB)     14.0 / 41.6 (8)
//   8 x 32 of 128256 (66 MB)     14.0 / 21.0 (8)    18.2 / 73.2 (all 32)
//   64 x 8 of 128256 (131 MB)    26.6 / 10.4 (1)    27.7 / 56.2 (all 8)
//   16 x 64 of 128256 (263 MB)   48.3 / 22.8 (8)    58.1 / 185 (all 64)
//   1 x 1024 of 33001 (68 MB)    22.6 / 21.6 (8)    197 / 2521 (all 1024)
// So small logits are scanned.  Of larger ones most trees' paths are cheaper to
// walk, but nothing on the host bounds a path below the number of nodes: where a
// walk over all of them could cost more than four scans, it stops after as many
// steps as cost about one scan, and a scan of the nodes behind it ends the path
// (1 x 1024 of 33001: 25.2 (8), 210 (all); 4 x 70 of 64001 fp32, 72 MB: 24.1 (8),
// 42.4 (all), 164 by walking alone).  The launches that have nothing left to do
// cost 3 to 4 us.
constexpr int64_t kScanAllBytes = int64_t(64) << 20;
constexpr int64_t kStepBytes = 13000000;    // scanned in a step's time
int64_t accept_bytes(const slimkv_tree_accept_args* a) {
    return int64_t(a->batch) * a->nodes * a->vocab * (a->type == SLIMKV_FP32 ? 4 : 2);
}
bool accept_scans_all(const slimkv_tree_accept_args* a) { return accept_bytes(a) <= kScanAllBytes; }
// Steps of a walk: all, or those that cost about a scan.
int accept_steps(const slimkv_tree_accept_args* a) {
    const int64_t of_a_scan = std::max<int64_t>(8, accept_bytes(a) / kStepBytes);
    return a->nodes <= 4 * of_a_scan ? a->nodes : int(of_a_scan);
}

int accept_splits(const slimkv_tree_accept_args* a) {
    // Blocks of at least 4096 logits, about eight per SM over all rows.
    const int64_t rows = int64_t(a->batch) * a->nodes;
    const int64_t want = (int64_t(device_info().sm_count) * 8 + rows - 1) / rows;
    return int(std::max<int64_t>(1, std::min<int64_t>(want, a->vocab / 4096)));
}

void carve_accept(Carver& c, const slimkv_tree_accept_args* a, AcceptArgs& k) {
    k.nodes = a->nodes;
    k.splits = accept_splits(a);
    const bool all = accept_scans_all(a);
    k.max_steps = all ? a->nodes : accept_steps(a);
    const bool stops = k.max_steps < k.nodes;
    const size_t first = stops ? a->batch : 0;          // resume_of's entries
    if (all || stops) k.best = c.take<uint64_t>(first + size_t(a->batch) * a->nodes * k.splits) + first;
}

int check_accept(const slimkv_tree_accept_args* a) {
    if (!a) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->batch < 1 || a->batch > 65535 || a->nodes < 1 || a->nodes > 1024 || a->vocab < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree accept: batch in 1..65535, nodes in 1..1024, vocab >= 1");
    if (a->type != SLIMKV_BF16 && a->type != SLIMKV_FP16 && a->type != SLIMKV_FP32)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree accept: unknown logits type %d", a->type);
    return SLIMKV_OK;
}

// ---------------------------------------------------------------- commit --
struct CommitArgs {
    uint8_t *k, *v;
    CacheView cache;            // strides in bytes
    int64_t k_layer, v_layer;   // bytes
    int kv_heads, k_units, v_units, lanes;      // 16-byte units of a K / V row; lanes of one layer
    int layers, nodes;
    const int32_t *lengths, *path, *count;
    int32_t* new_lengths;
    unsigned int* status;
};

// Latency and HBM: one layer of one sequence 3.0 us in a graph, 32 layers of 16
// sequences with 1 to 7 accepted rows 5.6 us (2.1 us for their bytes).
constexpr int kCommitRows = 8;

// One thread per 16-byte column of a (layer, K or V, head): rows move in
// ascending order, kCommitRows loaded before they are stored.  path[i] >= i
// ascends, so a row is read before a later one is written over it.
__global__ void __launch_bounds__(256) tree_commit_kernel(CommitArgs a) {
    const int b = blockIdx.y;
    const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int len = __ldg(a.lengths + b), want = __ldg(a.count + b);
    const int count = min(max(want, 0), a.nodes);
    const int64_t cap = cache_capacity(a.cache);
    if (at == 0) {
        const int64_t end = int64_t(max(len, 0)) + count;
        a.new_lengths[b] = int(min(end, cap));
        if (want != count || len < 0 || end > cap) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    if (at >= int64_t(a.layers) * a.lanes || len < 0) return;
    const int layer = int(at / a.lanes);
    int lane = int(at - int64_t(layer) * a.lanes);
    const bool is_v = lane >= a.kv_heads * a.k_units;
    if (is_v) lane -= a.kv_heads * a.k_units;
    const int units = is_v ? a.v_units : a.k_units, head = lane / units;
    const int64_t* st = is_v ? a.cache.v_stride : a.cache.k_stride;
    uint8_t* base = (is_v ? a.v + layer * a.v_layer : a.k + layer * a.k_layer) + head * st[2] + int64_t(lane - head * units) * 16;
    const int32_t* path = a.path + int64_t(b) * a.nodes;
    for (int i0 = 0; i0 < count; i0 += kCommitRows) {
        uint4 row[kCommitRows];
        bool move[kCommitRows];
#pragma unroll
        for (int j = 0; j < kCommitRows; ++j) {
            const int i = i0 + j;
            move[j] = i < count;
            if (!move[j]) continue;
            const int p = __ldg(path + i);
            int64_t page;
            int r;
            // Both the row's place and its source (the same when p == i) have to exist.
            if (p < i || p >= a.nodes || int64_t(len) + p >= cap || !cache_row(a.cache, b, len + i, page, r) ||
                !cache_row(a.cache, b, len + p, page, r)) {
                report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
                move[j] = false;
                continue;
            }
            move[j] = p != i;
            if (!move[j]) continue;
            row[j] = *reinterpret_cast<const uint4*>(base + page * st[0] + r * st[1]);
        }
#pragma unroll
        for (int j = 0; j < kCommitRows; ++j) {
            int64_t page;
            int r;
            if (move[j] && cache_row(a.cache, b, len + i0 + j, page, r))
                *reinterpret_cast<uint4*>(base + page * st[0] + r * st[1]) = row[j];
        }
    }
}

}  // namespace

// Checks of a cache whose rows are moved as 16-byte units; see host_utils.h.
int check_cache(const slimkv_cache& c, int batch, int dim_k, int dim_v, int elem_bytes, bool need_v, const char* what) {
    if (!c.k || (need_v && !c.v)) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: null cache", what);
    if (c.rows < 1) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: the cache needs rows", what);
    if (c.table && (c.table_pages < 1 || c.num_pages < 1 || (batch > 1 && c.table_stride < c.table_pages && c.table_stride != 0) ||
                    int64_t(c.rows) * c.table_pages > 0x7fffffffLL))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: block tables need pages, their stride and fewer than 2^31 rows", what);
    if (dim_k < 1 || (need_v && dim_v < 1)) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: dims must be positive", what);
    bool ok = aligned16(c.k) && int64_t(dim_k) * elem_bytes % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && c.k_stride[i] * elem_bytes % 16 == 0 && c.k_stride[i] >= 0;
    if (need_v) {
        ok = ok && aligned16(c.v) && int64_t(dim_v) * elem_bytes % 16 == 0;
        for (int i = 0; i < 3; ++i) ok = ok && c.v_stride[i] * elem_bytes % 16 == 0 && c.v_stride[i] >= 0;
    }
    return ok ? SLIMKV_OK : fail(SLIMKV_ERR_ALIGNMENT, "%s: cache pointers, strides and rows must be multiples of 16 bytes", what);
}

}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_tree_masks(const int32_t* parents, int batch, int nodes, int32_t* masks, void* stream) {
    if (!parents || !masks) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree masks: null pointer");
    if (batch < 1 || batch > 65535 || nodes < 1 || nodes > 1024)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree masks: batch in 1..65535, nodes in 1..1024");
    const int threads = std::min(256, (nodes + 31) / 32 * 32);
    tree_masks_kernel<<<dim3((nodes + threads - 1) / threads, batch), threads, 0, static_cast<cudaStream_t>(stream)>>>(
        parents, nodes, (nodes + 31) / 32, masks);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "tree masks launch failed: %s", cudaGetErrorString(e));
}

extern "C" size_t slimkv_tree_accept_workspace_size(const slimkv_tree_accept_args* a) {
    if (check_accept(a) != SLIMKV_OK) return 0;
    AcceptArgs k{};
    Carver c(nullptr, 0);
    carve_accept(c, a, k);
    return std::max<size_t>(c.used, 256);
}

extern "C" int slimkv_tree_accept(const slimkv_tree_accept_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_accept(a)) return rc;
    if (!a->logits || !a->tokens || !a->parents || !a->path || !a->count || !a->next)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree accept: null pointer");
    if (a->logits_stride[0] < 0 || a->logits_stride[1] < 0)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree accept: negative strides");
    AcceptArgs k{};
    Carver c(workspace, workspace_bytes);
    carve_accept(c, a, k);
    if (!workspace || workspace_bytes < std::max<size_t>(c.used, 256) || reinterpret_cast<uintptr_t>(workspace) % 8)
        return fail(SLIMKV_ERR_WORKSPACE, "tree accept: workspace too small or misaligned");
    k.vocab = a->vocab;
    k.logits = a->logits;
    k.stride_batch = a->logits_stride[0];
    k.stride_node = a->logits_stride[1];
    k.tokens = a->tokens;
    k.parents = a->parents;
    k.nodes_len = a->nodes_len;
    k.path = a->path;
    k.count = a->count;
    k.next = a->next;
    cudaError_t e = cudaSuccess;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = &attr;
    // The kernel of the logits' type.
    auto launch = [&](int attrs, dim3 grid, int threads, auto bf16, auto fp16, auto fp32) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.numAttrs = attrs;
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, a->type == SLIMKV_BF16 ? bf16 : a->type == SLIMKV_FP16 ? fp16 : fp32, k);
    };
    const bool walks = !accept_scans_all(a);
    if (walks) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kPathCtas;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        launch(1, dim3(unsigned(a->batch) * kPathCtas), kPathThreads, accept_path_kernel<__nv_bfloat16>, accept_path_kernel<__half>,
               accept_path_kernel<float>);
    }
    if (!walks || k.max_steps < k.nodes) {
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        launch(walks, dim3(k.splits, a->nodes, a->batch), kScanThreads, accept_scan_kernel<__nv_bfloat16>, accept_scan_kernel<__half>,
               accept_scan_kernel<float>);
        launch(1, dim3(a->batch), kWalkThreads, accept_walk_kernel, accept_walk_kernel, accept_walk_kernel);
    }
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "tree accept launch failed: %s", cudaGetErrorString(e));
}

extern "C" int slimkv_tree_commit(const slimkv_tree_commit_args* a, void* stream) {
    if (!a || !a->lengths || !a->path || !a->count || !a->new_lengths)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree commit: null pointer");
    if (a->layers < 1 || a->batch < 1 || a->batch > 65535 || a->nodes < 1 || a->nodes > 1024 || a->kv_heads < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree commit: layers, heads >= 1, batch in 1..65535, nodes in 1..1024");
    if (a->elem_bytes != 1 && a->elem_bytes != 2 && a->elem_bytes != 4)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree commit: elements of 1, 2 or 4 bytes");
    if (int rc = check_cache(a->cache, a->batch, a->dim_qk, a->dim_v, a->elem_bytes, true, "tree commit")) return rc;
    const int e = a->elem_bytes;
    if (a->k_layer_stride * e % 16 || a->v_layer_stride * e % 16)
        return fail(SLIMKV_ERR_ALIGNMENT, "tree commit: layer strides must be multiples of 16 bytes");
    if (a->batch > 1 && !a->cache.table && (a->cache.k_stride[0] == 0 || a->cache.v_stride[0] == 0))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree commit: one cache for each sequence, none shared by the batch");
    // A block would read a length that another has written.
    const size_t lengths_bytes = size_t(a->batch) * sizeof(int32_t);
    if (share_bytes(a->lengths, lengths_bytes, a->new_lengths, lengths_bytes))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree commit: new_lengths must not be lengths");
    // K and V may be (parts of) the same rows, which then move once: two threads would each read
    // what the other has moved.
    const slimkv_cache& c = a->cache;
    const Rows k_rows = cache_rows(c.k, c.k_stride, int64_t(a->dim_qk) * e, e, c, a->batch, a->kv_heads, a->layers, a->k_layer_stride);
    const Rows v_rows = cache_rows(c.v, c.v_stride, int64_t(a->dim_v) * e, e, c, a->batch, a->kv_heads, a->layers, a->v_layer_stride);
    int64_t k_bytes = k_rows.width, v_bytes = v_rows.width;
    uint8_t *first = static_cast<uint8_t*>(const_cast<void*>(c.k)), *v = static_cast<uint8_t*>(const_cast<void*>(c.v));
    if (share_rows(k_rows, v_rows)) {
        bool same = share_bytes(first, k_bytes, v, v_bytes);
        uint8_t* end = std::max(first + k_bytes, v + v_bytes);
        first = std::min(first, v);
        k_bytes = end - first;
        v_bytes = 0;
        for (int i = 0; i < 4; ++i)
            same = same && (k_rows.n[i] == 1 || (k_rows.stride[i] == v_rows.stride[i] && std::abs(k_rows.stride[i]) >= k_bytes));
        if (!same) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "tree commit: K and V must be apart, or (parts of) the same rows");
    }
    CommitArgs k{};
    k.k = first;
    k.v = v;
    k.cache = cache_view(a->cache);
    for (int i = 0; i < 3; ++i) { k.cache.k_stride[i] *= e; k.cache.v_stride[i] *= e; }
    k.k_layer = a->k_layer_stride * e;
    k.v_layer = a->v_layer_stride * e;
    k.kv_heads = a->kv_heads;
    k.k_units = int(k_bytes / 16);
    k.v_units = int(v_bytes / 16);
    k.lanes = a->kv_heads * (k.k_units + k.v_units);
    k.layers = a->layers;
    k.nodes = a->nodes;
    k.lengths = a->lengths;
    k.path = a->path;
    k.count = a->count;
    k.new_lengths = a->new_lengths;
    k.status = status_word();
    const int64_t blocks = (int64_t(a->layers) * k.lanes + 255) / 256;
    if (blocks > 0x7fffffff) return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "tree commit: too many rows in one call");
    tree_commit_kernel<<<dim3(unsigned(blocks), a->batch), 256, 0, static_cast<cudaStream_t>(stream)>>>(k);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "tree commit launch failed: %s", cudaGetErrorString(err));
}
