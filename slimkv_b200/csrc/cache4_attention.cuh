// What the two kernels of attention over a 4-bit cache share: the call, its work
// in pieces, and the merge of the pieces.
#pragma once

#include "bounded_wait.cuh"
#include "cache4.cuh"
#include "cache_view.cuh"
#include "host_utils.h"
#include "key_shares.cuh"
#include "node_mask.cuh"

namespace slimkv {
namespace attention4 {

constexpr float kLazyLog2 = 8.f;                 // O is rescaled when a score passes the row's maximum by 2^8
// P = 2^(s - m), m this far below the maximum: of fp16's exponents P uses those up to 2^15.
template <bool kHalf>
constexpr float kDownLog2 = kHalf ? 7.f : 0.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994530942f;

struct Job {
    int batch, nodes, heads, kv_heads, group;
    FastDiv group_div, page_div;    // by the query heads of a KV head, by the rows of a page
    int rows, row_groups;       // query rows of a KV head, and groups of row_tile of them
    int row_tile;
    int kg, vg;                 // groups of 32 dims of a K and a V row
    int k_pitch, v_pitch;       // bytes of a row
    int context_only, paged, shared_cache, box;
    CacheView cache;
    const uint8_t* v;
    int64_t capacity;
    const int32_t *lengths, *nodes_len, *mask;
    int64_t mask_stride;
    int words;
    float scale_log2;
    const uint16_t* q;
    int64_t q_sb, q_st, q_sh;
    uint16_t* out;
    int64_t o_sb, o_st, o_sh;
    float* lse;
    float* part_o;              // [2 ctas][8 NT][dim_v]
    float* part_lse;            // [2 ctas][8 NT], log2
    int ctas;
    unsigned int* status;
    uint64_t wait_ns;
};

// ------------------------------------------------------------- schedule --
struct Seq {
    int len, nodes, end;        // keys: rows [0, end), the context and then the nodes' own
    int tiles, groups;          // groups of row tiles with live rows
};
// NT: row tiles (8 rows) of a segment, kKeys: keys of a tile.
template <int NT, int kKeys>
struct Plan {
    // What a further piece costs, in tiles.
    static constexpr int kPieceUnits = NT >= 4 ? 4 : 2;
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
        s.groups = (s.nodes * J.group + 8 * NT - 1) / (8 * NT);
        return s;
    }
};

template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kHalf) {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        return pack_bf16x2(lo, hi);
    }
}
// Merges the pieces of a segment's rows (a block each), and writes the rows
// that see nothing.  The four warps take the pieces by turns, a lane four dims.
// Pieces whose weight underflows to 0 stay out of the sums (what overflowed in
// them must not count); only NaN of theirs is looked for afterwards, since 0 x NaN
// is NaN, as it is within a piece.
template <int NT, int kKeys, bool kHalf>
__global__ void __launch_bounds__(128) combine_kernel(const __grid_constant__ Job J) {
    constexpr int kRows = 8 * NT;
    __shared__ int range[3];                // first and last CTA of the segment's pieces, slot of the first
    __shared__ float4 acc[4][kMaxDims4 / 4];
    __shared__ float tops[4], sums[4], lows[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int at = blockIdx.x;
    const int group = at % J.row_groups;
    at /= J.row_groups;
    const int g = at % J.kv_heads, b = at / J.kv_heads, r = group * kRows + blockIdx.y;
    const Plan<NT, kKeys> plan(J);
    const Seq s = plan.sequence(b);
    const bool some = group < s.groups && s.tiles > 0;
    if (some && warp == 0) {
        uint32_t total, before;
        sum_units(plan, b, total, before);
        if (lane == 0) {
            const uint32_t units = segment_units(plan, s), u0 = before + uint32_t(g * s.groups + group) * units;
            const uint32_t ctas = share_count(total, J.ctas), c0 = share_of(total, u0 + Plan<NT, kKeys>::kPieceUnits, ctas);
            range[0] = int(c0);
            range[1] = int(share_of(total, u0 + units - 1, ctas));
            range[2] = 2 * int(c0) + (share_begin(total, c0, ctas) < u0 ? 1 : 0);   // a piece of another segment before it
        }
    }
    if (tid == 32 && g == 0 && group == 0 && blockIdx.y == 0) {
        const int len = __ldg(J.lengths + b), nodes = J.nodes_len ? __ldg(J.nodes_len + b) : J.nodes;
        if (len != s.len || nodes != s.nodes || (!J.context_only && s.end != s.len + s.nodes)) report(J.status, SLIMKV_DEVICE_BAD_LENGTH);
    }
    __syncthreads();
    const int c0 = some ? range[0] : 0, c1 = some ? range[1] : 0, slot0 = some ? range[2] : 0;
    grid_dependency_wait();                 // every block: what follows this grid counts on the one before it too
    if (r >= J.rows || (some && c0 == c1)) return;
    const int node = r / J.group, h = g * J.group + r - node * J.group, dims = J.vg * kGroupDims;
    uint16_t* out = J.out + b * J.o_sb + node * J.o_st + h * J.o_sh;
    float* lse = J.lse + (int64_t(b) * J.nodes + node) * J.heads + h;
    if (!some || node >= s.nodes) {
        for (int d = 8 * tid; d < dims; d += 8 * 128) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
        if (tid == 0) *lse = -INFINITY;
        return;
    }
    // In one pass, the largest exponent so far taken out: a piece's lse and rows are one latency.
    constexpr int kAhead = 4, kSpan = (kMaxDims4 + 127) / 128;
    float m = -INFINITY, sum = 0.f, low = INFINITY;     // low: of the pieces that saw anything
    float4 x[kSpan];
#pragma unroll
    for (int k = 0; k < kSpan; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0 + warp; c <= c1; c += 4 * kAhead) {
        float w[kAhead];
        float4 y[kAhead][kSpan];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            w[a] = -INFINITY;
            const int cc = c + 4 * a;
            if (cc > c1) continue;
            const int64_t row = int64_t(cc == c0 ? slot0 : 2 * cc) * kRows + blockIdx.y;
            w[a] = __ldcg(J.part_lse + row);
#pragma unroll
            for (int k = 0; k < kSpan; ++k)
                if (4 * lane + 128 * k < dims) y[a][k] = __ldcg(reinterpret_cast<const float4*>(J.part_o + row * dims) + lane + 32 * k);
        }
        const float before = m;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            m = fmaxf(m, w[a]);
            if (w[a] != -INFINITY) low = fminf(low, w[a]);
        }
        const float shift = m == -INFINITY ? 0.f : m, old = before == -INFINITY ? 0.f : sfu_exp2(before - shift);
        if (before != -INFINITY) {
            sum *= old;
#pragma unroll
            for (int k = 0; k < kSpan; ++k) { x[k].x *= old; x[k].y *= old; x[k].z *= old; x[k].w *= old; }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const float f = sfu_exp2(w[a] - shift);
            sum += f;
            if (f == 0.f) continue;
#pragma unroll
            for (int k = 0; k < kSpan; ++k)
                if (4 * lane + 128 * k < dims) {
                    x[k].x = fmaf(f, y[a][k].x, x[k].x); x[k].y = fmaf(f, y[a][k].y, x[k].y);
                    x[k].z = fmaf(f, y[a][k].z, x[k].z); x[k].w = fmaf(f, y[a][k].w, x[k].w);
                }
        }
    }
#pragma unroll
    for (int k = 0; k < kSpan; ++k)
        if (4 * lane + 128 * k < dims) acc[warp][lane + 32 * k] = x[k];
    if (lane == 0) { tops[warp] = m; sums[warp] = sum; lows[warp] = low; }
    __syncthreads();
    const float all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), shift = all == -INFINITY ? 0.f : all;
    float f[4], l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        f[k] = tops[k] == -INFINITY ? (sums[k] == 0.f ? 0.f : sums[k]) : sfu_exp2(tops[k] - shift);     // (NaN stays)
        l += tops[k] == -INFINITY ? sums[k] : f[k] * sums[k];
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const bool light = fminf(fminf(lows[0], lows[1]), fminf(lows[2], lows[3])) < all - 120.f;      // (of some the weight may be 0)
    for (int d = 8 * tid; d < dims; d += 8 * 128) {
        float4 y[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            y[half] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (f[k] == 0.f) continue;
                const float4 z = acc[k][d / 4 + half];
                y[half].x = fmaf(f[k], z.x, y[half].x); y[half].y = fmaf(f[k], z.y, y[half].y);
                y[half].z = fmaf(f[k], z.z, y[half].z); y[half].w = fmaf(f[k], z.w, y[half].w);
            }
        }
        for (int c = c0; light && c <= c1; ++c) {
            const int64_t row = int64_t(c == c0 ? slot0 : 2 * c) * kRows + blockIdx.y;
            if (__ldcg(J.part_lse + row) == -INFINITY) continue;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float4 z = __ldcg(reinterpret_cast<const float4*>(J.part_o + row * dims + d) + half);
                if (z.x != z.x) y[half].x = z.x;
                if (z.y != z.y) y[half].y = z.y;
                if (z.z != z.z) y[half].z = z.z;
                if (z.w != z.w) y[half].w = z.w;
            }
        }
        *reinterpret_cast<uint4*>(out + d) =
            make_uint4(pack2<kHalf>(y[0].x * inv, y[0].y * inv), pack2<kHalf>(y[0].z * inv, y[0].w * inv),
                       pack2<kHalf>(y[1].x * inv, y[1].y * inv), pack2<kHalf>(y[1].z * inv, y[1].w * inv));
    }
    if (tid == 0) *lse = l != 0.f ? (shift + log2f(l)) * kLn2 : -INFINITY;
}

// The launch of the merge behind a kernel.
template <int NT, int kKeys, bool kHalf>
int launch_combine(const Job& J, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(J.batch * J.kv_heads * J.row_groups, J.rows < 8 * NT ? J.rows : 8 * NT);
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute dependent{};
    dependent.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    dependent.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &dependent;
    cfg.numAttrs = 1;
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, combine_kernel<NT, kKeys, kHalf>, J);
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "4-bit attention launch failed: %s", cudaGetErrorString(e));
}

// Many query rows and dims (cache4_attention_wide.cu): query rows of a pass, keys of a tile, and
// rows of a TMA box at most.
constexpr int kWideRows = 32, kWideKeys = 128, kWideBox = 64;
int launch_wide(const CUtensorMap& km, const CUtensorMap& vm, const Job& J, bool half, cudaStream_t stream);

}  // namespace attention4
}  // namespace slimkv
