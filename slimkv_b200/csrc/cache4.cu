// Rows quantised into the 4-bit cache, and read back (C ABI
// slimkv_cache4_write, slimkv_cache4_read).
//
// For each group of 32 dims x of a row, in the rows' 16-bit type T:
//   low = min x,  scale = T((max x - low) / 15),  code = rint((x - low) / scale)
// and back T(code * scale + low).  Four neighbouring lanes hold a group, eight
// dims (one 16-byte load) each; the least and largest value go between them by
// two shuffles, and every lane writes the four bytes of its codes.
//
// Bound: reading, HBM (2.625 bytes a value either way); writing, instructions.  So
// a thread keeps its column and a block looks its rows' places up once (with two
// divisions and a table look-up for every eight values reading 16 x 8k latents took
// 62 us), and the quotient is a product with 1 / scale, put right by its exact
// remainder (Markstein's division), which leaves a half a half: a rule of its own
// for ties made the chunk below 56 us in place of 47.  Measured in a graph (bf16): 4
// sequences of 4608 rows of 8 heads of 128 dims, write 31 us = 3.2 TB/s, read 19 us
// = 5.2 TB/s; 4 of 4097 to 5120 rows written and read back 47 us; 16 x 8k latents of
// 320 dims out of pages read 38 us = 5.4 TB/s.
#include <algorithm>
#include <type_traits>

#include "cache4.cuh"
#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

constexpr int kThreads = 256;           // at most
constexpr int kAhead = 4;               // rows that a thread has under way
constexpr int kMaxTurns = 8;            // rows of a thread
constexpr int kMaxRows = kThreads / 4 * kMaxTurns;

// Columns are the eight-dim units of a row's heads; a block has up to 256 of them and as many
// rows side by side as it has threads for, so a thread keeps its column.
struct Part4 {
    int dim, cols, block_cols, side;    // columns in all and of a block, rows side by side
    FastDiv per_block, per_head;        // by block_cols and by a head's columns
    uint16_t* dense;                    // 16-bit rows: read by write, written by read
    int64_t stride[3];
    uint8_t* cache;
    int64_t c_stride[3];                // bytes
};
struct Args4 {
    Part4 part[2];                      // K and V
    int rows, turns;                    // rows of a thread
    FastDiv page;
    CacheView view;
    int64_t capacity;
    const int32_t *starts, *counts;
    int zero_rest;
    unsigned int* status;
};

// A sequence's rows: cache rows [start, start + count), without what the cache cannot hold
// (behind a negative start: none).
__device__ __forceinline__ bool span_of(const Args4& a, int b, int& start, int& count) {
    const int s = a.starts ? __ldg(a.starts + b) : 0, c = a.counts ? __ldg(a.counts + b) : a.rows;
    start = max(s, 0);
    count = s < 0 ? 0 : min(max(c, 0), a.rows);
    const bool fits = s >= 0 && c >= 0 && c <= a.rows && int64_t(start) + count <= a.capacity;
    count = int(max(min(int64_t(count), a.capacity - start), int64_t(0)));
    return fits;
}

// A thread's column, and the places of its block's cache rows (in shared memory).
struct Place {
    int start, count;           // the sequence's
    int first, rows;            // the block's rows
    int row, head, unit;        // the thread's first row of the block; its column
    bool some;                  // it has a column
};
__device__ __forceinline__ Place place_of(const Args4& a, const Part4& p, int chunk, int64_t* at, bool for_write) {
    Place w;
    const int b = blockIdx.y, tid = threadIdx.x;
    if (!span_of(a, b, w.start, w.count) && blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
    // (The grid is the longer row's: of the shorter one's blocks some lie behind all rows, up to 2^32.)
    w.first = int(min(int64_t(blockIdx.x) * (p.side * a.turns), int64_t(a.rows)));
    w.rows = min(p.side * a.turns, w.count - w.first);
    for (int i = tid; i < w.rows; i += blockDim.x) {
        int page = b, r = w.start + w.first + i;
        bool ok = true;
        if (a.view.table) {
            const int n = r, k = int(a.page.div(uint32_t(n)));
            page = __ldg(a.view.table + b * a.view.table_stride + k);
            r = n - k * a.view.rows;
            ok = page >= 0 && page < a.view.num_pages;
            if (!ok) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
            page = min(max(page, 0), a.view.num_pages - 1);
        }
        at[i] = ok || !for_write ? page * p.c_stride[0] + r * p.c_stride[1] : -1;
    }
    w.row = int(p.per_block.div(uint32_t(tid)));
    const int col = chunk * p.block_cols + tid - w.row * p.block_cols;
    w.head = int(p.per_head.div(uint32_t(col)));
    w.unit = col - w.head * (p.dim / 8);
    w.some = w.row < p.side && col < p.cols;
    __syncthreads();
    return w;
}

// The pair and the eight codes of a unit (four lanes: a group).
template <bool kHalf>
__device__ __forceinline__ void quantise(const uint4& raw, uint32_t& word, uint32_t& pair) {
    using P = Pair<kHalf>;
    using T2 = typename P::T2;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    T2 lo = P::as(w[0]), hi = lo;
#pragma unroll
    for (int e = 1; e < 4; ++e) { lo = __hmin2_nan(lo, P::as(w[e])); hi = __hmax2_nan(hi, P::as(w[e])); }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = __hmin2_nan(lo, P::as(__shfl_xor_sync(0xffffffffu, P::bits(lo), o)));
        hi = __hmax2_nan(hi, P::as(__shfl_xor_sync(0xffffffffu, P::bits(hi), o)));
    }
    auto lo1 = __hmin_nan(lo.x, lo.y), hi1 = __hmax_nan(hi.x, hi.y);
    const float low = float(lo1), high = float(hi1);
    // In halves: the difference of two large values has to stay finite.
    decltype(lo1) scale_t;
    if constexpr (kHalf) scale_t = __float2half_rn((0.5f * high - 0.5f * low) / 7.5f);
    else scale_t = __float2bfloat16_rn((0.5f * high - 0.5f * low) / 7.5f);
    float scale = float(scale_t);
    constexpr float kLargest = kHalf ? 65504.f : 3.3895313892515355e38f;
    // What code 15 stands for must not pass the type's largest value: a scale rounded up that far goes one step down.
    if (scale <= kLargest && fmaf(15.f, scale, low) > kLargest) {
        if constexpr (kHalf) scale_t = __ushort_as_half(__half_as_ushort(scale_t) - 1);
        else scale_t = __ushort_as_bfloat16(__bfloat16_as_ushort(scale_t) - 1);
        scale = float(scale_t);
    }
    const bool finite = scale <= kLargest;                  // (of infinities and NaN the scale is one)
    if (scale < 1.17549435e-38f) scale = 0.f;
    // Distances and steps in halves too (those of tiny scales times 2^60, out of the subnormals).
    const float f = scale > 0.f && scale < 0x1p-60f ? 0x1p59f : 0.5f, low2 = -f * low, s2 = f * scale;
    const float inv = scale > 0.f ? __fdividef(1.f, s2) : 0.f;
    // Nearest whole number: added to 1.5 2^23, whose last bit is 1.
    constexpr float kMagic = 12582912.f;
    word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float x;
        if constexpr (kHalf) x = e & 1 ? __high2float(P::as(w[e / 2])) : __low2float(P::as(w[e / 2]));
        else x = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        const float d = fmaf(x, f, low2);                   // the distance, rounded once
        // The quotient, put right by its exact remainder: a half stays a half (in bf16 two of three
        // warps have one), and nothing else becomes one.
        float q = d * inv;
        q = fmaf(fmaf(-q, s2, d), inv, q);
        float t = q + kMagic;
        // (bf16: the scale's rounding takes a quotient to 15.06 at most, and it has no small scales of few bits.)
        if constexpr (kHalf) t = fminf(t, kMagic + 15.f);
        word += __float_as_uint(t) << (16 * (e & 1) + 4 * (e / 2));
    }
    constexpr uint32_t kBits = 0x4b400000u;                 // kMagic's, as they were added up
    word -= (kBits + (kBits << 4) + (kBits << 8) + (kBits << 12)) + ((kBits << 16) + (kBits << 20) + (kBits << 24) + (kBits << 28));
    // scale, low; a group with an infinity or a NaN is NaN throughout.
    if constexpr (kHalf) pair = uint32_t(__half_as_ushort(__float2half_rn(scale))) | uint32_t(__half_as_ushort(lo1)) << 16;
    else pair = uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(scale))) | uint32_t(__bfloat16_as_ushort(lo1)) << 16;
    if (!finite) { word = 0; pair = 0x7fff7fffu; }
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) cache4_write_kernel(const __grid_constant__ Args4 a) {
    __shared__ int64_t at[kMaxRows];
    const Part4& p = a.part[blockIdx.z & 1];
    const Place w = place_of(a, p, blockIdx.z >> 1, at, true);
    const uint16_t* src = p.dense + blockIdx.y * p.stride[0] + (w.first + w.row) * p.stride[1] + w.head * p.stride[2] + 8 * w.unit;
    const int64_t step = p.side * p.stride[1];
    uint8_t* dst = p.cache + w.head * p.c_stride[2] + 4 * w.unit;
    const int pair_at = codes_bytes(p.dim) - 3 * w.unit;    // of the first lane of a group: D / 2 + unit, seen from its codes
    for (int i0 = 0; i0 * p.side < w.rows; i0 += kAhead) {
        uint4 raw[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            raw[k] = make_uint4(0, 0, 0, 0);
            if (w.some && w.row + (i0 + k) * p.side < w.rows) raw[k] = __ldcs(reinterpret_cast<const uint4*>(src + (i0 + k) * step));
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = w.row + (i0 + k) * p.side;
            if (!__any_sync(0xffffffffu, w.some && i < w.rows)) continue;
            uint32_t word, pair;
            quantise<kHalf>(raw[k], word, pair);
            if (!w.some || i >= w.rows || at[i] < 0) continue;
            uint8_t* row = dst + at[i];
            *reinterpret_cast<uint32_t*>(row) = word;
            if ((w.unit & 3) == 0) *reinterpret_cast<uint32_t*>(row + pair_at) = pair;
        }
    }
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const __grid_constant__ Args4 a) {
    using P = Pair<kHalf>;
    __shared__ int64_t at[kMaxRows];
    const Part4& p = a.part[blockIdx.z & 1];
    const Place w = place_of(a, p, blockIdx.z >> 1, at, false);
    if (!w.some) return;
    const uint8_t* src = p.cache + w.head * p.c_stride[2] + 4 * w.unit;
    const int pair_at = codes_bytes(p.dim) + (w.unit & ~3) - 4 * w.unit;
    uint16_t* dst = p.dense + blockIdx.y * p.stride[0] + (w.first + w.row) * p.stride[1] + w.head * p.stride[2] + 8 * w.unit;
    const int64_t step = p.side * p.stride[1];
    const int rows = a.zero_rest ? min(p.side * a.turns, a.rows - w.first) : w.rows;
    const typename P::Constants constants;
    for (int i0 = 0; i0 * p.side < rows; i0 += kAhead) {
        uint32_t code[kAhead], pair[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = w.row + (i0 + k) * p.side;
            code[k] = pair[k] = 0;                          // zeros: scale and low of 0
            if (i < w.rows) {
                const uint8_t* row = src + at[i];
                code[k] = __ldcs(reinterpret_cast<const uint32_t*>(row));
                pair[k] = __ldcs(reinterpret_cast<const uint32_t*>(row + pair_at));
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (w.row + (i0 + k) * p.side >= rows) break;
            const auto scale = P::as(low_twice(pair[k])), low = P::as(high_twice(pair[k]));
            __stcs(reinterpret_cast<uint4*>(dst + (i0 + k) * step),
                   make_uint4(P::template values<0>(constants, code[k], scale, low), P::template values<1>(constants, code[k], scale, low),
                              P::template values<2>(constants, code[k], scale, low), P::template values<3>(constants, code[k], scale, low)));
        }
    }
}

// ------------------------------------------------------------------- host --
int check_rows4(const slimkv_cache4_rows_args* a, const char* what) {
    if (!a || !a->k || !a->v) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
    if (a->batch < 1 || a->batch > 65535 || a->rows < 1 || a->kv_heads < 1)
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: batch in 1..65535, rows and heads", what);
    if (a->type != SLIMKV_BF16 && a->type != SLIMKV_FP16) return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: bf16 or fp16 rows", what);
    for (int dim : {a->dim_qk, a->dim_v})
        if (dim < kGroupDims || dim > kMaxDims4 || dim % kGroupDims)
            return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: dims must be multiples of 32 up to 320", what);
    if (a->rows > (1 << 28) || a->kv_heads > 4096)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: at most 2^28 rows of 4096 heads in one call", what);
    if (int rc = check_cache(a->cache, a->batch, row4_bytes(a->dim_qk), row4_bytes(a->dim_v), 1, true, what)) return rc;
    if (!aligned16(a->k) || !aligned16(a->v)) return fail(SLIMKV_ERR_ALIGNMENT, "%s: 16-byte aligned rows", what);
    for (int i = 0; i < 3; ++i)
        if (a->k_stride[i] % 8 || a->v_stride[i] % 8 || a->k_stride[i] < 0 || a->v_stride[i] < 0)
            return fail(SLIMKV_ERR_ALIGNMENT, "%s: strides must be multiples of 8 elements", what);
    return SLIMKV_OK;
}

Rows dense_rows(const slimkv_cache4_rows_args* a, bool is_v) {
    const int64_t* s = is_v ? a->v_stride : a->k_stride;
    return Rows{is_v ? a->v : a->k, int64_t(is_v ? a->dim_v : a->dim_qk) * 2, {1, a->batch, a->rows, a->kv_heads}, {0, s[0] * 2, s[1] * 2, s[2] * 2}};
}
Rows stored_rows(const slimkv_cache4_rows_args* a, bool is_v) {
    const slimkv_cache& c = a->cache;
    return cache_rows(is_v ? c.v : c.k, is_v ? c.v_stride : c.k_stride, row4_bytes(is_v ? a->dim_v : a->dim_qk), 1, c, a->batch, a->kv_heads);
}
// Rows that are written need a place of their own: no stride shorter than a row over more than one entry.
bool own_places(const Rows& r) {
    for (int i = 0; i < 4; ++i)
        if (r.n[i] > 1 && r.stride[i] < r.width) return false;
    return true;
}

Args4 args_of(const slimkv_cache4_rows_args* a) {
    Args4 k{};
    for (int i = 0; i < 2; ++i) {
        Part4& p = k.part[i];
        p.dim = i ? a->dim_v : a->dim_qk;
        p.cols = a->kv_heads * p.dim / 8;
        p.block_cols = p.cols < kThreads ? p.cols : kThreads;
        p.side = kThreads / p.block_cols;
        p.per_block = FastDiv(uint32_t(p.block_cols));
        p.per_head = FastDiv(uint32_t(p.dim / 8));
        p.dense = static_cast<uint16_t*>(const_cast<void*>(i ? a->v : a->k));
        p.cache = static_cast<uint8_t*>(const_cast<void*>(i ? a->cache.v : a->cache.k));
        for (int s = 0; s < 3; ++s) {
            p.stride[s] = (i ? a->v_stride : a->k_stride)[s];
            p.c_stride[s] = (i ? a->cache.v_stride : a->cache.k_stride)[s];
        }
    }
    k.rows = a->rows;
    k.page = FastDiv(uint32_t(a->cache.rows));
    k.view = cache_view(a->cache);
    k.capacity = cache_capacity(k.view);
    k.starts = a->starts;
    k.counts = a->counts;
    k.zero_rest = a->zero_rest;
    k.status = status_word();
    return k;
}

template <class Kernel>
int launch_rows4(Kernel kernel, Args4 k, int batch, const char* what, void* stream) {
    // K and V by turns; where their rows differ, the blocks that the longer one needs.
    int chunks = 0, row_blocks = 0, threads = 0;
    for (const Part4& p : k.part) {
        chunks = std::max(chunks, (p.cols + p.block_cols - 1) / p.block_cols);
        row_blocks = std::max(row_blocks, (k.rows - 1) / p.side + 1);
        threads = std::max(threads, (p.block_cols * p.side + 31) / 32 * 32);
    }
    // Few rows: a row to a thread, as long as that fills the GPU; many: several, for one look at their places.
    const int64_t fill = int64_t(row_blocks) * batch * 2 * chunks / (2 * device_info().sm_count);
    k.turns = int(std::max<int64_t>(1, std::min<int64_t>(kMaxTurns, fill)));
    row_blocks = (row_blocks - 1) / k.turns + 1;
    kernel<<<dim3(row_blocks, batch, 2 * chunks), threads, 0, static_cast<cudaStream_t>(stream)>>>(k);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SLIMKV_OK : fail(SLIMKV_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

}  // namespace
}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_row4_bytes(int dim) {
    return dim < kGroupDims || dim > kMaxDims4 || dim % kGroupDims ? 0 : row4_bytes(dim);
}

extern "C" int slimkv_cache4_write(const slimkv_cache4_rows_args* a, void* stream) {
    const char* what = "4-bit write";
    if (int rc = check_rows4(a, what)) return rc;
    if (!own_places(stored_rows(a, false)) || !own_places(stored_rows(a, true)))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: each cache row needs its own place (no stride below a row's bytes)", what);
    if (share_rows(stored_rows(a, false), stored_rows(a, true)))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: K and V need caches of their own", what);
    for (bool stored : {false, true})
        for (bool dense : {false, true})
            if (share_rows(stored_rows(a, stored), dense_rows(a, dense)))
                return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: the cache must not overlap the rows", what);
    const Args4 k = args_of(a);
    return a->type == SLIMKV_FP16 ? launch_rows4(cache4_write_kernel<true>, k, a->batch, what, stream)
                                  : launch_rows4(cache4_write_kernel<false>, k, a->batch, what, stream);
}

extern "C" int slimkv_cache4_read(const slimkv_cache4_rows_args* a, void* stream) {
    const char* what = "4-bit read";
    if (int rc = check_rows4(a, what)) return rc;
    if (!own_places(dense_rows(a, false)) || !own_places(dense_rows(a, true)))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: each row needs its own place (no stride below a row's length)", what);
    if (share_rows(dense_rows(a, false), dense_rows(a, true)))
        return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: K and V need rows of their own", what);
    for (bool stored : {false, true})
        for (bool dense : {false, true})
            if (share_rows(stored_rows(a, stored), dense_rows(a, dense)))
                return fail(SLIMKV_ERR_INVALID_ARGUMENT, "%s: the rows must not overlap the cache", what);
    const Args4 k = args_of(a);
    return a->type == SLIMKV_FP16 ? launch_rows4(cache4_read_kernel<true>, k, a->batch, what, stream)
                                  : launch_rows4(cache4_read_kernel<false>, k, a->batch, what, stream);
}
