// Rows quantised into the 4-bit cache, and read back (C ABI
// slimkv_cache4_write, slimkv_cache4_read).
//
// For each group of 32 dims x of a row, in the rows' 16-bit type T:
//   low = min x,  scale = T((max x - low) / 15),  code = rint((x - low) / scale)
// and back T(code * scale + low).  Four neighbouring lanes hold a group, eight
// dims (one 16-byte load) each; the least and largest value go between them by
// two shuffles, and every lane writes the four bytes of its codes.
//
// Bound: HBM (2.625 bytes a value either way); the codes cost about ten
// operations each, so what is exact is bought cheaply: the nearest code comes from
// a product with 1 / scale, whose error shows in the exact remainder
// x - low - code * scale (one fused operation); a remainder of half a scale or more
// sends the lane's codes through the exact rule.
#include <type_traits>

#include "cache4.cuh"
#include "cache_view.cuh"
#include "host_utils.h"

namespace slimkv {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;               // units of eight dims a thread has under way

struct Job4 {
    int rows, dim, units, upr;          // units of eight dims of a sequence (rows x heads x upr), and of a row
    FastDiv per_row, per_head;          // by heads * upr and by upr
    const uint16_t* dense;              // 16-bit rows: read by write, written by read
    uint16_t* out;
    int64_t stride[3];
    uint8_t* cache;
    int64_t c_stride[3];                // bytes
};
struct Args4 {
    Job4 part[2];                       // K and V
    CacheView view;
    int64_t capacity;
    const int32_t *starts, *counts;
    int zero_rest;
    unsigned int* status;
};

// A sequence's rows: cache rows [start, start + count), without what the cache cannot hold
// (behind a negative start: none).
__device__ __forceinline__ bool span_of(const Args4& a, int b, int rows, int& start, int& count) {
    const int s = a.starts ? __ldg(a.starts + b) : 0, c = a.counts ? __ldg(a.counts + b) : rows;
    start = max(s, 0);
    count = s < 0 ? 0 : min(max(c, 0), rows);
    const bool fits = s >= 0 && c >= 0 && c <= rows && int64_t(start) + count <= a.capacity;
    count = int(max(min(int64_t(count), a.capacity - start), int64_t(0)));
    return fits;
}

// The place of a unit: its row, head, and the byte address of the cache row.
__device__ __forceinline__ bool place_of(const Args4& a, const Job4& p, int b, uint32_t unit, int start, int& row, int& head, int& u,
                                         int64_t& at) {
    row = int(p.per_row.div(unit));
    const uint32_t in_row = unit - uint32_t(row) * p.per_row.d;
    head = int(p.per_head.div(in_row));
    u = int(in_row) - head * p.upr;
    int64_t page;
    int r;
    const bool ok = cache_row(a.view, b, start + row, page, r);
    at = page * p.c_stride[0] + r * p.c_stride[1] + head * p.c_stride[2];
    return ok;
}

// Code of a value whose quick code (of remainder r, with the sign of value minus what the code
// stands for) is at most one off: the nearest, an even one at a tie.
__device__ __noinline__ float exact_code(float c, float r, float scale) {
    const float half = 0.5f * scale;
    if (r > half || (r == half && (int(c) & 1))) c += 1.f;
    else if (r < -half || (r == -half && (int(c) & 1))) c -= 1.f;
    return fminf(fmaxf(c, 0.f), 15.f);
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) cache4_write_kernel(const __grid_constant__ Args4 a) {
    using P = Pair<kHalf>;
    using T2 = typename P::T2;
    const Job4& p = a.part[blockIdx.z];
    const int b = blockIdx.y, lane = threadIdx.x & 31;
    int start, count;
    if (!span_of(a, b, p.rows, start, count) && blockIdx.x == 0 && threadIdx.x == 0) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
    const uint32_t units = uint32_t(count) * p.per_row.d, first = blockIdx.x * (kThreads * kUnits) + threadIdx.x;
    if (first - threadIdx.x >= units) return;
    uint4 raw[kUnits];
    int64_t at[kUnits];
    int u[kUnits];
    // Whole groups of four lanes have work or none (a row's units are a multiple of four).
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        raw[k] = make_uint4(0, 0, 0, 0);
        u[k] = -1;
        const uint32_t unit = first + k * kThreads;
        if (unit >= units) continue;
        int row, head;
        const bool ok = place_of(a, p, b, unit, start, row, head, u[k], at[k]);
        raw[k] = __ldcs(reinterpret_cast<const uint4*>(p.dense + b * p.stride[0] + row * p.stride[1] + head * p.stride[2]) + u[k]);
        if (!ok) {
            report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
            u[k] = -1;
        }
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        if (first + k * kThreads - lane >= units) break;        // the whole warp
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
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
        const float s2 = 0.5f * scale, inv = scale > 0.f ? 1.f / s2 : 0.f, half = scale > 0.f ? 0.5f * s2 : INFINITY;
        // Nearest whole number: added to 1.5 2^23, whose last bit is 1.
        constexpr float kMagic = 12582912.f;
        float c[8], r[8];
        uint32_t word = 0;
        bool off = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 x = [&] {
                if constexpr (kHalf) return __half22float2(P::as(w[e / 2]));
                else return __bfloat1622float2(P::as(w[e / 2]));
            }();
            const float d = fmaf(e & 1 ? x.y : x.x, 0.5f, -0.5f * low);     // half the distance, rounded once
            const float t = fminf(fmaf(d, inv, kMagic), kMagic + 15.f);
            c[e] = t - kMagic;
            r[e] = fmaf(-c[e], s2, d);                          // exact where it matters
            off |= fabsf(r[e]) >= half;
            word += __float_as_uint(t) << (16 * (e & 1) + 4 * (e / 2));
        }
        constexpr uint32_t kBits = 0x4b400000u;                 // kMagic's, as they were added up
        word -= (kBits + (kBits << 4) + (kBits << 8) + (kBits << 12)) + ((kBits << 16) + (kBits << 20) + (kBits << 24) + (kBits << 28));
        if (off && finite && u[k] >= 0) {
            word = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) word |= uint32_t(exact_code(c[e], r[e], s2)) << (16 * (e & 1) + 4 * (e / 2));
        }
        if (u[k] < 0) continue;
        uint8_t* row = p.cache + at[k];
        reinterpret_cast<uint32_t*>(row)[u[k]] = finite ? word : 0u;
        if ((lane & 3) == 0) {
            // scale, low; a group with an infinity or a NaN is NaN throughout.
            uint32_t pair = 0x7fff7fffu;
            if (finite) {
                if constexpr (kHalf) pair = uint32_t(__half_as_ushort(__float2half_rn(scale))) | uint32_t(__half_as_ushort(lo1)) << 16;
                else pair = uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(scale))) | uint32_t(__bfloat16_as_ushort(lo1)) << 16;
            }
            *reinterpret_cast<uint32_t*>(row + codes_bytes(p.dim) + u[k]) = pair;
        }
    }
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) cache4_read_kernel(const __grid_constant__ Args4 a) {
    using P = Pair<kHalf>;
    const Job4& p = a.part[blockIdx.z];
    const int b = blockIdx.y;
    int start, count;
    if (!span_of(a, b, p.rows, start, count) && blockIdx.x == 0 && threadIdx.x == 0) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
    const uint32_t units = uint32_t(a.zero_rest ? p.rows : count) * p.per_row.d, first = blockIdx.x * (kThreads * kUnits) + threadIdx.x;
    uint32_t code[kUnits], pair[kUnits];
    uint4* dst[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        dst[k] = nullptr;
        code[k] = pair[k] = 0;
        const uint32_t unit = first + k * kThreads;
        if (unit >= units) continue;
        const int row = int(p.per_row.div(unit));
        const uint32_t in_row = unit - uint32_t(row) * p.per_row.d;
        const int head = int(p.per_head.div(in_row)), u = int(in_row) - head * p.upr;
        dst[k] = reinterpret_cast<uint4*>(p.out + b * p.stride[0] + row * p.stride[1] + head * p.stride[2]) + u;
        if (row >= count) continue;                             // zeros: scale and low of 0
        int64_t page;
        int r;
        if (!cache_row(a.view, b, start + row, page, r)) report(a.status, SLIMKV_DEVICE_BAD_LENGTH);
        const uint8_t* from = p.cache + page * p.c_stride[0] + r * p.c_stride[1] + head * p.c_stride[2];
        code[k] = __ldcs(reinterpret_cast<const uint32_t*>(from) + u);
        pair[k] = __ldcs(reinterpret_cast<const uint32_t*>(from + codes_bytes(p.dim) + (u & ~3)));
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
        if (!dst[k]) continue;
        const typename P::Constants constants;
        const auto scale = P::as(low_twice(pair[k])), low = P::as(high_twice(pair[k]));
        __stcs(dst[k], make_uint4(P::template values<0>(constants, code[k], scale, low), P::template values<1>(constants, code[k], scale, low),
                                  P::template values<2>(constants, code[k], scale, low), P::template values<3>(constants, code[k], scale, low)));
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
    if (double(a->rows) * a->kv_heads * (a->dim_qk > a->dim_v ? a->dim_qk : a->dim_v) / 8 >= 2147483648.0 - kThreads * kUnits)
        return fail(SLIMKV_ERR_UNSUPPORTED_SHAPE, "%s: too many rows in one call", what);
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
        Job4& p = k.part[i];
        p.rows = a->rows;
        p.dim = i ? a->dim_v : a->dim_qk;
        p.upr = p.dim / 8;
        p.units = a->rows * a->kv_heads * p.upr;
        p.per_row = FastDiv(uint32_t(a->kv_heads * p.upr));
        p.per_head = FastDiv(uint32_t(p.upr));
        p.out = static_cast<uint16_t*>(const_cast<void*>(i ? a->v : a->k));
        p.dense = p.out;
        p.cache = static_cast<uint8_t*>(const_cast<void*>(i ? a->cache.v : a->cache.k));
        for (int s = 0; s < 3; ++s) {
            p.stride[s] = (i ? a->v_stride : a->k_stride)[s];
            p.c_stride[s] = (i ? a->cache.v_stride : a->cache.k_stride)[s];
        }
    }
    k.view = cache_view(a->cache);
    k.capacity = cache_capacity(k.view);
    k.starts = a->starts;
    k.counts = a->counts;
    k.zero_rest = a->zero_rest;
    k.status = status_word();
    return k;
}

template <class Kernel>
int launch_rows4(Kernel kernel, const Args4& k, int batch, const char* what, void* stream) {
    const int units = k.part[0].units > k.part[1].units ? k.part[0].units : k.part[1].units;
    kernel<<<dim3((units - 1) / (kThreads * kUnits) + 1, batch, 2), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(k);
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
