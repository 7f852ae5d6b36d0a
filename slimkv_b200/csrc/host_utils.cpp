#include "host_utils.h"

#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

namespace slimkv {

static thread_local std::string g_last_error;

void set_error(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
}

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}

const DeviceInfo& device_info() {
    static thread_local DeviceInfo info;
    int dev = 0;
    cudaGetDevice(&dev);
    if (info.device != dev) {
        info.device = dev;
        cudaDeviceGetAttribute(&info.sm_count, cudaDevAttrMultiProcessorCount, dev);
        cudaDeviceGetAttribute(&info.smem_optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    }
    return info;
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        cudaDriverEntryPointQueryResult q;
        void* p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

int encode_map_4d(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2,
                  uint64_t d3, uint64_t s1, uint64_t s2, uint64_t s3, uint32_t box_rows) {
    return encode_map_4d_box(map, base, d0, d1, d2, d3, s1, s2, s3, 1, box_rows);
}

int encode_map_4d_box(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t d3,
                      uint64_t s1, uint64_t s2, uint64_t s3, uint32_t box1, uint32_t box2) {
    auto fn = encode_fn();
    if (!fn) return fail(SLIMKV_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[4] = {d0, d1, d2, d3};
    cuuint64_t strides[3] = {s1, s2, s3};
    cuuint32_t box[4] = {64, box1, box2, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
                    estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(SLIMKV_ERR_TENSOR_MAP,
                    "cuTensorMapEncodeTiled failed (%d): dims {%llu,%llu,%llu,%llu} strides {%llu,%llu,%llu}",
                    int(r), (unsigned long long)d0, (unsigned long long)d1, (unsigned long long)d2,
                    (unsigned long long)d3, (unsigned long long)s1, (unsigned long long)s2,
                    (unsigned long long)s3);
    return SLIMKV_OK;
}

int encode_map_words_4d(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t d3,
                        uint64_t s1, uint64_t s2, uint64_t s3, uint32_t box_rows) {
    auto fn = encode_fn();
    if (!fn) return fail(SLIMKV_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[4] = {d0, d1, d2, d3};
    cuuint64_t strides[3] = {s1, s2, s3};
    cuuint32_t box[4] = {cuuint32_t(d0), 1, box_rows, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(SLIMKV_ERR_TENSOR_MAP,
                    "cuTensorMapEncodeTiled (words) failed (%d): dims {%llu,%llu,%llu,%llu} strides {%llu,%llu,%llu}", int(r),
                    (unsigned long long)d0, (unsigned long long)d1, (unsigned long long)d2, (unsigned long long)d3,
                    (unsigned long long)s1, (unsigned long long)s2, (unsigned long long)s3);
    return SLIMKV_OK;
}

int encode_map_f32_3d(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1,
                      uint64_t s2, uint32_t box0, uint32_t box1) {
    auto fn = encode_fn();
    if (!fn) return fail(SLIMKV_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[3] = {d0, d1, d2};
    cuuint64_t strides[2] = {s1, s2};
    cuuint32_t box[3] = {box0, box1, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(SLIMKV_ERR_TENSOR_MAP, "cuTensorMapEncodeTiled (f32) failed (%d): dims {%llu,%llu,%llu}", int(r),
                    (unsigned long long)d0, (unsigned long long)d1, (unsigned long long)d2);
    return SLIMKV_OK;
}

Rows cache_rows(const void* at, const int64_t* strides, int64_t width_bytes, int elem_bytes, const slimkv_cache& cache,
                int batch, int heads, int layers, int64_t layer_stride) {
    return Rows{at, width_bytes, {layers, cache.table ? cache.num_pages : batch, cache.rows, heads},
                {layer_stride * elem_bytes, strides[0] * elem_bytes, strides[1] * elem_bytes, strides[2] * elem_bytes}};
}

namespace {

using Wide = __int128;          // strides are the caller's: no product of them may overflow

// A set of rows with its dimensions (of more than one entry, positive strides) from the widest on.
struct Sorted {
    int dims = 0;
    Wide at, width, n[4], stride[4], span[5];       // span[d]: bytes from the first to the last of dimensions d..
    explicit Sorted(const Rows& r) : at(reinterpret_cast<uintptr_t>(r.at)), width(r.width) {
        for (int i = 0; i < 4; ++i) {
            if (r.n[i] <= 1) continue;
            const Wide s = r.stride[i];
            if (s < 0) at += s * (r.n[i] - 1);
            int d = dims++;
            for (; d > 0 && stride[d - 1] < (s < 0 ? -s : s); --d) { stride[d] = stride[d - 1]; n[d] = n[d - 1]; }
            stride[d] = s < 0 ? -s : s;
            n[d] = r.n[i];
        }
        span[dims] = width;
        for (int d = dims - 1; d >= 0; --d) span[d] = span[d + 1] + stride[d] * (n[d] - 1);
    }
};

// First byte of a set of rows, and the one behind its last.
void range_of(const Rows& r, Wide& from, Wide& to) {
    from = reinterpret_cast<uintptr_t>(r.at);
    to = from + r.width;
    for (int i = 0; i < 4; ++i) {
        const Wide far = Wide(r.stride[i]) * (r.n[i] - 1);
        if (far < 0) from += far;
        else to += far;
    }
}

// The dimensions d.. of a and b, b `gap` bytes behind a.
bool share_from(const Sorted& a, const Sorted& b, int d, Wide gap) {
    if (gap >= a.span[std::min(d, a.dims)] || -gap >= b.span[std::min(d, b.dims)]) return false;
    if (d >= a.dims || d >= b.dims) return true;    // (one row against several: taken as shared)
    const Wide s = a.stride[d];
    if (s != b.stride[d] || s < a.span[d + 1] || s < b.span[d + 1]) return true;
    // Entry i of a and j of b are gap - (i - j) s apart: only the two differences that leave
    // less than s can share bytes.
    Wide q = gap / s;
    if (gap % s < 0) --q;
    for (Wide m = q; m <= q + 1; ++m)
        if (m > -b.n[d] && m < a.n[d] && share_from(a, b, d + 1, gap - m * s)) return true;
    return false;
}

}  // namespace

bool share_rows(const Rows& a, const Rows& b) {
    Wide a0, a1, b0, b1;
    range_of(a, a0, a1);
    range_of(b, b0, b1);
    if (a1 <= b0 || b1 <= a0) return false;         // what nearly every call has
    const Sorted x(a), y(b);
    return share_from(x, y, 0, y.at - x.at);
}

}  // namespace slimkv

extern "C" const char* slimkv_last_error(void) { return slimkv::g_last_error.c_str(); }
extern "C" int slimkv_version(void) { return 100; }
