// Device view of a batch's cache rows (slimkv_cache): dense [sequence, row,
// head] strides, or pages reached through block tables.
#pragma once

#include "common.cuh"

namespace slimkv {

struct CacheView {
    int64_t k_stride[3], v_stride[3];
    int rows;                 // rows of a sequence (dense) or of a page
    const int32_t* table;
    int64_t table_stride;
    int table_pages, num_pages;
};

inline CacheView cache_view(const slimkv_cache& c) {
    CacheView v{};
    for (int i = 0; i < 3; ++i) { v.k_stride[i] = c.k_stride[i]; v.v_stride[i] = c.v_stride[i]; }
    v.rows = c.rows;
    v.table = c.table;
    v.table_stride = c.table_stride;
    v.table_pages = c.table_pages;
    v.num_pages = c.num_pages;
    return v;
}

// Rows one sequence can hold.
__host__ __device__ __forceinline__ int64_t cache_capacity(const CacheView& c) {
    return c.table ? int64_t(c.rows) * c.table_pages : int64_t(c.rows);
}

// Which page (dense: sequence) row n of sequence b lies in, and its row
// there; false when the table names no page.
__device__ __forceinline__ bool cache_row(const CacheView& c, int b, int n, int64_t& page, int& row) {
    if (!c.table) {
        page = b;
        row = n;
        return true;
    }
    const int i = n / c.rows;
    const int p = __ldg(c.table + b * c.table_stride + i);
    page = min(max(p, 0), c.num_pages - 1);
    row = n - i * c.rows;
    return p >= 0 && p < c.num_pages;
}

}  // namespace slimkv
