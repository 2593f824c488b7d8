// Addressing of the paged key-value cache, shared by the kernels and the host.
#pragma once

#include "common.cuh"

namespace rgd {
namespace paged {

// Position p of a sequence lies in page table_row[p / page], slot p % page.  What a table holds is only known
// on the device, so every lookup is checked there: an index past the table's row or a page outside the pool is
// never followed.
struct PagedView {
    const int32_t *table;
    int64_t table_stride;
    int64_t pages;              // in the pool
    FastDiv page;               // tokens per page
    int max_pages;              // entries of a table row
};

__host__ __device__ __forceinline__ void split_position(const PagedView &v, uint32_t pos, int &index, int &slot) {
    const uint32_t q = fdiv(pos, v.page);
    index = (int)q;
    slot = (int)(pos - q * v.page.div);
}
__host__ __device__ __forceinline__ bool page_ok(const PagedView &v, int page) { return page >= 0 && page < v.pages; }

// Tokens a table row can address; positions are 31-bit.
__host__ __device__ __forceinline__ int64_t capacity(const PagedView &v) { return (int64_t)v.max_pages * v.page.div; }

inline PagedView make_view(const rgd_paged &c) {
    return {c.page_table, c.table_stride, c.num_pages, make_fastdiv((uint32_t)c.page_size), (int)c.max_pages};
}

inline int check_paged(const rgd_paged *c, int64_t B, bool cache_needed) {
    if (!c) return RGD_E_NULL;
    if (c->num_pages < 0 || c->max_pages < 0 || c->page_size < 1 || c->table_stride < 0) return RGD_E_INVALID;
    if (c->k_stride_p < 0 || c->k_stride_s < 0 || c->k_stride_h < 0 || c->v_stride_p < 0 || c->v_stride_s < 0 || c->v_stride_h < 0)
        return RGD_E_STRIDE;
    if (c->num_pages > INT32_MAX || c->page_size > INT32_MAX || c->max_pages > INT32_MAX ||
        c->max_pages * c->page_size > INT32_MAX - 1024)
        return RGD_E_SIZE;
    if (B > 0 && (!c->lengths || (c->max_pages > 0 && !c->page_table))) return RGD_E_NULL;
    if (cache_needed && c->num_pages > 0 && (!c->k || !c->v)) return RGD_E_NULL;
    return RGD_OK;
}

inline bool cache_vec16(const rgd_paged &c) {
    return is_aligned(c.k, 16) && is_aligned(c.v, 16) && c.k_stride_p % 8 == 0 && c.k_stride_s % 8 == 0 && c.k_stride_h % 8 == 0 &&
           c.v_stride_p % 8 == 0 && c.v_stride_s % 8 == 0 && c.v_stride_h % 8 == 0;
}
inline bool heads_vec16(const rgd_heads &v) {
    return is_aligned(v.ptr, 16) && v.stride_b % 8 == 0 && v.stride_h % 8 == 0 && v.stride_n % 8 == 0;
}

}  // namespace paged
}  // namespace rgd
