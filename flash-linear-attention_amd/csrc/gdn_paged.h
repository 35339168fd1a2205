// A paged cache of keys and values as the kernels see it.
#pragma once
#include "gdn_common.h"
#include "gdn_paged_index.h"

namespace gdn {

struct PagedCache {
    char* k; char* v;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;      // strides in elements
    PageTable pages;
    const void* context;                                          // [N]: slots that held a token before this step's rows
    bool context_i32;
};

// What every entry checks of a cache before a kernel indexes it.
inline int check_cache(const char* who, const gdn_paged_cache* c, int64_t N, PagedCache& out) {
    GDN_CHECK_ARG(c, GDN_ERR_INVALID, "%s: no cache", who);
    GDN_CHECK_ARG(c->pages >= 0 && c->page_size >= 1 && c->heads >= 1 && c->dim >= 1 && c->table_cols >= 0 && c->table_stride >= c->table_cols, GDN_ERR_INVALID,
                  "%s: bad sizes of the cache", who);
    GDN_CHECK_ARG(c->pages < (1ll << 31) && c->page_size < (1ll << 31) && c->table_cols < (1ll << 31) && c->table_cols * c->page_size < (1ll << 31) && N < (1ll << 31),
                  GDN_ERR_UNSUPPORTED, "%s: pages, slots of a page and of a sequence are below 2^31", who);
    GDN_CHECK_ARG(c->dtype == GDN_DTYPE_BF16 || c->dtype == GDN_DTYPE_F16 || c->dtype == GDN_DTYPE_F32, GDN_ERR_UNSUPPORTED, "%s: unsupported dtype %d", who, c->dtype);
    GDN_CHECK_ARG(N <= 0 || (c->context && (c->pages == 0 || (c->k && c->v)) && (c->table_cols == 0 || c->page_table)), GDN_ERR_INVALID, "%s: missing tensors of the cache", who);
    out = PagedCache{(char*)c->k, (char*)c->v, c->k_stride[0], c->k_stride[1], c->k_stride[2], c->v_stride[0], c->v_stride[1], c->v_stride[2],
                     PageTable{c->page_table, c->table_stride, c->table_cols * c->page_size, (int32_t)c->pages, (int32_t)c->page_size}, c->context, c->context_int32 != 0};
    return GDN_OK;
}

inline int size_of_dtype(int dtype) { return dtype == GDN_DTYPE_F32 ? 4 : 2; }

}  // namespace gdn
