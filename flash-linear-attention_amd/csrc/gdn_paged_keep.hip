// The accepted path of a tree of drafts, moved to the front of its slots.
//
//   slot context + i = slot context + rows[i], i < kept, rows[i] >= i
//
// In place: a thread owns 16 bytes (or less, by alignment) of one head of the keys or values in all slots of a sequence and takes them in order, eight
// slots read before eight are written.  A slot that is written (i) was a source of rows up to i only, because rows[j] >= j.  Launch time bounds it: a few rows.  One path
// of 8 rows 4.5 us a call, 256 of up to 64 rows 8.1.
#include "gdn_paged.h"
#include <algorithm>

namespace gdn {

struct KeepParams {
    PagedCache cache;
    const int32_t* rows; const int32_t* kept;
    int64_t rows_stride;
    int R, chunks, heads, all_heads;                              // all_heads: of keys and values
};

template <typename U>
__global__ __launch_bounds__(256) void paged_keep_kernel(KeepParams p, int per_unit) {
    constexpr int AHEAD = 8;
    const int64_t n = blockIdx.y;
    const int lane = blockIdx.x * 256 + threadIdx.x;
    if (lane >= p.all_heads * p.chunks) return;
    const int c = lane % p.chunks, kh = lane / p.chunks, h = kh % p.heads;
    const bool values = kh >= p.heads;
    char* const data = values ? p.cache.v : p.cache.k;
    const int64_t page_stride = (values ? p.cache.v_page : p.cache.k_page), slot_stride = (values ? p.cache.v_slot : p.cache.k_slot),
                  inside = h * (values ? p.cache.v_head : p.cache.k_head);
    const int64_t context = load_index(p.cache.context, n, p.cache.context_i32);
    const int kept = std::min(p.kept[n], p.R);
    const int32_t* rows = p.rows + n * p.rows_stride;
    auto place = [&](int64_t slot) -> U* {
        const int page = page_of(p.cache.pages, n, slot);
        if (page < 0) return nullptr;
        return (U*)data + (page * page_stride + (int64_t)place_in_page(p.cache.pages, slot) * slot_stride + inside) / per_unit + c;
    };
    for (int i = 0; i < kept; i += AHEAD) {
        U held[AHEAD];
        U* to[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            to[e] = nullptr;
            if (i + e >= kept) continue;
            const int64_t row = rows[i + e];
            if (row <= i + e || context < 0) continue;            // (in its place, or no row that may move here)
            const U* from = place(context + row);
            if (!from) continue;
            to[e] = place(context + i + e);
            held[e] = *from;
        }
#pragma unroll
        for (int e = 0; e < AHEAD; ++e)
            if (to[e]) *to[e] = held[e];
    }
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_paged_keep(const gdn_paged_cache* cache, const int32_t* rows, int64_t rows_stride, int64_t R, const int32_t* kept, int64_t N, void* stream) {
    const char* who = "gdn_paged_keep";
    KeepParams p{};
    const int rc = check_cache(who, cache, N, p.cache);
    if (rc != GDN_OK) return rc;
    GDN_CHECK_ARG(N >= 0 && R >= 0 && R < (1ll << 31) && rows_stride >= R && N <= 65535, GDN_ERR_INVALID, "%s: bad sizes (up to 65535 sequences)", who);
    if (N == 0 || R == 0 || cache->pages == 0) return GDN_OK;
    GDN_CHECK_ARG(rows && kept, GDN_ERR_INVALID, "%s: rows and kept are required", who);
    const int size = size_of_dtype(cache->dtype);
    const int64_t row_bytes = cache->dim * size;
    const PagedCache& c = p.cache;
    const uint64_t places = (uint64_t)row_bytes | (uint64_t)c.k | (uint64_t)c.v | (uint64_t)(c.k_page | c.k_slot | c.k_head | c.v_page | c.v_slot | c.v_head) * size;
    const int unit = places % 16 == 0 ? 16 : places % 4 == 0 ? 4 : 2;
    p.rows = rows; p.kept = kept; p.rows_stride = rows_stride; p.R = (int)R;
    GDN_CHECK_ARG(2 * cache->heads * (row_bytes / unit) < (1ll << 30), GDN_ERR_UNSUPPORTED, "%s: rows too long", who);
    p.heads = (int)cache->heads; p.chunks = (int)(row_bytes / unit);
    // (one tensor for keys and values, as of latent vectors, is moved once: two threads on the same slots would read what the other has written)
    p.all_heads = c.k == c.v && c.k_page == c.v_page && c.k_slot == c.v_slot && c.k_head == c.v_head ? p.heads : 2 * p.heads;
    const dim3 grid((unsigned)((p.all_heads * p.chunks + 255) / 256), (unsigned)N);
    auto go = [&](auto u) { hipLaunchKernelGGL(paged_keep_kernel<decltype(u)>, grid, dim3(256), 0, (hipStream_t)stream, p, unit / size); };
    if (unit == 16) go(u32x4{});
    else if (unit == 4) go(uint32_t{});
    else go(uint16_t{});
    return check_launch("paged_keep_kernel");
}
