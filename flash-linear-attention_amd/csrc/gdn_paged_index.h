// Where a slot of a paged cache lies.  Without HIP headers: the same code runs in a program of the host, where its limits can be tested.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define GDN_ANYWHERE __host__ __device__ __forceinline__
#else
#define GDN_ANYWHERE inline
#endif

namespace gdn {

// The pages of the sequences: slot p of sequence n is slot p % page_size of page table[n * table_stride + p / page_size].
struct PageTable {
    const int32_t* table;
    int64_t table_stride;
    int64_t capacity;                // slots that a row of the table can name: table_cols * page_size, below 2^31
    int32_t pages, page_size;
};

// The page of a slot, or -1: the slot lies outside the table's row, or the table names no page of the cache there.  Nothing is read
// for a slot outside the row.
template <typename Load>
GDN_ANYWHERE int32_t page_of(const PageTable& t, int64_t n, int64_t slot, Load load) {
    if (slot < 0 || slot >= t.capacity) return -1;
    const int32_t page = load(t.table, n * t.table_stride + (uint32_t)slot / (uint32_t)t.page_size);
    return page >= 0 && page < t.pages ? page : -1;
}
GDN_ANYWHERE int32_t page_of(const PageTable& t, int64_t n, int64_t slot) {
    return page_of(t, n, slot, [](const int32_t* at, int64_t i) { return at[i]; });
}
// The slot's place in its page (of a slot that has one).
GDN_ANYWHERE uint32_t place_in_page(const PageTable& t, int64_t slot) { return (uint32_t)slot % (uint32_t)t.page_size; }

// The sequence that a row of a packed batch belongs to, or -1: cu [N + 1] are the boundaries, rows before the first and behind the last
// belong to none.  (Boundaries that decrease give some sequence or none, and read nothing else.)
template <typename Load>
GDN_ANYWHERE int64_t sequence_of(int64_t row, int64_t N, Load cu) {
    int64_t lo = 0, hi = N;                                       // cu(lo) <= row < cu(hi), if at all
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        if (cu(mid) <= row) lo = mid; else hi = mid;
    }
    return cu(lo) <= row && row < cu(lo + 1) ? lo : -1;
}

}  // namespace gdn
