// Attention of a step's rows (one token, a chain or a tree of drafts) over a paged cache.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   s_ij = scale q_i . k_j over the keys that row i sees, m_i their maximum
//
// One pass over the keys with the running maximum and sum.  The rows of a sequence that share a head of the cache (its tokens times the heads of a group, row m = token * group +
// head) stand side by side, so a key is read once for all of them.  Both products have the rows as columns:
//
//   S^T [keys x rows] = K Q^T,   O^T [elements x rows] += V^T P^T,
//
// so a lane has the scores of one row, which are the second product's operand where they are (the order of the keys in a contraction is free, as long as V has
// the same), the row's statistics are the lane's, and nothing goes through LDS: K is the first operand as it lies in memory; a lane asks for eight elements of
// eight keys of V and exchanges them in its registers (one v_perm_b32 per pair).
//
// A wave takes tiles of 32 keys by itself, without barriers: K of the next tile is asked for when the scores of this one are formed, V of the next when it is added up, the
// pages' numbers a tile earlier.  From 33 rows on the four waves of a workgroup take the same keys, 64 at a time, from two stages in LDS (four waves asking for the same rows:
// 417 us for the long trees below, through LDS 318).  Waves that share rows are joined through LDS at the end, workgroups by paged_attn_join_kernel.
//
// The weights are rounded to the operands' type for their product with V, once, as the matrix cores take them; their sum, the statistics and the sums of V are fp32.  (In fp32
// the second product would have a sixteenth of the rate, by the published peaks.  With bf16 rows the result is 1.2 to 1.4 times as far from the exact one as its own rounding puts it.)
//
// The memory system bounds it up to 128 rows.  Measured (bf16, heads of 128, 32 query heads on 8): 64 sequences of 3300 keys, a row each 162 to 168 us (5.2 to 5.4 TB/s), of up to
// 8192 keys 176; eight trees of 32 rows over 32768 keys 220 to 240, by machine (4.5 to 4.9 TB/s), of it the join 12; four of 8000 with 256 rows 248 (551 TFLOP/s).  Heads of 256, 16 on 4,
// up to 8000 keys: 32 rows 115 us (4.7 TB/s), 16 trees of 16 rows 99 (3.7 TB/s, 232 TFLOP/s), 128 rows each 724 (374 TFLOP/s).  Heads of 80 in pages of 10 are bound by the wait for
// each tile: 33 chains of 7 over 3001 keys 27 us.  Whole prompts run, at half the rate of a chunk behind a context and less: seven of 2048 rows 1244 us (193 TFLOP/s), because
// a unit counts as all keys of its sequence while it stops at its last row.
#include "gdn_paged.h"
#include "gdn_chunk_common.h"
#include <algorithm>
#include <cmath>
#include <type_traits>

namespace gdn {

constexpr int PA_MAX_DIM = 256, PA_TILE = 32;

struct PagedAttnParams {
    PagedCache cache;
    const void* q; void* o; const void* cu; const uint8_t* mask;
    int64_t* before;                         // [N + 1]: the work of the sequences before (PagedWork), for the join
    float* part_o; float* part_ml;           // [2 workgroups][height][D], [..][2]: sums, maximum and sum of the weights of a part of a unit's keys
    int64_t qb, qt, qh;
    int64_t mask_seq, mask_row;
    int64_t T, total;                        // rows of a sequence (dense), of the batch
    uint32_t page_magic; int page_shift;     // slot / page_size = slot * page_magic >> page_shift
    int N, HQ, HK, D, group, mask_cols;
    int height, step, overhead, groups, row_groups, odd_at;      // rows of a unit; keys of a step, what a unit's beginning and end count as; workgroups; of four waves, those with rows of their own
    uint32_t k_page, k_slot, k_head, v_page, v_slot, v_head;     // the cache's strides where they are below 2^32 (UNIFORM)
    float scale2;                            // |scale| log2(e)
    bool cu_i32, negative;                   // negative: of a negative scale the queries take the sign
};

typedef uint16_t pa_whole __attribute__((ext_vector_type(8), aligned(2)));
typedef uint16_t pa_aligned __attribute__((ext_vector_type(8)));

// Infinities and NaN: an exponent of ones.  In a pair: its upper bit carries into the sign's place.
template <typename T> constexpr uint32_t PA_EXPONENT = std::is_same_v<T, bf16_t> ? 0x7f80 : 0x7c00;
template <typename T> constexpr uint32_t PA_CARRY = std::is_same_v<T, bf16_t> ? 0x0080 : 0x0400;
// Weights are 2^PA_LIFT at the row's maximum, and up to 2^8 times that before the maximum moves, below fp16's 2^16: rounded to fp16 a weight loses what is below 2^-32 of
// the maximum's, of which two million keys together make half a step of the largest value. (Without the lift 2^-25: 131071 keys 17.4 below one in their score, 0.36 % of
// the result, were 0.)  The factor is in the weights' sum, too.  bf16 has the range of fp32.
template <typename T> constexpr float PA_LIFT = std::is_same_v<T, bf16_t> ? 0.f : 7.f;
template <typename T> __device__ __forceinline__ bool not_a_number(uint16_t bits) { return (bits & PA_EXPONENT<T>) == PA_EXPONENT<T>; }

// (the same in every lane by construction)
__device__ __forceinline__ int64_t scalar(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T two __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, two));
}

// What a step's sequence is.
struct PagedSequence {
    int64_t first;                           // its first row in the batch
    int rows;
    int64_t context;
    int keys;                                // slots that may be seen: [0, keys)
    int whole;                               // tiles that lie in the context
};
template <bool UNIFORM = true>
__device__ __forceinline__ PagedSequence paged_sequence(const PagedAttnParams& p, int64_t n) {
    auto load = [](const void* at, int64_t i, bool is_i32) { return UNIFORM ? load_index_uniform(at, i, is_i32) : load_index(at, i, is_i32); };
    PagedSequence s;
    s.first = n * p.T;
    int64_t rows = p.T;
    if (p.cu) {
        s.first = load(p.cu, n, p.cu_i32);
        rows = load(p.cu, n + 1, p.cu_i32) - s.first;
        if (s.first < 0 || s.first > p.total) { s.first = 0; rows = 0; }
        rows = min(rows, p.total - s.first);
    }
    s.rows = (int)max(rows, (int64_t)0);
    s.context = load(p.cache.context, n, p.cache.context_i32);
    const int64_t capacity = p.cache.pages.pages > 0 ? p.cache.pages.capacity : 0;
    // (in this order: a context near the end of 64 bits does not overflow)
    s.context = max(min(s.context, capacity), (int64_t)-0x40000000);
    s.keys = (int)max(min(s.context + s.rows, capacity), (int64_t)0);
    s.whole = (int)max(s.context, (int64_t)0) / PA_TILE;
    return s;
}

// How the work is shared out.  A unit is `height` rows of a sequence at a head of the cache; it counts as its steps of keys and `overhead` (for its beginning and end).
// The units stand in a row, by sequence, head and rows, and every workgroup takes as much of the row as any other, wherever that begins and ends: contexts of all lengths
// keep all of them busy to the end, in one round of the chip.  What a workgroup has of a unit that others have parts of goes to the workspace: at most the end of one unit
// (part 2 w) and the beginning of another (part 2 w + 1).
struct PagedWork {
    int tiles, steps;                        // units per head; steps of each
    int64_t all;
};
__device__ __forceinline__ PagedWork paged_work(const PagedAttnParams& p, const PagedSequence& s) {
    PagedWork w;
    w.tiles = (s.rows * p.group + p.height - 1) / p.height;
    w.steps = (s.keys + p.step - 1) / p.step;
    w.all = (int64_t)p.HK * w.tiles * (w.steps + p.overhead);
    return w;
}
// Workgroup w of `groups` has all w / groups (rounded down) and up to where the next begins: none is empty, because no more of them work than there are places.
__device__ __forceinline__ int64_t paged_groups(const PagedAttnParams& p, int64_t all) { return min((int64_t)p.groups, all); }
__device__ __forceinline__ int paged_owner(int64_t x, int64_t all, int64_t groups) { return (int)(((x + 1) * groups - 1) / all); }

// Where a workgroup begins: the sequence with place `from` of the row, and the work before it.  by all 256 threads
struct PagedStart { int64_t n, before, from, to; };
__device__ __forceinline__ PagedStart paged_start(const PagedAttnParams& p, int group) {
    __shared__ int64_t sums[4], found[2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    auto work = [&](int64_t n) { return n < p.N ? paged_work(p, paged_sequence<false>(p, n)).all : (int64_t)0; };
    auto share = [&](int64_t all) {
        const int64_t groups = max(paged_groups(p, all), (int64_t)1);
        return PagedStart{p.N, 0, group < groups ? all * group / groups : all, group < groups ? all * (group + 1) / groups : all};
    };
    if (p.N <= 64) {                                             // every wave by itself
        const int64_t x = work(lane);
        int64_t upto = x;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t y = __shfl_up(upto, d, 64);
            if (lane >= d) upto += y;
        }
        const int64_t all = __shfl(upto, 63, 64);
        if (group == 0 && wave == 0) {
            if (lane < p.N) p.before[lane] = upto - x;
            if (lane == 0) p.before[p.N] = all;
        }
        PagedStart at = share(all);
        const uint64_t has = __ballot(upto - x <= at.from && at.from < upto);
        if (has) {
            at.n = __builtin_ctzll(has);
            at.before = __shfl(upto - x, (int)at.n, 64);
        }
        return at;
    }
    const int64_t first = work(threadIdx.x);
    int64_t mine = first;
    for (int64_t n = threadIdx.x + 256; n < p.N; n += 256) mine += work(n);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d, 64);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    const int64_t all = sums[0] + sums[1] + sums[2] + sums[3];
    PagedStart at = share(all);
    if (group == 0 && threadIdx.x == 0) p.before[p.N] = all;
    int64_t before = 0;
    for (int64_t n0 = 0; n0 < p.N; n0 += 256) {
        const int64_t n = n0 + threadIdx.x, x = n0 ? work(n) : first;
        int64_t upto = x;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t y = __shfl_up(upto, d, 64);
            if (lane >= d) upto += y;
        }
        __syncthreads();
        if (lane == 63) sums[wave] = upto;
        if (threadIdx.x == 0) found[0] = -1;
        __syncthreads();
        upto += before;
        for (int w = 0; w < wave; ++w) upto += sums[w];
        if (group == 0 && n < p.N) p.before[n] = upto - x;
        if (upto - x <= at.from && at.from < upto) { found[0] = n; found[1] = upto - x; }
        before += sums[0] + sums[1] + sums[2] + sums[3];
        __syncthreads();
        if (found[0] >= 0) { at.n = found[0]; at.before = found[1]; }
        if (group != 0 && before > at.from) break;
    }
    return at;
}

// The places of a tile's keys.  UNIFORM (pages of a multiple of 16 slots): a page for each 16 keys, the same for all lanes.  Else a place for each key, in lane key % 32.
template <bool UNIFORM> struct TilePlaces;
template <> struct TilePlaces<true> {
    uint64_t k[2], v[2];                     // first key of either half, in elements
    uint32_t there;                          // bit per key: its page is one of the cache
};
template <> struct TilePlaces<false> {
    int64_t k, v;
    uint32_t there;
};

template <typename T, int DT, int RT, bool UNIFORM, bool FULL, bool SHARED>
struct PagedWave {
    typedef typename Mma<T>::V8 V8;
    static constexpr int LD = DT + 4, ODD = DT / 32, ROW = 2 * DT, PIECES = ROW / 16;   // LDS: floats of a row of sums, words of odd_bits, bytes and 16-byte pieces of a key
    static constexpr int KS = DT / 32, VE = DT >= 128 ? 8 : 4, VC = DT / 16 / VE, MT = DT / 16;     // steps of a score; elements of V at a place, places, products per row tile
    const PagedAttnParams& p;
    const PagedSequence& s;
    const int64_t n;
    const int hk, lane, c16, g;
    typedef uint32_t VPiece __attribute__((ext_vector_type(VE / 2), aligned(2)));
    V8 q[RT][KS], k[2][KS];
    uint32_t v[DT / 4];                      // pairs: of elements of a key as they lie in memory (operand()), or of keys of an element (SHARED)
    f32x4 o[RT][MT];
    float m[RT], l[RT];
    int token[RT];                           // row of the sequence that the lane's column is; -1: none
    bool odd;                                // infinities and NaN of V are in LDS
    uint64_t* const odd_bits;                // the wave's place there, [16 RT][ODD]: for each 64 elements those up, those down

    __device__ __forceinline__ PagedWave(const PagedAttnParams& p, const PagedSequence& s, int64_t n, int hk, uint64_t* odd_bits)
        : p(p), s(s), n(n), hk(hk), lane(threadIdx.x & 63), c16(lane & 15), g(lane >> 4), odd(false), odd_bits(odd_bits) {}

    __device__ __forceinline__ int page_index(int slot) const { return (int)(((uint64_t)(uint32_t)slot * p.page_magic) >> p.page_shift); }

    __device__ __forceinline__ uint64_t k_place(uint32_t page, uint32_t inside) const { return (uint64_t)page * p.k_page + (uint64_t)inside * p.k_slot + (uint64_t)hk * p.k_head; }
    __device__ __forceinline__ uint64_t v_place(uint32_t page, uint32_t inside) const { return (uint64_t)page * p.v_page + (uint64_t)inside * p.v_slot + (uint64_t)hk * p.v_head; }

    __device__ __forceinline__ TilePlaces<UNIFORM> places(int tile) const {
        TilePlaces<UNIFORM> t;
        const PagedCache& c = p.cache;
        if constexpr (UNIFORM) {
            t.there = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int slot = tile * PA_TILE + 16 * b, index = page_index(slot);
                int page = -1;
                if (slot < s.keys) page = (int)load_index_uniform(c.pages.table, n * c.pages.table_stride + index, true);
                const bool there = page >= 0 && page < c.pages.pages;
                const int inside = there ? slot - index * c.pages.page_size : 0;
                page = there ? page : 0;
                t.there |= there ? 0xffffu << 16 * b : 0;
                t.k[b] = k_place(page, inside);
                t.v[b] = v_place(page, inside);
            }
        } else {
            const int slot = tile * PA_TILE + (lane & 31), index = page_index(slot);
            int page = -1;
            if (slot < s.keys) page = c.pages.table[n * c.pages.table_stride + index];
            const bool there = page >= 0 && page < c.pages.pages;
            const int inside = there ? slot - index * c.pages.page_size : 0;
            page = there ? page : 0;
            t.there = (uint32_t)__ballot(there);
            t.k = page * c.k_page + inside * c.k_slot + hk * c.k_head;
            t.v = page * c.v_page + inside * c.v_slot + hk * c.v_head;
        }
        return t;
    }

    __device__ __forceinline__ void load_k(const TilePlaces<UNIFORM>& t) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint16_t* at;
            if constexpr (UNIFORM) at = (const uint16_t*)p.cache.k + t.k[b] + (c16 * p.k_slot + 8 * g);
            else at = (const uint16_t*)p.cache.k + __shfl(t.k, 16 * b + c16, 64) + 8 * g;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                // (behind the head: nothing, from a place that is there)
                const bool inside = FULL || 32 * ks + 8 * g < p.D;
                const pa_whole x = *(const pa_whole*)(at + (inside ? 32 * ks : -8 * g));
                k[b][ks] = __builtin_bit_cast(V8, inside ? x : pa_whole{});
            }
        }
    }

    // Lane (c16, g): elements VE c16 .. of keys 16 b + 4 g + e, which are contraction indices 8 g + 4 b + e.
    __device__ __forceinline__ void load_v(const TilePlaces<UNIFORM>& t) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint16_t* at;
                if constexpr (UNIFORM) at = (const uint16_t*)p.cache.v + (t.v[b] + (uint64_t)(e * p.v_slot)) + (4 * g * p.v_slot + VE * c16);
                else at = (const uint16_t*)p.cache.v + __shfl(t.v, 16 * b + 4 * g + e, 64) + VE * c16;
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    const VPiece x = *(const VPiece*)(at + (FULL || 128 * c + VE * c16 < p.D ? 128 * c : -VE * c16));
#pragma unroll
                    for (int t = 0; t < VE / 2; ++t) v[pair(4 * b + e, c, t)] = x[t];
                }
            }
    }
    static constexpr int pair(int j, int c, int t) { return (j * VC + c) * (VE / 2) + t; }

    // The first operand of product t of a row tile, V^T: 16 elements of the eight keys of the lane's contraction indices.
    __device__ __forceinline__ V8 operand(int t) const {
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (SHARED) a[j] = v[4 * t + j];
            else a[j] = __builtin_amdgcn_perm(v[pair(2 * j + 1, t / VE, t % VE / 2)], v[pair(2 * j, t / VE, t % VE / 2)], t % 2 ? 0x07060302u : 0x05040100u);
        }
        return __builtin_bit_cast(V8, a);
    }

    __device__ __forceinline__ void start(int row0) {
        const int rows = s.rows * p.group;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = row0 + 16 * r + c16;
            token[r] = row < rows ? row / p.group : -1;
            const int h = hk * p.group + (row < rows ? row - token[r] * p.group : 0);
            const int64_t t = token[r] < 0 ? 0 : token[r];
            const uint16_t* at = (const uint16_t*)p.q + (p.cu ? (s.first + t) * p.qt : n * p.qb + t * p.qt) + h * p.qh + 8 * g;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                pa_whole x = {};
                if (token[r] >= 0 && 32 * ks + 8 * g < p.D) x = *(const pa_whole*)(at + 32 * ks);
                q[r][ks] = __builtin_bit_cast(V8, p.negative ? x ^ (uint16_t)0x8000 : x);
            }
            m[r] = -INFINITY; l[r] = 0.f;
#pragma unroll
            for (int t2 = 0; t2 < MT; ++t2) o[r][t2] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // What is formed of the result is formed where it is used: the rare paths' places held in registers through the whole loop would not leave the loop enough.
    static __device__ __forceinline__ int unhoisted(int x) {
        asm volatile("" : "+v"(x));
        return x;
    }

    // Which keys of a tile row token[r] sees of those whose pages are there: bit 4 b + e for key 16 b + 4 g + e.
    __device__ __forceinline__ uint32_t seen(int r, int tile, uint32_t there) const {
        const int g = unhoisted(lane) >> 4, fresh = (int)(tile * PA_TILE + 4 * g - s.context), most = p.mask ? min(p.mask_cols, s.rows) : token[r] + 1;
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = 16 * (i / 4) + i % 4;
            bits |= fresh + at < most && there >> (4 * g + at) & 1 ? 1u << i : 0;
        }
        if (p.mask) {
            // (all asked for at once, inside of the row)
            const int64_t row = max(unhoisted(token[r]), 0);
            const uint8_t* mask = p.mask + (p.cu ? (s.first + row) * p.mask_row : n * p.mask_seq + row * p.mask_row);
            uint8_t is[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) is[i] = mask[min(max(fresh + 16 * (i / 4) + i % 4, 0), most - 1)];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (fresh + 16 * (i / 4) + i % 4 >= 0 && !is[i]) bits &= ~(1u << i);
        }
        return bits;
    }

    // stage: where the tile lies in LDS (NULL: nowhere); next_k: asked for between the two products
    template <typename Next>
    __device__ __forceinline__ void tile(int tile, const TilePlaces<UNIFORM>& at, const char* stage, Next&& next_k) {
        // The keys of the context whose pages are there are seen by every row; the tiles behind them are few.
        const bool whole = tile < s.whole && at.there == 0xffffffffu;
        uint32_t bits[RT];
        if (!whole) {
#pragma unroll
            for (int r = 0; r < RT; ++r) bits[r] = seen(r, tile, at.there);
        }
        f32x4 x[RT][2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < RT; ++r) x[r][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (a product waits for the one before it in its own sum: the sums take turns)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < RT; ++r) x[r][b] = Mma<T>::run(k[b][ks], q[r][ks], x[r][b]);
        next_k();
        if (!whole) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[r][i / 4][i % 4] = bits[r] >> i & 1 ? x[r][i / 4][i % 4] : -INFINITY;
        }
        V8 w[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, x[r][i / 4][i % 4]);
            // m is a maximum that was passed by 2^8 at most: it is the same in the four lanes of a row and moves a few times only (as the true maximum it would move in
            // four tiles of ten of the first 4000 keys).  The sums' terms are up to 2^8 then (of fp16 2^15, PA_LIFT), of 2^128.
            if (__any((most - m[r]) * p.scale2 > 8.f || (m[r] == -INFINITY && most > m[r]))) {
                most = fmaxf(most, __shfl_xor(most, 16, 64));
                most = fmaxf(most, __shfl_xor(most, 32, 64));
                const float now = fmaxf(m[r], most), keep = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[r] - now) * p.scale2);
                m[r] = now;
                l[r] *= keep;
#pragma unroll
                for (int t = 0; t < MT; ++t) o[r][t] *= keep;
            }
            // (no maximum yet: nothing is seen, or what is seen is not a number and makes the row's sums so)
            // (the distance from it before the scale: a large score's steps may be far above 1, its distance from itself is 0)
            const float base = m[r] == -INFINITY ? 0.f : m[r];
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r][i / 4][i % 4] - base, p.scale2, PA_LIFT<T>));
            if (!whole) {                                                   // (of a scale of zero nothing is -inf)
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[r][i / 4][i % 4] == -INFINITY ? 0.f : y[i];
            }
            l[r] += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
            w[r] = __builtin_bit_cast(V8, u32x4{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])});
        }
        if (!whole && __any(odd_values())) clean(bits, at, stage);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const V8 a = operand(t);
#pragma unroll
            for (int r = 0; r < RT; ++r) o[r][t] = Mma<T>::run(a, w[r], o[r][t]);
        }
    }

    static __device__ __forceinline__ uint32_t carry(uint32_t pair) { return ((pair & PA_EXPONENT<T> * 0x10001u) + PA_CARRY<T> * 0x10001u) & 0x80008000u; }
    // Infinities and NaN in V, in tiles whose keys not every row sees: a weight of zero does not keep them out of a product.
    __device__ __forceinline__ bool odd_values() const {
        uint32_t carried = 0;
#pragma unroll
        for (int i = 0; i < DT / 4; ++i) carried |= carry(v[i]);
        return carried;
    }
    // They are taken out of V and kept in LDS for the rows that see the key (bits, seen()), however little it weighs: a bit for each row and element: what a sum of
    // infinities and NaN will be, whatever is added to it (both bits: NaN).
    __device__ __forceinline__ void clean(const uint32_t (&bits)[RT], const TilePlaces<UNIFORM>& at, const char* stage) {
        const int lane = unhoisted(this->lane), c16 = lane & 15, g = lane >> 4;
        uint64_t* const mine = odd_bits + (16 * g + c16) * ODD;                 // (lanes of g < RT: row 16 g + c16)
        if (!odd) {
            if (g < RT)
                for (int i = 0; i < ODD; ++i) mine[i] = 0;
            odd = true;
        }
        uint32_t row = 0;                                                   // the keys that the lane's row sees
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            uint32_t keys = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) keys |= bits[r] >> i & 1 ? 1u << (16 * (i / 4) + 4 * g + i % 4) : 0;
            keys |= __shfl_xor(keys, 16, 64);
            keys |= __shfl_xor(keys, 32, 64);
            if (g == r) row = keys;
        }
#pragma unroll
        for (int i = 0; i < DT / 4; ++i) v[i] &= ~((carry(v[i]) >> 15) * 0xffffu);
#pragma nounroll
        for (int key = 0; key < PA_TILE; ++key) {
            if (!(at.there >> key & 1)) continue;
            const uint16_t* from;
            if (stage) from = (const uint16_t*)(stage + TILE + key * ROW);
            else if constexpr (UNIFORM) from = (const uint16_t*)p.cache.v + (key < 16 ? at.v[0] : at.v[1]) + (key & 15) * p.cache.v_slot;
            else from = (const uint16_t*)p.cache.v + __shfl(at.v, key, 64);
#pragma nounroll
            for (int i = 0; i < DT / 64; ++i) {
                const int d = 64 * i + lane;
                uint16_t bits = 0;
                if (d < p.D) bits = from[stage ? d ^ swizzle(key) * 8 : d];
                const bool is = not_a_number<T>(bits), nan = is && (bits & ~PA_EXPONENT<T> & 0x7fffu);
                const uint64_t up = __ballot(is && (nan || !(bits >> 15))), down = __ballot(is && (nan || bits >> 15));
                if ((up | down) && g < RT && row >> key & 1) { mine[2 * i] |= up; mine[2 * i + 1] |= down; }
            }
        }
    }
    // What they make of element d of a row of the wave: infinity, minus infinity, NaN, or nothing.
    __device__ __forceinline__ float odd_sum(int row, int d) const {
        const uint64_t* at = odd_bits + row * ODD + 2 * (d / 64);
        const bool up = at[0] >> (d & 63) & 1, down = at[1] >> (d & 63) & 1;
        return up && down ? __builtin_nanf("") : up ? INFINITY : down ? -INFINITY : 0.f;
    }

    // ---- four waves on the same keys: 64 at a time through LDS ----
    // A stage holds K, then V, of two tiles as they lie in memory, the 16-byte pieces of row r in places XORed with twice r
    // (so that eight rows of a piece, and four rows of two pieces, meet no bank twice).  Copies are
    // of 1 KB, straight into LDS, asked for by inline assembly and waited for by hand; a wave makes those of 16 keys, so of one page.
    static constexpr int TILE = PA_TILE * ROW, STAGE = 4 * TILE, STAGES = 2;

    static __device__ __forceinline__ int swizzle(int row) { return (2 * (row & 7) + (row >> 3 & 1)) & (PIECES - 1) & 15; }
    struct Block { int page, inside; };
    __device__ __forceinline__ Block block_of(int stage, int wave) const {
        const int slot = 64 * stage + 16 * wave, index = page_index(slot);
        int page = -1;
        if (slot < s.keys) page = (int)load_index_uniform(p.cache.pages.table, n * p.cache.pages.table_stride + index, true);
        return Block{page, slot - index * p.cache.pages.page_size};
    }
    // there: a half word for each wave's keys, all ones where their page is one of the cache
    __device__ __forceinline__ void ask(const Block& from, uint32_t to, uint16_t* there, int wave) {
        const bool is = from.page >= 0 && from.page < p.cache.pages.pages;
        const uint32_t page = is ? from.page : 0, inside = is ? from.inside : 0;
        const char* kb = p.cache.k + 2 * k_place(page, inside);
        const char* vb = p.cache.v + 2 * v_place(page, inside);
        constexpr int EACH = 16 * ROW / 1024, KEYS = 1024 / ROW;            // copies of K (and of V), keys of one
        const uint32_t k0 = to + wave / 2 * (2 * TILE) + (wave & 1) * 16 * ROW;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int key = i * KEYS + lane * 16 / ROW;
            int element = 8 * ((lane % PIECES) ^ swizzle(key));
            if (!FULL && element >= p.D) element = 0;
            gather_1k_to_lds(kb, 2 * (key * p.k_slot + element), k0 + i * 1024);
            gather_1k_to_lds(vb, 2 * (key * p.v_slot + element), k0 + TILE + i * 1024);
        }
        if (lane == 0) there[wave] = is ? 0xffff : 0;
    }
    __device__ __forceinline__ void read_k(const char* at) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const pa_aligned x = *(const pa_aligned*)(at + (16 * b + c16) * ROW + 16 * ((4 * ks + g) ^ swizzle(c16)));
                k[b][ks] = __builtin_bit_cast(V8, FULL || 32 * ks + 8 * g < p.D ? x : pa_aligned{});
            }
    }
    // Transposed on the way: lane c16 of a group of 16 names four elements of key 4 g + c16 / 4 and receives element 16 t + c16 of the group's four keys.
    __device__ __forceinline__ void read_v(const char* at) {
        const int row = 4 * g + c16 / 4;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const auto x = Mma<T>::tr_read((const T*)(at + TILE + (16 * b + row) * ROW + 16 * ((2 * t + (c16 & 3) / 2) ^ swizzle(row)) + 8 * (c16 & 1)));
                const u32x2 two = __builtin_bit_cast(u32x2, x);
                v[4 * t + 2 * b] = two[0]; v[4 * t + 2 * b + 1] = two[1];
            }
    }

    // Stages first .. last - 1, all four waves on each.  there: [STAGES][4]
    __device__ __forceinline__ void run_shared(int first, int last, int wave, char* stages, uint16_t* there) {
        if (first >= last) return;
        const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)stages;
        ask(block_of(first, wave), base, there, wave);
        Block next = block_of(first + 1, wave);
        int now = 0;
        for (int i = first; i < last; ++i) {
            wait_vm_at_most<0>();
            lds_barrier();
            const uint64_t all = *(const uint64_t*)(there + 4 * now);
            if (i + 1 < last) ask(next, base + (now ^ 1) * STAGE, there + 4 * (now ^ 1), wave);
            next = block_of(i + 2, wave);
            TilePlaces<true> at = {};
#pragma nounroll
            for (int half = 0; half < 2; ++half) {
                const char* from = stages + now * STAGE + half * (2 * TILE);
                at.there = __builtin_amdgcn_readfirstlane((uint32_t)(all >> 32 * half));
                if (!at.there) continue;
                read_k(from);
                tile(2 * i + half, at, from, [&] { read_v(from); });
            }
            now ^= 1;
        }
    }

    __device__ __forceinline__ void run(int first, int last, int step) {
        if (first >= last) return;
        TilePlaces<UNIFORM> now = places(first), next = places(first + step);
        load_k(now);
        load_v(now);
        for (int t = first; t < last; t += step) {
            const bool more = t + step < last;
            tile(t, now, nullptr, [&] { if (more) load_k(next); });
            if (more) load_v(next);
            now = next;
            next = places(t + 2 * step);
        }
    }
};

template <typename T, int DT, int RT, bool UNIFORM, bool FULL, bool SHARED>
__global__ __launch_bounds__(256, DT == 256 ? 1 : 2) void paged_attn_kernel(PagedAttnParams p) {
    typedef PagedWave<T, DT, RT, UNIFORM, FULL, SHARED> Wave;
    static_assert(!SHARED || UNIFORM, "copies of whole pieces");
    constexpr int VE = Wave::VE, LD = Wave::LD;
    extern __shared__ float lds[];                               // [4 waves][16 RT][LD], then [4 waves][16 RT][2]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), group = blockIdx.x;
    const int rg = wave % p.row_groups, kg = wave / p.row_groups, key_groups = 4 / p.row_groups, height = p.height;
    if (p.cu) {
        // rows of no sequence
        const int64_t first = max(min(load_index_uniform(p.cu, 0, p.cu_i32), p.total), (int64_t)0), last = max(load_index_uniform(p.cu, p.N, p.cu_i32), first), width = (int64_t)p.HQ * p.D;
        for (int64_t row = group; row < p.total; row += p.groups)
            if (row < first || row >= last)
                for (int64_t d = threadIdx.x; d < width; d += 256) ((T*)p.o)[row * width + d] = (T)0.f;
    }
    const PagedStart start = paged_start(p, group);
    int64_t n = scalar(start.n), before = scalar(start.before), x = scalar(start.from);
    const int64_t to = scalar(start.to);
    while (x < to && n < p.N) {
        const PagedSequence s = paged_sequence(p, n);
        const PagedWork work = paged_work(p, s);
        if (x >= before + work.all) { before += work.all; ++n; continue; }
        const int per = work.steps + p.overhead, unit = (int)((x - before) / per);
        const int64_t begins = before + (int64_t)unit * per, ends = min(to, begins + per);
        const int first = max((int)(x - begins) - p.overhead, 0), last = max((int)(ends - begins) - p.overhead, 0);
        const bool all_of_it = first == 0 && last == work.steps;
        const int hk = unit / work.tiles, tile = unit - hk * work.tiles, rows = s.rows * p.group;
        const bool its_start = x == begins;
        x = ends;
        if (first == last && !(work.steps == 0 && its_start)) continue;
        Wave w(p, s, n, hk, (uint64_t*)((char*)lds + p.odd_at) + wave * 16 * RT * Wave::ODD);
        w.start(tile * height + rg * 16 * RT);
        // (without a mask a row sees no row behind it: nor do the keys behind the last row's matter)
        const int last_token = min((tile * height + height - 1) / p.group, s.rows - 1);
        const int keys = p.mask ? s.keys : (int)min((int64_t)s.keys, max(s.context + last_token + 1, (int64_t)0));
        if constexpr (SHARED) {
            w.run_shared(first, min(last, (keys + 2 * PA_TILE - 1) / (2 * PA_TILE)), wave, (char*)lds, (uint16_t*)((char*)lds + p.odd_at - 64));
            __syncthreads();
        } else {
            w.run(first * key_groups + kg, min(last * key_groups, (keys + PA_TILE - 1) / PA_TILE), key_groups);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            w.l[r] += __shfl_xor(w.l[r], 16, 64);
            w.l[r] += __shfl_xor(w.l[r], 32, 64);
        }
        // The waves that share rows, joined: each leaves its sums with its maximum.
        float* const ml = lds + 4 * 16 * RT * LD;
        const int lane = Wave::unhoisted(w.lane), c16 = lane & 15, g = lane >> 4;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = wave * 16 * RT + 16 * r + c16;
            auto put = [&](int d, f32x4 sum) {
                if (w.odd) sum += f32x4{w.odd_sum(16 * r + c16, d), w.odd_sum(16 * r + c16, d + 1), w.odd_sum(16 * r + c16, d + 2), w.odd_sum(16 * r + c16, d + 3)};
                *(f32x4*)(lds + row * LD + d) = sum;
            };
            if constexpr (SHARED) {
#pragma unroll
                for (int t = 0; t < Wave::MT; ++t) put(16 * t + 4 * g, w.o[r][t]);
            } else {
#pragma unroll
                for (int t = 0; t < Wave::MT; t += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e) put(128 * (t / VE) + VE * (4 * g + e) + t % VE, f32x4{w.o[r][t][e], w.o[r][t + 1][e], w.o[r][t + 2][e], w.o[r][t + 3][e]});
            }
            if (g == 0) { ml[2 * row] = w.m[r] == -INFINITY ? -INFINITY : w.m[r] * p.scale2; ml[2 * row + 1] = w.l[r]; }
        }
        __syncthreads();
        constexpr int PIECES = DT / 4;
        for (int i = threadIdx.x; i < height * PIECES; i += 256) {
            const int row = i / PIECES, d = 4 * (i % PIECES), at = row + tile * height;
            if (at >= rows || d >= p.D) continue;
            float m = -INFINITY;
            for (int k = 0; k < key_groups; ++k) m = fmaxf(m, ml[2 * (row + k * height)]);
            const float base = m == -INFINITY ? 0.f : m;
            float l = 0.f;
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < key_groups; ++k) {
                const int from = row + k * height;
                const float keep = __builtin_amdgcn_exp2f(ml[2 * from] - base);
                l += ml[2 * from + 1] * keep;
                sum += *(const f32x4*)(lds + from * LD + d) * keep;
            }
            const int token = at / p.group;
            const int64_t out = (s.first + token) * p.HQ + hk * p.group + (at - token * p.group);
            if (all_of_it) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
                typedef T piece __attribute__((ext_vector_type(4)));
                *(piece*)((T*)p.o + out * p.D + d) = piece{(T)(sum[0] * inv), (T)(sum[1] * inv), (T)(sum[2] * inv), (T)(sum[3] * inv)};
            } else {
                const int64_t part = (int64_t)(2 * group + (first == 0)) * height + row;
                *(f32x4*)(p.part_o + part * p.D + d) = sum;
                if (d == 0) { p.part_ml[2 * part] = m; p.part_ml[2 * part + 1] = l; }
            }
        }
        __syncthreads();
    }
}

// The parts of a row's keys, joined, where several workgroups have some: by a wave, or by four where a unit has many parts.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnParams p) {
    constexpr int AHEAD = 4;
    __shared__ f32x4 sums[WAVES][64];
    __shared__ float weights[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), sub = wave % WAVES;
    const int64_t row = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
    if (row >= p.total * p.HQ) return;                           // (four waves of a row end together)
    const int64_t token = row / p.HQ;
    const int h = (int)(row - token * p.HQ), hk = h / p.group;
    const int64_t n = p.cu ? sequence_of(token, p.N, [&](int64_t j) { return load_index(p.cu, j, p.cu_i32); }) : token / p.T;
    if (n < 0) return;
    const PagedSequence s = paged_sequence<false>(p, n);
    const PagedWork work = paged_work(p, s);
    const int64_t i = (token - s.first) * p.group + h - hk * p.group;
    if (work.steps == 0 || i < 0 || i >= (int64_t)s.rows * p.group) return;
    const int tile = (int)(i / p.height), at = (int)(i - (int64_t)tile * p.height);
    const int64_t all = p.before[p.N], groups = paged_groups(p, all), begins = p.before[n] + ((int64_t)hk * work.tiles + tile) * (work.steps + p.overhead) + p.overhead;
    const int first = paged_owner(begins, all, groups), last = paged_owner(begins + work.steps - 1, all, groups);
    if (first == last) return;
    auto part = [&](int w) { return (int64_t)(2 * w + (w == first)) * p.height + at; };
    float m = -INFINITY;
    for (int w = first + lane; w <= last; w += 64) m = fmaxf(m, p.part_ml[2 * part(w)]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d, 64));
    const float base = m == -INFINITY ? 0.f : m;
    const int d = 4 * lane;
    float l = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int w = first + sub; w <= last; w += AHEAD * WAVES) {
        f32x4 x[AHEAD];
        float ml[AHEAD][2];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int we = w + e * WAVES;
            const int64_t from = part(min(we, last));
            ml[e][0] = we <= last ? p.part_ml[2 * from] : -INFINITY;
            ml[e][1] = p.part_ml[2 * from + 1];
            x[e] = d < p.D ? *(const f32x4*)(p.part_o + from * p.D + d) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            if (w + e * WAVES > last) continue;
            const float keep = __builtin_amdgcn_exp2f(ml[e][0] - base);
            l += ml[e][1] * keep;
            sum += x[e] * keep;
        }
    }
    if constexpr (WAVES > 1) {
        sums[sub][lane] = sum;
        if (lane == 0) weights[sub] = l;
        __syncthreads();
        if (sub) return;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) { sum += sums[k][lane]; l += weights[k]; }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typedef T piece __attribute__((ext_vector_type(4)));
    if (d < p.D) *(piece*)((T*)p.o + row * p.D + d) = piece{(T)(sum[0] * inv), (T)(sum[1] * inv), (T)(sum[2] * inv), (T)(sum[3] * inv)};
}

static int check_attn(const char* who, const gdn_paged_cache* cache, const gdn_paged_attn_call* c, PagedCache& out) {
    GDN_CHECK_ARG(c && c->B >= 0 && c->T >= 0 && c->HQ >= 0 && c->max_rows >= 0 && (c->cu_seqlens ? c->B == 1 && c->N >= 1 : c->N == c->B), GDN_ERR_INVALID, "%s: bad sizes", who);
    const int rc = check_cache(who, cache, c->N, out);
    if (rc != GDN_OK) return rc;
    GDN_CHECK_ARG(c->HQ % cache->heads == 0, GDN_ERR_INVALID, "%s: the queries' heads are a multiple of the cache's", who);
    // (a row's bytes are asked for before it is known which of them count: one of them has to be there)
    GDN_CHECK_ARG(!c->mask || c->mask_cols >= 1, GDN_ERR_INVALID, "%s: a mask has columns", who);
    GDN_CHECK_ARG(cache->dtype != GDN_DTYPE_F32 && cache->dim <= PA_MAX_DIM && cache->dim % 8 == 0, GDN_ERR_UNSUPPORTED, "%s: bf16 or fp16 heads of a multiple of 8 up to %d elements", who, PA_MAX_DIM);
    // (a launch has fewer than 2^32 threads: 64 for each row of a head, in blocks of 256)
    GDN_CHECK_ARG(c->B < (1ll << 26) && c->T < (1ll << 26) && c->HQ < (1ll << 26) && c->B * c->T < (1ll << 26) && c->B * c->T * c->HQ <= (1ll << 26) - 4 && cache->table_cols * cache->page_size <= (1ll << 30) && c->mask_cols < (1ll << 31), GDN_ERR_UNSUPPORTED,
                  "%s: rows times heads up to 2^26 - 4, up to 2^30 slots of a sequence", who);
    // (the work is counted in 64 bits, times the workgroups)
    GDN_CHECK_ARG((double)c->N * (double)cache->heads * (double)(c->T * (c->HQ / cache->heads) / 16 + 1) * (double)(cache->table_cols * cache->page_size / 32 + 8) < 4e15, GDN_ERR_UNSUPPORTED,
                  "%s: too much work for one call", who);
    return GDN_OK;
}

struct PagedAttnPlan { int dim, row_tiles, row_groups, height, step, overhead, groups; bool shares, many_parts; size_t bytes; };
static PagedAttnPlan attn_plan(const gdn_paged_cache* cache, const gdn_paged_attn_call* c, bool uniform, bool shares) {
    PagedAttnPlan plan;
    const int64_t rows = std::max<int64_t>(1, std::min(c->max_rows, c->T)) * (c->HQ / cache->heads);
    plan.dim = cache->dim <= 64 ? 64 : cache->dim <= 128 ? 128 : 256;
    // More than 32 rows: the four waves on the same keys, through LDS.  Else by themselves, two row tiles where the registers hold them beside the keys under way (heads
    // of the whole 64 or 128 elements in pages of whole tiles).
    plan.shares = shares && rows > 32;
    plan.row_tiles = plan.dim < 256 && (plan.shares ? rows > 64 : rows > 16 && uniform && cache->dim == plan.dim) ? 2 : 1;
    const int64_t each = 16 * plan.row_tiles;
    plan.row_groups = plan.shares || rows > 2 * each ? 4 : rows > each ? 2 : 1;
    plan.height = (int)(each * plan.row_groups);
    plan.step = plan.shares ? 2 * PA_TILE : PA_TILE * (4 / plan.row_groups);
    // What a unit costs besides its keys, in steps.  Measured, us a call (1, 2, 4, 6, 8 steps): 16 sequences of up to 8000 keys with trees of 64 rows 219, 189, 166, 148, 149 (through
    // LDS); 32 of up to 8000 with 8 rows of 4 heads 142, 129, 131, 131, 133, 33 of up to 3001 with 7 rows of 2 heads 29.4, 27.7, 27.3; 256 of up to 1000 with one row of 4 heads 115,
    // 117, 123, 123, 124, one of 4000 15.6, 16.6, 16.9.
    plan.overhead = plan.shares ? 6 : rows > 8 ? 2 : 1;
    // One round of the chip: two workgroups share a CU (one where a head of 256 takes a wave's registers), but no more than there can be steps.
    const int64_t units = std::max<int64_t>(1, c->N) * cache->heads * ((rows + plan.height - 1) / plan.height);
    const int64_t steps = std::max<int64_t>(1, (cache->table_cols * cache->page_size + plan.step - 1) / plan.step);
    plan.groups = (int)std::min<int64_t>(plan.dim == 256 ? 256 : 512, units * steps);
    // The join of a row's parts by four waves in place of one: measured, us a call of a replayed graph (parts that a unit may have), heads of 128: 32 rows on one head of the
    // cache 18.3 and 18.3 (3), 19.2 and 18.6 (8), 30.8 and 27.0 (16), 50.6 and 42.5 (32), 64.9 and 31.6 (256); four on each of 8 heads 24.4 and 24.3 (4), 21.3 and 20.6 (8), 26.1 and
    // 24.1 (16), 43.8 and 35.7 (64).  It has four times the workgroups, so it is for few rows.
    plan.many_parts = plan.groups > 8 * units && c->B * c->T * c->HQ < (1 << 24);
    plan.bytes = ((size_t)c->N + 2) / 2 * 16 + (size_t)2 * plan.groups * plan.height * (cache->dim + 2) * sizeof(float);
    return plan;
}
// Rows on 16-byte boundaries: copies into LDS.
static bool whole_pieces(const PagedCache& v) {
    return (((uintptr_t)v.k | (uintptr_t)v.v) & 15) == 0 && ((v.k_page | v.k_slot | v.k_head | v.v_page | v.v_slot | v.v_head) & 7) == 0;
}
// A page for 16 keys; strides in 32 bits.
static bool uniform_tiles(const gdn_paged_cache* c) {
    bool is = c->page_size % 16 == 0 && std::max(c->k_stride[1], c->v_stride[1]) < (1ll << 24);
    for (int i = 0; i < 3; ++i)
        for (int64_t stride : {c->k_stride[i], c->v_stride[i]}) is = is && stride >= 0 && stride < (1ll << 32);
    return is;
}

}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_paged_attn_workspace_bytes(const gdn_paged_cache* cache, const gdn_paged_attn_call* c) {
    PagedCache view;
    if (check_attn("gdn_paged_attn_workspace_bytes", cache, c, view) != GDN_OK || c->B * c->T * c->HQ == 0) return 0;
    const bool uniform = uniform_tiles(cache);
    return attn_plan(cache, c, uniform, uniform && whole_pieces(view)).bytes;
}

extern "C" int gdn_paged_attn(const gdn_paged_cache* cache, const gdn_paged_attn_call* c, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "gdn_paged_attn";
    PagedAttnParams p{};
    const int rc = check_attn(who, cache, c, p.cache);
    if (rc != GDN_OK) return rc;
    if (c->B * c->T * c->HQ == 0) return GDN_OK;
    GDN_CHECK_ARG(c->q && c->o, GDN_ERR_INVALID, "%s: missing tensors", who);
    const bool uniform = uniform_tiles(cache);
    const PagedAttnPlan plan = attn_plan(cache, c, uniform, uniform && whole_pieces(p.cache));
    GDN_CHECK_ARG(workspace && workspace_bytes >= plan.bytes && (uintptr_t)workspace % 16 == 0, GDN_ERR_WORKSPACE, "%s: workspace of %zu bytes, 16-byte aligned", who, plan.bytes);
    p.q = c->q; p.o = c->o; p.cu = c->cu_seqlens; p.mask = c->mask;
    p.qb = c->q_stride[0]; p.qt = c->q_stride[1]; p.qh = c->q_stride[2];
    p.mask_seq = c->mask_seq_stride; p.mask_row = c->mask_row_stride; p.mask_cols = (int)c->mask_cols;
    p.T = c->T; p.total = c->B * c->T; p.N = (int)c->N; p.HQ = (int)c->HQ; p.HK = (int)cache->heads; p.D = (int)cache->dim; p.group = p.HQ / p.HK;
    p.cu_i32 = c->flags & GDN_FLAG_CU_INT32;
    p.scale2 = std::fabs(c->scale) * 1.4426950408889634f; p.negative = c->scale < 0;
    p.overhead = plan.overhead; p.height = plan.height; p.step = plan.step; p.groups = plan.groups; p.row_groups = plan.row_groups;
    p.before = (int64_t*)workspace;
    p.part_o = (float*)((char*)workspace + (c->N + 2) / 2 * 16);
    p.part_ml = p.part_o + (size_t)2 * plan.groups * plan.height * (size_t)p.D;
    // slot / page_size for slots below 2^31: ceil(2^(31 + l) / page_size), l = ceil(log2 page_size), is below 2^32 and exact
    int l = 0;
    while ((1ll << l) < cache->page_size) ++l;
    p.page_shift = 31 + l;
    p.page_magic = (uint32_t)(((1ull << p.page_shift) + cache->page_size - 1) / cache->page_size);
    p.k_page = (uint32_t)cache->k_stride[0]; p.k_slot = (uint32_t)cache->k_stride[1]; p.k_head = (uint32_t)cache->k_stride[2];
    p.v_page = (uint32_t)cache->v_stride[0]; p.v_slot = (uint32_t)cache->v_stride[1]; p.v_head = (uint32_t)cache->v_stride[2];
    auto go = [&](auto t, auto dim, auto row_tiles) {
        typedef decltype(t) T;
        constexpr int DT = decltype(dim)::value, RT = decltype(row_tiles)::value;
        auto launch = [&](auto uniform_, auto full_, auto shared_) {
            constexpr bool UNIFORM = decltype(uniform_)::value, FULL = decltype(full_)::value, SHARED = decltype(shared_)::value;
            typedef PagedWave<T, DT, RT, UNIFORM, FULL, SHARED> Wave;
            const size_t joined = (size_t)4 * 16 * RT * (DT + 4 + 2) * sizeof(float), room = 64 + (SHARED ? std::max<size_t>(joined, Wave::STAGES * Wave::STAGE) : joined),
                         smem = room + (size_t)4 * 16 * RT * Wave::ODD * sizeof(uint64_t);
            p.odd_at = (int)room;
            const auto kernel = paged_attn_kernel<T, DT, RT, UNIFORM, FULL, SHARED>;
            const int made = ensure_dynamic_smem_for((const void*)kernel, smem, who);
            if (made == GDN_OK) hipLaunchKernelGGL(kernel, dim3((unsigned)plan.groups), dim3(256), smem, (hipStream_t)stream, p);
            return made;
        };
        const std::true_type yes;
        const std::false_type no;
        const bool whole_head = p.D == DT;
        int made = GDN_ERR_UNSUPPORTED;
        if (plan.shares) made = whole_head ? launch(yes, yes, yes) : launch(yes, no, yes);
        if (!plan.shares) {
            if constexpr (RT == 2) made = launch(yes, yes, no);
            else if (uniform) made = whole_head ? launch(yes, yes, no) : launch(yes, no, no);
            else made = whole_head ? launch(no, yes, no) : launch(no, no, no);
        }
        if (made != GDN_OK) return made;
        const int ran = check_launch("paged_attn_kernel");
        if (ran != GDN_OK || plan.groups == 1) return ran;
        if (plan.many_parts) hipLaunchKernelGGL((paged_attn_join_kernel<T, 4>), dim3((unsigned)(p.total * p.HQ)), dim3(256), 0, (hipStream_t)stream, p);
        else hipLaunchKernelGGL((paged_attn_join_kernel<T, 1>), dim3((unsigned)((p.total * p.HQ + 3) / 4)), dim3(256), 0, (hipStream_t)stream, p);
        return check_launch("paged_attn_join_kernel");
    };
    auto dims = [&](auto t) {
        if (plan.dim == 256) return go(t, std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
        auto tiles = [&](auto dim) { return plan.row_tiles == 1 ? go(t, dim, std::integral_constant<int, 1>()) : go(t, dim, std::integral_constant<int, 2>()); };
        return plan.dim == 64 ? tiles(std::integral_constant<int, 64>()) : tiles(std::integral_constant<int, 128>());
    };
    return cache->dtype == GDN_DTYPE_BF16 ? dims(bf16_t{}) : dims(f16_t{});
}
