// Rotary positions, and keys and values on their way into a paged cache.
//
//   (y1, y2) = (x1 c - x2 s, x1 s + x2 c)      c, s = cos, sin of the row's position, pair (j, j + R/2) or (2j, 2j + 1), j < R/2 <= D/2
//
// The gradient is the turn back (s negated).  Every element is read once and written once; the rows of the tables are read once per row of heads.  The memory system bounds
// it: a thread turns 16 bytes of either half (or of pairs side by side) for two or three heads of its token, asked for before anything that says where the token stands, and
// keeps the tables' values in registers for them.  Loads and stores past the caches: 32768 tokens of 20 heads of 128 83 -> 64 us (5.5 TB/s), prompts of 14000 tokens of
// 48 heads into the cache 116 -> 89, with the rows asked for first 75, with scalar loads of the places 68.7 (5.2 TB/s).
#include "gdn_paged.h"
#include <algorithm>
#include <type_traits>

namespace gdn {

struct RotaryRows {
    const char* x; char* y;
    int64_t xb, xt, xh, yb, yt, yh;       // strides in elements
    int end;                              // heads of this and of the tensors before
    int turn;
    int cache;                            // 0: y [B,T,heads,D]; 1, 2: the keys, the values of the cache
};

struct RotaryParams {
    RotaryRows rows[3];
    int heads;
    const void* cos; const void* sin;
    int64_t table_stride, table_rows;
    const void* positions; const void* offsets; const void* cu;
    int64_t offset, B, T, N;
    int half, D;
    float sign;
    bool pos_i32, off_i32, cu_i32;
    int chunks, chunk_lanes, head_lanes, tokens, each;           // each: heads of a thread at a time
    PagedCache cache;
};

template <typename T, int V, int ALIGN = (V * sizeof(T) > 16 ? 16 : V * sizeof(T))> struct alignas(ALIGN) Pack { T e[V]; };

// (past the caches: a call's rows are more than they hold, or too few to matter)
template <typename P, typename T> __device__ __forceinline__ P load_streamed(const T* at) {
    if constexpr (sizeof(P) == 16) return __builtin_bit_cast(P, __builtin_nontemporal_load((const u32x4*)at));
    else return *(const P*)at;
}
template <typename P, typename T> __device__ __forceinline__ void store_streamed(T* at, const P& x) {
    if constexpr (sizeof(P) == 16) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x), (u32x4*)at);
    else *(P*)at = x;
}

// HEADS: of a thread at a time, at most
template <typename T, typename TT, int V, bool INTER, bool CACHE, int HEADS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
    // (the narrowest form of the interleaved layout takes pairs at any address)
    typedef std::conditional_t<INTER && V == 2, Pack<T, V, sizeof(T)>, Pack<T, V>> P;
    constexpr int PAIRS = INTER ? V / 2 : V;
    const int lanes = p.head_lanes * p.chunk_lanes, local = threadIdx.x / lanes, at = threadIdx.x - local * lanes;
    const int64_t token = (int64_t)blockIdx.x * p.tokens + local;
    if (local >= p.tokens || token >= p.B * p.T) return;
    const int64_t b = p.B == 1 ? 0 : (uint32_t)token / (uint32_t)p.T, t = token - b * p.T;
    const int h0 = at / p.chunk_lanes, c0 = at - h0 * p.chunk_lanes;
    const int turned = INTER ? 2 * p.half / V : p.half / V;
    P a[HEADS], z[HEADS];
    auto place = [&](int c) { return c < turned ? c * V : 2 * p.half + (c - turned) * V; };
    auto load = [&](int c, int h) {
#pragma unroll
        for (int u = 0; u < HEADS; ++u) {
            const int hu = h + u * p.head_lanes;
            if (u >= p.each || hu >= p.heads) continue;
            const int s = hu < p.rows[0].end ? 0 : hu < p.rows[1].end ? 1 : 2;
            const RotaryRows& r = p.rows[s];
            const T* x = (const T*)r.x + b * r.xb + t * r.xt + (hu - (s ? p.rows[s - 1].end : 0)) * r.xh + place(c);
            a[u] = load_streamed<P>(x);
            if (!INTER && c < turned) z[u] = load_streamed<P>(x + p.half);
        }
    };
    // The rows are asked for before what says where they stand, which takes several loads one after the other.
    if (c0 < p.chunks && h0 < p.heads) load(c0, h0);
    int64_t n = b, i = t, slot = -1, pos = 0, to[2] = {0, 0};
    bool stored = false;
    auto stand = [&](int64_t token, auto&& index) {
        if (p.cu) {
            n = sequence_of(token, p.N, [&](int64_t j) { return index(p.cu, j, p.cu_i32); });
            i = n < 0 ? 0 : token - index(p.cu, n, p.cu_i32);
        }
        if (n >= 0) {
            const int64_t before = p.offsets ? index(p.offsets, n, p.off_i32) : p.offset;
            pos = p.positions ? index(p.positions, token, p.pos_i32) : before + i;
            slot = before + i;
        }
        if constexpr (CACHE) {
            const int page = n >= 0 ? page_of(p.cache.pages, n, slot, [&](const int32_t* at, int64_t j) { return (int32_t)index(at, j, true); }) : -1;
            stored = page >= 0;
            const int64_t in_page = stored ? place_in_page(p.cache.pages, slot) : 0;
            to[0] = page * p.cache.k_page + in_page * p.cache.k_slot;
            to[1] = page * p.cache.v_page + in_page * p.cache.v_slot;
        }
    };
    // (a wave of one token: scalar loads, a third of the latency of the others)
    if (p.tokens == 1 || lanes % 64 == 0)
        stand((int64_t)blockIdx.x * p.tokens + __builtin_amdgcn_readfirstlane(local), [](const void* at, int64_t j, bool is_i32) { return load_index_uniform(at, j, is_i32); });
    else
        stand(token, [](const void* at, int64_t j, bool is_i32) { return load_index(at, j, is_i32); });
    // (a row of no sequence is handed on as it is; a position that the tables do not have gives NaN)
    const bool inside = n >= 0 && pos >= 0 && pos < p.table_rows;
    for (int c = c0; c < p.chunks; c += p.chunk_lanes) {
        const bool pair = c < turned;
        float cs[PAIRS], sn[PAIRS];
        if (pair && inside) {
            const int64_t from = pos * p.table_stride + c * PAIRS;
            const auto pc = *(const Pack<TT, PAIRS>*)((const TT*)p.cos + from), ps = *(const Pack<TT, PAIRS>*)((const TT*)p.sin + from);
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) { cs[e] = (float)pc.e[e]; sn[e] = p.sign * (float)ps.e[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) cs[e] = sn[e] = __builtin_nanf("");
        }
        const int first = place(c);
        for (int h = h0; h < p.heads; h += p.each * p.head_lanes) {
            if (c != c0 || h != h0) load(c, h);
#pragma unroll
            for (int u = 0; u < HEADS; ++u) {
                const int hu = h + u * p.head_lanes;
                if (u >= p.each || hu >= p.heads) continue;
                const int s = hu < p.rows[0].end ? 0 : hu < p.rows[1].end ? 1 : 2;
                const RotaryRows& r = p.rows[s];
                const int64_t head = hu - (s ? p.rows[s - 1].end : 0);
                T* y;
                if (CACHE && r.cache) {
                    if (!stored) continue;
                    y = r.cache == 1 ? (T*)p.cache.k + to[0] + head * p.cache.k_head : (T*)p.cache.v + to[1] + head * p.cache.v_head;
                } else {
                    y = (T*)r.y + b * r.yb + t * r.yt + head * r.yh;
                }
                if (pair && r.turn && n >= 0) {
#pragma unroll
                    for (int e = 0; e < PAIRS; ++e) {
                        const float x1 = (float)(INTER ? a[u].e[2 * e] : a[u].e[e]), x2 = (float)(INTER ? a[u].e[2 * e + 1] : z[u].e[e]);
                        const T y1 = (T)(x1 * cs[e] - x2 * sn[e]), y2 = (T)(x1 * sn[e] + x2 * cs[e]);
                        if (INTER) { a[u].e[2 * e] = y1; a[u].e[2 * e + 1] = y2; }
                        else { a[u].e[e] = y1; z[u].e[e] = y2; }
                    }
                }
                store_streamed(y + first, a[u]);
                if (!INTER && pair) store_streamed(y + first + p.half, z[u]);
            }
        }
    }
}

template <typename T, typename TT, int V>
static int launch_rotary(const char* who, RotaryParams& p, bool inter, bool cache, hipStream_t stream) {
    const int64_t tokens = p.B * p.T;
    p.chunks = (inter ? 2 * p.half : p.half) / V + (p.D - 2 * p.half) / V;
    p.chunk_lanes = std::min(p.chunks, 256);
    // Heads of a thread: one where the chip is not full, else two or three, as leaves the fewest of a block's threads idle (of equals two).  Measured, us a call of a replayed graph
    // with one, two and three: 32768 tokens of 20 heads of 128 elements 78.0, 65.5, 70.4; 14000 tokens of 48 heads into the cache 76.0, 70.1, 66.5, of 24 heads 44.6, 38.5, 35.2; 8192
    // tokens of 24 heads of 64 15.9, 15.8, 12.9, of 9 heads of 256 22.3, 21.4, 19.9; 8191 tokens of 40 heads of 64 interleaved and 64 other elements 45.9, 43.0, 44.2 (three is taken).
    // Fewer tokens of 20 heads: 820 (131000 threads of a head each) 5.3, 6.2, 7.1, 1640 (262000) 6.8, 7.1, 7.8, 3280 11.1, 9.5, 11.3.
    auto lay_out = [&](int each) {
        p.head_lanes = std::max(1, std::min((p.heads + each - 1) / each, 256 / p.chunk_lanes));
        p.tokens = std::max(1, 256 / (p.head_lanes * p.chunk_lanes));
        const int rounds = (p.heads + p.head_lanes * each - 1) / (p.head_lanes * each);
        return (double)(p.tokens * p.heads * p.chunk_lanes) / (256.0 * each * rounds);
    };
    int each = 1;
    if (tokens * p.heads * p.chunks > 256 * 1024) {
        const double two = lay_out(2);
        each = V * sizeof(T) == 16 && lay_out(3) > 1.02 * two ? 3 : 2;
    }
    lay_out(each);
    p.each = each;
    const int64_t blocks = (tokens + p.tokens - 1) / p.tokens;
    GDN_CHECK_ARG(blocks < (1 << 24), GDN_ERR_UNSUPPORTED, "%s: fewer than 2^24 workgroups of tokens", who);     // (a launch has fewer than 2^32 threads)
    auto go = [&](auto inter_, auto cache_) {
        constexpr bool I = decltype(inter_)::value, C = decltype(cache_)::value;
        if constexpr (!I || V >= 2) {
            if constexpr (V * sizeof(T) == 16) {
                if (each == 3) {
                    hipLaunchKernelGGL((rotary_kernel<T, TT, V, I, C, 3>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
                    return;
                }
            }
            hipLaunchKernelGGL((rotary_kernel<T, TT, V, I, C, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
        }
    };
    auto with_cache = [&](auto inter_) { cache ? go(inter_, std::true_type()) : go(inter_, std::false_type()); };
    inter ? with_cache(std::true_type()) : with_cache(std::false_type());
    return check_launch("rotary_kernel");
}

// V: as many elements (16 bytes at most) as every place of the call is a multiple of.
template <typename T, typename TT>
static int rotary_width(const char* who, RotaryParams& p, int count, bool inter, bool cache, hipStream_t stream) {
    const int64_t parts = (int64_t)(p.D - 2 * p.half) | (inter ? 2 * p.half : p.half);
    int64_t units = parts;
    uintptr_t bytes = 0;
    for (int s = 0; s < count; ++s) {
        const RotaryRows& r = p.rows[s];
        units |= r.xb | r.xt | r.xh;
        bytes |= (uintptr_t)r.x;
        if (!(cache && r.cache)) { units |= r.yb | r.yt | r.yh; bytes |= (uintptr_t)r.y; }
    }
    if (cache) {
        const PagedCache& c = p.cache;
        units |= c.k_page | c.k_slot | c.k_head | c.v_page | c.v_slot | c.v_head;
        bytes |= (uintptr_t)c.k | (uintptr_t)c.v;
    }
    constexpr int MOST = 16 / sizeof(T);
    int V = MOST;
    auto fits = [&](int v) {
        const int pairs = inter ? v / 2 : v;
        const size_t load = std::min<size_t>(16, pairs * sizeof(TT));
        return ((units % v == 0 && bytes % (v * sizeof(T)) == 0) || (inter && v == 2 && parts % 2 == 0)) &&
               (p.half == 0 || (((uintptr_t)p.cos | (uintptr_t)p.sin) % load == 0 && p.table_stride * sizeof(TT) % load == 0));
    };
    const int least = inter ? 2 : 1;
    while (V > least && !fits(V)) V /= 2;
    GDN_CHECK_ARG(!inter || p.D % 2 == 0, GDN_ERR_UNSUPPORTED, "%s: the interleaved layout takes heads of an even number of elements", who);
    if constexpr (MOST == 8)
        if (V == 8) return launch_rotary<T, TT, 8>(who, p, inter, cache, stream);
    if (V == 4) return launch_rotary<T, TT, 4>(who, p, inter, cache, stream);
    if (V == 2) return launch_rotary<T, TT, 2>(who, p, inter, cache, stream);
    return launch_rotary<T, TT, 1>(who, p, inter, cache, stream);
}

static int rotary_types(const char* who, RotaryParams& p, int count, int dtype, int table_dtype, bool inter, bool cache, hipStream_t stream) {
    const bool f32 = table_dtype == GDN_DTYPE_F32;
    GDN_CHECK_ARG(f32 || table_dtype == dtype, GDN_ERR_INVALID, "%s: the tables are fp32 or of the rows' type", who);
    if (dtype == GDN_DTYPE_BF16) return f32 ? rotary_width<bf16_t, float>(who, p, count, inter, cache, stream) : rotary_width<bf16_t, bf16_t>(who, p, count, inter, cache, stream);
    if (dtype == GDN_DTYPE_F16) return f32 ? rotary_width<f16_t, float>(who, p, count, inter, cache, stream) : rotary_width<f16_t, f16_t>(who, p, count, inter, cache, stream);
    return rotary_width<float, float>(who, p, count, inter, cache, stream);
}

// What both entries check; the tables' part of the parameters.
static int rotary_checks(const char* who, RotaryParams& p, const gdn_rotary_call* c) {
    GDN_CHECK_ARG(c && c->B >= 0 && c->T >= 0 && c->N >= 0 && c->D >= 1 && c->rotary_dim >= 0 && c->rotary_dim % 2 == 0 && c->rotary_dim <= c->D, GDN_ERR_INVALID,
                  "%s: bad sizes (the turned part of a head is even and at most the head)", who);
    GDN_CHECK_ARG(c->D <= GDN_ROTARY_MAX_DIM, GDN_ERR_UNSUPPORTED, "%s: heads of up to %d elements", who, GDN_ROTARY_MAX_DIM);
    GDN_CHECK_ARG(c->dtype == GDN_DTYPE_BF16 || c->dtype == GDN_DTYPE_F16 || c->dtype == GDN_DTYPE_F32, GDN_ERR_UNSUPPORTED, "%s: unsupported dtype %d", who, c->dtype);
    GDN_CHECK_ARG(c->B < (1ll << 31) && c->T < (1ll << 31) && c->B * c->T < (1ll << 31), GDN_ERR_UNSUPPORTED, "%s: fewer than 2^31 tokens", who);
    GDN_CHECK_ARG(!c->cu_seqlens || (c->B == 1 && c->N >= 1), GDN_ERR_INVALID, "%s: a packed batch is one row of tokens with N >= 1 sequences", who);
    GDN_CHECK_ARG(c->rotary_dim == 0 || (c->table_rows >= 0 && (c->table_rows == 0 || (c->cos && c->sin)) && c->table_stride >= c->rotary_dim / 2), GDN_ERR_INVALID, "%s: cos and sin are missing", who);
    p.cos = c->cos; p.sin = c->sin; p.table_stride = c->table_stride; p.table_rows = c->rotary_dim ? c->table_rows : (1ll << 62);
    p.positions = c->positions; p.offsets = c->offsets; p.offset = c->offset; p.cu = c->cu_seqlens;
    p.B = c->B; p.T = c->T; p.N = c->cu_seqlens ? c->N : c->B; p.half = (int)(c->rotary_dim / 2); p.D = (int)c->D;
    p.sign = c->flags & GDN_ROTARY_BACK ? -1.f : 1.f;
    p.pos_i32 = c->flags & GDN_ROTARY_POSITIONS_INT32; p.off_i32 = c->flags & GDN_ROTARY_OFFSETS_INT32; p.cu_i32 = c->flags & GDN_FLAG_CU_INT32;
    return GDN_OK;
}

static void rotary_rows(RotaryParams& p, int s, const gdn_rotary_rows& r, bool turn, int cache) {
    p.rows[s] = RotaryRows{(const char*)r.x, (char*)r.y, r.x_stride[0], r.x_stride[1], r.x_stride[2], r.y_stride[0], r.y_stride[1], r.y_stride[2], p.heads + (int)r.heads, turn, cache};
    p.heads += (int)r.heads;
    for (int k = s + 1; k < 3; ++k) p.rows[k].end = p.heads;
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_rotary(const gdn_rotary_rows* rows, int count, const gdn_rotary_call* call, void* stream) {
    const char* who = "gdn_rotary";
    RotaryParams p{};
    const int rc = rotary_checks(who, p, call);
    if (rc != GDN_OK) return rc;
    GDN_CHECK_ARG(rows && count >= 1 && count <= 2, GDN_ERR_INVALID, "%s: one or two tensors", who);
    for (int s = 0; s < count; ++s) {
        GDN_CHECK_ARG(rows[s].heads >= 0 && rows[s].heads <= GDN_ROTARY_MAX_HEADS && ((rows[s].x && rows[s].y) || rows[s].heads * p.B * p.T == 0), GDN_ERR_INVALID, "%s: bad tensor %d", who, s);
        rotary_rows(p, s, rows[s], true, 0);
    }
    if (p.B * p.T * p.heads == 0) return GDN_OK;
    return rotary_types(who, p, count, call->dtype, call->table_dtype, call->flags & GDN_ROTARY_INTERLEAVED, false, (hipStream_t)stream);
}

extern "C" int gdn_paged_append(const gdn_paged_cache* cache, const gdn_rotary_rows* q, const gdn_rotary_rows* k, const gdn_rotary_rows* v,
                                const gdn_rotary_call* call, void* stream) {
    const char* who = "gdn_paged_append";
    RotaryParams p{};
    int rc = rotary_checks(who, p, call);
    if (rc != GDN_OK) return rc;
    rc = check_cache(who, cache, p.N, p.cache);
    if (rc != GDN_OK) return rc;
    GDN_CHECK_ARG(k && v && k->heads == cache->heads && v->heads == cache->heads && call->dtype == cache->dtype && call->D == cache->dim, GDN_ERR_INVALID,
                  "%s: keys and values have the cache's heads, size and type", who);
    GDN_CHECK_ARG(cache->heads <= GDN_ROTARY_MAX_HEADS && (!q || (q->heads >= 0 && q->heads <= GDN_ROTARY_MAX_HEADS)), GDN_ERR_INVALID, "%s: too many heads", who);
    GDN_CHECK_ARG(p.B * p.T == 0 || (k->x && v->x && (!q || q->heads == 0 || (q->x && q->y))), GDN_ERR_INVALID, "%s: missing tensors", who);
    int s = 0;
    if (q) rotary_rows(p, s++, *q, true, 0);
    rotary_rows(p, s++, *k, true, 1);
    rotary_rows(p, s++, *v, false, 2);
    p.offsets = p.cache.context; p.off_i32 = p.cache.context_i32;
    if (p.B * p.T == 0) return GDN_OK;
    return rotary_types(who, p, s, call->dtype, call->table_dtype, call->flags & GDN_ROTARY_INTERLEAVED, true, (hipStream_t)stream);
}
