// Attention of a step's rows (one token, a chain or a tree of drafts) over a paged cache.
//
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   s_ij = scale q_i . k_j over the keys that row i sees, m_i their maximum
//
// One pass over the keys with the running maximum and sum: a wave for a row and a head, a lane for a key of 64, then for the head's elements.
#include "gdn_paged.h"
#include <algorithm>

namespace gdn {

constexpr int PA_MAX_DIM = 256;

struct PagedAttnParams {
    PagedCache cache;
    const void* q; void* o; const void* cu; const uint8_t* mask;
    int64_t qb, qt, qh;
    int64_t mask_seq, mask_row, mask_cols;
    int64_t B, T, N;
    int HQ, HK, D;
    float scale;
    bool cu_i32;
};

template <typename T>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttnParams p) {
    __shared__ float sq[PA_MAX_DIM], sp[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x;
    const int64_t token = blockIdx.x;
    const int h = blockIdx.y, hk = h / (p.HQ / p.HK);
    const int64_t b = token / p.T, t = token - b * p.T;
    int64_t n = b, i = t, rows = p.T;
    if (p.cu) {
        n = sequence_of(token, p.N, [&](int64_t j) { return load_index(p.cu, j, p.cu_i32); });
        if (n < 0) {
            for (int d = lane; d < p.D; d += 64) ((T*)p.o)[(token * p.HQ + h) * p.D + d] = (T)0.f;
            return;
        }
        const int64_t first = load_index(p.cu, n, p.cu_i32);
        i = token - first;
        rows = load_index(p.cu, n + 1, p.cu_i32) - first;
    }
    const T* q = (const T*)p.q + b * p.qb + t * p.qt + h * p.qh;
    for (int d = lane; d < p.D; d += 64) sq[d] = (float)q[d];
    __syncthreads();
    const int64_t context = load_index(p.cache.context, n, p.cache.context_i32);
    const uint8_t* mask = p.mask ? p.mask + (p.cu ? token * p.mask_row : n * p.mask_seq + i * p.mask_row) : nullptr;
    const int64_t keys = std::min<int64_t>(context + rows, p.cache.pages.capacity);
    float m = -INFINITY, l = 0.f, acc[PA_MAX_DIM / 64] = {};
    for (int64_t from = 0; from < keys; from += 64) {
        const int64_t key = from + lane, fresh = key - context;
        bool sees = key < keys;
        if (sees && fresh >= 0) sees = mask ? fresh < p.mask_cols && mask[fresh] : fresh <= i;
        const int page = sees ? page_of(p.cache.pages, n, key) : -1;
        sees = page >= 0;
        float s = -INFINITY;
        if (sees) {
            const int64_t in_page = key % p.cache.pages.page_size;
            const T* k = (const T*)p.cache.k + page * p.cache.k_page + in_page * p.cache.k_slot + hk * p.cache.k_head;
            s = 0.f;
            for (int d = 0; d < p.D; ++d) s += sq[d] * (float)k[d];
            s *= p.scale;
            at[lane] = page * p.cache.v_page + in_page * p.cache.v_slot + hk * p.cache.v_head;
        } else {
            at[lane] = -1;
        }
        float most = s;
        for (int x = 1; x < 64; x *= 2) most = fmaxf(most, __shfl_xor(most, x, 64));
        const float now = fmaxf(m, most);
        // (no maximum yet: nothing is seen, or what is seen is not a number and makes the row's sums so)
        const float base = now == -INFINITY ? 0.f : now, keep = expf(m - base), w = sees ? expf(s - base) : 0.f;
        float sum = w;
        for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x, 64);
        l = l * keep + sum;
        m = now;
        __syncthreads();
        sp[lane] = w;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < PA_MAX_DIM / 64; ++e) acc[e] *= keep;
        for (int j = 0; j < 64; ++j) {
            if (at[j] < 0) continue;
            const T* v = (const T*)p.cache.v + at[j];
#pragma unroll
            for (int e = 0; e < PA_MAX_DIM / 64; ++e)
                if (e * 64 + lane < p.D) acc[e] += sp[j] * (float)v[e * 64 + lane];
        }
        __syncthreads();
    }
    T* o = (T*)p.o + (token * p.HQ + h) * p.D;
#pragma unroll
    for (int e = 0; e < PA_MAX_DIM / 64; ++e)
        if (e * 64 + lane < p.D) o[e * 64 + lane] = (T)(l == 0.f ? 0.f : acc[e] / l);
}

static int check_attn(const char* who, const gdn_paged_cache* cache, const gdn_paged_attn_call* c, PagedCache& out) {
    GDN_CHECK_ARG(c && c->B >= 0 && c->T >= 0 && c->HQ >= 0 && c->max_rows >= 0 && (c->cu_seqlens ? c->B == 1 && c->N >= 1 : c->N == c->B), GDN_ERR_INVALID, "%s: bad sizes", who);
    const int rc = check_cache(who, cache, c->N, out);
    if (rc != GDN_OK) return rc;
    GDN_CHECK_ARG(c->HQ % cache->heads == 0, GDN_ERR_INVALID, "%s: the queries' heads are a multiple of the cache's", who);
    GDN_CHECK_ARG(cache->dtype != GDN_DTYPE_F32 && cache->dim <= PA_MAX_DIM, GDN_ERR_UNSUPPORTED, "%s: bf16 or fp16 heads of up to %d elements", who, PA_MAX_DIM);
    return GDN_OK;
}

}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_paged_attn_workspace_bytes(const gdn_paged_cache*, const gdn_paged_attn_call*) { return 0; }

extern "C" int gdn_paged_attn(const gdn_paged_cache* cache, const gdn_paged_attn_call* c, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "gdn_paged_attn";
    PagedAttnParams p{};
    const int rc = check_attn(who, cache, c, p.cache);
    if (rc != GDN_OK) return rc;
    if (c->B * c->T * c->HQ == 0) return GDN_OK;
    GDN_CHECK_ARG(c->q && c->o, GDN_ERR_INVALID, "%s: missing tensors", who);
    GDN_CHECK_ARG(c->B * c->T < (1ll << 31) && c->HQ <= 65535, GDN_ERR_UNSUPPORTED, "%s: too many rows", who);
    p.q = c->q; p.o = c->o; p.cu = c->cu_seqlens; p.mask = c->mask;
    p.qb = c->q_stride[0]; p.qt = c->q_stride[1]; p.qh = c->q_stride[2];
    p.mask_seq = c->mask_seq_stride; p.mask_row = c->mask_row_stride; p.mask_cols = c->mask_cols;
    p.B = c->B; p.T = c->T; p.N = c->N; p.HQ = (int)c->HQ; p.HK = (int)cache->heads; p.D = (int)cache->dim; p.scale = c->scale; p.cu_i32 = c->flags & GDN_FLAG_CU_INT32;
    const dim3 grid((unsigned)(c->B * c->T), (unsigned)c->HQ);
    if (cache->dtype == GDN_DTYPE_BF16) hipLaunchKernelGGL(paged_attn_kernel<bf16_t>, grid, dim3(64), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(paged_attn_kernel<f16_t>, grid, dim3(64), 0, (hipStream_t)stream, p);
    return check_launch("paged_attn_kernel");
}
