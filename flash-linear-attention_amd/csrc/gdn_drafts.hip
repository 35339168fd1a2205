// Which drafted tokens stand, and the token after them.
//
// From row 0 of a sequence the drafts that follow the row come to are asked in order: draft c, a word x, stands where u_c q(x) < p(x).  A draft that does not
// takes its part of the probabilities with it, p <- (p - q)+ / sum, and the next one is asked; the token after the last row that stands is drawn from what is
// left.  However many were refused, what is left is a weight of the two rows alone,
//
//   w(v) = (a p(v) - b q(v))+,   (a, b) = (1, 0), then (a, b + 1) / sum of w after each refusal,
//
// (or a p(v) without the refused words where the drafts were not sampled), so a refusal costs one pass over p and q for the sum, and nothing is stored.
// The sums are kept for every SEGMENT words: the token is found in the segment where the running sum crosses u_0 times the whole, by reading it again.
//
// Everything that decides is in 64 bits and in a fixed order.  Bounded by the memory system for many sequences and words, by latency for few: the first pass, for most
// sequences the only one, is shared out over workgroups (drafts_round_kernel), each of which walks to it by itself, and one workgroup per sequence finishes.
// Measured: 16 chains of five drafts over 32000 fp32 words 12.3 us; 32 trees of 15 over 131072 words 45 to 65 (three shared passes of 8.5, then 27; one workgroup per sequence for all: 71 to 83).
#include "gdn_common.h"
#include <algorithm>
#include <type_traits>

namespace gdn {

constexpr int DRAFT_SEGMENT = 2048, DRAFT_SEGMENTS = GDN_DRAFTS_MAX_WORDS / DRAFT_SEGMENT, DRAFT_ROWS = GDN_DRAFTS_MAX_ROWS;

struct DraftParams {
    const void* p; const void* q; const void* tokens; const float* u; const int32_t* parents; const int32_t* lengths;
    int64_t* next; int32_t* accepted; int32_t* rows;
    int64_t p_seq, p_row, q_seq, q_row, parents_stride;
    int R, V, segments;
    bool tokens64;
    double* sums;                                  // [rounds][N][segments]: of the first passes
    int64_t N;
    int rounds;
};

// Where a sequence has come to.
struct DraftWalk {
    int here, last, depth, refused;                // row come to, row asked last, rows that stand, refusals here
    int asks;                                      // 1: the last draft was refused, its pass is due
    double a, b;
};

struct DraftShared {
    int parent[DRAFT_ROWS], word[DRAFT_ROWS], path[DRAFT_ROWS], refused[DRAFT_ROWS];
    float u[DRAFT_ROWS];
    double p[DRAFT_ROWS], q[DRAFT_ROWS];           // of the draft's word after the row it follows
    double sums[DRAFT_SEGMENTS];
    DraftWalk walk;
    double total;
};

template <typename T> __device__ __forceinline__ double mass_of(T x) { const float f = (float)x; return f > 0.f ? (double)f : 0.0; }

__device__ __forceinline__ double weight(bool sampled, double a, double b, double p, double q) {
    const double w = sampled ? a * p - b * q : a * p;
    return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ int rows_of(const DraftParams& p, int64_t n) { return p.lengths ? min(max(p.lengths[n], 1), p.R) : p.R; }

template <typename T>
__device__ void draft_tests(const DraftParams& p, int64_t n, int rows, DraftShared& s) {
    for (int r = threadIdx.x; r < rows; r += blockDim.x) {
        int parent = r - 1;
        if (p.parents) parent = p.parents[n * p.parents_stride + r];
        const int64_t word = p.tokens64 ? ((const int64_t*)p.tokens)[n * p.R + r] : (int64_t)((const int32_t*)p.tokens)[n * p.R + r];
        const bool known = word >= 0 && word < p.V;
        // (a word outside the vocabulary was drawn from nothing and takes nothing: its row follows none)
        if (r == 0 || parent < 0 || parent >= r || !known) parent = -1;
        s.parent[r] = parent;
        s.word[r] = (int)word;
        s.u[r] = p.u[n * p.R + r];
        s.p[r] = parent >= 0 ? mass_of(((const T*)p.p)[n * p.p_seq + parent * p.p_row + word]) : 0.0;
        s.q[r] = !p.q ? 1.0 : parent >= 0 ? mass_of(((const T*)p.q)[n * p.q_seq + parent * p.q_row + word]) : 0.0;
    }
}

// The first row after `last` that follows `here` (rows: none); by a whole wave.
__device__ __forceinline__ int next_draft(const DraftShared& s, int here, int last, int rows) {
    const int lane = threadIdx.x & 63;
    for (int from = last + 1; from < rows; from += 64) {
        const int r = from + lane;
        const uint64_t found = __ballot(r < rows && s.parent[r < rows ? r : 0] == here);
        if (found) return from + __builtin_ctzll(found);
    }
    return rows;
}

// Asks drafts until one is refused or none is left (by wave 0).
__device__ void draft_walk(const DraftParams& p, int rows, DraftShared& s) {
    DraftWalk w = s.walk;
    w.asks = 0;
    for (;;) {
        const int c = next_draft(s, w.here, w.last, rows);
        if (c >= rows) break;
        w.last = c;
        const int word = s.word[c];
        double left = weight(p.q != nullptr, w.a, w.b, s.p[c], s.q[c]);
        if (!p.q)
            for (int k = 0; k < w.refused; ++k)
                if (s.refused[k] == word) left = 0.0;
        if ((double)s.u[c] * s.q[c] < left) {
            s.path[w.depth++] = c;
            w.here = c; w.refused = 0; w.a = 1.0; w.b = 0.0;
            continue;
        }
        s.refused[w.refused] = word;
        w.asks = 1;
        break;
    }
    s.walk = w;
}

// What is left, word by word: the weights that the due pass adds up (asks: with the draft that was just refused).
struct DraftWeights {
    double a, b;
    int refused, here;
};
__device__ __forceinline__ DraftWeights weights_of(const DraftWalk& w, int asks) { return {w.a, w.b + (asks ? 1.0 : 0.0), w.refused + (asks ? 1 : 0), w.here}; }

template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Words { T e[V]; };

// The sum of one segment, by a wave: lane l takes 16 bytes in every kilobyte.
template <typename T, bool SAMPLED>
__device__ double segment_sum(const DraftParams& p, int64_t n, const DraftShared& s, const DraftWeights& w, int segment) {
    constexpr int VEC = 16 / sizeof(T), STEPS = DRAFT_SEGMENT / (64 * VEC);
    const int lane = threadIdx.x & 63;
    const T* pr = (const T*)p.p + n * p.p_seq + w.here * p.p_row;
    const T* qr = (const T*)p.q + n * p.q_seq + w.here * p.q_row;
    const int first = segment * DRAFT_SEGMENT;
    Words<T, VEC> x[STEPS], y[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const int v = first + (k * 64 + lane) * VEC;
        if (v + VEC <= p.V) {
            x[k] = *(const Words<T, VEC>*)(pr + v);
            if (SAMPLED) y[k] = *(const Words<T, VEC>*)(qr + v);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                x[k].e[e] = v + e < p.V ? pr[v + e] : (T)0.f;
                if (SAMPLED) y[k].e[e] = v + e < p.V ? qr[v + e] : (T)0.f;
            }
        }
    }
    if (!SAMPLED)
        for (int j = 0; j < w.refused; ++j) {
            const int at = s.refused[j] - first;
            if (at < 0 || at >= DRAFT_SEGMENT) continue;
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if ((k * 64 + lane) * VEC + e == at) x[k].e[e] = (T)0.f;
        }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < STEPS; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += weight(SAMPLED, w.a, w.b, mass_of(x[k].e[e]), SAMPLED ? mass_of(y[k].e[e]) : 0.0);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
    return sum;
}

__device__ __forceinline__ double scan_add(double x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    return x;
}

// The first word where the running sum of the weights passes t, by wave 0; where none does (u at 1, the last bit of a sum) the last word with a weight.
template <typename T>
__device__ int draft_word(const DraftParams& p, int64_t n, const DraftShared& s, const DraftWeights& w, double t) {
    const int lane = threadIdx.x & 63;
    double before = 0.0;
    int segment = -1, filled = -1;
    for (int from = 0; from < p.segments; from += 64) {
        const double x = from + lane < p.segments ? s.sums[from + lane] : 0.0;
        const double upto = before + scan_add(x);
        const uint64_t passed = __ballot(upto > t && x > 0.0), some = __ballot(x > 0.0);
        if (some) filled = from + 63 - __builtin_clzll(some);
        if (passed) {
            const int at = __builtin_ctzll(passed);
            segment = from + at;
            before = at ? __shfl(upto, at - 1, 64) : before;
            break;
        }
        before = __shfl(upto, 63, 64);
    }
    const bool found = segment >= 0;
    if (!found) segment = filled;
    if (segment < 0) return -1;
    constexpr int EACH = DRAFT_SEGMENT / 64;
    constexpr int VEC = 16 / sizeof(T);
    const T* pr = (const T*)p.p + n * p.p_seq + w.here * p.p_row;
    const T* qr = (const T*)p.q + n * p.q_seq + w.here * p.q_row;
    const int first = segment * DRAFT_SEGMENT + lane * EACH;
    double x[EACH], sum = 0.0;
    int last = -1;
#pragma unroll
    for (int k = 0; k < EACH; k += VEC) {
        Words<T, VEC> a = {}, b = {};
        if (first + k + VEC <= p.V) {
            a = *(const Words<T, VEC>*)(pr + first + k);
            if (p.q) b = *(const Words<T, VEC>*)(qr + first + k);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                a.e[e] = first + k + e < p.V ? pr[first + k + e] : (T)0.f;
                if (p.q) b.e[e] = first + k + e < p.V ? qr[first + k + e] : (T)0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[k + e] = weight(p.q != nullptr, w.a, w.b, mass_of(a.e[e]), p.q ? mass_of(b.e[e]) : 0.0);
    }
    if (!p.q)
        for (int j = 0; j < w.refused; ++j) {
            const int at = s.refused[j] - first;
#pragma unroll
            for (int e = 0; e < EACH; ++e)
                if (e == at) x[e] = 0.0;
        }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        sum += x[e];
        if (x[e] > 0.0) last = first + e;
    }
    const double upto = before + scan_add(sum);
    const uint64_t passed = __ballot(found && upto > t && sum > 0.0);
    if (passed) {
        const int at = __builtin_ctzll(passed);
        double run = __shfl_up(upto, 1, 64);
        if (lane == 0) run = before;
        int word = last;
        bool done = false;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            run += x[e];
            if (!done && x[e] > 0.0 && run > t) { word = first + e; done = true; }
        }
        return __shfl(word, at, 64);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) last = max(last, __shfl_xor(last, d, 64));
    return last;
}


// A sequence's walk from pass to pass, the same in every workgroup that makes it: pass i is taken from memory where an earlier launch made it, else `make(weights)` makes
// it, or says that it ends here (false).  `finish(walk, weights)`: the last pass has been made.
template <typename T, typename Make, typename Finish>
__device__ __forceinline__ void draft_passes(const DraftParams& p, int64_t n, DraftShared& s, int made, Make&& make, Finish&& finish) {
    const int rows = rows_of(p, n);
    draft_tests<T>(p, n, rows, s);
    if (threadIdx.x == 0) {
        s.walk = DraftWalk{0, 0, 1, 0, 0, 1.0, 0.0};
        s.path[0] = 0;
    }
    __syncthreads();
    bool again = false;                                            // nothing was left: what was there before, added up again
    for (int pass = 0;; ++pass) {
        if (!again) {
            if (threadIdx.x < 64) draft_walk(p, rows, s);
            __syncthreads();
        }
        DraftWalk walk = s.walk;
        const DraftWeights w = weights_of(walk, walk.asks);
        if (pass < made) {
            const double* from = p.sums + (pass * p.N + n) * p.segments;
            for (int k = threadIdx.x; k < p.segments; k += blockDim.x) s.sums[k] = from[k];
        } else if (!make(w)) {
            return;
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            double sum = 0.0;
            for (int k = threadIdx.x; k < p.segments; k += 64) sum += s.sums[k];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
            if (threadIdx.x == 0) s.total = sum;
        }
        __syncthreads();
        // (every wave looks: rows asked later that follow the same row)
        const bool more = walk.asks && next_draft(s, walk.here, walk.last, rows) < rows;
        const bool some = s.total > 0.0;
        if (again || (!more && (some || !walk.asks))) {
            finish(walk, w);
            return;
        }
        if (some) { walk.a /= s.total; walk.b = (walk.b + 1.0) / s.total; ++walk.refused; }
        again = !more;
        walk.asks = 0;
        __syncthreads();
        if (threadIdx.x == 0) s.walk = walk;
        __syncthreads();
    }
}

// Pass p.rounds of every sequence (blockIdx.y) that comes to it, its segments shared out.
template <typename T>
__global__ __launch_bounds__(256) void drafts_round_kernel(DraftParams p) {
    __shared__ DraftShared s;
    const int64_t n = blockIdx.y;
    draft_passes<T>(p, n, s, p.rounds, [&](const DraftWeights& w) {
        double* const to = p.sums + (p.rounds * p.N + n) * p.segments;
        for (int k = blockIdx.x * 4 + threadIdx.x / 64; k < p.segments; k += gridDim.x * 4) {
            const double sum = p.q ? segment_sum<T, true>(p, n, s, w, k) : segment_sum<T, false>(p, n, s, w, k);
            if ((threadIdx.x & 63) == 0) to[k] = sum;
        }
        return false;
    }, [](const DraftWalk&, const DraftWeights&) {});
}

template <typename T>
__global__ __launch_bounds__(1024) void drafts_kernel(DraftParams p) {
    __shared__ DraftShared s;
    const int64_t n = blockIdx.x;
    draft_passes<T>(p, n, s, p.rounds, [&](const DraftWeights& w) {
        for (int k = threadIdx.x / 64; k < p.segments; k += 16) {
            const double sum = p.q ? segment_sum<T, true>(p, n, s, w, k) : segment_sum<T, false>(p, n, s, w, k);
            if ((threadIdx.x & 63) == 0) s.sums[k] = sum;
        }
        return true;
    }, [&](const DraftWalk& walk, const DraftWeights& w) {
        if (threadIdx.x < 64) {
            const int word = s.total > 0.0 && s.total < __builtin_inf() ? draft_word<T>(p, n, s, w, (double)s.u[0] * s.total) : -1;
            if (threadIdx.x == 0) {
                p.next[n] = word;
                p.accepted[n] = walk.depth;
            }
        }
        for (int r = threadIdx.x; r < p.R; r += 1024) p.rows[n * p.R + r] = r < walk.depth ? s.path[r] : -1;
    });
}

static int check_drafts(const char* who, const gdn_drafts_call* c) {
    GDN_CHECK_ARG(c && c->N >= 0 && c->R >= 1 && c->V >= 1, GDN_ERR_INVALID, "%s: bad sizes", who);
    GDN_CHECK_ARG(c->R <= GDN_DRAFTS_MAX_ROWS && c->V <= GDN_DRAFTS_MAX_WORDS && c->N <= 65535, GDN_ERR_UNSUPPORTED, "%s: up to 65535 sequences of %d rows, and %d words", who,
                  GDN_DRAFTS_MAX_ROWS, GDN_DRAFTS_MAX_WORDS);
    GDN_CHECK_ARG(c->p_dtype == GDN_DTYPE_BF16 || c->p_dtype == GDN_DTYPE_F16 || c->p_dtype == GDN_DTYPE_F32, GDN_ERR_UNSUPPORTED, "%s: unsupported dtype %d", who, c->p_dtype);
    GDN_CHECK_ARG(!c->q || c->q_dtype == c->p_dtype, GDN_ERR_INVALID, "%s: p and q are of one type", who);
    return GDN_OK;
}

// Passes that are shared out over workgroups, a launch for each, and workgroups per sequence: the first one, of which a chain has no other, and two more of trees.
// Measured, us a call of a replayed graph, one workgroup per sequence and shared (5 drafts of a chain, 15 of a tree, fp32):
//   sequences           1             8             32            48            64            96            192
//   chain,  32000       11.8  12.8    12.5  14.1    13.2  15.2    13.6  16.4    14.6  16.6    15.8  19.4    18.3  23.1
//   chain,  65536       14.8  12.8    15.8  14.2    17.6  15.9    18.1  18.2    18.2  19.2    18.9  21.9    24.8  31.9
//   chain, 131072       21.6  12.8    22.5  14.1    25.8  19.5    25.9  21.7    26.4  26.1    30.7  31.1    50.4  52.1
//   tree,   32000       22.4  29.6    27.8  35.8    28.2  37.8    29.6  39.1    30.1  40.4    30.9  44.3    34.0  51.3
//   tree,   65536       27.8  28.9    32.2  30.3    43.7  43.1    43.6  46.8    44.1  49.4    46.4  55.1    55.3  83.8
//   tree,  131072       59.8  36.3    67.5  46.2    70.7  55.7    74.0  61.8    74.9  76.0    82.2  95.4   108.0 133.8
// One or two shared passes of 32 trees of 131072 words: 66.4 and 61.1, five 56.3.  512 workgroups in all are as fast as 2048 up to 48 sequences.
struct DraftPlan { int rounds, parts; };
static DraftPlan draft_plan(const gdn_drafts_call* c) {
    const int64_t segments = (c->V + DRAFT_SEGMENT - 1) / DRAFT_SEGMENT;
    if (segments <= 32 || c->N >= 64) return {0, 0};
    return {c->parents ? 3 : 1, (int)std::min<int64_t>((segments + 3) / 4, std::max<int64_t>(1, 512 / std::max<int64_t>(1, c->N)))};
}

}  // namespace gdn

using namespace gdn;

extern "C" size_t gdn_verify_drafts_workspace_bytes(const gdn_drafts_call* c) {
    if (check_drafts("gdn_verify_drafts_workspace_bytes", c) != GDN_OK || c->N == 0) return 0;
    return (size_t)draft_plan(c).rounds * (size_t)(c->N * ((c->V + DRAFT_SEGMENT - 1) / DRAFT_SEGMENT)) * sizeof(double);
}

extern "C" int gdn_verify_drafts(const gdn_drafts_call* c, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "gdn_verify_drafts";
    const int rc = check_drafts(who, c);
    if (rc != GDN_OK) return rc;
    if (c->N == 0) return GDN_OK;
    GDN_CHECK_ARG(c->p && c->tokens && c->uniforms && c->next_token && c->accepted && c->rows, GDN_ERR_INVALID, "%s: missing tensors", who);
    const size_t need = gdn_verify_drafts_workspace_bytes(c);
    GDN_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0), GDN_ERR_WORKSPACE, "%s: workspace of %zu bytes, 8-byte aligned", who, need);
    DraftParams p{c->p, c->q, c->tokens, c->uniforms, c->parents, c->lengths, c->next_token, c->accepted, c->rows, c->p_stride[0], c->p_stride[1], c->q_stride[0], c->q_stride[1],
                  c->parents_stride, (int)c->R, (int)c->V, (int)((c->V + DRAFT_SEGMENT - 1) / DRAFT_SEGMENT), (c->flags & GDN_DRAFTS_TOKENS_INT64) != 0, (double*)workspace, c->N, 0};
    auto go = [&](auto t) {
        typedef decltype(t) T;
        const DraftPlan plan = draft_plan(c);
        for (; p.rounds < plan.rounds; ++p.rounds) {
            hipLaunchKernelGGL(drafts_round_kernel<T>, dim3((unsigned)plan.parts, (unsigned)c->N), dim3(256), 0, (hipStream_t)stream, p);
            const int ran = check_launch("drafts_round_kernel");
            if (ran != GDN_OK) return ran;
        }
        hipLaunchKernelGGL(drafts_kernel<T>, dim3((unsigned)c->N), dim3(1024), 0, (hipStream_t)stream, p);
        return check_launch("drafts_kernel");
    };
    if (c->p_dtype == GDN_DTYPE_BF16) return go(bf16_t{});
    if (c->p_dtype == GDN_DTYPE_F16) return go(f16_t{});
    return go(float{});
}
