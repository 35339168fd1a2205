// The gated feed-forward block (fla/modules/mlp.py: GatedMLP) and its gradients:
//
//   g = x Wg^T, u = x Wu^T;  h = act(g) u;  y = h Wd^T             x [M][D]; Wg, Wu [F][D]; Wd [D][F]
//   dh = dy Wd;  dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Forward two launches (both projections with the activation and the product on top; the down projection), backward three (dh with dg and du on top; dx;
// the weights' gradients together).  Many rows are bound by the matrix cores: gdn_gemm.h.
#include "gdn_gemm.h"

namespace gdn {

// act(g) and act'(g)
__device__ __forceinline__ void mlp_act(int act, float g, float& a, float& da) {
    if (act == GDN_ACT_GELU_TANH) {
        // (tanh has reached 1 long before 16; beyond, g^2 times its vanishing slope could be infinity times zero)
        const float c = g > 16.f ? 16.f : g < -16.f ? -16.f : g, z = 0.7978845608028654f * (c + 0.044715f * c * c * c);
        const float s = sigmoid_f(2.f * z);                          // (1 + tanh z) / 2
        a = g * s;
        da = s + c * 2.f * s * (1.f - s) * 0.7978845608028654f * (1.f + 0.134145f * c * c);
    } else {
        const float s = sigmoid_f(g);
        if (act == GDN_ACT_SIGMOID) { a = s; da = s * (1.f - s); }
        else { a = g * s; da = s * (1.f + g * (1.f - s)); }
    }
}

struct MlpGemm {
    GemmOperands op[3];
    int ops, tiles;
    void* C[3];                          // results (of a DUAL product's epilogue: h, g, u; of dh's: dg, du)
    const void* G; const void* U;
    float* part;                         // splits > 1: [splits][1 or 2 (both products of a DUAL)][M][N]
    int act;
};

enum MlpEpilogue { MLP_PLAIN, MLP_GATE, MLP_GRAD };

typedef float f32x8 __attribute__((ext_vector_type(8)));

// What becomes of eight neighbours of a result (of both products where there are two), at offset `at` of the outputs.
template <typename T, int EPI>
__device__ __forceinline__ void mlp_result(const MlpGemm& p, int which, int64_t at, f32x8 x, f32x8 u) {
    typedef typename Mma<T>::V8 V8;
    auto rounded = [](f32x8 v) { return V8{(T)v[0], (T)v[1], (T)v[2], (T)v[3], (T)v[4], (T)v[5], (T)v[6], (T)v[7]}; };
    if constexpr (EPI == MLP_PLAIN) {
        *(V8*)((T*)p.C[which] + at) = rounded(x);
    } else if constexpr (EPI == MLP_GATE) {
        V8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float a, da;
            mlp_act(p.act, x[e], a, da);
            h[e] = (T)(a * u[e]);
        }
        *(V8*)((T*)p.C[0] + at) = h;
        if (p.C[1]) {
            *(V8*)((T*)p.C[1] + at) = rounded(x);
            *(V8*)((T*)p.C[2] + at) = rounded(u);
        }
    } else {
        const V8 gv = *(const V8*)((const T*)p.G + at), uv = *(const V8*)((const T*)p.U + at);
        V8 dg, du;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float a, da;
            mlp_act(p.act, (float)gv[e], a, da);
            dg[e] = (T)(x[e] * (float)uv[e] * da);
            du[e] = (T)(x[e] * a);
        }
        *(V8*)((T*)p.C[0] + at) = dg;
        *(V8*)((T*)p.C[1] + at) = du;
    }
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool A_DOWN, bool B_DOWN, int EPI>
__global__ __launch_bounds__(64 * WM * WN, 2) void mlp_gemm_kernel(MlpGemm p) {
    typedef Gemm<T, BM, BN, WM, WN, STAGES, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    extern __shared__ __align__(16) char smem[];
    int tile = gemm_tile_of((int)blockIdx.x, p.tiles), which = 0;
    while (which + 1 < p.ops && tile >= p.op[which + 1].first) ++which;
    const GemmOperands& o = p.op[which];
    tile -= o.first;
    // (the parts of a tile one after the other: they share nothing, their neighbours in the band share rows and columns)
    const int area = o.tiles_m * o.tiles_n, part = tile / area;
    int tm, tn;
    gemm_place(tile - part * area, o.tiles_m, o.tiles_n, tm, tn);
    f32x16 acc[G::NT][G::MT];
    G::run(o, tm, tn, part, smem, acc);

    const int lane = threadIdx.x & 63, w = (int)threadIdx.x >> 6, wm = w % WM, wn = w / WM;
    constexpr int KINDS = EPI == MLP_GATE ? 2 : 1, COLS = G::NT / KINDS;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        const int m = tm * BM + 32 * (wm * G::MT + i) + (lane & 31);
        if (m >= o.M) continue;
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
#pragma unroll
            for (int q = 0; q < 16; q += 8) {
                const int n = tn * G::COLUMNS + 32 * G::column_tile(wn, j) + 16 * (lane >> 5) + q;
                if (n >= o.N) continue;
                const int64_t at = (int64_t)m * o.N + n;
                f32x8 x, u;
#pragma unroll
                for (int e = 0; e < 8; ++e) { x[e] = acc[j][i][q + e]; u[e] = acc[j + (KINDS - 1) * COLS][i][q + e]; }
                if (o.splits > 1) {
                    float* to = p.part + (int64_t)part * KINDS * o.M * o.N + at;
                    *(f32x8*)to = x;
                    if (KINDS == 2) *(f32x8*)(to + (int64_t)o.M * o.N) = u;
                } else
                    mlp_result<T, EPI>(p, which, at, x, u);
            }
        }
    }
}

// The parts of a contraction added up, in order, and what becomes of the sums.
template <typename T, int EPI>
__global__ __launch_bounds__(256) void mlp_join_kernel(MlpGemm p) {
    constexpr int KINDS = EPI == MLP_GATE ? 2 : 1;
    const int64_t size = (int64_t)p.op[0].M * p.op[0].N;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (at >= size) return;
    f32x8 x = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, u = x;
    for (int s = 0; s < p.op[0].splits; ++s) {
        x += *(const f32x8*)(p.part + s * KINDS * size + at);
        if (KINDS == 2) u += *(const f32x8*)(p.part + (s * KINDS + 1) * size + at);
    }
    mlp_result<T, EPI>(p, 0, at, x, u);
}

static GemmOperands operands(const void* A, const void* B, int64_t lda, int64_t ldb, int64_t M, int64_t N, int64_t K) {
    GemmOperands o{};
    o.A[0] = A; o.B[0] = B; o.lda = lda; o.ldb = ldb; o.M = (int)M; o.N = (int)N; o.K = (int)K; o.segments = 1; o.splits = 1;
    return o;
}

// How a product (or several in a launch) is cut: the tile, and into how many parts the contraction.
struct MlpPlan { int large; int splits; };
static MlpPlan plan_gemm(const MlpGemm& p, int kinds) {
    int64_t large = 0, small = 0;
    for (int i = 0; i < p.ops; ++i) {
        const int64_t M = p.op[i].M, N = (int64_t)p.op[i].N * kinds;
        large += ((M + 255) / 256) * ((N + 255) / 256);
        small += ((M + 127) / 128) * ((N + 127) / 128);
    }
    MlpPlan plan{large >= 160, 1};
    if (getenv("MLP_LARGE")) plan.large = atoi(getenv("MLP_LARGE"));
    if (!plan.large && p.ops == 1) {
        const int64_t steps = (int64_t)((p.op[0].K + GM_K - 1) / GM_K) * p.op[0].segments;
        plan.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(512 / std::max<int64_t>(small, 1), steps / 8), 16));
        if (getenv("MLP_SPLIT")) plan.splits = atoi(getenv("MLP_SPLIT"));
    }
    return plan;
}
static size_t plan_bytes(const MlpGemm& p, int kinds) {
    const MlpPlan plan = plan_gemm(p, kinds);
    return plan.splits > 1 ? (size_t)plan.splits * kinds * p.op[0].M * p.op[0].N * 4 : 0;
}

struct Workspace { void* at; size_t bytes; };

template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_tiles(MlpGemm& p, hipStream_t stream) {
    typedef Gemm<T, BM, BN, WM, WN, STAGES, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    int64_t tiles = 0;
    for (int i = 0; i < p.ops; ++i) {
        GemmOperands& o = p.op[i];
        o.first = (int)tiles;
        o.tiles_m = (o.M + BM - 1) / BM; o.tiles_n = (o.N + G::COLUMNS - 1) / G::COLUMNS;
        tiles += (int64_t)o.tiles_m * o.tiles_n * o.splits;
        GDN_CHECK_ARG(tiles < (1ll << 32) / G::THREADS, GDN_ERR_UNSUPPORTED, "the gated feed-forward block: %lld x %lld results are too many for one launch",
                      (long long)o.M, (long long)o.N);
    }
    if (tiles == 0) return GDN_OK;
    p.tiles = (int)tiles;
    auto kernel = mlp_gemm_kernel<T, BM, BN, WM, WN, STAGES, A_DOWN, B_DOWN, EPI>;
    const int rc = ensure_dynamic_smem_for((const void*)kernel, G::LDS, "mlp_gemm_kernel");
    if (rc != GDN_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.tiles), dim3(G::THREADS), G::LDS, stream, p);
    return check_launch("mlp_gemm_kernel");
}

template <typename T, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_gemm(MlpGemm& p, Workspace ws, hipStream_t stream) {
    constexpr int KINDS = EPI == MLP_GATE ? 2 : 1;
    const MlpPlan plan = plan_gemm(p, KINDS);
    p.op[0].splits = plan.splits;
    if (plan.splits > 1) {
        GDN_CHECK_ARG(ws.at && ws.bytes >= plan_bytes(p, KINDS), GDN_ERR_WORKSPACE, "the gated feed-forward block: workspace too small (%zu bytes, %zu needed)", ws.bytes,
                      plan_bytes(p, KINDS));
        p.part = (float*)ws.at;
    }
    int rc = plan.large == 1 ? launch_tiles<T, 256, 256, 2, 4, 2, A_DOWN, B_DOWN, EPI>(p, stream) : plan.large == 2 ? launch_tiles<T, 256, 128, 2, 2, 2, A_DOWN, B_DOWN, EPI>(p, stream) :
                                                                                                                    launch_tiles<T, 128, 128, 2, 2, 2, A_DOWN, B_DOWN, EPI>(p, stream);
    if (rc != GDN_OK || plan.splits <= 1) return rc;
    const int64_t size = (int64_t)p.op[0].M * p.op[0].N;
    hipLaunchKernelGGL((mlp_join_kernel<T, EPI>), dim3((unsigned)((size / 8 + 255) / 256)), dim3(256), 0, stream, p);
    return check_launch("mlp_join_kernel");
}

// The products of a forward and a backward pass.
static MlpGemm gate_up(const void* x, const void* wg, const void* wu, int64_t M, int64_t D, int64_t F) {
    MlpGemm p{};
    p.ops = 1;
    p.op[0] = operands(x, wg, D, D, M, F, D);
    p.op[0].B[1] = wu;
    return p;
}
static MlpGemm down(const void* h, const void* wd, int64_t M, int64_t D, int64_t F) {
    MlpGemm p{};
    p.ops = 1;
    p.op[0] = operands(h, wd, F, F, M, D, F);
    return p;
}
static MlpGemm grad_inner(const void* dy, const void* wd, int64_t M, int64_t D, int64_t F) {
    MlpGemm p{};
    p.ops = 1;
    p.op[0] = operands(dy, wd, D, F, M, F, D);
    return p;
}
static MlpGemm grad_x(const void* dg, const void* du, const void* wg, const void* wu, int64_t M, int64_t D, int64_t F) {
    MlpGemm p{};
    p.ops = 1;
    p.op[0] = operands(dg, wg, F, D, M, D, F);
    p.op[0].A[1] = du; p.op[0].B[1] = wu; p.op[0].segments = 2;
    return p;
}

template <typename T>
static int mlp_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* y, void* g, void* u, void* h, Workspace ws, int64_t M, int64_t D, int64_t F,
                   int act, hipStream_t stream) {
    MlpGemm p = gate_up(x, wg, wu, M, D, F);
    p.act = act; p.C[0] = h; p.C[1] = g; p.C[2] = u;
    const int rc = launch_gemm<T, false, false, MLP_GATE>(p, ws, stream);
    if (rc != GDN_OK) return rc;
    MlpGemm q = down(h, wd, M, D, F);
    q.C[0] = y;
    return launch_gemm<T, false, false, MLP_PLAIN>(q, ws, stream);
}

template <typename T>
static int mlp_bwd(const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* g, const void* u, const void* h,
                   void* dg, void* du, void* dx, void* dwg, void* dwu, void* dwd, Workspace ws, int64_t M, int64_t D, int64_t F, int act, hipStream_t stream) {
    int rc = GDN_OK;
    if (M > 0 && (dx || dwg || dwu)) {
        MlpGemm p = grad_inner(dy, wd, M, D, F);
        p.act = act; p.G = g; p.U = u; p.C[0] = dg; p.C[1] = du;
        rc = launch_gemm<T, false, true, MLP_GRAD>(p, ws, stream);
        if (rc != GDN_OK) return rc;
    }
    if (M > 0 && dx) {
        MlpGemm p = grad_x(dg, du, wg, wu, M, D, F);
        p.C[0] = dx;
        rc = launch_gemm<T, false, true, MLP_PLAIN>(p, ws, stream);
        if (rc != GDN_OK) return rc;
    }
    MlpGemm p{};
    auto add = [&](const void* A, const void* B, int64_t rows, int64_t cols, void* C) {
        if (!C) return;
        p.op[p.ops] = operands(A, B, rows, cols, rows, cols, M);
        p.C[p.ops++] = C;
    };
    add(dg, x, F, D, dwg);
    add(du, x, F, D, dwu);
    add(dy, h, D, F, dwd);
    return p.ops ? launch_gemm<T, true, true, MLP_PLAIN>(p, ws, stream) : GDN_OK;
}

}  // namespace gdn

using namespace gdn;

static int check_mlp(const char* who, int64_t M, int64_t D, int64_t F, int act, int dtype) {
    GDN_CHECK_ARG(M >= 0 && D >= 1 && F >= 1, GDN_ERR_INVALID, "%s: bad sizes M=%lld D=%lld F=%lld", who, (long long)M, (long long)D, (long long)F);
    GDN_CHECK_ARG(dtype == GDN_DTYPE_BF16 || dtype == GDN_DTYPE_F16, GDN_ERR_UNSUPPORTED, "%s: bf16 or f16 only", who);
    GDN_CHECK_ARG(act == GDN_ACT_SILU || act == GDN_ACT_SIGMOID || act == GDN_ACT_GELU_TANH, GDN_ERR_UNSUPPORTED, "%s: unknown activation", who);
    GDN_CHECK_ARG(D % 8 == 0 && F % 8 == 0, GDN_ERR_UNSUPPORTED, "%s: D and F must be multiples of 8 (got %lld, %lld)", who, (long long)D, (long long)F);
    GDN_CHECK_ARG(D <= GDN_MLP_MAX_FEATURES && F <= GDN_MLP_MAX_FEATURES && M < (1ll << 30), GDN_ERR_UNSUPPORTED,
                  "%s: D and F up to %d and fewer than 2^30 rows (got M=%lld D=%lld F=%lld)", who, GDN_MLP_MAX_FEATURES, (long long)M, (long long)D, (long long)F);
    return GDN_OK;
}

extern "C" size_t gdn_gated_mlp_workspace_bytes(int64_t M, int64_t D, int64_t F, int backward) {
    if (check_mlp("gdn_gated_mlp_workspace_bytes", M, D, F, GDN_ACT_SILU, GDN_DTYPE_BF16) != GDN_OK || M == 0) return 0;
    if (!backward) return std::max(plan_bytes(gate_up(nullptr, nullptr, nullptr, M, D, F), 2), plan_bytes(down(nullptr, nullptr, M, D, F), 1));
    return std::max(plan_bytes(grad_inner(nullptr, nullptr, M, D, F), 1), plan_bytes(grad_x(nullptr, nullptr, nullptr, nullptr, M, D, F), 1));
}

extern "C" int gdn_gated_mlp_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* y, void* g, void* u, void* h,
                                 void* workspace, size_t workspace_bytes, int64_t M, int64_t D, int64_t F, int activation, int dtype, void* stream) {
    const char* who = "gdn_gated_mlp_fwd";
    const int rc = check_mlp(who, M, D, F, activation, dtype);
    if (rc != GDN_OK) return rc;
    if (M == 0) return GDN_OK;
    GDN_CHECK_ARG(x && wg && wu && wd && y && h && !g == !u, GDN_ERR_INVALID, "%s: x, the weights, y and h are required, g goes with u", who);
    GDN_CHECK_ARG((((uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu | (uintptr_t)wd | (uintptr_t)y | (uintptr_t)g | (uintptr_t)u | (uintptr_t)h) & 15) == 0,
                  GDN_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
    hipStream_t s = (hipStream_t)stream;
    const Workspace ws{workspace, workspace_bytes};
    return dtype == GDN_DTYPE_BF16 ? mlp_fwd<bf16_t>(x, wg, wu, wd, y, g, u, h, ws, M, D, F, activation, s)
                                   : mlp_fwd<f16_t>(x, wg, wu, wd, y, g, u, h, ws, M, D, F, activation, s);
}

extern "C" int gdn_gated_mlp_bwd(const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* g, const void* u, const void* h,
                                 void* dg, void* du, void* dx, void* dwg, void* dwu, void* dwd,
                                 void* workspace, size_t workspace_bytes, int64_t M, int64_t D, int64_t F, int activation, int dtype, void* stream) {
    const char* who = "gdn_gated_mlp_bwd";
    const int rc = check_mlp(who, M, D, F, activation, dtype);
    if (rc != GDN_OK) return rc;
    const bool inner = dx || dwg || dwu;
    GDN_CHECK_ARG(M == 0 || (dy && (!inner || (wd && g && u && dg && du)) && (!dx || (wg && wu)) && ((!dwg && !dwu) || x) && (!dwd || h)), GDN_ERR_INVALID,
                  "%s: a tensor that the asked gradients need is missing", who);
    GDN_CHECK_ARG((((uintptr_t)dy | (uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu | (uintptr_t)wd | (uintptr_t)g | (uintptr_t)u | (uintptr_t)h | (uintptr_t)dg |
                    (uintptr_t)du | (uintptr_t)dx | (uintptr_t)dwg | (uintptr_t)dwu | (uintptr_t)dwd) & 15) == 0,
                  GDN_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
    hipStream_t s = (hipStream_t)stream;
    const Workspace ws{workspace, workspace_bytes};
    return dtype == GDN_DTYPE_BF16 ? mlp_bwd<bf16_t>(dy, x, wg, wu, wd, g, u, h, dg, du, dx, dwg, dwu, dwd, ws, M, D, F, activation, s)
                                   : mlp_bwd<f16_t>(dy, x, wg, wu, wd, g, u, h, dg, du, dx, dwg, dwu, dwd, ws, M, D, F, activation, s);
}
