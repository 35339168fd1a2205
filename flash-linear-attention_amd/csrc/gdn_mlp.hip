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
    int act;
};

enum MlpEpilogue { MLP_PLAIN, MLP_GATE, MLP_GRAD };

template <typename T, int BM, int BN, int WM, int WN, bool A_DOWN, bool B_DOWN, int EPI>
__global__ __launch_bounds__(64 * WM * WN, 2) void mlp_gemm_kernel(MlpGemm p) {
    typedef Gemm<T, BM, BN, WM, WN, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    typedef typename Mma<T>::V4 V4;
    extern __shared__ __align__(16) char smem[];
    int tile = gemm_tile_of((int)blockIdx.x, p.tiles), which = 0;
    while (which + 1 < p.ops && tile >= p.op[which + 1].first) ++which;
    const GemmOperands& o = p.op[which];
    int tm, tn;
    gemm_place(tile - o.first, o.tiles_m, o.tiles_n, tm, tn);
    f32x4 acc[G::NT][G::MT];
    G::run(o, tm, tn, smem, acc);

    const int lane = threadIdx.x & 63, w = (int)threadIdx.x >> 6, wm = w % WM, wn = w / WM, c16 = lane & 15, g4 = 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        const int m = tm * BM + 16 * (wm * G::MT + i) + c16;
        if (m >= o.M) continue;
#pragma unroll
        for (int j = 0; j < (EPI == MLP_GATE ? G::NT / 2 : G::NT); ++j) {
            const int n = tn * G::COLUMNS + 16 * G::column_tile(wn, j) + g4;
            if (n >= o.N) continue;
            const int64_t at = (int64_t)m * o.N + n;
            const f32x4 x = acc[j][i];
            if constexpr (EPI == MLP_PLAIN) {
                *(V4*)((T*)p.C[which] + at) = V4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
            } else if constexpr (EPI == MLP_GATE) {
                const f32x4 u = acc[j + G::NT / 2][i];
                V4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float a, da;
                    mlp_act(p.act, x[e], a, da);
                    h[e] = (T)(a * u[e]);
                }
                *(V4*)((T*)p.C[0] + at) = h;
                if (p.C[1]) {
                    *(V4*)((T*)p.C[1] + at) = V4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
                    *(V4*)((T*)p.C[2] + at) = V4{(T)u[0], (T)u[1], (T)u[2], (T)u[3]};
                }
            } else {
                const V4 gv = *(const V4*)((const T*)p.G + at), uv = *(const V4*)((const T*)p.U + at);
                V4 dg, du;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float a, da;
                    mlp_act(p.act, (float)gv[e], a, da);
                    dg[e] = (T)(x[e] * (float)uv[e] * da);
                    du[e] = (T)(x[e] * a);
                }
                *(V4*)((T*)p.C[0] + at) = dg;
                *(V4*)((T*)p.C[1] + at) = du;
            }
        }
    }
}

static GemmOperands operands(const void* A, const void* B, int64_t lda, int64_t ldb, int64_t M, int64_t N, int64_t K) {
    GemmOperands o{};
    o.A[0] = A; o.B[0] = B; o.lda = lda; o.ldb = ldb; o.M = (int)M; o.N = (int)N; o.K = (int)K; o.segments = 1;
    return o;
}

template <typename T, int BM, int BN, int WM, int WN, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_tiles(MlpGemm& p, hipStream_t stream) {
    typedef Gemm<T, BM, BN, WM, WN, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    int64_t tiles = 0;
    for (int i = 0; i < p.ops; ++i) {
        GemmOperands& o = p.op[i];
        o.first = (int)tiles;
        o.tiles_m = (o.M + BM - 1) / BM; o.tiles_n = (o.N + G::COLUMNS - 1) / G::COLUMNS;
        tiles += (int64_t)o.tiles_m * o.tiles_n;
        GDN_CHECK_ARG(tiles < (1ll << 32) / G::THREADS, GDN_ERR_UNSUPPORTED, "the gated feed-forward block: %lld x %lld results are too many for one launch",
                      (long long)o.M, (long long)o.N);
    }
    if (tiles == 0) return GDN_OK;
    p.tiles = (int)tiles;
    auto kernel = mlp_gemm_kernel<T, BM, BN, WM, WN, A_DOWN, B_DOWN, EPI>;
    const int rc = ensure_dynamic_smem_for((const void*)kernel, G::LDS, "mlp_gemm_kernel");
    if (rc != GDN_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.tiles), dim3(G::THREADS), G::LDS, stream, p);
    return check_launch("mlp_gemm_kernel");
}

template <typename T, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_gemm(MlpGemm& p, hipStream_t stream) {
    return launch_tiles<T, 256, 256, 2, 4, A_DOWN, B_DOWN, EPI>(p, stream);
}

template <typename T>
static int mlp_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* y, void* g, void* u, void* h, int64_t M, int64_t D, int64_t F,
                   int act, hipStream_t stream) {
    MlpGemm p{};
    p.ops = 1; p.act = act;
    p.op[0] = operands(x, wg, D, D, M, F, D);
    p.op[0].B[1] = wu;
    p.C[0] = h; p.C[1] = g; p.C[2] = u;
    int rc = launch_gemm<T, false, false, MLP_GATE>(p, stream);
    if (rc != GDN_OK) return rc;
    MlpGemm q{};
    q.ops = 1;
    q.op[0] = operands(h, wd, F, F, M, D, F);
    q.C[0] = y;
    return launch_gemm<T, false, false, MLP_PLAIN>(q, stream);
}

template <typename T>
static int mlp_bwd(const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* g, const void* u, const void* h,
                   void* dg, void* du, void* dx, void* dwg, void* dwu, void* dwd, int64_t M, int64_t D, int64_t F, int act, hipStream_t stream) {
    int rc = GDN_OK;
    if (dx || dwg || dwu) {
        MlpGemm p{};
        p.ops = 1; p.act = act; p.G = g; p.U = u;
        p.op[0] = operands(dy, wd, D, F, M, F, D);
        p.C[0] = dg; p.C[1] = du;
        rc = launch_gemm<T, false, true, MLP_GRAD>(p, stream);
        if (rc != GDN_OK) return rc;
    }
    if (dx) {
        MlpGemm p{};
        p.ops = 1;
        p.op[0] = operands(dg, wg, F, D, M, D, F);
        p.op[0].A[1] = du; p.op[0].B[1] = wu; p.op[0].segments = 2;
        p.C[0] = dx;
        rc = launch_gemm<T, false, true, MLP_PLAIN>(p, stream);
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
    return p.ops ? launch_gemm<T, true, true, MLP_PLAIN>(p, stream) : GDN_OK;
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

extern "C" int gdn_gated_mlp_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* y, void* g, void* u, void* h,
                                 int64_t M, int64_t D, int64_t F, int activation, int dtype, void* stream) {
    const char* who = "gdn_gated_mlp_fwd";
    const int rc = check_mlp(who, M, D, F, activation, dtype);
    if (rc != GDN_OK) return rc;
    if (M == 0) return GDN_OK;
    GDN_CHECK_ARG(x && wg && wu && wd && y && h && !g == !u, GDN_ERR_INVALID, "%s: x, the weights, y and h are required, g goes with u", who);
    GDN_CHECK_ARG((((uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu | (uintptr_t)wd | (uintptr_t)y | (uintptr_t)g | (uintptr_t)u | (uintptr_t)h) & 15) == 0,
                  GDN_ERR_INVALID, "%s: tensors must be 16-byte aligned", who);
    hipStream_t s = (hipStream_t)stream;
    return dtype == GDN_DTYPE_BF16 ? mlp_fwd<bf16_t>(x, wg, wu, wd, y, g, u, h, M, D, F, activation, s)
                                   : mlp_fwd<f16_t>(x, wg, wu, wd, y, g, u, h, M, D, F, activation, s);
}

extern "C" int gdn_gated_mlp_bwd(const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* g, const void* u, const void* h,
                                 void* dg, void* du, void* dx, void* dwg, void* dwu, void* dwd,
                                 int64_t M, int64_t D, int64_t F, int activation, int dtype, void* stream) {
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
    return dtype == GDN_DTYPE_BF16 ? mlp_bwd<bf16_t>(dy, x, wg, wu, wd, g, u, h, dg, du, dx, dwg, dwu, dwd, M, D, F, activation, s)
                                   : mlp_bwd<f16_t>(dy, x, wg, wu, wd, g, u, h, dg, du, dx, dwg, dwu, dwd, M, D, F, activation, s);
}
