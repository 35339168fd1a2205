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
    int ops;
    int full, rest, parts;               // tiles with a workgroup each, and tiles after them whose contraction is shared out over `parts` workgroups
    void* C[3];                          // results (of a DUAL product's epilogue: h, g, u; of dh's: dg, du)
    const void* G; const void* U;
    float* sums;                         // [rest][parts][a tile's accumulators, as the lanes hold them]
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

struct MlpTile { int which, tm, tn; };
__device__ __forceinline__ MlpTile mlp_tile(const MlpGemm& p, int tile) {
    MlpTile t{0, 0, 0};
    while (t.which + 1 < p.ops && tile >= p.op[t.which + 1].first) ++t.which;
    const GemmOperands& o = p.op[t.which];
    gemm_place(tile - o.first, o.tiles_m, o.tiles_n, t.tm, t.tn);
    return t;
}

// Eight neighbours of this lane's results of a tile: fragment (i, j), its q-th half
template <typename T, typename G, int EPI>
__device__ __forceinline__ void mlp_chunk(const MlpGemm& p, MlpTile t, int i, int j, int q, f32x8 x, f32x8 u) {
    const GemmOperands& o = p.op[t.which];
    const int lane = threadIdx.x & 63, w = (int)threadIdx.x >> 6, wm = w % G::WAVES_M, wn = w / G::WAVES_M;
    const int m = t.tm * G::ROWS + 32 * (wm * G::MT + i) + (lane & 31), n = t.tn * G::COLUMNS + 32 * G::column_tile(wn, j) + 16 * (lane >> 5) + 8 * q;
    if (m < o.M && n < o.N) mlp_result<T, EPI>(p, t.which, (int64_t)m * o.N + n, x, u);
}

template <typename T, int BM, int BN, int WM, int WN, int KS, int STAGES, bool A_DOWN, bool B_DOWN, int EPI>
__global__ __launch_bounds__(64 * WM * WN, 2) void mlp_gemm_kernel(MlpGemm p) {
    typedef Gemm<T, BM, BN, WM, WN, KS, STAGES, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    extern __shared__ __align__(16) char smem[];
    const int id = (int)blockIdx.x, shared = id - p.full;
    int tile, part = 0;
    if (shared < 0) tile = gemm_tile_of(id, p.full);
    else {
        // (part by part: neighbours share rows and columns, the parts of a tile share nothing)
        const int at = gemm_tile_of(shared, p.rest * p.parts);
        part = at / p.rest; tile = p.full + at % p.rest;
    }
    f32x16 acc[G::NT][G::MT];
    const MlpTile at = mlp_tile(p, tile);
    G::run(p.op[at.which], at.tm, at.tn, part, shared < 0 ? 1 : p.parts, smem, acc);

    constexpr int KINDS = EPI == MLP_GATE ? 2 : 1, COLS = G::NT / KINDS;
    float* sums = shared < 0 || p.parts == 1 ? nullptr : p.sums + ((int64_t)(tile - p.full) * p.parts + part) * (BM * BN);
#pragma unroll
    for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int j = 0; j < COLS; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                f32x8 x, u;
#pragma unroll
                for (int e = 0; e < 8; ++e) { x[e] = acc[j][i][8 * q + e]; u[e] = acc[j + (KINDS - 1) * COLS][i][8 * q + e]; }
                if (sums) {
                    const int chunk = (i * COLS + j) * 2 + q;
                    *(f32x8*)(sums + ((int64_t)(chunk * KINDS) * G::THREADS + threadIdx.x) * 8) = x;
                    if (KINDS == 2) *(f32x8*)(sums + ((int64_t)(chunk * KINDS + 1) * G::THREADS + threadIdx.x) * 8) = u;
                } else
                    mlp_chunk<T, G, EPI>(p, at, i, j, q, x, u);
            }
}

// The parts of a shared tile added up, in order, and what becomes of the sums: a workgroup for eight results of every lane.
template <typename T, int BM, int BN, int WM, int WN, int KS, int STAGES, bool A_DOWN, bool B_DOWN, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void mlp_join_kernel(MlpGemm p) {
    typedef Gemm<T, BM, BN, WM, WN, KS, STAGES, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    constexpr int KINDS = EPI == MLP_GATE ? 2 : 1, COLS = G::NT / KINDS, CHUNKS = G::MT * COLS * 2;
    const int tile = (int)blockIdx.x / CHUNKS, chunk = (int)blockIdx.x % CHUNKS;
    const float* sums = p.sums + (int64_t)tile * p.parts * (BM * BN) + ((int64_t)(chunk * KINDS) * G::THREADS + threadIdx.x) * 8;
    f32x8 x = *(const f32x8*)sums, u = x;
    if (KINDS == 2) u = *(const f32x8*)(sums + G::THREADS * 8);
    for (int s = 1; s < p.parts; ++s) {
        x += *(const f32x8*)(sums + (int64_t)s * (BM * BN));
        if (KINDS == 2) u += *(const f32x8*)(sums + (int64_t)s * (BM * BN) + G::THREADS * 8);
    }
    mlp_chunk<T, G, EPI>(p, mlp_tile(p, p.full + tile), chunk / 2 / COLS, chunk / 2 % COLS, chunk % 2, x, u);
}

static GemmOperands operands(const void* A, const void* B, int64_t lda, int64_t ldb, int64_t M, int64_t N, int64_t K) {
    GemmOperands o{};
    o.A[0] = A; o.B[0] = B; o.lda = lda; o.ldb = ldb; o.M = (int)M; o.N = (int)N; o.K = (int)K; o.segments = 1;
    return o;
}

// How the products of a launch are cut: 256 x 256 tiles, a workgroup of eight waves a CU, or 128 x 128, two of four waves; and over how many workgroups the
// contraction of each tile is shared out that does not fill a round of the chip.  The least of the times that the launch would take by these figures:
//   a stage of 64 of a full round     1.7 us (256 x 256), 1.03 us (128 x 128: 512 tiles, half the area; 0.65 us where no two share a CU)
//   a round's begin and end           4 us; joining parts 5 us and their bytes, written and read, at 4 TB/s
// 8192 x 2048 x 5632, the weights' gradients (528 tiles of 256 x 256, two rounds and 16 tiles): the third round shared out over 16 workgroups a tile.
struct MlpPlan { bool large; int full, rest, parts; double us; };
static MlpPlan plan_gemm(const MlpGemm& p, int kinds) {
    MlpPlan best{true, 0, 0, 1, 1e30};
    for (int large = 0; large < 2; ++large) {
        const int64_t side = large ? 256 : 128, slots = large ? 256 : 512;
        int64_t tiles = 0, stages = 1;
        for (int i = 0; i < p.ops; ++i) {
            tiles += ((p.op[i].M + side - 1) / side) * (((int64_t)p.op[i].N * kinds + side - 1) / side);
            stages = std::max<int64_t>(stages, (int64_t)((p.op[i].K + 63) / 64) * p.op[i].segments);
        }
        if (tiles >= (1ll << 31)) continue;
        const int64_t rest = tiles % slots, rounds = tiles / slots;
        const double stage = large ? 1.7 : 1.03;
        const double before = rounds * (stages * stage + 4);
        auto tail = [&](int64_t workgroups) { return large || workgroups > 256 ? stage : 0.65; };
        for (int64_t parts = 1; parts <= 16 && (parts == 1 || (rest * parts <= slots && stages / parts >= 2)); ++parts) {
            double us = before + (rest ? ((stages + parts - 1) / parts) * tail(rest * parts) + 4 : 0);
            if (parts > 1) us += 5 + rest * parts * side * side * 8 / 4e6;
            if (us < best.us) best = MlpPlan{large != 0, parts > 1 ? (int)(tiles - rest) : (int)tiles, parts > 1 ? (int)rest : 0, (int)parts, us};
        }
    }
    return best;
}
static size_t plan_bytes(const MlpPlan& plan) { return (size_t)plan.rest * plan.parts * (plan.large ? 65536 : 16384) * 4; }
static size_t plan_bytes(const MlpGemm& p, int kinds) { return plan_bytes(plan_gemm(p, kinds)); }

struct Workspace { void* at; size_t bytes; };

template <typename T, int SIDE, int WN, int KS, int STAGES, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_tiles(MlpGemm& p, const MlpPlan& plan, hipStream_t stream) {
    typedef Gemm<T, SIDE, SIDE, 2, WN, KS, STAGES, A_DOWN, B_DOWN, EPI == MLP_GATE> G;
    int64_t tiles = 0;
    for (int i = 0; i < p.ops; ++i) {
        GemmOperands& o = p.op[i];
        o.first = (int)tiles;
        o.tiles_m = (o.M + SIDE - 1) / SIDE; o.tiles_n = (o.N + G::COLUMNS - 1) / G::COLUMNS;
        tiles += (int64_t)o.tiles_m * o.tiles_n;
        GDN_CHECK_ARG(tiles < (1ll << 32) / G::THREADS, GDN_ERR_UNSUPPORTED, "the gated feed-forward block: %lld x %lld results are too many for one launch",
                      (long long)o.M, (long long)o.N);
    }
    if (tiles == 0) return GDN_OK;
    p.full = plan.full; p.rest = plan.rest; p.parts = plan.parts;
    GDN_CHECK_ARG(tiles == (int64_t)p.full + p.rest, GDN_ERR_INVALID, "the gated feed-forward block: a plan for %d tiles, not %lld", p.full + p.rest, (long long)tiles);
    auto kernel = mlp_gemm_kernel<T, SIDE, SIDE, 2, WN, KS, STAGES, A_DOWN, B_DOWN, EPI>;
    const int rc = ensure_dynamic_smem_for((const void*)kernel, G::LDS, "mlp_gemm_kernel");
    if (rc != GDN_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.full + p.rest * p.parts)), dim3(G::THREADS), G::LDS, stream, p);
    if (p.rest == 0) return check_launch("mlp_gemm_kernel");
    const int rc2 = check_launch("mlp_gemm_kernel");
    if (rc2 != GDN_OK) return rc2;
    hipLaunchKernelGGL((mlp_join_kernel<T, SIDE, SIDE, 2, WN, KS, STAGES, A_DOWN, B_DOWN, EPI>), dim3((unsigned)(p.rest * G::MT * G::NT * 2 / (EPI == MLP_GATE ? 2 : 1))),
                       dim3(G::THREADS), 0, stream, p);
    return check_launch("mlp_join_kernel");
}

template <typename T, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_gemm(MlpGemm& p, Workspace ws, hipStream_t stream) {
    const MlpPlan plan = plan_gemm(p, EPI == MLP_GATE ? 2 : 1);
    const size_t need = plan_bytes(plan);
    GDN_CHECK_ARG(need == 0 || (ws.at && ws.bytes >= need), GDN_ERR_WORKSPACE, "the gated feed-forward block: workspace too small (%zu bytes, %zu needed)", ws.bytes, need);
    p.sums = (float*)ws.at;
    constexpr int KS = A_DOWN && B_DOWN ? 32 : 64, STAGES = 128 / KS;
    return plan.large ? launch_tiles<T, 256, 4, KS, STAGES, A_DOWN, B_DOWN, EPI>(p, plan, stream) : launch_tiles<T, 128, 2, KS, STAGES, A_DOWN, B_DOWN, EPI>(p, plan, stream);
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

static MlpGemm grad_weights(const void* dy, const void* x, const void* h, const void* dg, const void* du, void* dwg, void* dwu, void* dwd, int64_t M, int64_t D, int64_t F) {
    MlpGemm p{};
    auto add = [&](const void* A, const void* B, int64_t rows, int64_t cols, void* C) {
        if (!C) return;
        p.op[p.ops] = operands(A, B, rows, cols, rows, cols, M);
        p.C[p.ops++] = C;
    };
    add(dg, x, F, D, dwg);
    add(du, x, F, D, dwu);
    add(dy, h, D, F, dwd);
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
    MlpGemm p = grad_weights(dy, x, h, dg, du, dwg, dwu, dwd, M, D, F);
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
    size_t most = std::max(plan_bytes(grad_inner(nullptr, nullptr, M, D, F), 1), plan_bytes(grad_x(nullptr, nullptr, nullptr, nullptr, M, D, F), 1));
    // (which of the weights' gradients will be asked for is not known here: those of Wg and Wu are alike)
    char some;
    for (int asked = 1; asked < 6; ++asked) {
        const int alike = asked % 3;
        most = std::max(most, plan_bytes(grad_weights(nullptr, nullptr, nullptr, nullptr, nullptr, alike ? &some : nullptr, alike > 1 ? &some : nullptr, asked > 2 ? &some : nullptr, M, D, F), 1));
    }
    return most;
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
