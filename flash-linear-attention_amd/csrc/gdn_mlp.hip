// The gated feed-forward block (fla/modules/mlp.py: GatedMLP) and its gradients:
//
//   g = x Wg^T, u = x Wu^T;  h = act(g) u;  y = h Wd^T             x [M][D]; Wg, Wu [F][D]; Wd [D][F]
//   dh = dy Wd;  dg = dh s, du = dh a  with  s = act'(g) u, a = act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Roundings to 16 bits besides the results': h, dg and du, because they are operands of matrix products, whose instructions take 16-bit operands (with h in two halves of 16 bits the
// down projection would be two products); s and a, to hold half of what 32 bits would from the forward to the backward.  Each is rounded once, from 32-bit sums.  y and
// dWd come out 1.4 times as far from the exact ones as their own rounding, the other gradients 1.7 times (bf16: 2.3e-3 and 2.9e-3 against 1.7e-3, 2-norms).
//
// Three tensors of M x F are held for the backward, s, a and h: 541 MB at 8192 x 11008.  g and u would be two, 361 MB; but of those two roundings (and a slope's
// steepness) would go into dg, and the backward would work the activation out again, and h for dWd.
//
// Forward two launches (both projections with the activation and the product on top; the down projection), backward three (dh with dg and du on top; dx;
// the weights' gradients together).  Many rows are bound by the matrix cores: gdn_gemm.h.
#include "gdn_gemm.h"

namespace gdn {

// act(g) and act'(g).  (The hardware's reciprocal and base-2 exponential, 1 ulp each: what follows is rounded to 16 bits, and a tile's 32768 activations are 3 us
// of its eight waves' time this way, 10 with full division.)
__device__ __forceinline__ void mlp_act(int act, float g, float& a, float& da) {
    if (act == GDN_ACT_GELU_TANH) {
        // (tanh has reached 1 long before 16; beyond, g^2 times its vanishing slope could be infinity times zero)
        const float c = g > 16.f ? 16.f : g < -16.f ? -16.f : g, z = 0.7978845608028654f * (c + 0.044715f * c * c * c);
        const float s = sigmoid_stream(2.f * z);                     // (1 + tanh z) / 2
        a = g * s;
        da = s + c * 2.f * s * (1.f - s) * 0.7978845608028654f * (1.f + 0.134145f * c * c);
    } else {
        const float s = sigmoid_stream(g);
        if (act == GDN_ACT_SIGMOID) { a = s; da = s * (1.f - s); }
        else { a = g * s; da = s * (1.f + g * (1.f - s)); }
    }
}

struct MlpGemm {
    GemmOperands op[3];
    int ops;
    int full, rest, parts;               // tiles with a workgroup each, and tiles after them whose contraction is shared out over `parts` workgroups
    void* C[3];                          // results (of a DUAL product's epilogue: h, s, a; of dh's: dg, du)
    const void* S; const void* A;        // dh's epilogue: s and a of the forward
    float* sums;                         // [rest][parts][a tile's accumulators, as the lanes hold them]
};

// MLP_GATE + an activation's code: the epilogue of both projections (the activation is the kernel's, or its choice would be made for every result)
enum MlpEpilogue { MLP_PLAIN, MLP_GRAD, MLP_GATE };
constexpr bool is_gate(int epilogue) { return epilogue >= MLP_GATE; }

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x8_at16 __attribute__((ext_vector_type(8), aligned(16)));       // (in the workspace, which lies on 16-byte boundaries)

// What becomes of eight neighbours of a result (of both products where there are two), at offset `at` of the outputs; MLP_GRAD: sv, av are the
// forward's s and a there.
template <typename T, int EPI>
__device__ __forceinline__ void mlp_result(const MlpGemm& p, int which, int64_t at, f32x8 x, f32x8 u, typename Mma<T>::V8 sv, typename Mma<T>::V8 av) {
    typedef typename Mma<T>::V8 V8;
    auto rounded = [](f32x8 v) { return V8{(T)v[0], (T)v[1], (T)v[2], (T)v[3], (T)v[4], (T)v[5], (T)v[6], (T)v[7]}; };
    if constexpr (EPI == MLP_PLAIN) {
        *(V8*)((T*)p.C[which] + at) = rounded(x);
    } else if constexpr (is_gate(EPI)) {
        V8 h, s, a;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float act, slope;
            mlp_act(EPI - MLP_GATE, x[e], act, slope);
            h[e] = (T)(act * u[e]); s[e] = (T)(slope * u[e]); a[e] = (T)act;
        }
        *(V8*)((T*)p.C[0] + at) = h;
        if (p.C[1]) {
            // (not read again before the backward: past the caches, 2 - 3 % of the launch at 8192 x 2048 x 5632)
            __builtin_nontemporal_store(s, (V8*)((T*)p.C[1] + at));
            __builtin_nontemporal_store(a, (V8*)((T*)p.C[2] + at));
        }
    } else {
        V8 dg, du;
#pragma unroll
        for (int e = 0; e < 8; ++e) { dg[e] = (T)(x[e] * (float)sv[e]); du[e] = (T)(x[e] * (float)av[e]); }
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

// Where eight neighbours of this lane's results of a tile go - fragment (i, j), its q-th half - or -1: past the end of C.
template <typename G>
__device__ __forceinline__ int64_t mlp_place(const MlpGemm& p, MlpTile t, int i, int j, int q) {
    const GemmOperands& o = p.op[t.which];
    const int lane = threadIdx.x & 63, w = (int)threadIdx.x >> 6, wm = w % G::WAVES_M, wn = w / G::WAVES_M;
    const int m = t.tm * G::ROWS + 32 * (wm * G::MT + i) + (lane & 31), n = t.tn * G::COLUMNS + 32 * G::column_tile(wn, j) + 16 * q + 8 * (lane >> 5);
    return m < o.M && n < o.N ? (int64_t)m * o.N + n : -1;
}

template <typename T, int BM, int BN, int WM, int WN, int KS, int SLOTS, bool A_DOWN, bool B_DOWN, int EPI>
__global__ __launch_bounds__(64 * WM * WN, 2) void mlp_gemm_kernel(MlpGemm p) {
    typedef Gemm<T, BM, BN, WM, WN, KS, SLOTS, A_DOWN, B_DOWN, is_gate(EPI)> G;
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

    constexpr int KINDS = is_gate(EPI) ? 2 : 1, COLS = G::NT / KINDS, ROUND = 2 * COLS;
    auto result = [&](int i, int jq) {
        f32x8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = acc[jq / 2][i][8 * (jq % 2) + e];
        return x;
    };
    if (shared >= 0 && p.parts > 1) {
        float* sums = p.sums + ((int64_t)(tile - p.full) * p.parts + part) * (BM * BN) + threadIdx.x * 8;
#pragma unroll
        for (int i = 0; i < G::MT; ++i)
#pragma unroll
            for (int c = 0; c < ROUND; ++c)
#pragma unroll
                for (int kind = 0; kind < KINDS; ++kind) *(f32x8_at16*)(sums + (int64_t)((i * ROUND + c) * KINDS + kind) * G::THREADS * 8) = result(i, kind * ROUND + c);
        return;
    }
    // 32 rows at a time through this wave's share of the LDS, from the lanes' order into rows, so that the rows of 64 (32) columns leave in whole lines.  A row's
    // 16-byte slots are XORed with the row: no bank conflicts in tiles of 256 x 256, in the smaller ones of both projections 2 % of the LDS cycles.  s and a are asked for 32 rows before they are needed.  Straight from the lanes, 32 bytes
    // of a row at a time, 8192 x 2048 x 5632 took 988 us backward (this way 956), 32768 rows 3790 (3670), with four operand slots.
    typedef typename Mma<T>::V8 V8;
    constexpr int CW = 32 * COLS, QUADS = CW / 4, PER_ROW = CW / 8, ROWS = 64 / PER_ROW, PASSES = 32 / ROWS;
    static_assert(KINDS * 32 * CW * 4 * G::WAVES <= G::LDS, "32 rows of every wave fit in the LDS of the main loop");
    const GemmOperands& o = p.op[at.which];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = w % WM, wn = w / WM;
    float* area = (float*)smem + w * (KINDS * 32 * CW);
    const int row0 = at.tm * BM + 32 * (wm * G::MT) + lane / PER_ROW, n = at.tn * G::COLUMNS + 32 * G::column_tile(wn, 0) + 8 * (lane % PER_ROW);
    V8 sv[2][PASSES], av[2][PASSES];
    auto inner = [&](int i) {
        if constexpr (EPI == MLP_GRAD) {
#pragma unroll
            for (int r = 0; r < PASSES; ++r) {
                const int64_t to = (int64_t)min(row0 + 32 * i + ROWS * r, o.M - 1) * o.N + min(n, o.N - 8);
                sv[i % 2][r] = __builtin_nontemporal_load((const V8*)((const T*)p.S + to));
                av[i % 2][r] = __builtin_nontemporal_load((const V8*)((const T*)p.A + to));
            }
        }
    };
    inner(0);
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
        if (i + 1 < G::MT) inner(i + 1);
#pragma unroll
        for (int kind = 0; kind < KINDS; ++kind)
#pragma unroll
            for (int c = 0; c < ROUND; ++c) {
                const int m = lane & 31, slot = 4 * c + 2 * (lane >> 5);
                const f32x8 x = result(i, kind * ROUND + c);
                float* to = area + kind * 32 * CW + m * CW;
                *(f32x4*)(to + 4 * (slot ^ (m & (QUADS - 1)))) = f32x4{x[0], x[1], x[2], x[3]};
                *(f32x4*)(to + 4 * ((slot + 1) ^ (m & (QUADS - 1)))) = f32x4{x[4], x[5], x[6], x[7]};
            }
#pragma unroll
        for (int r = 0; r < PASSES; ++r) {
            const int m = ROWS * r + lane / PER_ROW, slot = 2 * (lane % PER_ROW);
            f32x8 x[KINDS];
#pragma unroll
            for (int kind = 0; kind < KINDS; ++kind) {
                const float* from = area + kind * 32 * CW + m * CW;
                const f32x4 lo = *(const f32x4*)(from + 4 * (slot ^ (m & (QUADS - 1)))), hi = *(const f32x4*)(from + 4 * ((slot + 1) ^ (m & (QUADS - 1))));
                x[kind] = f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            }
            if (row0 + 32 * i + ROWS * r < o.M && n < o.N)
                mlp_result<T, EPI>(p, at.which, (int64_t)(row0 + 32 * i + ROWS * r) * o.N + n, x[0], x[KINDS - 1], sv[i % 2][r], av[i % 2][r]);
        }
    }
}

// The parts of a shared tile added up, in order, and what becomes of the sums: a workgroup for eight results of every lane.
template <typename T, int BM, int BN, int WM, int WN, int KS, int SLOTS, bool A_DOWN, bool B_DOWN, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void mlp_join_kernel(MlpGemm p) {
    typedef Gemm<T, BM, BN, WM, WN, KS, SLOTS, A_DOWN, B_DOWN, is_gate(EPI)> G;
    constexpr int KINDS = is_gate(EPI) ? 2 : 1, COLS = G::NT / KINDS, CHUNKS = G::MT * COLS * 2;
    const int tile = (int)blockIdx.x / CHUNKS, chunk = (int)blockIdx.x % CHUNKS;
    const float* sums = p.sums + (int64_t)tile * p.parts * (BM * BN) + ((int64_t)(chunk * KINDS) * G::THREADS + threadIdx.x) * 8;
    f32x8 x = *(const f32x8_at16*)sums, u = x;
    if (KINDS == 2) u = *(const f32x8_at16*)(sums + G::THREADS * 8);
    for (int s = 1; s < p.parts; ++s) {
        x += *(const f32x8_at16*)(sums + (int64_t)s * (BM * BN));
        if (KINDS == 2) u += *(const f32x8_at16*)(sums + (int64_t)s * (BM * BN) + G::THREADS * 8);
    }
    const MlpTile at = mlp_tile(p, p.full + tile);
    const int64_t to = mlp_place<G>(p, at, chunk / 2 / COLS, chunk / 2 % COLS, chunk % 2);
    if (to < 0) return;
    typename Mma<T>::V8 sv{}, av{};
    if constexpr (EPI == MLP_GRAD) { sv = *(const decltype(sv)*)((const T*)p.S + to); av = *(const decltype(av)*)((const T*)p.A + to); }
    mlp_result<T, EPI>(p, at.which, to, x, u, sv, av);
}

static GemmOperands operands(const void* A, const void* B, int64_t lda, int64_t ldb, int64_t M, int64_t N, int64_t K) {
    GemmOperands o{};
    o.A[0] = A; o.B[0] = B; o.lda = lda; o.ldb = ldb; o.M = (int)M; o.N = (int)N; o.K = (int)K; o.segments = 1;
    return o;
}

// How the products of a launch are cut: the tiles, and over how many workgroups the contraction of each tile is shared out that does not fill a round of the
// chip (`rest` tiles of `parts` workgroups after `full` of one): the least of the times that the launch would take by these figures.
//   tiles       waves  workgroups   us for a stage of 64, the chip full   and at least (few workgroups)   a round's begin and end
//   256 x 256   8      1 a CU       1.54                                  1.18                            6
//   128 x 128   4      2 a CU       0.95                                  0.67                            4.3    five slots of LDS: half the CU's
//   128 x 128   8      1 a CU       0.55                                  0.55                            5      eight: more in flight, for few workgroups
//   64 x 64     2      2 a CU       0.42                                  0.42                            4.4    the same, where no operand is read down its columns
// In between a stage's time grows with the workgroups: a full chip is held back by its caches and its clock, too.  What a round's results are read and written with
// (8 bytes a result for the inner gradients, 2 otherwise: between those of h alone and of h, s and a) goes at 2.5 TB/s where all workgroups end together; of the rounds
// before the last a fifth of it is seen.  Joining parts takes 4.3 us, 0.3 a part and their bytes, written and read, at 5.2 TB/s.
// Fitted to 2481 cuts - every tile and up to 16 parts of the six launches of a forward and a training step, 29 sizes from 20 x 4096 x 11008 and 3000 x 512 x 1408 to
// 8192 x 4096 x 11008 and 30000 x 1024 x 1024 -, each the geometric mean of its times on operands in the caches and behind 600 MB of other data: met within a tenth
// (root mean square of the logarithms); the chosen cut takes 2 % longer than the best one in the mean, 24 % at worst (dh of 3000 x 512 x 1408).  Both projections of
// 48 x 2048 x 5632 take 16 us in 64 x 64 tiles, 21 in 128 x 128; down of 300 x 4096 x 11008 50 in 128 x 128 in four parts, 76 in 64 x 64; dh of 2999 x 1008 x 2696 41 in
// 128 x 128 in four parts, 48 in 132 of 256 x 256; the weights' gradients of 8192 x 2048 x 5632, 528 tiles of 256 x 256, 456 with the last 16 in ten parts, 569 in 128 x 128
// (operands in the caches).
struct MlpTiles { int side, waves_m, waves_n, slots, per_cu; double full, least, round; };
constexpr MlpTiles MLP_TILES[] = {{256, 2, 4, 5, 1, 1.54, 1.18, 6}, {128, 2, 2, 5, 2, 0.95, 0.67, 4.3}, {128, 4, 2, 8, 1, 0.55, 0.55, 5}, {64, 2, 1, 8, 2, 0.42, 0.42, 4.4}};
struct MlpPlan { int tiles, full, rest, parts; };
static MlpPlan plan_gemm(const MlpGemm& p, int epilogue, bool rows) {
    const int kinds = is_gate(epilogue) ? 2 : 1;
    MlpPlan best{0, 0, 0, 1};
    double best_us = 1e30;
    for (int t = 0; t < (rows ? 4 : 3); ++t) {
        const MlpTiles& k = MLP_TILES[t];
        const int64_t slots = 256 * k.per_cu;
        int64_t tiles = 0, stages = 1;
        for (int i = 0; i < p.ops; ++i) {
            tiles += ((p.op[i].M + k.side - 1ll) / k.side) * (((int64_t)p.op[i].N * kinds + k.side - 1) / k.side);
            stages = std::max<int64_t>(stages, (p.op[i].K + 63ll) / 64 * p.op[i].segments);
        }
        if (tiles >= (1ll << 31)) continue;
        const int64_t rest = tiles % slots;
        const double results = (double)k.side * k.side * (epilogue == MLP_GRAD ? 8 : 2) / 2.5e6;          // us, a tile's
        const double before = (double)(tiles / slots) * (stages * k.full + k.round + 0.2 * slots * results);
        for (int64_t parts = 1; parts <= 16 && (parts == 1 || (rest > 0 && rest * parts <= slots && stages / parts >= 2)); ++parts) {
            double us = before;
            if (rest) us += (stages + parts - 1) / parts * std::max(k.least, k.full * (rest * parts) / slots) + k.round + rest * results;
            if (parts > 1) us += 4.3 + 0.3 * parts + (double)(rest * parts) * k.side * k.side * 8 / 5.2e6;
            if (us < best_us) {
                best_us = us;
                best = MlpPlan{t, (int)(parts > 1 ? tiles - rest : tiles), (int)(parts > 1 ? rest : 0), (int)parts};
            }
        }
    }
    return best;
}
static size_t plan_bytes(const MlpPlan& plan) { return (size_t)plan.rest * plan.parts * MLP_TILES[plan.tiles].side * MLP_TILES[plan.tiles].side * 4; }

struct Workspace { void* at; size_t bytes; };

template <typename T, int TILES, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_tiles(MlpGemm& p, const MlpPlan& plan, hipStream_t stream) {
    // (both operands down their columns: stages of half the width, twice as many, an even number of slots)
    // (both projections in a 256 x 256 tile: 64 columns of each to a wave, a whole line of every result's row)
    constexpr bool WIDE = is_gate(EPI) && MLP_TILES[TILES].side == 256;
    constexpr int SIDE = MLP_TILES[TILES].side, WM = WIDE ? 4 : MLP_TILES[TILES].waves_m, WN = WIDE ? 2 : MLP_TILES[TILES].waves_n, KS = A_DOWN && B_DOWN ? 32 : 64, SLOTS = KS == 64 ? MLP_TILES[TILES].slots : 4 * (MLP_TILES[TILES].slots / 2);
    typedef Gemm<T, SIDE, SIDE, WM, WN, KS, SLOTS, A_DOWN, B_DOWN, is_gate(EPI)> G;
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
    auto kernel = mlp_gemm_kernel<T, SIDE, SIDE, WM, WN, KS, SLOTS, A_DOWN, B_DOWN, EPI>;
    const int rc = ensure_dynamic_smem_for((const void*)kernel, G::LDS, "mlp_gemm_kernel");
    if (rc != GDN_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.full + p.rest * p.parts)), dim3(G::THREADS), G::LDS, stream, p);
    if (p.rest == 0) return check_launch("mlp_gemm_kernel");
    const int rc2 = check_launch("mlp_gemm_kernel");
    if (rc2 != GDN_OK) return rc2;
    hipLaunchKernelGGL((mlp_join_kernel<T, SIDE, SIDE, WM, WN, KS, SLOTS, A_DOWN, B_DOWN, EPI>), dim3((unsigned)(p.rest * G::MT * G::NT * 2 / (is_gate(EPI) ? 2 : 1))),
                       dim3(G::THREADS), 0, stream, p);
    return check_launch("mlp_join_kernel");
}

template <typename T, bool A_DOWN, bool B_DOWN, int EPI>
static int launch_gemm(MlpGemm& p, Workspace ws, hipStream_t stream) {
    constexpr bool ROWS = !A_DOWN && !B_DOWN;
    const MlpPlan plan = plan_gemm(p, EPI, ROWS);
    const size_t need = plan_bytes(plan);
    GDN_CHECK_ARG(need == 0 || (ws.at && ws.bytes >= need), GDN_ERR_WORKSPACE, "the gated feed-forward block: workspace too small (%zu bytes, %zu needed)", ws.bytes, need);
    p.sums = (float*)ws.at;
    if (plan.tiles == 0) return launch_tiles<T, 0, A_DOWN, B_DOWN, EPI>(p, plan, stream);
    if (plan.tiles == 1) return launch_tiles<T, 1, A_DOWN, B_DOWN, EPI>(p, plan, stream);
    if constexpr (ROWS) {
        if (plan.tiles == 3) return launch_tiles<T, 3, A_DOWN, B_DOWN, EPI>(p, plan, stream);
    }
    return launch_tiles<T, 2, A_DOWN, B_DOWN, EPI>(p, plan, stream);
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

// ---------------------------------------------------------------------------------------------
// A few rows (a decode step): every weight is read once and little else, so what counts is how much of the weights is in flight.  A workgroup takes CT tiles of 16
// weight rows - eight of Wg and the eight of Wu at the same columns, or 16 rows of Wd - and its waves a share of
// the contraction each, operands straight from memory to registers, partial sums through LDS.  Rows may begin at any address and end anywhere.
// ---------------------------------------------------------------------------------------------
struct MlpFew {
    const void* x; const void* w[2];
    void* C[3];
    int M, N, K, act;
};

template <typename T, int EPI>
__device__ __forceinline__ void few_result(const MlpFew& p, int64_t at, float x, float u) {
    if constexpr (is_gate(EPI)) {
        float act, slope;
        mlp_act(p.act, x, act, slope);
        ((T*)p.C[0])[at] = (T)(act * u);
        if (p.C[1]) { ((T*)p.C[1])[at] = (T)(slope * u); ((T*)p.C[2])[at] = (T)act; }
    } else
        ((T*)p.C[0])[at] = (T)x;
}

template <typename T, int CT, int WAVES, int EPI, int COLS>
__global__ __launch_bounds__(64 * WAVES) void mlp_few_kernel(MlpFew p) {
    typedef typename Mma<T>::V8 V8;
    typedef T AnyV8 __attribute__((ext_vector_type(8), aligned(2)));
    constexpr int U = 8, PITCH = 16 * CT + 1;                      // U: steps of 32 requested together
    __shared__ float sums[WAVES][16][PITCH];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * COLS * CT, K = p.K;
    const int steps = (K + 31) / 32, whole = K / 32, s0 = w * steps / WAVES, s1 = (w + 1) * steps / WAVES;
    // (columns and rows past the end repeat the last ones, their results are dropped)
    const T* wr[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c)
        wr[c] = (const T*)(is_gate(EPI) && c16 >= 8 ? p.w[1] : p.w[0]) + (int64_t)min(n0 + COLS * c + c16 % COLS, p.N - 1) * K + 8 * g;
    const T* xr = (const T*)p.x + (int64_t)min(c16, p.M - 1) * K + 8 * g;
    f32x4 acc[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int end = min(s1, whole);
    for (int s = s0; s < end; s += U) {
        V8 fw[CT][U], fx[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < end) {                                     // (the same for the wave)
#pragma unroll
                for (int c = 0; c < CT; ++c) fw[c][u] = *(const AnyV8*)(wr[c] + 32 * (s + u));
            }
#pragma unroll
        for (int u = 0; u < U; ++u) if (s + u < end) fx[u] = *(const AnyV8*)(xr + 32 * (s + u));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < end) {
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[c] = Mma<T>::run(fw[c][u], fx[u], acc[c]);
            }
    }
    if (s1 > whole) {                                              // the last step of a contraction that is no multiple of 32: zeros from K on
        auto rest = [&](const T* at) {
            const int left = K - 32 * whole - 8 * g;
            V8 v{};
            if (left >= 8) v = *(const AnyV8*)(at + 32 * whole);
            else {
#pragma unroll
                for (int e = 0; e < 8; ++e) if (e < left) v[e] = at[32 * whole + e];
            }
            return v;
        };
        const V8 fx = rest(xr);
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c] = Mma<T>::run(rest(wr[c]), fx, acc[c]);
    }
    // lane (c16, g): row c16, columns 4g .. 4g + 3 of each tile
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[w][c16][16 * c + 4 * g + e] = acc[c][e];
    __syncthreads();
    for (int i = tid; i < COLS * CT * p.M; i += 64 * WAVES) {
        const int m = i / (COLS * CT), j = i % (COLS * CT), n = n0 + j, at16 = 16 * (j / COLS) + j % COLS;
        if (n >= p.N) continue;
        float x = 0.f, u = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            x += sums[v][m][at16];
            if (is_gate(EPI)) u += sums[v][m][at16 + 8];
        }
        few_result<T, EPI>(p, (int64_t)m * p.N + n, x, u);
    }
}

// Four rows and fewer: a wave reads whole kilobytes of weight rows (the tiles above take sixteen rows 64 bytes at a time), two columns' - of both projections or
// of the down projection -, and multiplies them with x two elements at a time, sums over its lanes at the end.
template <typename T> struct Dot;
template <> struct Dot<bf16_t> {
    static __device__ __forceinline__ float add(bf16x2 a, bf16x2 b, float c) { return __builtin_amdgcn_fdot2_f32_bf16(a, b, c, false); }
};
template <> struct Dot<f16_t> {
    typedef f16_t V2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float add(V2 a, V2 b, float c) { return __builtin_amdgcn_fdot2(a, b, c, false); }
};

template <typename T, int ROWS, int EPI>
__global__ __launch_bounds__(256) void mlp_vec_kernel(MlpFew p) {
    typedef typename Mma<T>::V8 V8;
    typedef T AnyV8 __attribute__((ext_vector_type(8), aligned(2)));
    constexpr int COLS = 2, KINDS = is_gate(EPI) ? 2 : 1, W = COLS * KINDS, U = 16 / W;      // W weight rows of a wave, U kilobytes of each requested together
    const int lane = threadIdx.x & 63, K = p.K, n0 = ((int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6)) * COLS;
    if (n0 >= p.N) return;
    const T* wr[W];                                                // (a column past the end repeats the last one, its result is dropped)
#pragma unroll
    for (int r = 0; r < W; ++r) wr[r] = (const T*)p.w[r / COLS] + (int64_t)min(n0 + r % COLS, p.N - 1) * K;
    float acc[W][ROWS] = {};
    auto load = [&](const T* row, int k) {
        V8 v{};
        if (k + 8 <= K) v = *(const AnyV8*)(row + k);
        else if (k < K) {
#pragma unroll
            for (int e = 0; e < 8; ++e) if (k + e < K) v[e] = row[k + e];
        }
        return v;
    };
    for (int k0 = 0; k0 < K; k0 += 512 * U) {
        V8 fw[W][U], fx[ROWS][U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + 512 * u < K) {                                // (the same for the workgroup)
#pragma unroll
                for (int r = 0; r < W; ++r) fw[r][u] = load(wr[r], k0 + 512 * u + 8 * lane);
#pragma unroll
                for (int m = 0; m < ROWS; ++m) fx[m][u] = load((const T*)p.x + (int64_t)min(m, p.M - 1) * K, k0 + 512 * u + 8 * lane);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + 512 * u < K) {
#pragma unroll
                for (int r = 0; r < W; ++r)
#pragma unroll
                    for (int m = 0; m < ROWS; ++m)
#pragma unroll
                        for (int e = 0; e < 8; e += 2) acc[r][m] = Dot<T>::add({fw[r][u][e], fw[r][u][e + 1]}, {fx[m][u][e], fx[m][u][e + 1]}, acc[r][m]);
            }
    }
    // every lane gets every sum; lane COLS m + c keeps those of row m, column c
    float x = 0.f, u = 0.f;
#pragma unroll
    for (int r = 0; r < W; ++r)
#pragma unroll
        for (int m = 0; m < ROWS; ++m) {
            float v = acc[r][m];
#pragma unroll
            for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s, 64);
            if (lane == COLS * m + r % COLS) (r < COLS ? x : u) = v;
        }
    const int m = lane / COLS, n = n0 + lane % COLS;
    if (m < p.M && m < ROWS && n < p.N) few_result<T, EPI>(p, (int64_t)m * p.N + n, x, u);
}

// Up to 16 rows (one matrix tile of them): 16 rows of 2048 x 5632 22.5 us, in 64 x 64 tiles 25.7.  Rows of x cost a workgroup as much as a tile of weights, so it
// takes three tiles of Wg and Wu.  Up to four rows by whole kilobytes of a row: one row 18.0 -> 14.5 us (69 MB in two launches: 4.8 TB/s), four 19.9 -> 17.7;
// one of 4096 x 11008 56.4 -> 53.3 us, of 1024 x 2816 10.2 -> 7.9.
constexpr int64_t MLP_FEW_ROWS = GDN_MLP_FEW_ROWS;

template <typename T, int EPI>
static int launch_few(const MlpFew& p, hipStream_t stream) {
    if (p.M <= 4) {
        const dim3 grid((unsigned)((p.N + 7) / 8));
        if (p.M == 1) hipLaunchKernelGGL((mlp_vec_kernel<T, 1, EPI>), grid, dim3(256), 0, stream, p);
        else if (p.M == 2) hipLaunchKernelGGL((mlp_vec_kernel<T, 2, EPI>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((mlp_vec_kernel<T, 4, EPI>), grid, dim3(256), 0, stream, p);
        return check_launch("mlp_vec_kernel");
    }
    constexpr int WAVES = 8, COLS = is_gate(EPI) ? 8 : 16, CT = is_gate(EPI) ? 3 : 1;
    hipLaunchKernelGGL((mlp_few_kernel<T, CT, WAVES, EPI, COLS>), dim3((unsigned)((p.N + COLS * CT - 1) / (COLS * CT))), dim3(64 * WAVES), 0, stream, p);
    return check_launch("mlp_few_kernel");
}

template <typename T>
static int mlp_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* y, void* s, void* a, void* h, Workspace ws, int64_t M, int64_t D, int64_t F,
                   int act, hipStream_t stream) {
    if (M <= MLP_FEW_ROWS) {
        const MlpFew first{x, {wg, wu}, {h, s, a}, (int)M, (int)F, (int)D, act};
        const int rc = launch_few<T, MLP_GATE>(first, stream);
        return rc != GDN_OK ? rc : launch_few<T, MLP_PLAIN>(MlpFew{h, {wd, wd}, {y, nullptr, nullptr}, (int)M, (int)D, (int)F, act}, stream);
    }
    MlpGemm p = gate_up(x, wg, wu, M, D, F);
    p.C[0] = h; p.C[1] = s; p.C[2] = a;
    const int rc = act == GDN_ACT_SILU ? launch_gemm<T, false, false, MLP_GATE + GDN_ACT_SILU>(p, ws, stream) :
                   act == GDN_ACT_SIGMOID ? launch_gemm<T, false, false, MLP_GATE + GDN_ACT_SIGMOID>(p, ws, stream) :
                                            launch_gemm<T, false, false, MLP_GATE + GDN_ACT_GELU_TANH>(p, ws, stream);
    if (rc != GDN_OK) return rc;
    MlpGemm q = down(h, wd, M, D, F);
    q.C[0] = y;
    return launch_gemm<T, false, false, MLP_PLAIN>(q, ws, stream);
}

template <typename T>
static int mlp_bwd(const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* s, const void* a, const void* h,
                   void* dg, void* du, void* dx, void* dwg, void* dwu, void* dwd, Workspace ws, int64_t M, int64_t D, int64_t F, hipStream_t stream) {
    int rc = GDN_OK;
    if (M > 0 && (dx || dwg || dwu)) {
        MlpGemm p = grad_inner(dy, wd, M, D, F);
        p.S = s; p.A = a; p.C[0] = dg; p.C[1] = du;
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

// Matrices of 16-bit elements with other row lengths and counts: zeros where the source has nothing, cut where the destination has less.  A thread for eight
// elements of a row of a destination, at any address.
struct PadSegments { gdn_pad_segment s[GDN_PAD_SEGMENTS]; uint32_t first[GDN_PAD_SEGMENTS + 1]; int n; };
__global__ __launch_bounds__(256) void pad_rows_kernel(PadSegments p) {
    typedef uint16_t Any8 __attribute__((ext_vector_type(8), aligned(2)));
    const uint32_t at = blockIdx.x * 256 + threadIdx.x;
    if (at >= p.first[p.n]) return;
    int i = 0;
    while (i + 1 < p.n && at >= p.first[i + 1]) ++i;
    const gdn_pad_segment& s = p.s[i];
    // (fewer than 2^32 pieces in all, so places count in 32 bits: their division takes a fifth of that in 64)
    const uint32_t pieces = (uint32_t)((s.dst_cols + 7) / 8), r = (at - p.first[i]) / pieces;
    const int64_t row = r, c = (int64_t)(at - p.first[i] - r * pieces) * 8;
    const int64_t have = row < s.src_rows ? s.src_cols - c : 0;
    const uint16_t* from = (const uint16_t*)s.src + row * s.src_cols + c;
    uint16_t* to = (uint16_t*)s.dst + row * s.dst_cols + c;
    Any8 v{};
    if (have >= 8) v = *(const Any8*)from;
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e < have) v[e] = from[e];
    }
    if (c + 8 <= s.dst_cols) *(Any8*)to = v;
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (c + e < s.dst_cols) to[e] = v[e];
    }
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_pad_rows(const gdn_pad_segment* segments, int count, void* stream) {
    const char* who = "gdn_pad_rows";
    GDN_CHECK_ARG(segments && count >= 1 && count <= GDN_PAD_SEGMENTS, GDN_ERR_INVALID, "%s: 1 to %d segments are required", who, GDN_PAD_SEGMENTS);
    PadSegments p{};
    p.n = count;
    int64_t pieces = 0;
    for (int i = 0; i < count; ++i) {
        const gdn_pad_segment& s = segments[i];
        const bool reads = s.src_rows > 0 && s.src_cols > 0, writes = s.dst_rows > 0 && s.dst_cols > 0;
        GDN_CHECK_ARG(s.src_rows >= 0 && s.src_cols >= 0 && s.dst_rows >= 0 && s.dst_cols >= 0 && (!writes || s.dst) && (!writes || !reads || s.src), GDN_ERR_INVALID,
                      "%s: segment %d has no tensor or a negative size", who, i);
        p.s[i] = s;
        pieces += writes ? s.dst_rows * ((s.dst_cols + 7) / 8) : 0;
        GDN_CHECK_ARG(s.dst_rows < (1ll << 32) && s.dst_cols < (1ll << 32) && pieces < (1ll << 32) - 256, GDN_ERR_UNSUPPORTED, "%s: too many elements for one launch", who);
        p.first[i + 1] = (uint32_t)pieces;
    }
    if (pieces == 0) return GDN_OK;
    hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream, p);
    return check_launch("pad_rows_kernel");
}

static int check_mlp(const char* who, int64_t M, int64_t D, int64_t F, int act, int dtype, bool any_width = false) {
    GDN_CHECK_ARG(M >= 0 && D >= 1 && F >= 1, GDN_ERR_INVALID, "%s: bad sizes M=%lld D=%lld F=%lld", who, (long long)M, (long long)D, (long long)F);
    GDN_CHECK_ARG(dtype == GDN_DTYPE_BF16 || dtype == GDN_DTYPE_F16, GDN_ERR_UNSUPPORTED, "%s: bf16 or f16 only", who);
    GDN_CHECK_ARG(act == GDN_ACT_SILU || act == GDN_ACT_SIGMOID || act == GDN_ACT_GELU_TANH, GDN_ERR_UNSUPPORTED, "%s: unknown activation", who);
    GDN_CHECK_ARG(any_width || (D % 8 == 0 && F % 8 == 0), GDN_ERR_UNSUPPORTED, "%s: D and F must be multiples of 8 (got %lld, %lld)", who, (long long)D, (long long)F);
    GDN_CHECK_ARG(D <= GDN_MLP_MAX_FEATURES && F <= GDN_MLP_MAX_FEATURES && M < (1ll << 30), GDN_ERR_UNSUPPORTED,
                  "%s: D and F up to %d and fewer than 2^30 rows (got M=%lld D=%lld F=%lld)", who, GDN_MLP_MAX_FEATURES, (long long)M, (long long)D, (long long)F);
    return GDN_OK;
}

extern "C" size_t gdn_gated_mlp_workspace_bytes(int64_t M, int64_t D, int64_t F, int backward) {
    if (check_mlp("gdn_gated_mlp_workspace_bytes", M, D, F, GDN_ACT_SILU, GDN_DTYPE_BF16, !backward && M <= MLP_FEW_ROWS) != GDN_OK || M == 0) return 0;
    auto bytes = [](const MlpGemm& p, int epilogue, bool rows) { return plan_bytes(plan_gemm(p, epilogue, rows)); };
    if (!backward) return M <= MLP_FEW_ROWS ? 0 : std::max(bytes(gate_up(nullptr, nullptr, nullptr, M, D, F), MLP_GATE, true), bytes(down(nullptr, nullptr, M, D, F), MLP_PLAIN, true));
    size_t most = std::max(bytes(grad_inner(nullptr, nullptr, M, D, F), MLP_GRAD, false), bytes(grad_x(nullptr, nullptr, nullptr, nullptr, M, D, F), MLP_PLAIN, false));
    // (which of the weights' gradients will be asked for is not known here: none, one or both of Wg's and Wu's, which are alike, with Wd's or without)
    char some;
    for (int inner = 0; inner < 3; ++inner)
        for (int with_down = inner == 0; with_down < 2; ++with_down)
            most = std::max(most, bytes(grad_weights(nullptr, nullptr, nullptr, nullptr, nullptr, inner > 0 ? &some : nullptr, inner > 1 ? &some : nullptr,
                                                     with_down ? &some : nullptr, M, D, F), MLP_PLAIN, false));
    return most;
}

extern "C" int gdn_gated_mlp_fwd(const void* x, const void* wg, const void* wu, const void* wd, void* y, void* s, void* a, void* h,
                                 void* workspace, size_t workspace_bytes, int64_t M, int64_t D, int64_t F, int activation, int dtype, void* stream) {
    const char* who = "gdn_gated_mlp_fwd";
    const bool few = M <= MLP_FEW_ROWS;
    const int rc = check_mlp(who, M, D, F, activation, dtype, few);
    if (rc != GDN_OK) return rc;
    if (M == 0) return GDN_OK;
    GDN_CHECK_ARG(x && wg && wu && wd && y && h && !s == !a, GDN_ERR_INVALID, "%s: x, the weights, y and h are required, s goes with a", who);
    GDN_CHECK_ARG(few || (((uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu | (uintptr_t)wd | (uintptr_t)y | (uintptr_t)s | (uintptr_t)a | (uintptr_t)h |
                           (uintptr_t)workspace) & 15) == 0, GDN_ERR_INVALID, "%s: tensors and workspace must be 16-byte aligned", who);
    hipStream_t q = (hipStream_t)stream;
    const Workspace ws{workspace, workspace_bytes};
    return dtype == GDN_DTYPE_BF16 ? mlp_fwd<bf16_t>(x, wg, wu, wd, y, s, a, h, ws, M, D, F, activation, q)
                                   : mlp_fwd<f16_t>(x, wg, wu, wd, y, s, a, h, ws, M, D, F, activation, q);
}

extern "C" int gdn_gated_mlp_bwd(const void* dy, const void* x, const void* wg, const void* wu, const void* wd, const void* s, const void* a, const void* h,
                                 void* dg, void* du, void* dx, void* dwg, void* dwu, void* dwd,
                                 void* workspace, size_t workspace_bytes, int64_t M, int64_t D, int64_t F, int dtype, void* stream) {
    const char* who = "gdn_gated_mlp_bwd";
    const int rc = check_mlp(who, M, D, F, GDN_ACT_SILU, dtype);
    if (rc != GDN_OK) return rc;
    const bool inner = dx || dwg || dwu;
    GDN_CHECK_ARG(M == 0 || (dy && (!inner || (wd && s && a && dg && du)) && (!dx || (wg && wu)) && ((!dwg && !dwu) || x) && (!dwd || h)), GDN_ERR_INVALID,
                  "%s: a tensor that the asked gradients need is missing", who);
    GDN_CHECK_ARG((((uintptr_t)dy | (uintptr_t)x | (uintptr_t)wg | (uintptr_t)wu | (uintptr_t)wd | (uintptr_t)s | (uintptr_t)a | (uintptr_t)h | (uintptr_t)dg |
                    (uintptr_t)du | (uintptr_t)dx | (uintptr_t)dwg | (uintptr_t)dwu | (uintptr_t)dwd | (uintptr_t)workspace) & 15) == 0,
                  GDN_ERR_INVALID, "%s: tensors and workspace must be 16-byte aligned", who);
    hipStream_t q = (hipStream_t)stream;
    const Workspace ws{workspace, workspace_bytes};
    return dtype == GDN_DTYPE_BF16 ? mlp_bwd<bf16_t>(dy, x, wg, wu, wd, s, a, h, dg, du, dx, dwg, dwu, dwd, ws, M, D, F, q)
                                   : mlp_bwd<f16_t>(dy, x, wg, wu, wd, s, a, h, dg, du, dx, dwg, dwu, dwd, ws, M, D, F, q);
}
