// Matrix products of 16-bit operands for large row counts: C[m][n] = sum_k A(m, k) B(n, k), fp32 accumulators, with either operand stored with the
// contraction along its rows (A[m][k]) or down its columns (A[k][m]).  What becomes of an accumulator is an epilogue's business.
//
// A workgroup takes a BM x BN tile of C and walks over k in steps of 32.  A step's operands are (BM + BN) * 64 bytes of LDS; GM_STAGES of them are in
// flight or in use: at step t the wave's matrix instructions work on fragments of t in registers, the fragments of t + 1 leave LDS for the other set of
// registers, and the stage that t has just been read from is filled with t + GM_STAGES straight from memory (buffer_load ... lds).  One barrier a step.
// Places past the end of a row, a column or the contraction are requested beyond the buffer's extent and arrive as zeros, so every size
// that is a multiple of 8 along rows runs the same code.
//
// LDS layout (a CU serves 256 bytes a cycle; of a 16-byte read the lanes {0-3, 12-15, 20-27} and {4-11, 16-19, 28-31} of each half wave together, of
// an 8-byte transposing read a half wave):
//   contraction along rows   a row of the tile is 64 bytes, piece c (16 bytes) of row r in slot c ^ (-(r >> 2) & 3)
//   down columns             row k of the stage is 2 BM (BN) bytes, its 32-byte pieces (16 columns) XORed with 3 bits of k
// Neither meets a bank conflict, and both are whole 1 KB runs for the copies.
#pragma once
#include "gdn_chunk_common.h"

namespace gdn {

constexpr int GM_STAGES = 4, GM_K = 32;

// One product of a launch.  A second pair of operands (A1, B1) continues the contraction of the first (segments == 2, K columns each).
struct GemmOperands {
    const void* A[2]; const void* B[2];
    int64_t lda, ldb;                    // elements from row to row
    int M, N, K, segments;
    int tiles_m, tiles_n;
    int first;                           // the launch's tile where this product begins
    int splits;                          // parts of the contraction, a workgroup each
};

typedef uint32_t gm_rsrc __attribute__((ext_vector_type(4)));

// 64 x 16 bytes from a buffer into LDS at lds_off + 16 lane; places at or past `extent` arrive as zeros
__device__ __forceinline__ void buffer_1k_to_lds(uint64_t base, uint32_t extent, uint32_t voff, uint32_t lds_off) {
    gm_rsrc r;
    r[0] = __builtin_amdgcn_readfirstlane((uint32_t)base);
    r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)) & 0xffff;
    r[2] = __builtin_amdgcn_readfirstlane(extent);
    r[3] = 0x00020000;
    lds_off = __builtin_amdgcn_readfirstlane(lds_off);
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds_off), "v"(voff), "s"(r));
}

constexpr uint32_t GM_NOWHERE = 0xffff0000u;
constexpr int64_t GM_EXTENT = 1ll << 31;

// One operand's share in a step: how its tile of ROWS rows (or columns) comes from memory and how its fragments are read.
// DOWN: the contraction runs down the columns of the stored matrix.
template <typename T, int ROWS, bool DOWN>
struct GemmSide {
    static constexpr int BYTES = ROWS * 64, PIECES = BYTES / 1024;
    static constexpr int SLOTS = ROWS / 16;                          // DOWN: 32-byte pieces of a stage's row
    static_assert(!DOWN || SLOTS >= 4, "at least four pieces to a row");
    static __device__ __forceinline__ int flip(int k) {              // DOWN: the XOR of row k's pieces
        return SLOTS >= 8 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1;
    }
    // byte offset of this lane's 16 bytes of piece p from the tile's corner, GM_NOWHERE where the matrix ends before
    static __device__ __forceinline__ uint32_t source(int p, int lane, int64_t ld, int left) {
        if constexpr (!DOWN) {
            const int row = 16 * p + (lane >> 2), c = (lane & 3) ^ (-(lane >> 4) & 3);
            return row < left ? (uint32_t)(row * (int)ld * 2 + 16 * c) : GM_NOWHERE;
        } else {
            constexpr int LANES = 2 * SLOTS;                         // 16-byte pieces of a row
            const int k = (64 / LANES) * p + lane / LANES, s = lane % LANES, c = 2 * ((s >> 1) ^ flip(k)) + (s & 1);
            return 8 * c < left ? (uint32_t)(k * (int)ld * 2 + 16 * c) : GM_NOWHERE;
        }
    }
    // this lane's share of the place of a fragment, and the fragment of the 16 rows (columns) 16 i ..
    static __device__ __forceinline__ uint32_t share(int lane) {
        const int c16 = lane & 15, g = lane >> 4;
        if constexpr (!DOWN) return (uint32_t)(c16 * 64 + 16 * (g ^ (-(c16 >> 2) & 3)));
        else {
            const int k = 8 * g + (c16 >> 2);                        // (and k + 4: the same XOR)
            return (uint32_t)(k * 2 * ROWS + 32 * flip(k) + 8 * (c16 & 3));
        }
    }
    static __device__ __forceinline__ typename Mma<T>::V8 fragment(const char* stage, uint32_t share, int i) {
        typedef typename Mma<T>::V8 V8;
        if constexpr (!DOWN) return *(const V8*)(stage + share + 1024 * i);
        else {
            const char* at = stage + (share ^ (uint32_t)(32 * i));
            return join<V8>(Mma<T>::tr_read((const T*)at), Mma<T>::tr_read((const T*)(at + 8 * ROWS)));
        }
    }
};

// The workgroup's tile of C.  DUAL: the tile's first BN / 2 columns come from B[0], the others from B[1] at the same columns (two products of the same A,
// side by side in every wave); else B[1] is the second segment's.
template <typename T, int BM, int BN, int WM, int WN, bool A_DOWN, bool B_DOWN, bool DUAL>
struct Gemm {
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, MT = BM / WM / 16, NT = BN / WN / 16;
    static constexpr int STAGE = (BM + BN) * 64, LDS = GM_STAGES * STAGE;
    static constexpr int COLUMNS = DUAL ? BN / 2 : BN;               // columns of C (of each product)
    typedef GemmSide<T, BM, A_DOWN> SideA;
    typedef GemmSide<T, BN, B_DOWN> SideB;
    static constexpr int PA = SideA::PIECES / WAVES, PB = SideB::PIECES / WAVES;
    static_assert(SideA::PIECES % WAVES == 0 && SideB::PIECES % WAVES == 0 && !(DUAL && B_DOWN), "whole pieces to every wave");
    static_assert(!DUAL || NT % 2 == 0, "both products in every wave");
    typedef typename Mma<T>::V8 V8;

    // the column (of C, in the tile) of a wave's fragment j, in tiles of 16; DUAL: j and j + NT / 2 are the same column of the two products
    static __device__ __forceinline__ int column_tile(int wn, int j) {
        return DUAL ? (j < NT / 2 ? wn * (NT / 2) + j : BN / 32 + wn * (NT / 2) + j - NT / 2) : wn * NT + j;
    }

    // `part` of p.splits: that share of the contraction's steps
    static __device__ __forceinline__ void run(const GemmOperands& p, int tm, int tn, int part, char* smem, f32x4 (&acc)[NT][MT]) {
        const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wm = w % WM, wn = w / WM;
        const int m0 = tm * BM, n0 = tn * COLUMNS;
        uint32_t va[PA], vb[PB];
#pragma unroll
        for (int i = 0; i < PA; ++i) va[i] = SideA::source(w * PA + i, lane, p.lda, p.M - m0);
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            const int piece = w * PB + i;
            vb[i] = SideB::source(DUAL ? piece % (SideB::PIECES / 2) : piece, lane, p.ldb, p.N - n0);
        }
        const int chunk8 = 8 * ((lane & 3) ^ (-(lane >> 4) & 3));    // where this lane's piece of a row along k begins
        const int steps = max(1, (p.K + GM_K - 1) / GM_K), all = steps * p.segments;      // (no contraction at all: one step on zeros)
        const int begin = (int)((int64_t)all * part / p.splits), total = (int)((int64_t)all * (part + 1) / p.splits) - begin;

        // where the next step's tiles begin, kept in scalar registers: a load of a parameter inside the loop would be waited for with the LDS reads
        struct Walk { uint64_t at, second; uint32_t stride; };
        auto walk = [&](const void* first, const void* second, bool down, int64_t ld, int corner) {
            const int64_t offset = 2 * (down ? (int64_t)corner : corner * ld), stride = 2 * (down ? GM_K * ld : GM_K);
            const bool in_second = begin >= steps;
            return Walk{(uint64_t)(in_second ? second : first) + offset + (uint64_t)stride * (begin - (in_second ? steps : 0)), (uint64_t)second + offset, (uint32_t)stride};
        };
        Walk wa = walk(p.A[0], p.A[1], A_DOWN, p.lda, m0);
        const void* b0 = DUAL ? p.B[w * PB >= SideB::PIECES / 2] : p.B[0];          // (all pieces of a wave are of one product)
        Walk wb = walk(b0, p.B[1], B_DOWN, p.ldb, n0);
        const int K = p.K, lda2 = 2 * (int)p.lda, ldb2 = 2 * (int)p.ldb;
        int asked = 0, left = K - GM_K * (begin % steps), until_second = p.segments == 2 && begin < steps ? steps - begin : -1;
        uint32_t to = 0;
        auto extent = [&](bool down, int ld2, int corner) {
            const uint32_t whole = (uint32_t)GM_EXTENT, rest = (uint32_t)(left * ld2 - 2 * corner);
            return asked >= total || left <= 0 ? 0u : down && left < GM_K ? rest : whole;
        };
        // the copies of one more step: this wave's piece i of PA + PB, and then on to the next step
        uint32_t ea = 0, eb = 0;
        auto request = [&](int i) {
            if (i == 0) { ea = extent(A_DOWN, lda2, m0); eb = extent(B_DOWN, ldb2, n0); }
            if (i < PA) buffer_1k_to_lds(wa.at, ea, !A_DOWN && chunk8 >= left ? GM_NOWHERE : va[i < PA ? i : 0], to + 1024 * (w * PA + i));
            else buffer_1k_to_lds(wb.at, eb, !B_DOWN && chunk8 >= left ? GM_NOWHERE : vb[i < PA ? 0 : i - PA], to + SideA::BYTES + 1024 * (w * PB + i - PA));
            if (i < PA + PB - 1) return;
            ++asked;
            const bool second = asked == until_second;
            wa.at = second ? wa.second : wa.at + wa.stride;
            wb.at = second ? wb.second : wb.at + wb.stride;
            left = second ? K : left - GM_K;
            to = to + STAGE == LDS ? 0 : to + STAGE;
        };
        const uint32_t sa = SideA::share(lane), sb = SideB::share(lane);
        V8 fa[2][MT], fb[2][NT];
        // fragment i of NT + MT of step t
        auto fetch = [&](int t, int i, V8 (&a)[MT], V8 (&b)[NT]) {
            const char* stage = smem + (t % GM_STAGES) * STAGE;
            if (i < NT) b[i < NT ? i : 0] = SideB::fragment(stage + SideA::BYTES, sb, column_tile(wn, i));
            else a[i < NT ? 0 : i - NT] = SideA::fragment(stage, sa, wm * MT + i - NT);
        };
        // A step's products in MT rounds, each with its share of the fragments of the next step and of the copies in front of its NT products: whatever they take
        // to issue hides behind the products, which one after the other keep the matrix core busy.
        auto step = [&](int t, V8 (&a)[MT], V8 (&b)[NT], V8 (&a1)[MT], V8 (&b1)[NT]) {
            wait_vm_at_most<(GM_STAGES - 2) * (PA + PB)>();          // this wave's share of stage t + 1 is there
            lds_barrier();                                           // ... everyone's is, and everyone has read stage t
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int f = i * (NT + MT) / MT; f < (i + 1) * (NT + MT) / MT; ++f) fetch(t + 1, f, a1, b1);
#pragma unroll
                for (int r = i * (PA + PB) / MT; r < (i + 1) * (PA + PB) / MT; ++r) request(r);
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][i] = Mma<T>::run(b[j], a[i], acc[j][i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < GM_STAGES; ++t)
#pragma unroll
            for (int r = 0; r < PA + PB; ++r) request(r);
        wait_vm_at_most<(GM_STAGES - 1) * (PA + PB)>();
        lds_barrier();
#pragma unroll
        for (int f = 0; f < NT + MT; ++f) fetch(0, f, fa[0], fb[0]);
        // (an odd number of steps: one more on zeros)
        for (int t = 0; t < total; t += 2) {
            step(t, fa[0], fb[0], fa[1], fb[1]);
            step(t + 1, fa[1], fb[1], fa[0], fb[0]);
        }
        wait_vm_at_most<0>();                                        // no copy into LDS outlives the workgroup, or meets the epilogue's use of it
        lds_barrier();
    }
};

// The launch's workgroup `id` of `count` -> a tile of tiles_m x tiles_n.  Workgroups go round the eight XCDs; each XCD gets a run of tiles, walked in
// bands of GM_BAND tiles of rows, so that the tiles at work on it at one time share rows and columns in its L2.
constexpr int GM_BAND = 4;
__device__ __forceinline__ int gemm_tile_of(int id, int count) {
    const int per = count / 8, more = count % 8, x = id % 8;
    return x * per + min(x, more) + id / 8;
}
__device__ __forceinline__ void gemm_place(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int band = tile / (GM_BAND * tiles_n), m0 = band * GM_BAND, rows = min(GM_BAND, tiles_m - m0), in = tile - band * GM_BAND * tiles_n;
    tn = in / rows;
    tm = m0 + in % rows;
}

}  // namespace gdn
