// Matrix products of 16-bit operands for large row counts: C[m][n] = sum_k A(m, k) B(n, k), fp32 accumulators, with either operand stored with the
// contraction along its rows (A[m][k]) or down its columns (A[k][m]).  What becomes of an accumulator is an epilogue's business.
//
// A workgroup takes a BM x BN tile of C and walks over k in stages of KS (64; 32 where both operands are read down their columns): (BM + BN) * 2 KS
// bytes of LDS each, filled straight from memory (buffer_load ... lds) into a ring of SLOTS operand shares, A's and B's in turn.  Stages are 64 wide because a
// row's share is then a whole 128-byte line: with stages of 32 every line was asked for twice, in halves, and both projections of 8192 x 4096 x 11008 took 1214 us
// where whole lines took 1178.  Where both operands have the contraction down their columns a stage of 32 asks for whole lines as well, and four of those
// keep requests in flight longer.  The matrix cores work through a stage in halves of 32, each on fragments in registers while those of the next half leave LDS
// for another set of registers: a barrier a stage, after which the stage before is filled again.  Places past the end of a row, a column or the
// contraction are requested beyond the buffer's extent and arrive as zeros, so every size that is a multiple of 8 along rows runs the same code.
//
// With an odd number of slots (five of 32 KB fill the LDS) A's copies go out in one half of a stage, A a half stage earlier, and B's in the other, spread
// over three quarters of it; with four slots both operands' went out together in a quarter of a stage.  8192 x 4096 x 11008, four slots and five: both projections
// 1243 -> 1174 us, down 588 -> 539, dh 694 -> 665, dx 1109 -> 1044 (the down projection's matrix cores busy 66 and 81 % of the cycles).  With four slots and no copies at
// all after the first ones the down projection took 481 us, with all copies from lines that stay in the caches 567 of 606: the copies cost more than the way
// to memory.  Four waves of 128 x 128 results, with a third fewer LDS reads, take the same time, and so do ten slots of 32 for operands down their columns.
//
// LDS layout (a CU serves 256 bytes a cycle; of a 16-byte read the lanes {0-3, 12-15, 20-27} and {4-11, 16-19, 28-31} of each half wave together, of
// an 8-byte transposing read a half wave):
//   contraction along rows   a row of the tile is 128 bytes, piece c (16 bytes) of row r in slot c ^ ((r >> 1) & 7)
//   down columns             row k of the stage is 2 BM (BN) bytes, its 64-byte pieces (32 columns) XORed with k & 3
// Neither meets a bank conflict (counted: none in tiles of 256 x 256), and both are whole 1 KB runs for the copies.
#pragma once
#include "gdn_chunk_common.h"

namespace gdn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
// 32 x 32 results, 16 deep: lane l holds index l % 32 and the contraction indices 8 (l / 32) .. + 7 of either operand; of the result column l % 32 (b's
// index) and, in element 4 q + e, row 8 q + 4 (l / 32) + e (a's index).  Half the operand registers per product of the 16 x 16 form.
__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// One product of a launch.  A second pair of operands (A1, B1) continues the contraction of the first (segments == 2, K columns each).
struct GemmOperands {
    const void* A[2]; const void* B[2];
    int64_t lda, ldb;                    // elements from row to row
    int M, N, K, segments;
    int tiles_m, tiles_n;
    int first;                           // the launch's tile where this product begins
};

typedef uint32_t gm_rsrc __attribute__((ext_vector_type(4)));

// 64 x 16 bytes from a buffer into LDS at slot + place + 16 lane; places at or past `extent` arrive as zeros.  (A load into LDS needs one wait state after the
// scalar write of M0, which the compiler does not see to inside assembly: s_nop, made up for by the addition straight into M0 - 48 rows of 2048 x 5632 29.5 us
// against 31 with the sum made outside, 8192 x 4096 x 11008 with its gradients 5107 and 5129.  M0 is a reserved register: the compiler writes it itself before every use.)
__device__ __forceinline__ void buffer_1k_to_lds(uint64_t base, uint32_t extent, uint32_t voff, uint32_t slot, uint32_t place) {
    gm_rsrc r;
    r[0] = __builtin_amdgcn_readfirstlane((uint32_t)base);
    r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)) & 0xffff;
    r[2] = __builtin_amdgcn_readfirstlane(extent);
    r[3] = 0x00020000;
    slot = __builtin_amdgcn_readfirstlane(slot); place = __builtin_amdgcn_readfirstlane(place);
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" : : "s"(slot), "s"(place), "v"(voff), "s"(r) : "scc");
}

constexpr uint32_t GM_NOWHERE = 0xffff0000u;
constexpr int64_t GM_EXTENT = 1ll << 31;

// One operand's share in a step: how its tile of ROWS rows (or columns) comes from memory and how its fragments are read.
// DOWN: the contraction runs down the columns of the stored matrix.
// SPREAD (the operand whose index becomes the rows of a result): row i of a fragment is row 16 (i >> 4) + 8 ((i >> 2) & 1) + 4 ((i >> 3) & 1) + (i & 3) of its
// 32, so that results 8q .. 8q + 7 of lane l are neighbours, and those of lane l + 32 are the next eight.
template <typename T, int ROWS, int KS, bool DOWN, bool SPREAD>
struct GemmSide {
    static constexpr int BYTES = ROWS * 2 * KS, PIECES = BYTES / 1024;
    static constexpr int SLOTS = ROWS / 16;                          // DOWN: 32-byte pieces of a stage's row
    static_assert(DOWN ? SLOTS >= 8 : KS == 64, "256 bytes to a row of k at least, whole lines of a row along k");
    // !DOWN: where along k this lane's 16 bytes of piece p begin
    static __device__ __forceinline__ int first_k(int p, int lane) { return 8 * ((lane & 7) ^ (4 * (p & 1) + (lane >> 4))); }
    // byte offset of this lane's 16 bytes of piece p from the tile's corner, GM_NOWHERE where the matrix ends before
    static __device__ __forceinline__ uint32_t source(int p, int lane, int64_t ld, int left) {
        if constexpr (!DOWN) {
            const int row = 8 * p + (lane >> 3);
            return row < left ? (uint32_t)(row * (int)ld * 2 + 2 * first_k(p, lane)) : GM_NOWHERE;
        } else {
            constexpr int LANES = 2 * SLOTS;                         // 16-byte pieces of a row
            const int k = (64 / LANES) * p + lane / LANES, s = lane % LANES, c = s ^ (4 * (k & 3));
            return 8 * c < left ? (uint32_t)(k * (int)ld * 2 + 16 * c) : GM_NOWHERE;
        }
    }
    // this lane's share of the place of a fragment, and the fragment of the 32 rows (columns) 32 i .., contraction indices 16 kk ..
    static __device__ __forceinline__ uint32_t share(int lane) {
        if constexpr (!DOWN) {
            const int l = lane & 31, r = SPREAD ? 16 * (l >> 4) + 8 * ((l >> 2) & 1) + 4 * ((l >> 3) & 1) + (l & 3) : l;
            return (uint32_t)(r * 128 + 16 * ((lane >> 5) ^ ((r >> 1) & 7)));
        } else {
            // sixteen lanes read four rows of k, four runs of four columns each; run t of a fragment's eight
            const int k = 8 * (lane >> 5) + ((lane & 15) >> 2), t = 4 * ((lane >> 4) & 1) + (lane & 3), run = SPREAD ? (t & 4) + 2 * (t & 1) + ((t >> 1) & 1) : t;
            return (uint32_t)(k * 2 * ROWS + 64 * (k & 3) + 8 * run);
        }
    }
    static __device__ __forceinline__ typename Mma<T>::V8 fragment(const char* stage, uint32_t share, int i, int kk) {
        typedef typename Mma<T>::V8 V8;
        if constexpr (!DOWN) return *(const V8*)(stage + (share ^ (uint32_t)(32 * kk)) + 4096 * i);
        else {
            const char* at = stage + (share ^ (uint32_t)(64 * i)) + 32 * ROWS * kk;
            return join<V8>(Mma<T>::tr_read((const T*)at), Mma<T>::tr_read((const T*)(at + 8 * ROWS)));      // (k and k + 4: the same XOR)
        }
    }
};

// The workgroup's tile of C.  DUAL: the tile's first BN / 2 columns come from B[0], the others from B[1] at the same columns (two products of the same A,
// side by side in every wave); else B[1] is the second segment's.
template <typename T, int BM, int BN, int WM, int WN, int KS, int SLOTS, bool A_DOWN, bool B_DOWN, bool DUAL>
struct Gemm {
    static constexpr int ROWS = BM, WAVES_M = WM, WAVES = WM * WN, THREADS = 64 * WAVES, MT = BM / WM / 32, NT = BN / WN / 32;
    static constexpr int SLOT = BM * 2 * KS, LDS = SLOTS * SLOT;
    static constexpr bool TURNS = SLOTS % 2 == 1;                    // A's copies in one half of a stage, B's in the other
    static_assert(BM == BN && SLOTS >= 4 && !(TURNS && KS != 64), "a slot holds either operand's share of a stage");
    static constexpr int COLUMNS = DUAL ? BN / 2 : BN;               // columns of C (of each product)
    typedef GemmSide<T, BM, KS, A_DOWN, false> SideA;
    typedef GemmSide<T, BN, KS, B_DOWN, true> SideB;
    static constexpr int PA = SideA::PIECES / WAVES, PB = SideB::PIECES / WAVES;
    static_assert(SideA::PIECES % WAVES == 0 && SideB::PIECES % WAVES == 0 && !(DUAL && B_DOWN), "whole pieces to every wave");
    static_assert(!DUAL || NT % 2 == 0, "both products in every wave");
    typedef typename Mma<T>::V8 V8;

    // the column (of C, in the tile) of a wave's fragment j, in tiles of 32; DUAL: j and j + NT / 2 are the same column of the two products
    static __device__ __forceinline__ int column_tile(int wn, int j) {
        return DUAL ? (j < NT / 2 ? wn * (NT / 2) + j : BN / 64 + wn * (NT / 2) + j - NT / 2) : wn * NT + j;
    }

    // `part` of `parts`: that share of the contraction's stages
    static __device__ __forceinline__ void run(const GemmOperands& p, int tm, int tn, int part, int parts, char* smem, f32x16 (&acc)[NT][MT]) {
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
        const int steps = max(1, (p.K + KS - 1) / KS), all = steps * p.segments;      // (no contraction at all: one step on zeros)
        const int begin = (int)((int64_t)all * part / parts), total = (int)((int64_t)all * (part + 1) / parts) - begin;

        // where the next step's tiles begin, kept in scalar registers: a load of a parameter inside the loop would be waited for with the LDS reads
        struct Walk { uint64_t at, second; uint32_t stride; };
        auto walk = [&](const void* first, const void* second, bool down, int64_t ld, int corner) {
            const int64_t offset = 2 * (down ? (int64_t)corner : corner * ld), stride = 2 * (down ? KS * ld : KS);
            const bool in_second = begin >= steps;
            return Walk{(uint64_t)(in_second ? second : first) + offset + (uint64_t)stride * (begin - (in_second ? steps : 0)), (uint64_t)second + offset, (uint32_t)stride};
        };
        Walk wa = walk(p.A[0], p.A[1], A_DOWN, p.lda, m0);
        const void* b0 = DUAL ? p.B[w * PB >= SideB::PIECES / 2] : p.B[0];          // (all pieces of a wave are of one product)
        Walk wb = walk(b0, p.B[1], B_DOWN, p.ldb, n0);
        const int K = p.K, lda2 = 2 * (int)p.lda, ldb2 = 2 * (int)p.ldb;
        int asked = 0, left = K - KS * (begin % steps), until_second = p.segments == 2 && begin < steps ? steps - begin : -1;
        uint32_t to = 0;
        auto extent = [&](bool down, int ld2, int corner) {
            // (unsigned: `rest` is formed, and not used, where more rows are left than 32 bits of bytes hold)
            const uint32_t whole = (uint32_t)GM_EXTENT, rest = (uint32_t)left * (uint32_t)ld2 - 2u * (uint32_t)corner;
            return asked >= total || left <= 0 ? 0u : down && left < KS ? rest : whole;
        };
        auto next_slot = [](uint32_t at) { return at + SLOT == LDS ? 0u : at + SLOT; };
        auto slot_of_b = [&](uint32_t at) { return TURNS ? next_slot(at) : at + SLOT; };      // (of a stage whose A is at `at`)
        auto next_step = [&](uint32_t at) { return TURNS ? next_slot(next_slot(at)) : at + 2 * SLOT == LDS ? 0u : at + 2 * SLOT; };
        // the copies of one more step: this wave's piece i of PA + PB, and then on to the next step
        uint32_t ea = 0, eb = 0;
        auto request = [&](int i) {
            if (i == 0) { ea = extent(A_DOWN, lda2, m0); eb = extent(B_DOWN, ldb2, n0); }
            if (i < PA) buffer_1k_to_lds(wa.at, ea, !A_DOWN && SideA::first_k(w * PA + i, lane) >= left ? GM_NOWHERE : va[i < PA ? i : 0], to, 1024 * (w * PA + i));
            else buffer_1k_to_lds(wb.at, eb, !B_DOWN && SideB::first_k(w * PB + i - PA, lane) >= left ? GM_NOWHERE : vb[i < PA ? 0 : i - PA], slot_of_b(to), 1024 * (w * PB + i - PA));
            if (i < PA + PB - 1) return;
            ++asked;
            const bool second = asked == until_second;
            wa.at = second ? wa.second : wa.at + wa.stride;
            wb.at = second ? wb.second : wb.at + wb.stride;
            left = second ? K : left - KS;
            to = next_step(to);
        };
        const uint32_t sa = SideA::share(lane), sb = SideB::share(lane);
        struct Fragments { V8 a[2][MT], b[2][NT]; } f0, f1;              // of the two halves of a stage
        constexpr int FRAGMENTS = 2 * (NT + MT), ROUNDS = 2 * MT, COPIES = PA + PB, SPREAD = (ROUNDS * 6 + 7) / 8;      // SPREAD: rounds that the copies of a half are spread over
        // fragment i of a half of the stage at `from`: in the order in which the products ask for them
        auto fetch = [&](uint32_t from, int half, int i, Fragments& f) {
            const int kk = i / (NT + MT), x = i % (NT + MT);
            if (x < NT) f.b[kk][x < NT ? x : 0] = SideB::fragment(smem + slot_of_b(from), sb, column_tile(wn, x), 2 * half + kk);
            else f.a[kk][x < NT ? 0 : x - NT] = SideA::fragment(smem + from, sa, wm * MT + x - NT, 2 * half + kk);
        };
        // The products of half a stage in rounds of NT, each with its share of the next half's fragments in front (and, early on, of the copies): whatever
        // they take to issue hides behind the products, which one after the other keep the matrix core busy.
        auto half = [&](Fragments& now, uint32_t from, int which, Fragments& next, int first, int count) {
#pragma unroll
            for (int i = 0; i < ROUNDS; ++i) {
#pragma unroll
                for (int f = i * FRAGMENTS / ROUNDS; f < (i + 1) * FRAGMENTS / ROUNDS; ++f) fetch(from, which, f, next);
#pragma unroll
                for (int r = min(count, i * count / SPREAD); r < min(count, (i + 1) * count / SPREAD); ++r) request(first + r);
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][i % MT] = mma32(now.b[i / MT][j], now.a[i / MT][i % MT], acc[j][i % MT]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
#pragma unroll
        for (int t = 0; t < SLOTS / 2; ++t)
#pragma unroll
            for (int r = 0; r < COPIES; ++r) request(r);
        wait_vm_at_most<(SLOTS / 2 - 1) * COPIES>();
        lds_barrier();
#pragma unroll
        for (int f = 0; f < FRAGMENTS; ++f) fetch(0, 0, f, f0);
        uint32_t from = 0;
        auto next_stage = [&]() {
            wait_vm_at_most<(SLOTS / 2 - 2) * COPIES + (TURNS ? PA : 0)>();                // this wave's share of the next stage is there
            lds_barrier();                                           // ... everyone's is, and everyone has read this stage
            from = next_step(from);
        };
        if constexpr (KS == 64) {
            for (int s = 0; s < total; ++s) {
                half(f0, from, 1, f1, 0, TURNS ? PA : 0);
                next_stage();
                half(f1, from, 0, f0, TURNS ? PA : 0, TURNS ? PB : COPIES);
            }
        } else {
            // (an odd number of stages: one more, on zeros)
            for (int s = 0; s < total; s += 2) {
                next_stage();
                half(f0, from, 0, f1, 0, COPIES);
                next_stage();
                half(f1, from, 0, f0, 0, COPIES);
            }
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
