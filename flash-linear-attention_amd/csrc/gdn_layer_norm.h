// Layer / RMS normalisation of rows of D features with the residual stream added first (fla/modules/layernorm.py): what the forward and the
// backward kernels share.
//
//   r = x (+ residual), rounded to the stream's type RT;  mean = sum r / D (rms norm: 0);  rstd = 1 / sqrt(sum (r - mean)^2 / D + eps)
//   xh = (r - mean) rstd;  y = xh w + b
//   dr = rstd (dy w - xh mean(dy w xh) - [layer norm: mean(dy w)]) + dstream;  dw = sum over rows of dy xh;  db = sum over rows of dy
//
// The stream is a tensor of its own type, and that tensor is normalised, whether it is handed on or not: forward and backward see the same numbers (the
// backward keeps one tensor of the stream's type, not two), y is the same with prenorm and without, and the gradients of the parameters are as exact as their sums.
//
// A few operations an element: bound by memory, every element read and written once.  Measured with the stream handed on: 32768 x 2048 bf16 forward 96 us
// (5.6 TB/s; a copy of 1 GB runs at 5.1), with the backward 207 to 217 us (5.2 to 4.9); 16384 x 4096 bf16 with an fp32 stream, both, 343 to 347 us (4.7).  A row belongs to LANES lanes - part of a wave, a wave, a
// workgroup - each of which holds PIECES pieces of 16 bytes (of x) in registers.
#pragma once
#include "gdn_common.h"
#include <algorithm>
#include <type_traits>

namespace gdn {

template <typename T, int LANES, bool ALIGNED>
struct NormRow {
    static constexpr int VEC = 16 / sizeof(T), THREADS = LANES < 256 ? 256 : LANES, GROUPS = THREADS / LANES;
    // the column of element e of lane l's piece i
    static __device__ __forceinline__ int column(int l, int i, int e) { return (l + LANES * i) * VEC + e; }

    template <typename S> using Piece = S __attribute__((ext_vector_type(VEC)));
    // (in memory, of rows that begin on 16-byte boundaries: eight fp32 values lie on no others, either)
    template <typename S> using WholePiece = S __attribute__((ext_vector_type(VEC), aligned(16)));
    // (rows that do not begin on 16-byte boundaries: the same wide loads and stores at any address, and element by element only where a row ends inside a piece)
    template <typename S> using AnyPiece = S __attribute__((ext_vector_type(VEC), aligned(sizeof(S))));

    template <typename S>
    static __device__ __forceinline__ Piece<S> load(const S* row, int l, int i, int D) {
        const int c = column(l, i, 0);
        Piece<S> v{};
        if constexpr (ALIGNED) {
            if (c < D) v = *(const WholePiece<S>*)(row + c);
        } else if (c + VEC <= D) {
            v = *(const AnyPiece<S>*)(row + c);
        } else if (c < D) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (c + e < D) v[e] = row[c + e];
        }
        return v;
    }
    template <typename S>
    static __device__ __forceinline__ void store(S* row, int l, int i, int D, Piece<S> v) {
        const int c = column(l, i, 0);
        if constexpr (ALIGNED) {
            if (c < D) *(WholePiece<S>*)(row + c) = v;
        } else if (c + VEC <= D) {
            *(AnyPiece<S>*)(row + c) = v;
        } else if (c < D) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (c + e < D) row[c + e] = v[e];
        }
    }
    // weight or bias, of T's type or fp32: `fill` where there is none, zeros past the end of the one there is
    static __device__ __forceinline__ void params(const void* w, int dtype, float fill, int l, int i, int D, float (&out)[VEC]) {
        if (!w) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = fill;
        } else if (dtype == GDN_DTYPE_F32) {
            const Piece<float> v = load((const float*)w, l, i, D);
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = v[e];
        } else {
            const Piece<T> v = load((const T*)w, l, i, D);
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = (float)v[e];
        }
    }
    // The same registers as values that the compiler knows nothing about: what follows is worked out from the pieces again and not kept, widened to fp32, from
    // before a reduction until after it.
    template <typename P> static __device__ __forceinline__ void forget(P& v) {
        if constexpr (sizeof(P) == 16) { u32x4 t = __builtin_bit_cast(u32x4, v); asm("" : "+v"(t)); v = __builtin_bit_cast(P, t); }
        else {
            struct Two { u32x4 a, b; } t = __builtin_bit_cast(Two, v);
            asm("" : "+v"(t.a)); asm("" : "+v"(t.b));
            v = __builtin_bit_cast(P, t);
        }
    }
    // sums over the lanes of a row.  `red`: a place for this sum that the last sum of the same workgroup did not use (LANES > 64)
    static __device__ __forceinline__ void sum2(float& a, float& b, float (*red)[2]) {
#pragma unroll
        for (int m = (LANES < 64 ? LANES : 64) / 2; m >= 1; m >>= 1) { a += __shfl_xor(a, m, 64); b += __shfl_xor(b, m, 64); }
        if constexpr (LANES > 64) {
            if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6][0] = a; red[threadIdx.x >> 6][1] = b; }
            __syncthreads();
            a = 0.f; b = 0.f;
#pragma unroll
            for (int w = 0; w < LANES / 64; ++w) { a += red[w][0]; b += red[w][1]; }
        }
    }
};

// The forms of a row that there are kernels for, by the pieces of 16 bytes in it: f(LANES, PIECES, ALIGNED) as integral constants.  The lanes that a row does not
// fill wait: 8000 x 4097 bf16 (513 pieces) forward and backward 191 us on 512 lanes of two pieces, 143 us on 256 of three.  Rows that begin on 16-byte
// boundaries would run as the others do, too: forward the same, backward 2 % slower (32768 x 2048 bf16 207 -> 211 us).  Element by element, as the others once
// ran, 1929 x 7837 fp32 took 223 us, now 105.
template <int LANES, int PIECES, bool ALIGNED, typename F>
static int norm_form_is(F&& f) {
    return f(std::integral_constant<int, LANES>{}, std::integral_constant<int, PIECES>{}, std::integral_constant<bool, ALIGNED>{});
}
template <bool ALIGNED, typename F>
static int norm_form_of(int64_t pieces, F&& f) {
    if (pieces <= 16) return norm_form_is<16, 1, ALIGNED>(f);
    if (pieces <= 64) return norm_form_is<64, 1, ALIGNED>(f);
    if (pieces <= 128) return norm_form_is<64, 2, ALIGNED>(f);
    if (pieces <= 256) return norm_form_is<256, 1, ALIGNED>(f);
    if (pieces <= 512) return norm_form_is<256, 2, ALIGNED>(f);
    if (pieces <= 768) return norm_form_is<256, 3, ALIGNED>(f);
    if (pieces <= 1024) return norm_form_is<512, 2, ALIGNED>(f);
    if (pieces <= 2048) return norm_form_is<1024, 2, ALIGNED>(f);
    return norm_form_is<1024, 4, ALIGNED>(f);
}
template <typename F>
static int norm_form(int64_t pieces, bool aligned, F&& f) { return aligned ? norm_form_of<true>(pieces, f) : norm_form_of<false>(pieces, f); }

// f(T, RT) as values of the row's and the stream's types
template <typename F>
static int norm_types(const char* who, int dtype, int stream_dtype, F&& f) {
    if (dtype == GDN_DTYPE_BF16 && stream_dtype == GDN_DTYPE_BF16) return f(bf16_t{}, bf16_t{});
    if (dtype == GDN_DTYPE_BF16 && stream_dtype == GDN_DTYPE_F32) return f(bf16_t{}, float{});
    if (dtype == GDN_DTYPE_F16 && stream_dtype == GDN_DTYPE_F16) return f(f16_t{}, f16_t{});
    if (dtype == GDN_DTYPE_F16 && stream_dtype == GDN_DTYPE_F32) return f(f16_t{}, float{});
    if (dtype == GDN_DTYPE_F32 && stream_dtype == GDN_DTYPE_F32) return f(float{}, float{});
    set_error("%s: rows in bf16, f16 or f32, the residual stream in the rows' type or f32", who);
    return GDN_ERR_UNSUPPORTED;
}

inline int check_norm(const char* who, int64_t rows, int64_t D, int dtype, int w_dtype) {
    GDN_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && D >= 1, GDN_ERR_INVALID, "%s: bad sizes rows=%lld D=%lld", who, (long long)rows, (long long)D);
    GDN_CHECK_ARG(D <= GDN_NORM_MAX_ROW_BYTES / (dtype == GDN_DTYPE_F32 ? 4 : 2), GDN_ERR_UNSUPPORTED, "%s: rows of more than 64 KB are not supported (D=%lld)",
                  who, (long long)D);
    GDN_CHECK_ARG(w_dtype == GDN_DTYPE_F32 || w_dtype == dtype, GDN_ERR_UNSUPPORTED, "%s: weight and bias in the rows' type or f32", who);
    return GDN_OK;
}

}  // namespace gdn
