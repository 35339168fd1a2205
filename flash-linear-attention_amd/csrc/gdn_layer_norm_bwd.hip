// Backward of the normalisation with the residual stream (gdn_layer_norm.h).  A workgroup walks over rows and keeps its share of the
// parameters' gradients in registers; they leave it as one row of partial sums, which gdn_sum_rows adds up in a fixed order.
#include "gdn_layer_norm.h"

namespace gdn {

struct LayerNormBwdParams {
    const void* dy; const void* r; const void* weight; const float* mean; const float* rstd; const void* dstream;
    void* dx; void* dresidual; float* part;      // part [gridDim.x][dw, then db][D]
    int64_t rows; int D;
    int w_dtype;
    bool rms, with_dw, with_db;
};

// Registers: up to 512 lanes a row's pieces and its parameters' sums fit (asked to leave room for a second workgroup of 512 lanes a CU, rows at any address spilled 118 to
// 319 registers: 8192 x 7001 bf16 627 us, 762 with a bias, now 175 and 177).  1024 lanes have 128 registers each.  Two pieces spill a few of them where there is a bias
// or an fp32 stream (8192 x 16384 bf16 none, 195 us, 5.5 TB/s; with a bias 1, 206 us; with a bias and an fp32 stream 54, 590 us, 3.6 TB/s; 167 at
// any address, 8192 x 8203 490 us, 2.2 TB/s), and four pieces 100 to 600.
template <typename T, typename RT, int LANES, int PIECES, bool ALIGNED, bool BIAS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void layer_norm_bwd_kernel(LayerNormBwdParams p) {
    typedef NormRow<T, LANES, ALIGNED> R;
    constexpr int VEC = R::VEC, WIDTH = LANES * PIECES * VEC;
    __shared__ float red[2][16][2];
    extern __shared__ __align__(16) float rows_of_sums[];                    // [GROUPS][WIDTH] where a workgroup takes several rows at a time
    const int l = threadIdx.x % LANES, D = p.D;
    const int64_t step = (int64_t)gridDim.x * R::GROUPS;
    const float inv = 1.f / (float)D;
    constexpr bool KEEP = PIECES <= 3;                                       // longer rows read the weight (from the caches) for every row
    float dw[PIECES][VEC], db[BIAS ? PIECES : 1][VEC], w[PIECES][VEC];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        if constexpr (KEEP) R::params(p.weight, p.w_dtype, 1.f, l, i, D, w[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { dw[i][e] = 0.f; if (BIAS) db[i][e] = 0.f; }
    }
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * R::GROUPS + threadIdx.x / LANES; row < p.rows; row += step) {
        const int64_t base = row * D;
        typename R::template Piece<T> dyv[PIECES];
        typename R::template Piece<RT> rv[PIECES], sv[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) { dyv[i] = R::load((const T*)p.dy + base, l, i, D); rv[i] = R::load((const RT*)p.r + base, l, i, D); }
        if (p.dstream) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) sv[i] = R::load((const RT*)p.dstream + base, l, i, D);
        }
        const float rstd = p.rstd[row], mean = p.rms ? 0.f : p.mean[row];
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if constexpr (!KEEP) R::params(p.weight, p.w_dtype, 1.f, l, i, D, w[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float dy = (float)dyv[i][e], xh = ((float)rv[i][e] - mean) * rstd, g = dy * w[i][e];
                dw[i][e] += dy * xh;
                if (BIAS) db[i][e] += dy;
                c1 += g * xh; c2 += g;                                       // (dy is zero past the end of a row)
            }
            R::forget(dyv[i]); R::forget(rv[i]);
        }
        R::sum2(c1, c2, red[turn]);
        turn ^= 1;
        c1 *= inv; c2 = p.rms ? 0.f : c2 * inv;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if constexpr (!KEEP) R::params(p.weight, p.w_dtype, 1.f, l, i, D, w[i]);
            typename R::template Piece<T> dx;
            typename R::template Piece<RT> dr;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float d = rstd * ((float)dyv[i][e] * w[i][e] - c2 - ((float)rv[i][e] - mean) * rstd * c1);
                if (p.dstream) d += (float)sv[i][e];
                dx[e] = (T)d; dr[e] = (RT)d;
            }
            if (p.dx) R::store((T*)p.dx + base, l, i, D, dx);
            if (p.dresidual) R::store((RT*)p.dresidual + base, l, i, D, dr);
        }
    }
    const int kinds = (int)p.with_dw + (int)p.with_db;
#pragma unroll
    for (int kind = 0; kind < (BIAS ? 2 : 1); ++kind) {
        if (!(kind ? p.with_db : p.with_dw)) continue;                       // (the same for the whole grid)
        float* out = p.part + ((int64_t)blockIdx.x * kinds + (kind && p.with_dw)) * D;
        if constexpr (R::GROUPS == 1) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                typename R::template Piece<float> v;
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = kind ? db[i][e] : dw[i][e];
                R::store(out, l, i, D, v);
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) rows_of_sums[(threadIdx.x / LANES) * WIDTH + R::column(l, i, e)] = kind ? db[i][e] : dw[i][e];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += R::THREADS) {
                float s = 0.f;
#pragma unroll
                for (int r = 0; r < R::GROUPS; ++r) s += rows_of_sums[r * WIDTH + c];
                out[c] = s;
            }
        }
    }
}

}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_layer_norm_bwd_parts(int64_t rows, int64_t D, int dtype) {
    const int64_t pieces = (D * (dtype == GDN_DTYPE_F32 ? 4 : 2) + 15) / 16, at_once = pieces <= 16 ? 16 : pieces <= 128 ? 4 : 1;
    return std::max<int64_t>(1, std::min<int64_t>((rows + at_once - 1) / at_once, 512));
}

extern "C" int gdn_layer_norm_bwd(const void* dy, const void* r, const void* weight, const float* mean, const float* rstd, const void* dstream,
                                  void* dx, void* dresidual, float* part, int64_t rows, int64_t D, int64_t parts, int with_dweight, int with_dbias,
                                  int dtype, int stream_dtype, int w_dtype, int is_rms_norm, void* stream) {
    const char* who = "gdn_layer_norm_bwd";
    const int rc = check_norm(who, rows, D, dtype, w_dtype);
    if (rc != GDN_OK) return rc;
    GDN_CHECK_ARG(parts >= 1 && parts <= 65535, GDN_ERR_INVALID, "%s: parts must be in 1..65535", who);
    GDN_CHECK_ARG(!(with_dweight || with_dbias) || part, GDN_ERR_INVALID, "%s: the parameters' gradients need room for partial sums", who);
    GDN_CHECK_ARG(rows == 0 || (dy && r && rstd && (is_rms_norm || mean)), GDN_ERR_INVALID, "%s: dy, r and the rows' statistics are required", who);
    if (rows == 0 && !with_dweight && !with_dbias) return GDN_OK;
    LayerNormBwdParams p{dy, r, weight, mean, rstd, dstream, dx, dresidual, part, rows, (int)D, w_dtype, is_rms_norm != 0, with_dweight != 0, with_dbias != 0};
    const int64_t vec = dtype == GDN_DTYPE_F32 ? 4 : 8;
    const bool aligned = D % vec == 0 && (((uintptr_t)dy | (uintptr_t)r | (uintptr_t)weight | (uintptr_t)dstream | (uintptr_t)dx | (uintptr_t)dresidual | (uintptr_t)part) & 15) == 0;
    return norm_types(who, dtype, stream_dtype, [&](auto t, auto rt) {
        typedef decltype(t) T;
        typedef decltype(rt) RT;
        return norm_form((D + vec - 1) / vec, aligned, [&](auto lanes, auto pieces, auto al) {
            constexpr int LANES = decltype(lanes)::value, PIECES = decltype(pieces)::value, THREADS = LANES < 256 ? 256 : LANES;
            constexpr size_t sums = LANES < 256 ? (size_t)THREADS * PIECES * (16 / sizeof(T)) * 4 : 0;
            if (with_dbias) hipLaunchKernelGGL((layer_norm_bwd_kernel<T, RT, LANES, PIECES, decltype(al)::value, true>), dim3((unsigned)parts), dim3(THREADS), sums, (hipStream_t)stream, p);
            else hipLaunchKernelGGL((layer_norm_bwd_kernel<T, RT, LANES, PIECES, decltype(al)::value, false>), dim3((unsigned)parts), dim3(THREADS), sums, (hipStream_t)stream, p);
            return check_launch("layer_norm_bwd_kernel");
        });
    });
}
