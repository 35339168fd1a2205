// Forward of the normalisation with the residual stream (gdn_layer_norm.h).
#include "gdn_layer_norm.h"

namespace gdn {

struct LayerNormParams {
    const void* x; const void* residual; const void* weight; const void* bias;
    void* y; void* stream_out; float* mean; float* rstd;
    int64_t rows; int D;
    float eps;
    int w_dtype;
    bool rms;
};

template <typename T, typename RT, int LANES, int PIECES, bool ALIGNED>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void layer_norm_kernel(LayerNormParams p) {
    typedef NormRow<T, LANES, ALIGNED> R;
    constexpr int VEC = R::VEC;
    __shared__ float red[2][16][2];
    const int l = threadIdx.x % LANES, D = p.D;
    const int64_t step = (int64_t)gridDim.x * R::GROUPS;
    const float inv = 1.f / (float)D;
    constexpr bool KEEP = PIECES <= 3;                                       // longer rows read the parameters (from the caches) for every row
    float w[PIECES][VEC], b[PIECES][VEC];
    auto parameters = [&](int i) {
        R::params(p.weight, p.w_dtype, 1.f, l, i, D, w[i]);
        R::params(p.bias, p.w_dtype, 0.f, l, i, D, b[i]);
    };
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) parameters(i);
    }
    int turn = 0;
    // (a workgroup's rows end together: the barriers of LANES > 64 are met by all of it)
    for (int64_t row = (int64_t)blockIdx.x * R::GROUPS + threadIdx.x / LANES; row < p.rows; row += step) {
        const int64_t base = row * D;
        typename R::template Piece<T> xv[PIECES];
        typename R::template Piece<RT> rv[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) xv[i] = R::load((const T*)p.x + base, l, i, D);
        if (p.residual) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) rv[i] = R::load((const RT*)p.residual + base, l, i, D);
        }
        float v[PIECES][VEC], s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i][e] = (float)xv[i][e];
                if (p.residual) { rv[i][e] = (RT)(v[i][e] + (float)rv[i][e]); v[i][e] = (float)rv[i][e]; }
                else rv[i][e] = (RT)v[i][e];
                s += v[i][e]; q += v[i][e] * v[i][e];
            }
            if (p.stream_out) R::store((RT*)p.stream_out + base, l, i, D, rv[i]);
        }
        R::sum2(s, q, red[turn]);
        turn ^= 1;
        float mean = 0.f;
        if (!p.rms) {
            mean = s * inv;
            q = 0.f;
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e) { const float d = R::column(l, i, e) < D ? v[i][e] - mean : 0.f; q += d * d; }
            R::sum2(s, q, red[turn]);
            turn ^= 1;
        }
        const float rstd = 1.f / sqrtf(q * inv + p.eps);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if constexpr (!KEEP) parameters(i);
            typename R::template Piece<T> y;
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = (T)((v[i][e] - mean) * rstd * w[i][e] + b[i][e]);
            R::store((T*)p.y + base, l, i, D, y);
        }
        if (l == 0) {
            if (p.rstd) p.rstd[row] = rstd;
            if (p.mean) p.mean[row] = mean;
        }
    }
}

}  // namespace gdn

using namespace gdn;

extern "C" int gdn_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias,
                                  void* y, void* stream_out, float* mean, float* rstd, int64_t rows, int64_t D, float eps,
                                  int dtype, int stream_dtype, int w_dtype, int is_rms_norm, void* stream) {
    const char* who = "gdn_layer_norm_fwd";
    const int rc = check_norm(who, rows, D, dtype, w_dtype);
    if (rc != GDN_OK) return rc;
    if (rows == 0) return GDN_OK;
    GDN_CHECK_ARG(x && y && (!residual || stream_out), GDN_ERR_INVALID, "%s: x and y are required, and stream_out with a residual", who);
    LayerNormParams p{x, residual, weight, bias, y, stream_out, is_rms_norm ? nullptr : mean, rstd, rows, (int)D, eps, w_dtype, is_rms_norm != 0};
    const int64_t vec = dtype == GDN_DTYPE_F32 ? 4 : 8;
    const bool aligned = D % vec == 0 && (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)bias | (uintptr_t)y | (uintptr_t)stream_out) & 15) == 0;
    return norm_types(who, dtype, stream_dtype, [&](auto t, auto rt) {
        typedef decltype(t) T;
        typedef decltype(rt) RT;
        return norm_form((D + vec - 1) / vec, aligned, [&](auto lanes, auto pieces, auto al) {
            constexpr int LANES = decltype(lanes)::value, GROUPS = LANES < 256 ? 256 / LANES : 1;
            const int64_t blocks = std::min<int64_t>((rows + GROUPS - 1) / GROUPS, 8192);
            hipLaunchKernelGGL((layer_norm_kernel<T, RT, LANES, decltype(pieces)::value, decltype(al)::value>), dim3((unsigned)blocks), dim3(LANES < 256 ? 256 : LANES), 0,
                               (hipStream_t)stream, p);
            return check_launch("layer_norm_kernel");
        });
    });
}
