// Layer norm, forward and backward, over the rows' elements (dim 1: a node's features, the layout of a graph product's C)
// or the columns' (dim 0: a token's features, the layout of a pruned weight's B).
//
//   mean = sum x / n    rstd = 1 / sqrt(sum (x - mean)^2 / n + eps)    xh = (x - mean) rstd    y = w xh + b
//   g = w dy            dx = rstd (g - mean(g) - xh mean(g xh))        dw = sum dy xh          db = sum dy
#include <algorithm>
#include <climits>
#include <cmath>

#include "dense.h"

namespace tca {
namespace {

struct NormParams {
    const void *X;
    long long ldx;
    void *Y;
    long long ldy;
    int yt;
    const void *w, *b;  // one per feature, type pt, or NULL
    int pt;
    float *mean, *rstd;  // one per vector, or NULL
    long long vecs, n;   // vectors normalised, their length
    float eps;
};

struct NormGradParams {
    const void *dY;
    long long lddy;
    int dyt;
    const void *X;
    long long ldx;
    const float *mean, *rstd;
    const void *w;
    int pt;
    void *dX;
    long long lddx;
    void *dw, *db;  // type pt (fp32 without a weight), or NULL
    long long vecs, n;
};

// Sum over the block's threads, the same in all of them.  `s` holds a float per warp.
__device__ float block_sum(float v, float *s)
{
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    const int warps = blockDim.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < warps; ++i) t += s[i];
    return t;
}

// One block per vector; element i of vector v lies at v * sv + i * si.
template <typename T>
__global__ void __launch_bounds__(256) norm_fwd(const NormParams p, long long sv, long long si, long long yv, long long yi)
{
    __shared__ float s[8];
    for (long long v = blockIdx.x; v < p.vecs; v += gridDim.x) {
        const T *x = (const T *)p.X + v * sv;
        float a = 0.0f;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) a += to_float(x[i * si]);
        const float mean = block_sum(a, s) / (float)p.n;
        a = 0.0f;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float d = to_float(x[i * si]) - mean;
            a += d * d;
        }
        const float rstd = 1.0f / sqrtf(block_sum(a, s) / (float)p.n + p.eps);
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float xh = (to_float(x[i * si]) - mean) * rstd;
            store_as(p.Y, p.yt, v * yv + i * yi,
                     xh * (p.w ? load_as(p.w, p.pt, i) : 1.0f) + (p.b ? load_as(p.b, p.pt, i) : 0.0f));
        }
        if (threadIdx.x == 0 && p.mean) {
            p.mean[v] = mean;
            p.rstd[v] = rstd;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_bwd(const NormGradParams p, long long sv, long long si, long long gv, long long gi,
                                                long long dv, long long di)
{
    __shared__ float s[8];
    for (long long v = blockIdx.x; v < p.vecs; v += gridDim.x) {
        const T *x = (const T *)p.X + v * sv;
        const float mean = p.mean[v], rstd = p.rstd[v];
        float a = 0.0f, c = 0.0f;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float g = load_as(p.dY, p.dyt, v * gv + i * gi) * (p.w ? load_as(p.w, p.pt, i) : 1.0f);
            a += g;
            c += g * ((to_float(x[i * si]) - mean) * rstd);
        }
        a = block_sum(a, s) / (float)p.n;
        c = block_sum(c, s) / (float)p.n;
        for (long long i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float g = load_as(p.dY, p.dyt, v * gv + i * gi) * (p.w ? load_as(p.w, p.pt, i) : 1.0f);
            const float xh = (to_float(x[i * si]) - mean) * rstd;
            ((T *)p.dX)[v * dv + i * di] = from_float<T>(rstd * (g - a - xh * c));
        }
    }
}

// One block per feature: its weight's and bias's gradients over all vectors.
template <typename T>
__global__ void __launch_bounds__(256) norm_wgrad(const NormGradParams p, long long sv, long long si, long long gv, long long gi)
{
    __shared__ float s[8];
    for (long long i = blockIdx.x; i < p.n; i += gridDim.x) {
        float a = 0.0f, c = 0.0f;
        for (long long v = threadIdx.x; v < p.vecs; v += blockDim.x) {
            const float dy = load_as(p.dY, p.dyt, v * gv + i * gi);
            a += dy * ((to_float(((const T *)p.X)[v * sv + i * si]) - p.mean[v]) * p.rstd[v]);
            c += dy;
        }
        a = block_sum(a, s);
        c = block_sum(c, s);
        if (threadIdx.x == 0) {
            if (p.dw) store_as(p.dw, p.pt, i, a);
            if (p.db) store_as(p.db, p.pt, i, c);
        }
    }
}

unsigned blocks_of(long long n) { return (unsigned)std::min<long long>(n, INT_MAX); }

tcaspmm_status launched(const char *what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TCASPMM_OK : cuda_fail(e, what);
}

}  // namespace
}  // namespace tca

using namespace tca;

extern "C" tcaspmm_status tcaspmm_layer_norm(const void *dX, int64_t ldx, tcaspmm_dtype x_dt, void *dY, int64_t ldy,
                                             tcaspmm_dtype y_dt, const void *weight, const void *bias, tcaspmm_dtype p_dt,
                                             float *mean, float *rstd, int64_t rows, int64_t cols, int dim, double eps,
                                             void *stream)
{
    clear_error();
    if (!dtype_valid(x_dt) || !dtype_valid(y_dt) || !dtype_valid(p_dt))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: unknown dtype");
    if (dim != 0 && dim != 1) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: dim must be 0 or 1, not %d", dim);
    if (rows < 0 || cols < 0 || !matrix_ok(dX, rows, cols, ldx) || !matrix_ok(dY, rows, cols, ldy))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: bad sizes rows=%lld cols=%lld ldx=%lld ldy=%lld or NULL pointer",
                    (long long)rows, (long long)cols, (long long)ldx, (long long)ldy);
    if (!(eps >= 0.0) || std::isinf(eps)) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: eps must be finite and not negative");
    if (!mean != !rstd) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: mean and rstd go together");
    const long long vecs = dim == 1 ? rows : cols, n = dim == 1 ? cols : rows;
    if (vecs == 0) return TCASPMM_OK;
    if (n == 0) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm: the normalised dimension is empty");
    const NormParams p{dX, ldx, dY, ldy, type_code(y_dt), weight, bias, type_code(p_dt), mean, rstd, vecs, n, (float)eps};
    return with_type(type_code(x_dt), [&](auto t) {
        using T = decltype(t);
        norm_fwd<T><<<blocks_of(vecs), 256, 0, (cudaStream_t)stream>>>(p, dim ? ldx : 1, dim ? 1 : ldx, dim ? ldy : 1,
                                                                        dim ? 1 : ldy);
        return launched("layer_norm launch");
    });
}

extern "C" size_t tcaspmm_layer_norm_backward_workspace(int64_t rows, int64_t cols, int dim)
{
    (void)rows;
    (void)cols;
    (void)dim;
    return 0;
}

extern "C" tcaspmm_status tcaspmm_layer_norm_backward(const void *dDY, int64_t lddy, tcaspmm_dtype dy_dt, const void *dX,
                                                      int64_t ldx, tcaspmm_dtype x_dt, const float *mean, const float *rstd,
                                                      const void *weight, tcaspmm_dtype p_dt, void *dDX, int64_t lddx,
                                                      void *dweight, void *dbias, int64_t rows, int64_t cols, int dim,
                                                      void *workspace, size_t workspace_bytes, void *stream)
{
    clear_error();
    if (!dtype_valid(x_dt) || !dtype_valid(dy_dt) || !dtype_valid(p_dt))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: unknown dtype");
    if (dim != 0 && dim != 1) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: dim must be 0 or 1, not %d", dim);
    if (rows < 0 || cols < 0 || !matrix_ok(dX, rows, cols, ldx) || !matrix_ok(dDY, rows, cols, lddy) ||
        (dDX && lddx < cols))
        return fail(TCASPMM_ERR_INVALID_ARG,
                    "layer_norm_backward: bad sizes rows=%lld cols=%lld ldx=%lld lddy=%lld lddx=%lld or NULL pointer",
                    (long long)rows, (long long)cols, (long long)ldx, (long long)lddy, (long long)lddx);
    const long long vecs = dim == 1 ? rows : cols, n = dim == 1 ? cols : rows;
    if (n == 0) return vecs == 0 ? TCASPMM_OK : fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: the normalised dimension is empty");
    if (vecs > 0 && (!mean || !rstd)) return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: mean and rstd are needed");
    if (workspace_bytes < tcaspmm_layer_norm_backward_workspace(rows, cols, dim))
        return fail(TCASPMM_ERR_INVALID_ARG, "layer_norm_backward: workspace of %zu bytes is too small", workspace_bytes);
    (void)workspace;
    const NormGradParams p{dDY, lddy, type_code(dy_dt), dX, ldx, mean, rstd, weight, type_code(p_dt), dDX, lddx, dweight, dbias,
                           vecs, n};
    const cudaStream_t st = (cudaStream_t)stream;
    const long long sv = dim ? ldx : 1, si = dim ? 1 : ldx, gv = dim ? lddy : 1, gi = dim ? 1 : lddy;
    return with_type(type_code(x_dt), [&](auto t) {
        using T = decltype(t);
        if (dDX && vecs > 0)
            norm_bwd<T><<<blocks_of(vecs), 256, 0, st>>>(p, sv, si, gv, gi, dim ? lddx : 1, dim ? 1 : lddx);
        if (dweight || dbias) norm_wgrad<T><<<blocks_of(n), 256, 0, st>>>(p, sv, si, gv, gi);
        return launched("layer_norm_backward launch");
    });
}
