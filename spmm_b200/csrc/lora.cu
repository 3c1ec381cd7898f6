// Low-rank adapters of many requests beside a sparse product: C (M x N) gets, column by column, the two small factors of
// the column's own adapter.  With a = index[t], D_a (R x K), U_a (M x R) and the scale s_a:
//
//   H[:, t] = s_a D_a X[:, t]        Y[:, t] = base[:, t] + U_a H[:, t]
//   P[:, t] = s_a U_a^T dY[:, t]     dX[:, t] = base[:, t] + D_a^T P[:, t]
//   dD_a = sum_t P[:, t] X[:, t]^T   dU_a = sum_t dY[:, t] H[:, t]^T     (over the columns of adapter a)
//
// A column whose index is not in [0, L) has no adapter: H = P = 0 there and Y = base.
#include <algorithm>
#include <climits>

#include "dense.h"

namespace tca {
namespace {

struct Columns {
    const void *index;  // one per column, or NULL: adapter 0 for all
    int wide;           // 64-bit indices
    int L;
    __device__ int of(long long t) const
    {
        if (!index) return L > 0 ? 0 : -1;
        const long long a = wide ? __ldg((const long long *)index + t) : (long long)__ldg((const int *)index + t);
        return a >= 0 && a < L ? (int)a : -1;
    }
};

// S[r, t] = scale * sum_i F[a][r, i] In[i, t], element (r, i) of adapter a at a * R * n + r * fr + i * fi.
template <typename T>
__global__ void lora_shrink(const T *F, long long fr, long long fi, int R, long long n, const void *In, long long ldin, int intype,
                            Columns c, const float *scale, float *S, long long N)
{
    const long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int r = blockIdx.y;
    if (t >= N) return;
    const int a = c.of(t);
    float v = 0.0f;
    if (a >= 0) {
        const T *f = F + (long long)a * R * n + r * fr;
        for (long long i = 0; i < n; ++i) v += to_float(f[i * fi]) * load_as(In, intype, i * ldin + t);
        if (scale) v *= scale[a];
    }
    S[r * N + t] = v;
}

// Out[j, t] = base[j, t] + sum_r F[a][j, r] S[r, t].
template <typename T>
__global__ void lora_expand(const T *F, long long fj, long long fr, int R, long long n, const float *S, Columns c, const void *base,
                            long long ldbase, int basetype, void *Out, long long ldout, int outtype, long long N)
{
    const long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (t >= N) return;
    const int a = c.of(t);
    for (long long j = blockIdx.y; j < n; j += gridDim.y) {
        float v = 0.0f;
        if (a >= 0) {
            const T *f = F + (long long)a * R * n + j * fj;
            for (int r = 0; r < R; ++r) v += to_float(f[r * fr]) * S[r * N + t];
        }
        store_as(Out, outtype, j * ldout + t, base ? load_as(base, basetype, j * ldbase + t) + v : v);
    }
}

// G[a][j, r] = sum over the columns of adapter a of Z[j, t] S[r, t], stored at a * R * n + j * gj + r * gr.  A warp per element.
template <typename T>
__global__ void lora_grad(const void *Z, long long ldz, int ztype, const float *S, int R, long long n, Columns c, T *G, long long gj,
                          long long gr, long long N)
{
    const long long total = (long long)c.L * n * R;
    for (long long e = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; e < total;
         e += ((long long)gridDim.x * blockDim.x) >> 5) {
        const int a = (int)(e / (n * R));
        const long long j = e / R % n;
        const int r = (int)(e % R);
        float v = 0.0f;
        for (long long t = threadIdx.x & 31; t < N; t += 32)
            if (c.of(t) == a) v += load_as(Z, ztype, j * ldz + t) * S[r * N + t];
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        if ((threadIdx.x & 31) == 0) G[(long long)a * R * n + j * gj + r * gr] = from_float<T>(v);
    }
}

tcaspmm_status launched(const char *what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TCASPMM_OK : cuda_fail(e, what);
}

unsigned grid_y(long long n) { return (unsigned)std::min<long long>(std::max<long long>(n, 1), 65535); }

constexpr int64_t MAX_RANK = 256;

tcaspmm_status check(const tcaspmm_adapters *ad, int64_t N, const char *who)
{
    if (!ad) return fail(TCASPMM_ERR_INVALID_ARG, "%s: NULL adapters", who);
    if (!dtype_valid(ad->dt)) return fail(TCASPMM_ERR_INVALID_ARG, "%s: unknown dtype %d", who, (int)ad->dt);
    if (ad->count < 0 || ad->rank < 1 || ad->M < 0 || ad->K < 0 || N < 0)
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: bad sizes count=%lld rank=%lld M=%lld K=%lld N=%lld", who, (long long)ad->count,
                    (long long)ad->rank, (long long)ad->M, (long long)ad->K, (long long)N);
    if (ad->rank > MAX_RANK) return fail(TCASPMM_ERR_UNSUPPORTED, "%s: rank %lld is above %lld", who, (long long)ad->rank, (long long)MAX_RANK);
    if (ad->count > INT_MAX || N > INT_MAX - 65535 || ad->M > INT_MAX - 65535 || ad->K > INT_MAX - 65535)
        return fail(TCASPMM_ERR_UNSUPPORTED, "%s: adapters, M, K and N must be below 2^31 - 65535", who);
    if (ad->index && ad->index_bytes != 4 && ad->index_bytes != 8)
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: index_bytes must be 4 or 8, not %d", who, ad->index_bytes);
    if (ad->count > 0 && ((!ad->down && ad->K > 0) || (!ad->up && ad->M > 0)))
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: NULL factor", who);
    return TCASPMM_OK;
}

// Out = base + F2 (scale F1 In): the forward pass with (D, U), dX with (U^T, D^T).
template <typename T>
void apply(const tcaspmm_adapters *ad, bool forward, const void *In, int64_t ldin, int intype, float *S, const void *base,
           int64_t ldbase, int basetype, void *Out, int64_t ldout, int outtype, int64_t N, cudaStream_t st)
{
    const Columns c{ad->index, ad->index_bytes == 8, (int)ad->count};
    const long long R = ad->rank, M = ad->M, K = ad->K;
    const dim3 b(128), gs((unsigned)((N + 127) / 128), (unsigned)R);
    if (forward) {
        lora_shrink<T><<<gs, b, 0, st>>>((const T *)ad->down, K, 1, (int)R, K, In, ldin, intype, c, ad->scale, S, N);
        if (Out) lora_expand<T><<<dim3(gs.x, grid_y(M)), b, 0, st>>>((const T *)ad->up, R, 1, (int)R, M, S, c, base, ldbase, basetype, Out, ldout, outtype, N);
    } else {
        lora_shrink<T><<<gs, b, 0, st>>>((const T *)ad->up, 1, R, (int)R, M, In, ldin, intype, c, ad->scale, S, N);
        if (Out) lora_expand<T><<<dim3(gs.x, grid_y(K)), b, 0, st>>>((const T *)ad->down, 1, K, (int)R, K, S, c, base, ldbase, basetype, Out, ldout, outtype, N);
    }
}

}  // namespace
}  // namespace tca

using namespace tca;

extern "C" tcaspmm_status tcaspmm_lora(const tcaspmm_adapters *ad, const void *dX, int64_t ldx, int64_t N, const void *dBase,
                                       int64_t ldbase, void *dY, int64_t ldy, tcaspmm_dtype y_dt, float *dH, void *stream)
{
    clear_error();
    const tcaspmm_status s = check(ad, N, "lora");
    if (s != TCASPMM_OK) return s;
    if (!dtype_valid(y_dt)) return fail(TCASPMM_ERR_INVALID_ARG, "lora: unknown dtype %d", (int)y_dt);
    if (!matrix_ok(dX, ad->K, N, ldx) || !matrix_ok(dY, ad->M, N, ldy) || (dBase && ldbase < N))
        return fail(TCASPMM_ERR_INVALID_ARG, "lora: bad leading dimension ldx=%lld ldbase=%lld ldy=%lld or NULL pointer",
                    (long long)ldx, (long long)ldbase, (long long)ldy);
    if (N == 0) return TCASPMM_OK;
    if (!dH) return fail(TCASPMM_ERR_INVALID_ARG, "lora: NULL dH");
    return with_type(type_code(ad->dt), [&](auto t) {
        apply<decltype(t)>(ad, true, dX, ldx, type_code(ad->dt), dH, dBase, ldbase, type_code(y_dt), dY, ldy, type_code(y_dt), N,
                           (cudaStream_t)stream);
        return launched("lora launch");
    });
}

extern "C" tcaspmm_status tcaspmm_lora_backward(const tcaspmm_adapters *ad, const void *dDY, int64_t lddy, tcaspmm_dtype dy_dt,
                                                const void *dX, int64_t ldx, int64_t N, const float *dH, const float *dBase,
                                                int64_t ldbase, void *dDX, int64_t lddx, void *ddown, void *dup, float *dP,
                                                void *stream)
{
    clear_error();
    const tcaspmm_status s = check(ad, N, "lora_backward");
    if (s != TCASPMM_OK) return s;
    if (!dtype_valid(dy_dt)) return fail(TCASPMM_ERR_INVALID_ARG, "lora_backward: unknown dtype %d", (int)dy_dt);
    if (!matrix_ok(dDY, ad->M, N, lddy) || (ddown && !matrix_ok(dX, ad->K, N, ldx)) || (dBase && ldbase < N) ||
        (dDX && lddx < N) || (dup && !dH && N > 0) || (!dP && N > 0 && (dDX || ddown)))
        return fail(TCASPMM_ERR_INVALID_ARG,
                    "lora_backward: bad leading dimension lddy=%lld ldx=%lld ldbase=%lld lddx=%lld or NULL pointer",
                    (long long)lddy, (long long)ldx, (long long)ldbase, (long long)lddx);
    const cudaStream_t st = (cudaStream_t)stream;
    const Columns c{ad->index, ad->index_bytes == 8, (int)ad->count};
    const long long R = ad->rank;
    return with_type(type_code(ad->dt), [&](auto t) {
        using T = decltype(t);
        if ((dDX || ddown) && N > 0)
            apply<T>(ad, false, dDY, lddy, type_code(dy_dt), dP, dBase, ldbase, 0, dDX, lddx, type_code(ad->dt), N, st);
        const auto blocks = [&](long long n) { return (unsigned)std::min<long long>((c.L * n * R + 7) / 8, 1 << 20); };
        if (ddown && c.L > 0 && ad->K > 0)
            lora_grad<T><<<blocks(ad->K), 256, 0, st>>>(dX, ldx, type_code(ad->dt), dP, (int)R, ad->K, c, (T *)ddown, 1, ad->K, N);
        if (dup && c.L > 0 && ad->M > 0)
            lora_grad<T><<<blocks(ad->M), 256, 0, st>>>(dDY, lddy, type_code(dy_dt), dH, (int)R, ad->M, c, (T *)dup, R, 1, N);
        return launched("lora_backward launch");
    });
}
