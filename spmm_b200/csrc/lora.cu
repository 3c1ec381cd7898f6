// The C entries of the low-rank adapters (kernels: lora.cuh).
#include "lora.cuh"

namespace tca {

int sm_count();

#define TCA_LORA(k)                                                                         \
    tcaspmm_status lora_forward_##k(const ApplyParams &p, bool tokens, int sms, cudaStream_t st); \
    tcaspmm_status lora_input_grad_##k(const ApplyParams &p, bool in32, int sms, cudaStream_t st); \
    tcaspmm_status lora_factor_grads_##k(const GradParams &w, bool early, int sms, cudaStream_t st);
TCA_LORA(f32)
TCA_LORA(f16)
TCA_LORA(bf16)
#undef TCA_LORA

namespace {

constexpr int64_t MAX_RANK = 256;

tcaspmm_status check(const tcaspmm_adapters *ad, int64_t N, const char *who)
{
    if (!ad) return fail(TCASPMM_ERR_INVALID_ARG, "%s: NULL adapters", who);
    if (!dtype_valid(ad->dt)) return fail(TCASPMM_ERR_INVALID_ARG, "%s: unknown dtype %d", who, (int)ad->dt);
    if (ad->count < 0 || ad->rank < 1 || ad->M < 0 || ad->K < 0 || N < 0)
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: bad sizes count=%lld rank=%lld M=%lld K=%lld N=%lld", who, (long long)ad->count,
                    (long long)ad->rank, (long long)ad->M, (long long)ad->K, (long long)N);
    if (ad->rank > MAX_RANK) return fail(TCASPMM_ERR_UNSUPPORTED, "%s: rank %lld is above %lld", who, (long long)ad->rank, (long long)MAX_RANK);
    if (ad->count > INT_MAX - 65535 || N > INT_MAX - 65535 || ad->M > INT_MAX - 65535 || ad->K > INT_MAX - 65535)
        return fail(TCASPMM_ERR_UNSUPPORTED, "%s: adapters, M, K and N must be below 2^31 - 65535", who);
    if (ad->index && ad->index_bytes != 4 && ad->index_bytes != 8)
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: index_bytes must be 4 or 8, not %d", who, ad->index_bytes);
    if (ad->count > 0 && ((!ad->down && ad->K > 0) || (!ad->up && ad->M > 0)))
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: NULL factor", who);
    const int type = type_code(ad->dt);
    if (!pointer_ok(ad->down, type) || !pointer_ok(ad->up, type) || !pointer_ok(ad->scale, 0) || (uintptr_t)ad->index % (ad->index ? ad->index_bytes : 1))
        return fail(TCASPMM_ERR_INVALID_ARG, "%s: a misaligned factor, index or scale", who);
    return TCASPMM_OK;
}

// Rows of an array start where `bytes`-byte accesses may.
bool aligned(const void *p, int64_t ld, int type, int bytes)
{
    return (uintptr_t)p % bytes == 0 && ld * size_of(type) % bytes == 0;
}

}  // namespace
}  // namespace tca

using namespace tca;

extern "C" size_t tcaspmm_lora_hidden_bytes(int64_t count, int64_t rank, int64_t M, int64_t K, int64_t N, tcaspmm_dtype dt, int keep)
{
    if (rank < 1 || N < 1 || !dtype_valid(dt) || (!keep && by_token(count, rank, M, K, N))) return 0;
    return Hidden::bytes(rank, N, type_code(dt));
}

extern "C" tcaspmm_status tcaspmm_lora(const tcaspmm_adapters *ad, const void *dX, int64_t ldx, int64_t N, const void *dBase,
                                       int64_t ldbase, void *dY, int64_t ldy, tcaspmm_dtype y_dt, void *hidden, int keep, void *stream)
{
    clear_error();
    const tcaspmm_status s = check(ad, N, "lora");
    if (s != TCASPMM_OK) return s;
    if (!dtype_valid(y_dt)) return fail(TCASPMM_ERR_INVALID_ARG, "lora: unknown dtype %d", (int)y_dt);
    const int ft = type_code(ad->dt), yt = type_code(y_dt);
    if (!matrix_ok(dX, ad->K, N, ldx, ft) || !matrix_ok(dY, ad->M, N, ldy, yt) || (dBase && !matrix_ok(dBase, ad->M, N, ldbase, yt)))
        return fail(TCASPMM_ERR_INVALID_ARG, "lora: bad leading dimension ldx=%lld ldbase=%lld ldy=%lld, NULL or misaligned pointer",
                    (long long)ldx, (long long)ldbase, (long long)ldy);
    const int fs = size_of(ft), ys = size_of(yt);
    const Extent Y(dY, ad->M, N, ldy, ys), down(ad->down, ad->count * ad->rank, ad->K, ad->K, fs), up(ad->up, ad->count * ad->M, ad->rank, ad->rank, fs);
    if (overlaps_any(Y, {Extent(dX, ad->K, N, ldx, fs), down, up}) ||
        (!(dBase == dY && ldbase == ldy) && overlap(Y, Extent(dBase, ad->M, N, ldbase, ys))))
        return fail(TCASPMM_ERR_INVALID_ARG, "lora: Y shares memory with an input (it may be base itself, with base's ld)");
    if (N == 0) return TCASPMM_OK;
    const bool tokens = !keep && by_token(ad->count, ad->rank, ad->M, ad->K, N);
    if (!tokens && (!hidden || (uintptr_t)hidden % 16)) return fail(TCASPMM_ERR_INVALID_ARG, "lora: hidden must be a 16-byte aligned device pointer");
    ApplyParams p = {};
    p.F1 = ad->down;
    p.F2 = ad->up;
    p.scale = ad->scale;
    p.c = Columns{ad->index, ad->index_bytes == 8, (int)ad->count};
    p.R = (int)ad->rank;
    p.n1 = ad->K;
    p.n2 = ad->M;
    p.N = N;
    p.In = dX;
    p.ldin = ldx;
    p.base = dBase;
    p.ldbase = ldbase;
    p.basetype = yt;
    p.Out = dY;
    p.ldout = ldy;
    p.outtype = yt;
    p.hidden = hidden;
    p.vec_in = aligned(dX, ldx, ft, 16);
    p.vec_f1 = aligned(ad->down, ad->K, ft, 16);
    p.vec_f2 = aligned(ad->up, ad->rank, ft, 16);
    p.word_in = aligned(dX, ldx, ft, 4);
    p.word_f1 = aligned(ad->down, ad->K, ft, 4);
    p.word_f2 = aligned(ad->up, ad->rank, ft, 4);
    p.vec_base = aligned(dBase, ldbase, yt, 4 * size_of(yt));
    p.vec_out = aligned(dY, ldy, yt, 4 * size_of(yt));
    const auto run = ft == 0 ? lora_forward_f32 : ft == 1 ? lora_forward_f16 : lora_forward_bf16;
    return run(p, tokens, sm_count(), (cudaStream_t)stream);
}

extern "C" tcaspmm_status tcaspmm_lora_backward(const tcaspmm_adapters *ad, const void *dDY, int64_t lddy, tcaspmm_dtype dy_dt,
                                                const void *dX, int64_t ldx, int64_t N, const void *hidden, const float *dBase,
                                                int64_t ldbase, void *dDX, int64_t lddx, void *ddown, void *dup, void *scratch,
                                                void *stream)
{
    clear_error();
    const tcaspmm_status s = check(ad, N, "lora_backward");
    if (s != TCASPMM_OK) return s;
    if (!dtype_valid(dy_dt)) return fail(TCASPMM_ERR_INVALID_ARG, "lora_backward: unknown dtype %d", (int)dy_dt);
    const int ft = type_code(ad->dt), gt = type_code(dy_dt);
    if (gt != 0 && gt != ft) return fail(TCASPMM_ERR_INVALID_ARG, "lora_backward: dY must be fp32 or of the factors' type");
    if (!matrix_ok(dDY, ad->M, N, lddy, gt) || (ddown && !matrix_ok(dX, ad->K, N, ldx, ft)) || (dBase && !matrix_ok(dBase, ad->K, N, ldbase, 0)) ||
        (dDX && !matrix_ok(dDX, ad->K, N, lddx, ft)) || !pointer_ok(ddown, ft) || !pointer_ok(dup, ft))
        return fail(TCASPMM_ERR_INVALID_ARG,
                    "lora_backward: bad leading dimension lddy=%lld ldx=%lld ldbase=%lld lddx=%lld, NULL or misaligned pointer",
                    (long long)lddy, (long long)ldx, (long long)ldbase, (long long)lddx);
    const int fs = size_of(ft);
    const int64_t LR = ad->count * ad->rank;
    const Extent X(ddown ? dX : nullptr, ad->K, N, ldx, fs), DY(dDY, ad->M, N, lddy, size_of(gt)), DX(dDX, ad->K, N, lddx, fs);
    const Extent down(ad->down, LR, ad->K, ad->K, fs), up(ad->up, ad->count * ad->M, ad->rank, ad->rank, fs);
    const Extent base(dBase, ad->K, N, ldbase, 4), gdown(ddown, LR, ad->K, ad->K, fs), gup(dup, ad->count * ad->M, ad->rank, ad->rank, fs);
    const bool in_place = ft == 0 && dBase == dDX && ldbase == lddx;
    if (overlaps_any(DX, {X, DY, down, up, gdown, gup}) || (!in_place && overlap(DX, base)) || overlaps_any(gdown, {X, DY, down, up, base, gup}) ||
        overlaps_any(gup, {X, DY, down, up, base}))
        return fail(TCASPMM_ERR_INVALID_ARG, "lora_backward: an output shares memory with another argument (dX may be an fp32 base itself)");
    if (N > 0 && ((dup && !hidden) || ((dDX || ddown) && !scratch) || (uintptr_t)hidden % 16 || (uintptr_t)scratch % 16))
        return fail(TCASPMM_ERR_INVALID_ARG, "lora_backward: hidden and scratch must be 16-byte aligned device pointers");
    const cudaStream_t st = (cudaStream_t)stream;
    const Columns c{ad->index, ad->index_bytes == 8, (int)ad->count};
    if ((dDX || ddown) && N > 0) {
        ApplyParams p = {};
        p.F1 = ad->up;
        p.F2 = ad->down;
        p.scale = ad->scale;
        p.c = c;
        p.R = (int)ad->rank;
        p.n1 = ad->M;
        p.n2 = ad->K;
        p.N = N;
        p.In = dDY;
        p.ldin = lddy;
        p.base = dBase;
        p.ldbase = ldbase;
        p.Out = dDX;
        p.ldout = lddx;
        p.outtype = ft;
        p.hidden = scratch;
        p.vec_in = aligned(dDY, lddy, gt, 16);
        p.vec_f1 = aligned(ad->up, ad->rank, ft, 16);
        p.vec_f2 = aligned(ad->down, ad->K, ft, 16);
        p.word_in = aligned(dDY, lddy, gt, 4);
        p.word_f1 = aligned(ad->up, ad->rank, ft, 4);
        p.word_f2 = aligned(ad->down, ad->K, ft, 4);
        p.vec_base = aligned(dBase, ldbase, 0, 16);
        p.vec_out = aligned(dDX, lddx, ft, 4 * size_of(ft));
        const auto run = ft == 0 ? lora_input_grad_f32 : ft == 1 ? lora_input_grad_f16 : lora_input_grad_bf16;
        const tcaspmm_status e = run(p, gt == 0, sm_count(), st);
        if (e != TCASPMM_OK) return e;
    }
    GradParams w = {};
    w.c = c;
    w.R = (int)ad->rank;
    w.N = N;
    // The first needs nothing of this call; the second what dX's first kernel has made.
    w.p[0] = GradProblem{dDY, lddy, gt == 0, aligned(dDY, lddy, gt, 16), aligned(dDY, lddy, gt, 4), (const float *)hidden, ad->M, ad->M > 0 ? dup : nullptr, ad->rank, 1, 0};
    w.p[1] = GradProblem{dX, ldx, ft == 0, aligned(dX, ldx, ft, 16), aligned(dX, ldx, ft, 4), (const float *)scratch, ad->K, ad->K > 0 ? ddown : nullptr, 1, ad->K, 0};
    const auto run = ft == 0 ? lora_factor_grads_f32 : ft == 1 ? lora_factor_grads_f16 : lora_factor_grads_bf16;
    return run(w, (dDX || ddown) && N > 0, sm_count(), st);  // early only behind kernels of this call
}
