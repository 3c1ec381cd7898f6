// torch operators over the C entries of the dense operators: tcaspmm::layer_norm and tcaspmm::lora with their gradients.
//
// They are C++ so that a call costs the host about as much as one of torch's own operators: through ctypes and Python
// autograd a forward and backward pass of a small layer norm took 219 us of host time, several times its kernels.
#include <c10/cuda/CUDAGuard.h>
#include <ATen/cuda/CUDAContext.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "tcaspmm.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

void check(tcaspmm_status s)
{
    TORCH_CHECK(s == TCASPMM_OK, tcaspmm_status_string(s), ": ", tcaspmm_last_error());
}

bool known(ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

tcaspmm_dtype code(ScalarType t) { return t == at::kHalf ? TCASPMM_F16 : t == at::kBFloat16 ? TCASPMM_BF16 : TCASPMM_F32; }

void check_type(const Tensor &t, const char *name)
{
    TORCH_CHECK_VALUE(known(t.scalar_type()), name, " must be float32, float16 or bfloat16, not ", t.scalar_type());
}

// A matrix argument with contiguous rows (copied if they are not) and its leading dimension.
struct Matrix {
    Tensor t;
    int64_t ld = 0;
    Matrix(const Tensor &m, const char *name) : t(m)
    {
        check_type(m, name);
        TORCH_CHECK_VALUE(m.dim() == 2, name, " must be 2-D, not ", m.dim(), "-D");
        const int64_t rows = m.size(0), cols = m.size(1);
        if ((cols > 1 && m.stride(1) != 1) || (rows > 1 && m.stride(0) < cols)) t = m.contiguous();
        ld = std::max(t.stride(0), cols);
    }
    Matrix() = default;
    void *ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
};

void check_shape(const Tensor &t, const char *name, at::IntArrayRef shape)
{
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", not ", t.sizes());
}

void check_device(const Tensor &X)
{
    TORCH_CHECK_VALUE(X.is_cuda(), "X must be on a CUDA device");
}

void check_with(const Tensor &X, const Tensor &t, const char *name)
{
    TORCH_CHECK_VALUE(!t.defined() || t.device() == X.device(), name, " is on ", t.device(), ", not on ", X.device());
}

Tensor given(const MaybeTensor &t) { return t.has_value() && t->defined() ? *t : Tensor(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// The operators have no forward-mode derivatives; a tangent would be dropped without a word.
void refuse_tangents(const char *name, std::initializer_list<Tensor> inputs)
{
    for (const Tensor &t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), name, " has no forward-mode derivatives");
}

template <typename F>
auto op(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// ------------------------------------------------------------------ layer norm
struct Norm {
    Matrix X;
    Tensor w, b;
    ScalarType pt = at::kFloat;
    int64_t dim, n, vecs;
    Norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, int64_t d)
    {
        TORCH_CHECK_VALUE(d >= -2 && d <= 1, "dim must be 0 (columns) or 1 (rows), not ", d);
        X = Matrix(x, "X");
        dim = d < 0 ? d + 2 : d;
        n = X.t.size(dim);
        vecs = X.t.size(1 - dim);
        TORCH_CHECK_VALUE(n > 0 || vecs == 0, "the normalised dimension is empty");
        w = param(weight, "weight");
        b = param(bias, "bias");
        TORCH_CHECK_VALUE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                          "weight and bias must have one type, not ", w.scalar_type(), " and ", b.scalar_type());
        if (w.defined() || b.defined()) pt = (w.defined() ? w : b).scalar_type();
    }
    Tensor param(const MaybeTensor &p, const char *name) const
    {
        const Tensor t = given(p);
        if (!t.defined()) return t;
        check_type(t, name);
        check_shape(t, name, {n});
        return t.contiguous();
    }
};

std::tuple<Tensor, Tensor, Tensor> norm_call(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps,
                                             int64_t dim, ScalarType out, bool stats)
{
    const Norm a(x, weight, bias, dim);
    TORCH_CHECK_VALUE(known(out), "out_dtype must be float32, float16 or bfloat16, not ", out);
    TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "eps must be finite and not negative, not ", eps);
    check_device(x);
    check_with(x, a.w, "weight");
    check_with(x, a.b, "bias");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    Tensor Y = at::empty({rows, cols}, x.options().dtype(out)), mean, rstd;
    if (stats) {
        mean = at::empty({a.vecs}, x.options().dtype(at::kFloat));
        rstd = at::empty({a.vecs}, x.options().dtype(at::kFloat));
    }
    check(tcaspmm_layer_norm(a.X.ptr(), a.X.ld, code(x.scalar_type()), Y.data_ptr(), cols, code(out), ptr(a.w), ptr(a.b), code(a.pt),
                             stats ? mean.data_ptr<float>() : nullptr, stats ? rstd.data_ptr<float>() : nullptr, rows, cols,
                             (int)a.dim, eps, at::cuda::getCurrentCUDAStream().stream()));
    return {Y, mean, rstd};
}

Tensor layer_norm(const Tensor &X, const MaybeTensor &weight, const MaybeTensor &bias, double eps, int64_t dim, ScalarType out)
{
    return std::get<0>(norm_call(X, weight, bias, eps, dim, out, false));
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_stats(const Tensor &X, const MaybeTensor &weight, const MaybeTensor &bias, double eps,
                                                    int64_t dim, ScalarType out)
{
    return norm_call(X, weight, bias, eps, dim, out, true);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor &dy, const Tensor &x, const Tensor &mean, const Tensor &rstd,
                                                       const MaybeTensor &weight, int64_t dim, ScalarType param_dtype, bool need_input,
                                                       bool need_weight, bool need_bias)
{
    const Norm a(x, weight, std::nullopt, dim);
    const Matrix dY(dy, "dY");
    check_shape(dy, "dY", x.sizes());
    for (const auto &p : {std::make_pair(&mean, "mean"), std::make_pair(&rstd, "rstd")}) {
        check_shape(*p.first, p.second, {a.vecs});
        TORCH_CHECK_VALUE(p.first->scalar_type() == at::kFloat && p.first->is_contiguous(), p.second,
                          " must be the contiguous float32 tensor that layer_norm returned");
    }
    TORCH_CHECK_VALUE(known(param_dtype), "param_dtype must be float32, float16 or bfloat16, not ", param_dtype);
    TORCH_CHECK_VALUE(!a.w.defined() || a.pt == param_dtype, "param_dtype must be weight's type ", a.pt, ", not ", param_dtype);
    check_device(x);
    check_with(x, dy, "dY");
    check_with(x, mean, "mean");
    check_with(x, rstd, "rstd");
    check_with(x, a.w, "weight");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    // What is not needed comes back as an empty tensor.
    Tensor dX = at::empty(need_input ? at::IntArrayRef{rows, cols} : at::IntArrayRef{0}, x.options());
    Tensor dw = at::empty({need_weight ? a.n : 0}, x.options().dtype(param_dtype));
    Tensor db = at::empty({need_bias ? a.n : 0}, x.options().dtype(param_dtype));
    const size_t size = need_weight || need_bias ? tcaspmm_layer_norm_backward_workspace(rows, cols, (int)a.dim) : 0;
    Tensor ws;
    if (size) ws = at::empty({(int64_t)size}, x.options().dtype(at::kByte));
    check(tcaspmm_layer_norm_backward(dY.ptr(), dY.ld, code(dy.scalar_type()), a.X.ptr(), a.X.ld, code(x.scalar_type()),
                                      mean.data_ptr<float>(), rstd.data_ptr<float>(), ptr(a.w), code(param_dtype),
                                      need_input ? dX.data_ptr() : nullptr, cols, need_weight ? dw.data_ptr() : nullptr,
                                      need_bias ? db.data_ptr() : nullptr, rows, cols, (int)a.dim, ptr(ws), size,
                                      at::cuda::getCurrentCUDAStream().stream()));
    return {dX, dw, db};
}

using NormOp = Tensor(const Tensor &, const MaybeTensor &, const MaybeTensor &, double, int64_t, ScalarType);
using NormStatsOp = std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const MaybeTensor &, const MaybeTensor &, double, int64_t,
                                                       ScalarType);
using NormGradOp = std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                      const MaybeTensor &, int64_t, ScalarType, bool, bool, bool);

struct NormFunction : torch::autograd::Function<NormFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &X, const MaybeTensor &weight, const MaybeTensor &bias, double eps,
                          int64_t dim, ScalarType out)
    {
        static const auto run = op<NormStatsOp>("tcaspmm::layer_norm_stats");
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto [Y, mean, rstd] = run.call(X, weight, bias, eps, dim, out);
        const Tensor w = given(weight), b = given(bias);
        ctx->save_for_backward({X, w, mean, rstd});
        ctx->saved_data["dim"] = dim;
        ctx->saved_data["bias"] = b.defined();
        ctx->saved_data["param"] = (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat);
        ctx->set_materialize_grads(false);
        return Y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        static const auto run = op<NormGradOp>("tcaspmm::layer_norm_backward");
        const auto saved = ctx->get_saved_variables();
        // needs_input_grad counts the tensors that were given.
        const bool has_w = saved[1].defined(), has_b = ctx->saved_data["bias"].toBool();
        const bool need[3] = {ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1), has_b && ctx->needs_input_grad(1 + has_w)};
        const auto [dX, dw, db] =
            run.call(grads[0], saved[0], saved[2], saved[3], saved[1].defined() ? MaybeTensor(saved[1]) : std::nullopt,
                     ctx->saved_data["dim"].toInt(), (ScalarType)ctx->saved_data["param"].toInt(), need[0], need[1], need[2]);
        if (need[0]) out[0] = dX;
        if (need[1]) out[1] = dw;
        if (need[2]) out[2] = db;
        return out;
    }
};

Tensor layer_norm_autograd(const Tensor &X, const MaybeTensor &weight, const MaybeTensor &bias, double eps, int64_t dim, ScalarType out)
{
    refuse_tangents("layer_norm", {X, given(weight), given(bias)});
    if (at::GradMode::is_enabled() && (wants_grad(X) || wants_grad(given(weight)) || wants_grad(given(bias))))
        return NormFunction::apply(X, weight, bias, eps, dim, out);
    static const auto run = op<NormOp>("tcaspmm::layer_norm");
    const at::AutoDispatchBelowADInplaceOrView below;
    return run.call(X, weight, bias, eps, dim, out);
}

// ------------------------------------------------------------------ low-rank adapters
struct Adapters {
    Matrix X;
    Tensor down, up, index, scale;
    tcaspmm_adapters c = {};
    int64_t K, N, M, R, L;
    Adapters(const Tensor &x, const Tensor &d, const Tensor &u, const MaybeTensor &idx, const MaybeTensor &s)
        : X(x, "X"), index(given(idx)), scale(given(s))
    {
        K = x.size(0);
        N = x.size(1);
        for (const auto &f : {std::make_pair(&d, "down"), std::make_pair(&u, "up")}) {
            TORCH_CHECK_VALUE(f.first->dim() == 3, f.second, " must be 3-D (adapters first), not ", f.first->dim(), "-D");
            TORCH_CHECK_VALUE(f.first->scalar_type() == x.scalar_type(), f.second, " must have X's type ", x.scalar_type(), ", not ",
                              f.first->scalar_type());
        }
        L = d.size(0);
        R = d.size(1);
        M = u.size(1);
        check_shape(d, "down", {L, R, K});
        check_shape(u, "up", {L, M, R});
        TORCH_CHECK_VALUE(R >= 1 && R <= 256, "the rank must be between 1 and 256, not ", R);
        down = d.contiguous();
        up = u.contiguous();
        if (index.defined()) {
            check_shape(index, "index", {N});
            TORCH_CHECK_VALUE(index.scalar_type() == at::kInt || index.scalar_type() == at::kLong, "index must be int32 or int64, not ",
                              index.scalar_type());
            index = index.contiguous();
        }
        if (scale.defined()) {
            check_shape(scale, "scale", {L});
            TORCH_CHECK_VALUE(scale.scalar_type() == at::kFloat, "scale must be float32, not ", scale.scalar_type());
            scale = scale.contiguous();
        }
    }
    const tcaspmm_adapters *args()
    {
        c.down = down.data_ptr();
        c.up = up.data_ptr();
        c.index = ptr(index);
        c.scale = (const float *)ptr(scale);
        c.count = L;
        c.rank = R;
        c.M = M;
        c.K = K;
        c.dt = code(X.t.scalar_type());
        c.index_bytes = index.defined() && index.scalar_type() == at::kLong ? 8 : 4;
        return &c;
    }
    void check_devices(const Tensor &x) const
    {
        check_device(x);
        check_with(x, down, "down");
        check_with(x, up, "up");
        check_with(x, index, "index");
        check_with(x, scale, "scale");
    }
};

int64_t hidden_bytes(const Tensor &x, int64_t L, int64_t R, int64_t M, bool keep)
{
    return (int64_t)tcaspmm_lora_hidden_bytes(L, R, M, x.size(0), x.size(1), code(x.scalar_type()), keep);
}

Tensor hidden_buffer(const Tensor &x, int64_t L, int64_t R, int64_t M, bool keep)
{
    const int64_t size = hidden_bytes(x, L, R, M, keep);
    return size || keep ? at::empty({size}, x.options().dtype(at::kByte)) : Tensor();
}

// H: where the caller wants what the backward pass reads, or null.
Tensor lora_call(const Tensor &x, const Tensor &down, const Tensor &up, const MaybeTensor &index, const MaybeTensor &scale,
                 const MaybeTensor &base_, const Tensor *out, Tensor *H)
{
    Adapters a(x, down, up, index, scale);
    const Tensor b = given(base_);
    Matrix base, Y;
    ScalarType type = at::kFloat;
    if (b.defined()) {
        base = Matrix(b, "base");
        check_shape(b, "base", {a.M, a.N});
        type = b.scalar_type();
    }
    if (out) {
        Y = Matrix(*out, "out");
        check_shape(*out, "out", {a.M, a.N});
        TORCH_CHECK_VALUE(Y.t.is_same(*out), "out must have contiguous rows");
        TORCH_CHECK_VALUE(!b.defined() || out->scalar_type() == type, "out must have base's type ", type, ", not ", out->scalar_type());
        type = out->scalar_type();
    }
    a.check_devices(x);
    check_with(x, b, "base");
    if (out) check_with(x, *out, "out");
    const c10::cuda::CUDAGuard guard(x.device());
    if (!out) Y = Matrix(at::empty({a.M, a.N}, x.options().dtype(type)), "out");
    const Tensor hidden = hidden_buffer(x, a.L, a.R, a.M, H != nullptr);
    check(tcaspmm_lora(a.args(), a.X.ptr(), a.X.ld, a.N, base.ptr(), base.ld, Y.ptr(), Y.ld, code(type), ptr(hidden),
                       H != nullptr, at::cuda::getCurrentCUDAStream().stream()));
    if (H) *H = hidden;
    return Y.t;
}

Tensor lora(const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index, const MaybeTensor &scale,
            const MaybeTensor &base)
{
    return lora_call(X, down, up, index, scale, base, nullptr, nullptr);
}

std::tuple<Tensor, Tensor> lora_hidden(const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index,
                                       const MaybeTensor &scale, const MaybeTensor &base)
{
    Tensor H;
    const Tensor Y = lora_call(X, down, up, index, scale, base, nullptr, &H);
    return {Y, H};
}

// Into `out`, which may be base; returns H, or an empty tensor where it is not kept (few columns then go one by one).
Tensor lora_into(const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index, const MaybeTensor &scale,
                 const MaybeTensor &base, const Tensor &out, bool keep)
{
    Tensor H;
    lora_call(X, down, up, index, scale, base, &out, keep ? &H : nullptr);
    return keep ? H : at::empty({0}, X.options().dtype(at::kByte));
}

std::tuple<Tensor, Tensor, Tensor> lora_backward(const Tensor &dy, const Tensor &x, const Tensor &down, const Tensor &up, const Tensor &H,
                                                 const MaybeTensor &index, const MaybeTensor &scale, const MaybeTensor &base_,
                                                 bool need_input, bool need_down, bool need_up)
{
    Adapters a(x, down, up, index, scale);
    const Matrix dY(dy, "dY");
    check_shape(dy, "dY", {a.M, a.N});
    TORCH_CHECK_VALUE(dy.scalar_type() == at::kFloat || dy.scalar_type() == x.scalar_type(), "dY must be float32 or X's type ",
                      x.scalar_type(), ", not ", dy.scalar_type());
    TORCH_CHECK_VALUE(H.scalar_type() == at::kByte && H.dim() == 1 && H.is_contiguous() && H.numel() == hidden_bytes(x, a.L, a.R, a.M, true),
                      "H must be the tensor that lora returned with hidden");
    const Tensor b = given(base_);
    Matrix base;
    if (b.defined()) {
        TORCH_CHECK_VALUE(b.scalar_type() == at::kFloat, "base must be float32, not ", b.scalar_type());
        base = Matrix(b, "base");
        check_shape(b, "base", {a.K, a.N});
    }
    a.check_devices(x);
    check_with(x, dy, "dY");
    check_with(x, H, "H");
    check_with(x, b, "base");
    const c10::cuda::CUDAGuard guard(x.device());
    // What is not needed comes back as an empty tensor.
    Tensor dX = at::empty(need_input ? at::IntArrayRef{a.K, a.N} : at::IntArrayRef{0}, x.options());
    Tensor dD = at::empty(need_down ? a.down.sizes() : at::IntArrayRef{0}, x.options());
    Tensor dU = at::empty(need_up ? a.up.sizes() : at::IntArrayRef{0}, x.options());
    Tensor P;
    if (need_input || need_down) P = hidden_buffer(x, a.L, a.R, a.M, true);
    check(tcaspmm_lora_backward(a.args(), dY.ptr(), dY.ld, code(dy.scalar_type()), a.X.ptr(), a.X.ld, a.N, H.data_ptr(),
                                (const float *)base.ptr(), base.ld, need_input ? dX.data_ptr() : nullptr, a.N,
                                need_down ? dD.data_ptr() : nullptr, need_up ? dU.data_ptr() : nullptr, ptr(P),
                                at::cuda::getCurrentCUDAStream().stream()));
    return {dX, dD, dU};
}

using LoraOp = Tensor(const Tensor &, const Tensor &, const Tensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &);
using LoraHiddenOp = std::tuple<Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const MaybeTensor &,
                                                const MaybeTensor &, const MaybeTensor &);
using LoraIntoOp = Tensor(const Tensor &, const Tensor &, const Tensor &, const MaybeTensor &, const MaybeTensor &, const MaybeTensor &,
                          const Tensor &, bool);
using LoraGradOp = std::tuple<Tensor, Tensor, Tensor>(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const Tensor &,
                                                      const MaybeTensor &, const MaybeTensor &, const MaybeTensor &, bool, bool, bool);

MaybeTensor maybe(const Tensor &t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

struct LoraFunction : torch::autograd::Function<LoraFunction> {
    static Tensor forward(AutogradContext *ctx, const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index,
                          const MaybeTensor &scale, const MaybeTensor &base)
    {
        static const auto run = op<LoraHiddenOp>("tcaspmm::lora_hidden");
        const at::AutoDispatchBelowADInplaceOrView below;
        const auto [Y, H] = run.call(X, down, up, index, scale, base);
        ctx->save_for_backward({X, down, up, given(index), given(scale), H});
        ctx->saved_data["base"] = given(base).defined();
        ctx->set_materialize_grads(false);
        return Y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        variable_list out(6);
        Tensor dY = grads[0];
        if (!dY.defined()) return out;
        const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
        static const auto run = op<LoraGradOp>("tcaspmm::lora_backward");
        const auto v = ctx->get_saved_variables();
        // needs_input_grad counts the tensors that were given.
        if (ctx->saved_data["base"].toBool() && ctx->needs_input_grad(3 + v[3].defined() + v[4].defined())) out[5] = dY;
        if (!need[0] && !need[1] && !need[2]) return out;
        if (dY.scalar_type() != at::kFloat && dY.scalar_type() != v[0].scalar_type()) dY = dY.to(at::kFloat);
        const auto [dX, dD, dU] =
            run.call(dY, v[0], v[1], v[2], v[5], maybe(v[3]), maybe(v[4]), std::nullopt, need[0], need[1], need[2]);
        if (need[0]) out[0] = dX;
        if (need[1]) out[1] = dD;
        if (need[2]) out[2] = dU;
        return out;
    }
};

// `out` gets a new version, so that autograd sees what it saved change.
Tensor lora_into_versioned(const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index, const MaybeTensor &scale,
                           const MaybeTensor &base, const Tensor &out, bool keep)
{
    static const auto run = op<LoraIntoOp>("tcaspmm::lora_into");
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor H = run.call(X, down, up, index, scale, base, out, keep);
    if (!out.is_inference()) torch::autograd::impl::bump_version(out);
    return H;
}

Tensor lora_into_autograd(const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index, const MaybeTensor &scale,
                          const MaybeTensor &base, const Tensor &out, bool keep)
{
    refuse_tangents("lora", {X, down, up, given(scale), given(base), out});
    for (const Tensor &t : {X, down, up, given(scale), given(base), out})  // as torch's own out= forms
        TORCH_CHECK(!at::GradMode::is_enabled() || !wants_grad(t),
                    "lora with out does not support automatic differentiation, but one of the arguments requires grad");
    static const auto run = op<LoraIntoOp>("tcaspmm::lora_into");
    const at::AutoDispatchBelowAutograd below;
    return run.call(X, down, up, index, scale, base, out, keep);
}

Tensor lora_autograd(const Tensor &X, const Tensor &down, const Tensor &up, const MaybeTensor &index, const MaybeTensor &scale,
                     const MaybeTensor &base)
{
    refuse_tangents("lora", {X, down, up, given(scale), given(base)});
    const bool grad = at::GradMode::is_enabled();
    TORCH_CHECK_VALUE(!grad || !wants_grad(given(scale)), "the adapters' scale is a constant: it has no gradient");
    if (grad && (wants_grad(X) || wants_grad(down) || wants_grad(up) || wants_grad(given(base))))
        return LoraFunction::apply(X, down, up, index, scale, base);
    static const auto run = op<LoraOp>("tcaspmm::lora");
    const at::AutoDispatchBelowADInplaceOrView below;
    return run.call(X, down, up, index, scale, base);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tcaspmm, m)
{
    m.def("layer_norm(Tensor X, Tensor? weight, Tensor? bias, float eps, int dim, ScalarType out_dtype) -> Tensor");
    m.def("layer_norm_stats(Tensor X, Tensor? weight, Tensor? bias, float eps, int dim, ScalarType out_dtype) -> "
          "(Tensor, Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor dY, Tensor X, Tensor mean, Tensor rstd, Tensor? weight, int dim, ScalarType param_dtype, "
          "bool need_input, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
    m.def("lora(Tensor X, Tensor down, Tensor up, Tensor? index, Tensor? scale, Tensor? base) -> Tensor");
    m.def("lora_hidden(Tensor X, Tensor down, Tensor up, Tensor? index, Tensor? scale, Tensor? base) -> (Tensor, Tensor)");
    m.def("lora_into(Tensor X, Tensor down, Tensor up, Tensor? index, Tensor? scale, Tensor? base, Tensor(a!) out, "
          "bool keep=True) -> Tensor");
    m.def("lora_backward(Tensor dY, Tensor X, Tensor down, Tensor up, Tensor H, Tensor? index, Tensor? scale, Tensor? base, "
          "bool need_input, bool need_down, bool need_up) -> (Tensor, Tensor, Tensor)");
}

// The CPU entries are the same functions: they check the arguments and refuse the device.
#define TCASPMM_IMPL(key)                              \
    TORCH_LIBRARY_IMPL(tcaspmm, key, m)                \
    {                                                  \
        m.impl("layer_norm", layer_norm);              \
        m.impl("layer_norm_stats", layer_norm_stats);  \
        m.impl("layer_norm_backward", layer_norm_backward); \
        m.impl("lora", lora);                          \
        m.impl("lora_hidden", lora_hidden);            \
        m.impl("lora_into", lora_into);                \
        m.impl("lora_backward", lora_backward);        \
    }
TCASPMM_IMPL(CUDA)
TCASPMM_IMPL(CPU)

TORCH_LIBRARY_IMPL(tcaspmm, Autograd, m)
{
    m.impl("layer_norm", layer_norm_autograd);
    m.impl("lora", lora_autograd);
    // The parts have no derivatives of their own: differentiating through one raises, and out= is refused at once.
    m.impl("layer_norm_stats", torch::autograd::autogradNotImplementedFallback());
    m.impl("layer_norm_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("lora_hidden", torch::autograd::autogradNotImplementedFallback());
    m.impl("lora_backward", torch::autograd::autogradNotImplementedFallback());
    m.impl("lora_into", lora_into_autograd);
}

TORCH_LIBRARY_IMPL(tcaspmm, ADInplaceOrView, m)
{
    m.impl("lora_into", lora_into_versioned);
}
