"""Layer norm and low-rank adapters around a sparse product against plain 64-bit formulas.

Tolerances are bounds, element by element, from the arithmetic the kernels promise: fp32 sums
whose longest chain of additions is known, one rounding of the result to its type (half a step,
eps / 2), and for 16-bit adapters the stated roundings of the small intermediates.
"""
import ctypes as C

import pytest
import torch

import spmm_b200 as T
from spmm_b200 import dense, torch_op

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24  # half a step of fp32
TINY = 2.0 ** -126


def half_step(y, dt):
    """Half a step of type dt at y, with the fixed step below its normal range."""
    low = {F32: 2.0 ** -126, F16: 2.0 ** -14, BF16: 2.0 ** -126}[dt]
    return torch.finfo(dt).eps / 2 * torch.clamp(y.abs(), min=low)


def close(got, ref, tol):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at]} for {ref[at]} "
                             f"(tolerance {tol[at]})")


# ------------------------------------------------------------------ layer norm
def chain(n):
    """Additions on the longest path of a sum of n terms: at least 8 threads share a vector's terms (a warp a row's,
    8 a column's), then 5 levels in a warp, 32 warps and 8 blocks."""
    return n / 8 + 48


def norm_ref(X, w, b, eps, dim, out_dtype):
    """(Y, its tolerance, xhat, xhat's tolerance, rstd), vectors along the last dimension."""
    x = X.double().cpu()
    if dim == 0:
        x = x.T
    n = x.shape[1]
    D = chain(n) * U
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = d * rstd
    e_mean = D * x.abs().mean(1, keepdim=True) + U * mean.abs()
    # (x - m - e)^2 averages to var + e^2; the sum's own rounding is D relative, the root halves it.
    e_rstd = 0.5 * (D + 4 * U) + 0.5 * (e_mean * rstd) ** 2 + 4 * U
    e_xh = (e_mean + U * d.abs()) * rstd * (1 + e_rstd) + xh.abs() * (e_rstd + U)
    w = torch.ones(n, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if b is None else b.detach().double().cpu()
    y = xh * w + b
    tol = w.abs() * e_xh + 2 * U * ((xh * w).abs() + y.abs()) + TINY
    tol = tol + half_step(y.abs() + tol, out_dtype)
    if dim == 0:
        return y.T, tol.T, xh, e_xh, rstd, e_rstd
    return y, tol, xh, e_xh, rstd, e_rstd


def norm_grads_ref(X, w, b, eps, dim, dY, pdt):
    y, _, xh, e_xh, rstd, e_rstd = norm_ref(X, w, b, eps, dim, F32)
    dy = dY.double().cpu()
    if dim == 0:
        dy = dy.T
    v, n = dy.shape
    D = chain(n) * U
    ww = torch.ones(n, dtype=torch.float64) if w is None else w.detach().double().cpu()
    g = dy * ww
    mg, mgx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - mg - xh * mgx)
    e_g = U * g.abs()
    e_mg = (D + 2 * U) * g.abs().mean(1, keepdim=True)
    e_mgx = (D + 3 * U) * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    size = g.abs() + mg.abs() + (xh * mgx).abs()
    tol = rstd * (e_g + e_mg + xh.abs() * e_mgx + e_xh * mgx.abs() + 4 * U * size) * (1 + e_rstd) + e_rstd * dx.abs() + TINY
    tol = tol + half_step(dx.abs() + tol, X.dtype)
    Dv = chain(v) * U
    dw, db = (dy * xh).sum(0), dy.sum(0)
    e_dw = (Dv + 2 * U) * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0) + TINY
    e_db = Dv * dy.abs().sum(0) + TINY
    e_dw = e_dw + half_step(dw.abs() + e_dw, pdt)
    e_db = e_db + half_step(db.abs() + e_db, pdt)
    if dim == 0:
        dx, tol = dx.T, tol.T
    return (dx, tol), (dw, e_dw), (db, e_db)


def norm_inputs(rows, cols, dim, dt, pdt, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = cols if dim == 1 else rows
    X = (torch.randn(rows, cols, generator=g) * 1.5 + 0.7).to(dt).cuda()
    w = (1 + 0.2 * torch.randn(n, generator=g)).to(pdt).cuda()
    b = (0.3 * torch.randn(n, generator=g)).to(pdt).cuda()
    return X, w, b


NORM_SHAPES = [(1, 1), (1, 7), (5, 1), (3, 8), (64, 512), (33, 1000), (7, 5003), (300, 64), (129, 24), (2, 20000), (1000, 31),
               (2049, 17), (513, 264), (4100, 130), (20000, 3), (9, 4096), (3, 12000), (3, 9001), (70001, 5), (6000, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("dt,out,pdt", [(F32, F32, F32), (F16, F16, F32), (BF16, BF16, BF16), (F32, BF16, F32), (BF16, F32, F32),
                                        (F16, F32, F16)])
def test_norm_and_its_gradients(rows, cols, dim, dt, out, pdt):
    X, w, b = norm_inputs(rows, cols, dim, dt, pdt)
    y, tol, *_ = norm_ref(X, w, b, 1e-5, dim, out)
    Y, mean, rstd = T.layer_norm(X, w, b, 1e-5, dim, out, stats=True)
    assert Y.dtype == out and mean.dtype == rstd.dtype == F32
    close(Y, y, tol)
    assert torch.equal(Y, T.layer_norm(X, w, b, 1e-5, dim, out))  # the same without the statistics, and again
    dY = torch.randn(rows, cols, generator=torch.Generator().manual_seed(1)).to(out).cuda()
    got = T.layer_norm_backward(dY, X, mean, rstd, w, dim)
    assert [t.dtype for t in got] == [dt, pdt, pdt]
    for t, (ref, tol) in zip(got, norm_grads_ref(X, w, b, 1e-5, dim, dY, pdt)):
        close(t, ref, tol)
    again = T.layer_norm_backward(dY, X, mean, rstd, w, dim)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
def test_norm_without_parameters_and_partial_gradients(dim):
    X, w, b = norm_inputs(70, 90, dim, F32, F32)
    Y, mean, rstd = T.layer_norm(X, dim=dim, stats=True)
    y, tol, *_ = norm_ref(X, None, None, 1e-5, dim, F32)
    close(Y, y, tol)
    dY = torch.randn(70, 90, generator=torch.Generator().manual_seed(2)).cuda()
    refs = norm_grads_ref(X, None, None, 1e-5, dim, dY, F32)
    for need in [(True, False, False), (False, True, False), (False, False, True), (True, True, True)]:
        got = T.layer_norm_backward(dY, X, mean, rstd, None, dim, need_input=need[0], need_weight=need[1], need_bias=need[2])
        for t, n, (ref, tol) in zip(got, need, refs):
            assert (t is not None) == n
            if n:
                close(t, ref, tol)
    close(T.layer_norm(X, None, b, dim=dim), norm_ref(X, None, b, 1e-5, dim, F32)[0], norm_ref(X, None, b, 1e-5, dim, F32)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("view", ["padded", "offset", "transposed", "expanded"])
def test_norm_of_views(dim, dt, view):
    g = torch.Generator().manual_seed(3)
    big = torch.randn(200, 160, generator=g).to(dt).cuda()
    X = {"padded": big[:100, :96], "offset": big[3:100, 5:102], "transposed": big[:, :50].T,
         "expanded": big[:1, :64].expand(40, 64)}[view]
    dY = (0.5 * big.T[: X.shape[0], : X.shape[1]]) if view != "transposed" else torch.ones((), device="cuda", dtype=dt).expand(X.shape)
    Y, mean, rstd = T.layer_norm(X, dim=dim, stats=True)
    y, tol, *_ = norm_ref(X, None, None, 1e-5, dim, dt)
    close(Y, y, tol)
    got = T.layer_norm_backward(dY, X, mean, rstd, None, dim)
    for t, (ref, tol) in zip(got, norm_grads_ref(X, None, None, 1e-5, dim, dY, F32)):
        close(t, ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
def test_norm_keeps_bad_vectors_apart(dim):
    """A NaN or an infinity spoils its own row (column) and nothing beside it; a constant one gives the bias."""
    X, w, b = norm_inputs(50, 40, dim, F32, F32)
    V = X if dim == 1 else X.T
    V[3, 5] = float("nan")
    V[7, 0] = float("inf")
    V[9] = 2.5
    Y = T.layer_norm(X, w, b, 1e-5, dim)
    Yv = Y if dim == 1 else Y.T
    assert Yv[3].isnan().all() and Yv[7].isnan().all()
    assert torch.equal(Yv[9], b)
    keep = [i for i in range(V.shape[0]) if i not in (3, 7)]
    Xk = V[keep] if dim == 1 else V[keep].T
    y, tol, *_ = norm_ref(Xk, w, b, 1e-5, dim, F32)
    got = Yv[keep] if dim == 1 else Yv[keep].T
    close(got, y, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
def test_norm_of_values_far_from_zero(dim):
    """A mean a thousand times the deviation: the variance is of the differences, not of the squares."""
    X = (1000 + torch.randn(64, 64, generator=torch.Generator().manual_seed(4))).cuda()
    y, tol, *_ = norm_ref(X, None, None, 0.0, dim, F32)
    close(T.layer_norm(X, eps=0.0, dim=dim), y, tol)
    assert float(tol.max()) < 0.05


@pytest.mark.gpu
def test_norm_of_nothing():
    e = T.layer_norm(torch.empty(0, 16, device="cuda"), dim=1)
    assert e.shape == (0, 16)
    X = torch.empty(0, 16, device="cuda")
    _, mean, rstd = T.layer_norm(X, dim=1, stats=True)
    dX, dw, db = T.layer_norm_backward(X, X, mean, rstd, None, 1)
    assert dX.shape == (0, 16) and torch.equal(dw, torch.zeros(16, device="cuda")) and torch.equal(db, torch.zeros(16, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [0, 1])
def test_norm_autograd_matches_differences(dim):
    X, w, b = norm_inputs(12, 10, dim, F32, F32)
    leaves = [t.requires_grad_(True) for t in (X, w, b)]
    dY = torch.randn(12, 10, generator=torch.Generator().manual_seed(5)).cuda()
    Y = torch_op.layer_norm(X, w, b, 1e-3, dim)
    grads = torch.autograd.grad(Y, leaves, dY)

    def f(ts):
        x, ww, bb = (t.detach().double().cpu() for t in ts)
        x = x if dim == 1 else x.T
        m = x.mean(1, keepdim=True)
        y = (x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + 1e-3) * ww + bb
        return float(((y if dim == 1 else y.T) * dY.double().cpu()).sum())

    for k, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(6 + k), dtype=torch.float64)
        h = 1e-4
        ts = [[t.detach().double().cpu() + (s * h * v if j == k else 0) for j, t in enumerate(leaves)] for s in (1, -1)]
        num = (f(ts[0]) - f(ts[1])) / (2 * h)
        ana = float((grads[k].double().cpu() * v).sum())
        # Central difference in 64 bits: h^2 times a third derivative of order 100; the gradient's fp32 rounding.
        assert abs(num - ana) <= 1e-5 * (1 + abs(num)) + 200 * U * float((grads[k].double().cpu() * v).abs().sum())
    for k in range(3):  # one leaf at a time: the same gradient, and none for the others
        one = [t.detach().requires_grad_(j == k) for j, t in enumerate(leaves)]
        torch_op.layer_norm(*one, 1e-3, dim).backward(dY)
        assert [t.grad is not None for t in one] == [j == k for j in range(3)] and torch.equal(one[k].grad, grads[k])
    only_bias = torch_op.layer_norm(X.detach(), None, b, 1e-3, dim)
    assert torch.equal(torch.autograd.grad(only_bias, b, dY)[0], grads[2])
    with pytest.raises(RuntimeError):  # no second derivatives
        dX, = torch.autograd.grad(torch_op.layer_norm(X, w, b, 1e-3, dim), X, dY, create_graph=True)
        dX.sum().backward()


# --------------------------------------------------------- low-rank adapters
def lora_ref(X, down, up, index, scale, base, out_dtype):
    """(Y, tolerance, H)."""
    X, down, up = (t.detach().double().cpu() for t in (X, down, up))
    L, R, K = down.shape
    M, N = up.shape[1], X.shape[1]
    part = 2.0 ** -17 if out_dtype == BF16 else 2.0 ** -21
    idx = torch.zeros(N, dtype=torch.long) if index is None else index.cpu().long()
    Y = torch.zeros(M, N, dtype=torch.float64) if base is None else base.detach().double().cpu().clone()
    tol = U * Y.abs()
    H = torch.zeros(R, N, dtype=torch.float64)
    for a in range(L):
        at = (idx == a).nonzero().flatten()
        if not at.numel():
            continue
        s = 1.0 if scale is None else float(scale[a].double())
        h, ha = s * (down[a] @ X[:, at]), abs(s) * (down[a].abs() @ X[:, at].abs())
        H[:, at] = h
        d, da = up[a] @ h, up[a].abs() @ h.abs()
        Y[:, at] += d
        tol[:, at] += lora_sum_error(K) * (up[a].abs() @ ha) + lora_sum_error(R, part) * da + 2 * U * Y[:, at].abs()
    tol = tol + TINY
    return Y, tol + half_step(Y.abs() + tol, out_dtype), H


def lora_sum_error(n, parts=2.0 ** -21):
    """A sum of n products: the tensor cores may cut (not round) at each of up to n / 4 + 64 partial sums, a full step
    each; an intermediate is held in parts of its type: 22 bits or more of it, 2^-17 where a bf16 result needs no more."""
    return 2 * U * (n / 4 + 64) + parts


def lora_grads_ref(X, down, up, index, scale, dY, base=None):
    dt = X.dtype
    X, down, up, dY = (t.detach().double().cpu() for t in (X, down, up, dY))
    L, R, K = down.shape
    M, N = up.shape[1], X.shape[1]
    # With bf16 factors the fp32 operands of the gradients' products are rounded to TF32 (10 bits after the point), and the
    # intermediate of dX is held in two parts.
    tf, part = (2.0 ** -11, 2.0 ** -17) if dt == BF16 else (0.0, 2.0 ** -21)
    idx = torch.zeros(N, dtype=torch.long) if index is None else index.cpu().long()
    dX = torch.zeros(K, N, dtype=torch.float64) if base is None else base.double().cpu().clone()
    dD, dU = torch.zeros_like(down), torch.zeros_like(up)
    eX, eD, eU = 2 * U * dX.abs(), torch.zeros_like(down), torch.zeros_like(up)
    for a in range(L):
        at = (idx == a).nonzero().flatten()
        if not at.numel():
            continue
        s = 1.0 if scale is None else float(scale[a].double())
        x, g = X[:, at], dY[:, at]
        h, p = s * (down[a] @ x), s * (up[a].T @ g)
        e_h = lora_sum_error(K) * abs(s) * (down[a].abs() @ x.abs())
        e_p = (lora_sum_error(M) + tf) * abs(s) * (up[a].abs().T @ g.abs())
        d = down[a].T @ p
        dX[:, at] += d
        eX[:, at] += down[a].abs().T @ (e_p + lora_sum_error(R, part) * p.abs()) + 2 * U * dX[:, at].abs()
        n = at.numel()
        # The columns of other adapters in between count as zero terms of the sums.
        dD[a] = p @ x.T
        eD[a] = (e_p + (lora_sum_error(N) + tf) * p.abs()) @ x.abs().T
        dU[a] = g @ h.T
        eU[a] = (g.abs() @ e_h.T) + (lora_sum_error(N) + 2 * tf) * (g.abs() @ h.abs().T)
    out = []
    for ref, e in ((dX, eX), (dD, eD), (dU, eU)):
        e = e + TINY
        out.append((ref, e + half_step(ref.abs() + e, dt)))
    return out


def lora_inputs(M, K, N, R, L, dt, ydt=F32, mix="runs", seed=0, index_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(K, N, generator=g).to(dt).cuda()
    down = (torch.randn(L, R, K, generator=g) / max(K, 1) ** 0.5).to(dt).cuda()
    up = (torch.randn(L, M, R, generator=g) / R ** 0.5).to(dt).cuda()
    scale = (0.25 + torch.rand(L, generator=g)).cuda()
    base = torch.randn(M, N, generator=g).to(ydt).cuda()
    if mix == "runs":
        index = torch.sort(torch.randint(-1, L, (N,), generator=g)).values
    elif mix == "each":
        index = torch.randint(-1, L, (N,), generator=g)
    elif mix == "none":
        index = torch.full((N,), -1)
    elif mix == "wild":  # far outside, on both sides
        index = torch.randint(-1, L + 1, (N,), generator=g)
        index[index == L] = 2 ** 31 - 1
        index[index == -1] = -(2 ** 31)
    else:
        index = None
    if index is not None:
        index = index.to(index_dtype).cuda()
    return X, down, up, index, scale, base


LORA_SHAPES = [(1, 1, 1, 1, 1), (5, 3, 2, 1, 2), (64, 64, 1, 16, 4), (100, 72, 33, 8, 3), (257, 515, 70, 12, 5), (512, 256, 300, 16, 2),
               (96, 1000, 64, 64, 3), (130, 96, 200, 128, 2), (48, 40, 90, 200, 2), (1024, 2050, 9, 32, 9), (2048, 520, 130, 5, 3),
               (40, 200, 700, 24, 4), (131, 262, 333, 6, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("mix", ["runs", "each", "one"])
@pytest.mark.parametrize("M,K,N,R,L", LORA_SHAPES)
@pytest.mark.parametrize("dt,ydt", [(F32, F32), (F16, F32), (BF16, F32), (BF16, BF16), (F16, F16), (F32, BF16)])
def test_lora_and_its_gradients(M, K, N, R, L, dt, ydt, mix):
    X, down, up, index, scale, base = lora_inputs(M, K, N, R, L, dt, ydt, mix)
    y, tol, h = lora_ref(X, down, up, index, scale, base, ydt)
    Y, H = T.lora(X, down, up, index, scale, base, hidden=True)
    assert Y.dtype == ydt
    close(Y, y, tol)
    none = (torch.zeros(N) if index is None else index.cpu()) < 0
    assert torch.equal(Y.cpu()[:, none], base.cpu()[:, none])
    assert torch.equal(Y, T.lora(X, down, up, index, scale, base, hidden=True)[0])
    Z = T.lora(X, down, up, index, scale, base)  # nothing kept: few columns go another way
    close(Z, y, tol)
    assert torch.equal(Z.cpu()[:, none], base.cpu()[:, none]) and torch.equal(Z, T.lora(X, down, up, index, scale, base))
    dY = torch.randn(M, N, generator=torch.Generator().manual_seed(7)).to(dt if ydt != F32 else F32).cuda()
    got = T.lora_backward(dY, X, down, up, H, index, scale)
    for t, (ref, tol) in zip(got, lora_grads_ref(X, down, up, index, scale, dY)):
        assert t.dtype == dt
        close(t, ref, tol)
    again = T.lora_backward(dY, X, down, up, H, index, scale)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("mix", ["none", "wild"])
@pytest.mark.parametrize("N", [1, 40, 200])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_lora_columns_without_an_adapter(mix, N, index_dtype):
    X, down, up, index, scale, base = lora_inputs(90, 70, N, 16, 3, BF16, F32, mix, index_dtype=index_dtype)
    if index_dtype == torch.int64 and mix == "wild":
        index[0] = 2 ** 32  # its low half would be adapter 0
    Y, H = T.lora(X, down, up, index, scale, base, hidden=True)
    y, tol, _ = lora_ref(X, down, up, index, scale, base, F32)
    close(Y, y, tol)
    off = ((index < 0) | (index >= 3)).cpu()
    assert torch.equal(Y.cpu()[:, off], base.cpu()[:, off])
    dY = torch.randn(90, N, device="cuda")
    for t, (ref, tol) in zip(T.lora_backward(dY, X, down, up, H, index, scale), lora_grads_ref(X, down, up, index, scale, dY)):
        close(t, ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("N", [6, 80])
def test_lora_keeps_requests_apart(dt, N):
    """Adapters, inputs and gradients that are not finite reach their own columns and gradients, nobody else's."""
    X, down, up, _, scale, base = lora_inputs(60, 80, N, 16, 4, dt)
    index = (torch.arange(N) % 4).int().cuda()
    down[1, 2, 3] = float("nan")
    up[2, 5] = float("inf")
    X[4, 3] = float("nan")  # column 3 belongs to adapter 3
    clean = [t.clone() for t in (X, down, up)]
    clean[0][4, 3], clean[1][1, 2, 3], clean[2][2, 5] = 0, 0, 0
    Y, H = T.lora(X, down, up, index, scale, base, hidden=True)
    Yc, Hc = T.lora(*clean, index, scale, base, hidden=True)
    at = (index.cpu() == 0) | ((index.cpu() == 3) & (torch.arange(N) != 3))
    assert torch.equal(Y[:, at], Yc[:, at]) and Yc.isfinite().all()
    assert Y[:, (index == 1).cpu()].isnan().all() and not Y[5, (index == 2).cpu()].isfinite().any()
    dY = torch.randn(60, N, device="cuda")
    dX, dD, dU = T.lora_backward(dY, X, down, up, H, index, scale)
    cX, cD, cU = T.lora_backward(dY, *clean, Hc, index, scale)
    assert torch.equal(dX[:, at], cX[:, at]) and torch.equal(dD[0], cD[0]) and torch.equal(dU[0], cU[0])
    assert dD[3, :, 4].isnan().all() and torch.equal(dU[2], cU[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_lora_wide_range_intermediate(dt):
    """H above fp16's range and far below it in one column: nothing overflows, small parts keep their bits."""
    M, K, N, R = 32, 64, 40, 8
    X, down, up, _, _, base = lora_inputs(M, K, N, R, 1, dt)
    X[:, 0] *= 200
    scale = torch.tensor([2000.0]).cuda()
    down[0, 1] *= 2.0 ** -6
    y, tol, h = lora_ref(X, down, up, None, scale, base, F32)
    assert float(h.abs().max()) > 65504
    close(T.lora(X, down, up, None, scale, base), y, tol)
    close(T.lora(X, down, up, None, scale, base, hidden=True)[0], y, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("N", [9, 90])
@pytest.mark.parametrize("hidden", [False, True])
def test_lora_of_views_in_place_and_without_base(dt, N, hidden):
    def lora(*args, **kw):
        got = T.lora(*args, hidden=hidden, **kw)
        return got[0] if hidden else got

    X, down, up, index, scale, base = lora_inputs(120, 70, N, 16, 3, dt)
    y, tol, _ = lora_ref(X, down, up, index, scale, base, F32)
    pad = torch.zeros(75, N + 13, device="cuda", dtype=dt)
    pad[2:72, 5:5 + N] = X
    close(lora(pad[2:72, 5:5 + N], down, up, index, scale, base), y, tol)
    close(lora(X.T.contiguous().T, down.transpose(1, 2).contiguous().transpose(1, 2), up, index, scale, base), y, tol)
    out = torch.full((122, N + 7), 7.0, device="cuda")
    view = out[1:121, 3:3 + N]
    assert lora(X, down, up, index, scale, base, out=view) is view
    close(view, y, tol)
    view.fill_(7.0)
    assert torch.equal(out, torch.full_like(out, 7.0))  # nothing beside it was written
    view.copy_(base)
    lora(X, down, up, index, scale, view, out=view)
    close(view, y, tol)
    y0, tol0, _ = lora_ref(X, down, up, index, None, None, F32)
    close(lora(X, down, up, index), y0, tol0)


@pytest.mark.gpu
def test_lora_of_nothing():
    X, down, up, index, scale, base = lora_inputs(20, 30, 8, 4, 2, F32)
    assert torch.equal(T.lora(X, down[:0], up[:0], index, scale[:0], base), base)      # no adapters
    assert torch.equal(T.lora(X, down[:0], up[:0], None, None, base), base)
    assert T.lora(X[:, :0], down, up, index[:0], scale, base[:, :0]).shape == (20, 0)  # no columns
    assert torch.equal(T.lora(X[:0], down[:, :, :0], up, index, scale, base), base)    # no input features
    assert T.lora(X, down, up[:, :0], index, scale, base[:0]).shape == (0, 8)          # no output features
    H = torch.zeros(0, device="cuda", dtype=torch.uint8)
    dX, dD, dU = T.lora_backward(base[:, :0], X[:, :0], down, up, H, index[:0], scale)
    assert dX.shape == (30, 0) and not dD.any() and not dU.any()


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 100])
def test_lora_partial_gradients_and_base(N):
    X, down, up, index, scale, base = lora_inputs(60, 50, N, 8, 3, BF16)
    _, H = T.lora(X, down, up, index, scale, base, hidden=True)
    dY = torch.randn(60, N, device="cuda")
    add = torch.randn(50, N, device="cuda")
    full = T.lora_backward(dY, X, down, up, H, index, scale, add)
    for t, (ref, tol) in zip(full, lora_grads_ref(X, down, up, index, scale, dY, add)):
        close(t, ref, tol)
    for need in [(True, False, False), (False, True, False), (False, False, True)]:
        got = T.lora_backward(dY, X, down, up, H, index, scale, add, need_input=need[0], need_down=need[1], need_up=need[2])
        for t, n, f in zip(got, need, full):
            assert (t is not None) == n and (t is None or torch.equal(t, f))


@pytest.mark.gpu
def test_lora_autograd_matches_differences():
    X, down, up, index, scale, base = lora_inputs(14, 12, 9, 3, 2, F32)
    leaves = [t.requires_grad_(True) for t in (X, down, up, base)]
    dY = torch.randn(14, 9, generator=torch.Generator().manual_seed(8)).cuda()
    grads = torch.autograd.grad(torch_op.lora(X, down, up, index, scale, base), leaves, dY)

    def f(ts):
        return float((lora_ref(ts[0], ts[1], ts[2], index, scale, ts[3], F32)[0] * dY.double().cpu()).sum())

    for k, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(9 + k), dtype=torch.float64)
        h = 1e-3
        ts = [[t.detach().double().cpu() + (s * h * v if j == k else 0) for j, t in enumerate(leaves)] for s in (1, -1)]
        num = (f(ts[0]) - f(ts[1])) / (2 * h)  # linear in each leaf: exact up to rounding
        ana = (grads[k].double().cpu() * v)
        assert abs(num - float(ana.sum())) <= 1e-9 + 1e-4 * float(ana.abs().sum())
    for k in range(4):
        one = [t.detach().requires_grad_(j == k) for j, t in enumerate(leaves)]
        for idx, sc in ((index, scale), (None, scale), (index, None), (None, None)):
            Y = torch_op.lora(*one[:3], idx, sc, one[3])
            g, = torch.autograd.grad(Y, one[k], dY)
            if idx is not None and sc is not None:
                assert torch.equal(g, grads[k])
    with pytest.raises(ValueError, match="scale"):
        torch_op.lora(X, down, up, index, scale.clone().requires_grad_(True), base).sum().backward()


# --------------------------------------------------------------- in programs
def _weight(M, K, density=0.3, seed=0):
    A = T.gen_uniform(M, K, density, seed)
    return A, torch.from_numpy(A.row_ptr), torch.from_numpy(A.col), torch.from_numpy(A.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_adapted_block_trains(dt):
    """Norm of the tokens' features, a frozen sparse weight with adapters, and back: output and gradients of the whole
    block against 64 bits (roundings of the intermediate activations to the type included)."""
    K, M, N, R, L = 128, 192, 80, 8, 3
    A, crow, col, val = _weight(M, K)
    g = torch.Generator().manual_seed(11)
    x = torch.randn(K, N, generator=g).cuda().requires_grad_(True)
    norm = torch_op.LayerNorm(K, dim=0, out_dtype=dt, device="cuda")
    ad = torch_op.LowRankAdapters(L, R, M, K, alpha=16, device="cuda", dtype=dt)
    with torch.no_grad():
        ad.up.copy_(torch.randn(L, M, R, generator=g) / R ** 0.5)
    block = torch_op.AdaptedProduct(crow, col, val, ad)
    index = torch.sort(torch.randint(-1, L, (N,), generator=g)).values.cuda()
    Y = block(norm(x), index)
    dY = torch.randn(M, N, generator=g).cuda()
    leaves = [x, norm.weight, norm.bias, ad.down, ad.up]
    got = torch.autograd.grad(Y, leaves, dY)

    W = torch.from_numpy(A.to_scipy().toarray()).to(dt).double()
    ref = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    xr, w, b, D, Up = ref
    m = xr.mean(0, keepdim=True)
    z = (xr - m) / torch.sqrt(((xr - m) ** 2).mean(0, keepdim=True) + 1e-5) * w[:, None] + b[:, None]
    own = (index.cpu()[None, :] == torch.arange(L)[:, None]).double() * ad.scale.double().cpu()[:, None]
    Yr = W @ z + torch.einsum("amr,ark,kt,at->mt", Up, D, z, own)
    refs = torch.autograd.grad(Yr, ref, dY.double().cpu())
    # fp32: sums of at most a few hundred terms; bf16: activations and the gradient handed to A^T are rounded to bf16.
    tol = 1e-5 if dt == F32 else 4 * 2.0 ** -8
    for t, r in zip([Y, *got], [Yr.detach(), *refs]):
        assert float((t.detach().double().cpu() - r).norm() / r.norm()) <= tol
    torch_op.clear_plan_cache()


@pytest.mark.gpu
def test_gcn_layer_with_a_norm():
    A = T.gen_rmat(9, 4000, kind="gcn", seed=3)
    args = [torch.from_numpy(a) for a in (A.row_ptr, A.col, A.values())]
    X = torch.randn(A.ncol, 40, generator=torch.Generator().manual_seed(12)).cuda().requires_grad_(True)
    norm = torch_op.LayerNorm(40, device="cuda")
    layer = torch_op.GCNAggregate(*args, relu=True, norm=norm)
    Y = layer(X)
    G = torch.from_numpy(A.to_scipy().toarray()).double()
    x = X.detach().double().cpu().requires_grad_(True)
    z = G @ x
    m = z.mean(1, keepdim=True)
    Yr = torch.relu((z - m) / torch.sqrt(((z - m) ** 2).mean(1, keepdim=True) + 1e-5))
    dY = torch.randn(Y.shape, generator=torch.Generator().manual_seed(13))
    near = (Yr.detach().cpu().abs() < 1e-3) & (Yr.detach() > 0)
    dY[near] = 0  # where rounding could move a value across the border of the ReLU
    dx, dw = torch.autograd.grad(Y, [X, norm.weight], dY.cuda())
    dxr, = torch.autograd.grad(Yr, [x], dY.double())
    assert float((Y.detach().double().cpu() - Yr.detach()).norm() / Yr.detach().norm()) <= 1e-5
    assert float((dx.double().cpu() - dxr).norm() / dxr.norm()) <= 1e-4
    torch_op.clear_plan_cache()


@pytest.mark.gpu
def test_spmm_lora_is_the_product_and_its_adapters():
    A, crow, col, val = _weight(150, 96)
    X, down, up, index, scale, _ = lora_inputs(150, 96, 70, 16, 3, F16)
    C0 = torch.ops.tcaspmm.spmm(crow, col, val, X)
    Y = torch_op.spmm_lora(crow, col, val, X, down, up, index, scale)
    assert torch.equal(Y, T.lora(X, down, up, index, scale, C0, hidden=True)[0])
    with pytest.raises(ValueError, match="up"):
        torch_op.spmm_lora(crow, col, val, X, down, up[:, :149], index, scale)
    torch_op.clear_plan_cache()


@pytest.mark.gpu
def test_on_another_stream_and_captured():
    """The calls run on the current stream, and replay from a CUDA graph with other contents of the same tensors."""
    Xn, w, b = norm_inputs(64, 200, 0, F16, F32)
    X, down, up, index, scale, base = lora_inputs(96, 64, 200, 16, 3, F16)
    small = lora_inputs(96, 64, 4, 16, 3, F16, mix="each", seed=4)

    def step():
        Z = T.layer_norm(Xn, w, b, 1e-5, 0)
        Y, H = T.lora(Z, down, up, index, scale, base, hidden=True)
        dZ, dD, dU = T.lora_backward(Y, Z, down, up, H, index, scale)
        _, mean, rstd = T.layer_norm(Xn, w, b, 1e-5, 0, stats=True)
        return [Z, Y, dD, dU, *T.layer_norm_backward(dZ, Xn, mean, rstd, w, 0), T.lora(*small)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same tensors: each has its own scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, c) for a, c in zip(first, out))
    Xn.copy_(torch.randn_like(Xn))
    index.copy_(index.flip(0))
    small[3].fill_(1)
    want = [t.clone() for t in step()]
    s.wait_stream(torch.cuda.current_stream())
    graphs[1].replay()
    with torch.cuda.stream(s):
        graphs[0].replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, c) for a, c in zip(want, out))


@pytest.mark.gpu
def test_training_step_captured():
    """Forward and backward through autograd in one captured graph, on leaves that no other graph uses."""
    A, crow, col, val = _weight(64, 48)
    x = torch.randn(48, 40, device="cuda", dtype=F16)
    norm = torch_op.LayerNorm(48, dim=0, device="cuda")
    ad = torch_op.LowRankAdapters(2, 4, 64, 48, device="cuda", dtype=F16)
    with torch.no_grad():
        ad.up.normal_()
    block = torch_op.AdaptedProduct(crow, col, val, ad)
    dY = torch.randn(64, 40, device="cuda")
    leaves = [norm.weight, norm.bias, ad.down, ad.up]

    def step():
        Y = block(norm(x))
        return [Y.detach(), *torch.autograd.grad(Y, leaves, dY)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # plans are built before the capture
        want = [t.clone() for t in step()]
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, out))
    torch_op.clear_plan_cache()


@pytest.mark.gpu
def test_registered_operators():
    """Schemas and fake tensors agree with what the operators do."""
    check = ("test_schema", "test_faketensor")
    X, w, b = norm_inputs(12, 16, 1, BF16, F32)
    ops = torch.ops.tcaspmm
    for dim in (0, 1):
        p = w if dim == 1 else w[:12]
        torch.library.opcheck(ops.layer_norm.default, (X, p, p, 1e-5, dim, F32), test_utils=check)
        torch.library.opcheck(ops.layer_norm_stats.default, (X, p, None, 1e-5, dim, BF16), test_utils=check)
        _, mean, rstd = T.layer_norm(X, dim=dim, stats=True)
        torch.library.opcheck(ops.layer_norm_backward.default, (X, X, mean, rstd, None, dim, F32, True, False, True), test_utils=check)
    X, down, up, index, scale, base = lora_inputs(20, 12, 16, 4, 2, F16)
    torch.library.opcheck(ops.lora.default, (X, down, up, index, scale, base), test_utils=check)
    torch.library.opcheck(ops.lora_hidden.default, (X, down, up, None, None, None), test_utils=("test_faketensor",))
    torch.library.opcheck(ops.lora_into.default, (X, down, up, index, scale, base, base.clone()), test_utils=("test_faketensor",))
    _, H = T.lora(X, down, up, index, scale, base, hidden=True)
    torch.library.opcheck(ops.lora_backward.default, (base, X, down, up, H, index, scale, None, True, True, False), test_utils=check)


@pytest.mark.gpu
def test_calls_overlap_on_two_streams():
    """Calls share nothing: the same results when many run on two streams at once, in either order."""
    args = [lora_inputs(300, 200, n, 16, 5, F16, seed=n) for n in (500, 40, 130, 700)]
    norms = [norm_inputs(300, c, 0, F16, F32, seed=c) for c in (400, 33, 64, 256)]
    want = [(T.lora(*a), T.layer_norm(*n, 1e-5, 0)) for a, n in zip(args, norms)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], {}
    for turn in range(6):
        for k in range(4):
            s = (turn + k) % 2
            with torch.cuda.stream(streams[s]):
                got[turn, k] = (T.lora(*args[k]), T.layer_norm(*norms[k], 1e-5, 0))
    torch.cuda.synchronize()
    for (_, k), (y, z) in got.items():
        assert torch.equal(y, want[k][0]) and torch.equal(z, want[k][1])


@pytest.mark.gpu
def test_lora_past_32_bit_offsets():
    """A base of more than 2^31 elements: columns at both ends of the last rows."""
    M, N = 34000, 65600
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    X = torch.randn(16, N, device="cuda").to(BF16)
    down, up = torch.randn(1, 4, 16, device="cuda").to(BF16), torch.randn(1, M, 4, device="cuda").to(BF16)
    out = torch.empty(M, N, device="cuda", dtype=BF16)
    T.lora(X, down, up, out=out)
    for rows, cols in [(slice(0, 40), slice(0, 40)), (slice(M - 40, M), slice(N - 40, N)), (slice(M - 40, M), slice(0, 40))]:
        y, tol, _ = lora_ref(X[:, cols], down, up[:, rows], None, None, None, BF16)
        close(out[rows, cols], y, tol)
    Y = T.layer_norm(out, dim=1)
    y, tol, *_ = norm_ref(out[M - 3:], None, None, 1e-5, 1, BF16)
    close(Y[M - 3:], y, tol)


@pytest.mark.gpu
def test_on_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    X, down, up, index, scale, base = lora_inputs(60, 50, 90, 8, 3, BF16)
    there = [t.to("cuda:1") for t in (X, down, up, index, scale, base)]
    assert torch.equal(T.lora(*there).cpu(), T.lora(X, down, up, index, scale, base).cpu())
    assert torch.equal(T.layer_norm(there[0]).cpu(), T.layer_norm(X).cpu())
    with pytest.raises(ValueError, match="cuda"):
        T.lora(X, *there[1:])


# ------------------------------------------------------------------- refusals
def test_norm_refuses():
    X = torch.zeros(4, 6)
    for kw, word in [(dict(X=X), "CUDA"), (dict(X=X.long()), "float32"), (dict(X=X[0]), "2-D"), (dict(X=X, dim=2), "dim"),
                     (dict(X=X, weight=torch.ones(5)), "shape"), (dict(X=X, weight=torch.ones(6).double()), "float32"),
                     (dict(X=X, weight=torch.ones(6), bias=torch.ones(6, dtype=F16)), "one type"),
                     (dict(X=X, out_dtype=torch.float64), "out_dtype"), (dict(X=X, eps=-1.0), "eps"),
                     (dict(X=X, eps=float("nan")), "eps"), (dict(X=X, weight=torch.ones(4), dim=1), "shape"),
                     (dict(X=torch.zeros(4, 0)), "empty")]:
        with pytest.raises(ValueError, match=word):
            T.layer_norm(**kw)
    s = torch.zeros(4)
    for args, kw, word in [((torch.zeros(4, 5), X, s, s), {}, "shape"), ((X, X, s[:3], s), {}, "shape"),
                           ((X, X, s, s.double()), {}, "rstd"), ((X, X, s, s), {}, "CUDA"),
                           ((X, X, s, s), dict(param_dtype=torch.int8), "param_dtype")]:
        with pytest.raises(ValueError, match=word):
            T.layer_norm_backward(*args, **kw)
    with pytest.raises(ValueError, match="along dim 0"):
        torch_op.LayerNorm(6, dim=0)(X)


def test_lora_refuses():
    X, down, up = torch.zeros(6, 5), torch.zeros(2, 3, 6), torch.zeros(2, 4, 3)
    idx, sc, base = torch.zeros(5, dtype=torch.int32), torch.zeros(2), torch.zeros(4, 5)
    for args, kw, word in [((X, down, up, idx, sc, base), {}, "CUDA"), ((X, down[0], up), {}, "3-D"),
                           ((X, down.half(), up), {}, "type"), ((X, down, up[:1]), {}, "shape"),
                           ((X, down[:, :, :5], up), {}, "shape"), ((X, down, up[:, :, :2]), {}, "shape"),
                           ((X, down, up, idx[:4]), {}, "shape"), ((X, down, up, idx.float()), {}, "int32"),
                           ((X, down, up, idx, sc[:1]), {}, "shape"), ((X, down, up, idx, sc.half()), {}, "float32"),
                           ((X, down, up, idx, sc, base[:3]), {}, "shape"), ((X, down, up, idx, sc, base.long()), {}, "base"),
                           ((X, torch.zeros(2, 257, 6), torch.zeros(2, 4, 257)), {}, "rank"),
                           ((X, down[:, :0], up[:, :, :0]), {}, "rank"),
                           ((X, down, up, idx, sc, base), dict(out=base.half()), "type"),
                           ((X, down, up, idx, sc, base), dict(out=torch.zeros(5, 4).T), "contiguous")]:
        with pytest.raises(ValueError, match=word):
            T.lora(*args, **kw)
    H = torch.zeros(dense.hidden_bytes(2, 3, 4, 6, 5, F32), dtype=torch.uint8)
    for args, word in [((base.half(), X, down, up, H), "dY"), ((base[:3], X, down, up, H), "shape"),
                       ((base, X, down, up, H[:-1]), "H must"), ((base, X, down, up, H.float()), "H must"),
                       ((base, X, down, up, H, idx, sc, X.half()), "base"), ((base, X, down, up, H), "CUDA")]:
        with pytest.raises(ValueError, match=word):
            T.lora_backward(*args)


def test_c_entries_refuse_bad_arguments():
    """Refused on the host, before any launch: no device is needed."""
    lib, p = T.lib, 4096
    INV, UNS = T.Status.INVALID_ARG, T.Status.UNSUPPORTED

    def norm(x=p, ldx=8, xt=0, y=p, ldy=8, yt=0, pt=0, mean=None, rstd=None, rows=4, cols=8, dim=1, eps=1e-5):
        return lib.tcaspmm_layer_norm(x, ldx, xt, y, ldy, yt, None, None, pt, mean, rstd, rows, cols, dim, eps, None)

    for kw in [dict(xt=9), dict(yt=-1), dict(pt=7), dict(dim=2), dict(ldx=7), dict(ldy=7), dict(rows=-1), dict(cols=-1), dict(x=None),
               dict(y=None), dict(eps=-1.0), dict(eps=float("inf")), dict(eps=float("nan")), dict(mean=p), dict(rstd=p),
               dict(rows=0, dim=0)]:
        assert norm(**kw) == INV, kw
        assert T.last_error()
    assert norm(rows=0) == T.Status.OK and norm(cols=0, dim=0) == T.Status.OK

    def back(dy=p, lddy=8, dyt=0, x=p, ldx=8, xt=0, mean=p, rstd=p, pt=0, dx=p, lddx=8, rows=4, cols=8, dim=1):
        return lib.tcaspmm_layer_norm_backward(dy, lddy, dyt, x, ldx, xt, mean, rstd, None, pt, dx, lddx, None, None, rows, cols, dim,
                                               None, 0, None)

    for kw in [dict(dyt=5), dict(xt=5), dict(pt=5), dict(dim=-1), dict(dy=None), dict(x=None), dict(lddy=1), dict(ldx=1), dict(lddx=1),
               dict(mean=None), dict(rstd=None), dict(rows=0, dim=0)]:
        assert back(**kw) == INV, kw

    def ad(**kw):
        d = dict(down=p, up=p, index=p, scale=None, count=2, rank=4, M=8, K=8, dt=0, index_bytes=4)
        d.update(kw)
        return dense._Adapters(*(d[n] for n, _ in dense._Adapters._fields_))

    def lora(a=None, x=p, ldx=8, n=8, base=None, ldb=8, y=p, ldy=8, yt=0, h=p, **kw):
        a = ad(**kw) if a is None else a
        return lib.tcaspmm_lora(C.byref(a), x, ldx, n, base, ldb, y, ldy, yt, h, 1, None)

    for kw in [dict(dt=9), dict(yt=9), dict(count=-1), dict(rank=0), dict(M=-1), dict(K=-1), dict(n=-1), dict(index_bytes=2),
               dict(down=None), dict(up=None), dict(x=None), dict(y=None), dict(ldx=7), dict(ldy=7), dict(base=p, ldb=7), dict(h=None), dict(h=p + 4)]:
        assert lora(**kw) == INV, kw
    for kw in [dict(rank=257), dict(count=2 ** 31 - 1), dict(M=2 ** 31 - 1), dict(n=2 ** 31 - 1, ldx=2 ** 31, ldy=2 ** 31)]:
        assert lora(**kw) == UNS, kw
    assert lib.tcaspmm_lora(None, p, 8, 8, None, 8, p, 8, 0, p, 1, None) == INV

    def lback(dy=p, lddy=8, dyt=0, x=p, ldx=8, n=8, h=p, base=None, ldb=8, dx=p, lddx=8, dd=p, du=p, s=p, **kw):
        return lib.tcaspmm_lora_backward(C.byref(ad(**kw)), dy, lddy, dyt, x, ldx, n, h, base, ldb, dx, lddx, dd, du, s, None)

    for kw in [dict(dyt=9), dict(dy=None), dict(lddy=7), dict(x=None), dict(ldx=7), dict(h=None), dict(base=p, ldb=7), dict(lddx=7),
               dict(s=None), dict(rank=0)]:
        assert lback(**kw) == INV, kw


def test_c_entries_refuse_misaligned_pointers():
    """An element's own alignment is asked of every pointer, on the host: no device is needed."""
    lib, p, INV = T.lib, 4096, T.Status.INVALID_ARG

    def norm(x=p, y=p, w=p, b=p, m=p, r=p, t=0):
        return lib.tcaspmm_layer_norm(x, 8, t, y, 8, t, w, b, t, m, r, 4, 8, 1, 1e-5, None)

    def back(dy=p, x=p, m=p, r=p, w=p, dx=p, dw=p, db=p, t=0):
        return lib.tcaspmm_layer_norm_backward(dy, 8, t, x, 8, t, m, r, w, t, dx, 8, dw, db, 4, 8, 1, p, 1 << 30, None)

    def ad(t, wide, **kw):
        d = dict(down=p, up=p, index=p, scale=p, count=2, rank=4, M=8, K=8, dt=t, index_bytes=8 if wide else 4)
        d.update(kw)
        return C.byref(dense._Adapters(*(d[n] for n, _ in dense._Adapters._fields_)))

    def lora(x=p, base=p, y=p, t=0, wide=True, **kw):
        return lib.tcaspmm_lora(ad(t, wide, **kw), x, 8, 8, base, 8, y, 8, t, p, 1, None)

    def lback(dy=p, x=p, base=p, dx=p, dd=p, du=p, t=0, wide=True, **kw):
        return lib.tcaspmm_lora_backward(ad(t, wide, **kw), dy, 8, t, x, 8, 8, p, base, 8, dx, 8, dd, du, p, None)

    for call, names in [(norm, ["x", "y", "w", "b", "m", "r"]), (back, ["dy", "x", "m", "r", "w", "dx", "dw", "db"]),
                        (lora, ["x", "base", "y", "down", "up", "scale", "index"]),
                        (lback, ["dy", "x", "base", "dx", "dd", "du", "down", "up", "scale", "index"])]:
        for name in names:
            for t, off in [(0, 1), (0, 2), (1, 1), (2, 1)]:
                assert call(**{name: p + off}, t=t) == INV, (call.__name__, name, t)
                assert "aligned" in T.last_error()
    assert lora(index=p + 4) == INV


def test_c_entries_refuse_outputs_over_inputs():
    """Refused on the host: no device is needed.  The two in-place forms and windows side by side are on the GPU below."""
    lib, INV = T.lib, T.Status.INVALID_ARG
    at = lambda k: 65536 * (k + 1)  # noqa: E731  (far from one another)

    def norm(x=at(0), y=at(1), w=at(2), b=at(3), ldx=8, ldy=8):
        return lib.tcaspmm_layer_norm(x, ldx, 0, y, ldy, 0, w, b, 0, None, None, 4, 8, 1, 1e-5, None)

    # The same, a few elements on, the last element, another pitch, a window that runs into its neighbour.
    for kw in [dict(y=at(0)), dict(y=at(0) + 4), dict(y=at(0) + 4 * 31), dict(y=at(0) - 4 * 31), dict(y=at(0), ldy=9),
               dict(y=at(0) + 28, ldx=16, ldy=16), dict(y=at(2)), dict(y=at(3) - 4)]:
        assert norm(**kw) == INV and "shares memory" in T.last_error(), kw

    def back(dy=at(0), x=at(1), w=at(2), dx=at(3)):
        return lib.tcaspmm_layer_norm_backward(dy, 8, 0, x, 8, 0, at(4), at(5), w, 0, dx, 8, None, None, 4, 8, 1, None, 0, None)

    for kw in [dict(dx=at(0)), dict(dx=at(1)), dict(dx=at(2))]:
        assert back(**kw) == INV and "shares memory" in T.last_error(), kw

    def ad(down=at(10), up=at(11)):
        return C.byref(dense._Adapters(down, up, at(12), None, 2, 4, 8, 8, 0, 4))

    def lora(x=at(0), base=at(1), y=at(2), ldb=8, ldy=8, **kw):
        return lib.tcaspmm_lora(ad(**kw), x, 8, 8, base, ldb, y, ldy, 0, at(3), 1, None)

    for kw in [dict(y=at(0)), dict(y=at(1) + 4), dict(y=at(1), ldb=9), dict(y=at(10)), dict(y=at(11))]:
        assert lora(**kw) == INV and "shares memory" in T.last_error(), kw

    def lback(dy=at(0), x=at(1), base=at(2), dx=at(3), dd=at(4), du=at(5), **kw):
        return lib.tcaspmm_lora_backward(ad(**kw), dy, 8, 0, x, 8, 8, at(6), base, 8, dx, 8, dd, du, at(7), None)

    for kw in [dict(dx=at(0)), dict(dx=at(1)), dict(dx=at(2) + 4), dict(dx=at(4)), dict(dx=at(10)), dict(dd=at(0)), dict(dd=at(10)),
               dict(dd=at(5)), dict(du=at(11)), dict(du=at(2)), dict(du=at(1))]:
        assert lback(**kw) == INV and "shares memory" in T.last_error(), kw


@pytest.mark.gpu
def test_lora_in_place_and_beside_its_base():
    """Y as base itself, and Y and base as neighbouring windows of one matrix: the same bits as a new Y."""
    X, down, up, index, scale, base = lora_inputs(200, 96, 150, 16, 3, F32, F32, "runs")
    want = T.lora(X, down, up, index, scale, base)
    both = torch.zeros(200, 304, device="cuda")
    both[:, :150] = base
    got = T.lora(X, down, up, index, scale, both[:, :150], out=both[:, 150:300])
    assert torch.equal(got, want) and torch.equal(both[:, :150], base) and not both[:, 300:].any()
    assert torch.equal(T.lora(X, down, up, index, scale, both[:, :150], out=both[:, :150]), want)
    for out in (both[:, 1:151], both[:, 149:299]):
        with pytest.raises(RuntimeError, match="shares memory"):
            T.lora(X, down, up, index, scale, both[:, :150], out=out)


def test_adapters_struct_matches_the_header(tmp_path):
    import os
    import shutil
    import subprocess

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = [name for name, _ in dense._Adapters._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tcaspmm.h"\nint main(void) {\n'
                   '  printf("%zu\\n", sizeof(tcaspmm_adapters));\n'
                   + "".join(f'  printf("%zu\\n", offsetof(tcaspmm_adapters, {f}));\n' for f in fields) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    root = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [C.sizeof(dense._Adapters)] + [getattr(dense._Adapters, f).offset for f in fields]
