"""Layer norm and low-rank adapters where the arithmetic, autograd and the build can go wrong at the edges.

Values are chosen so that the formula's result is known exactly, or the bound stands beside the check.
"""
import os
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import spmm_b200 as T
from spmm_b200 import dense, torch_op
from test_dense_ops import BF16, F16, F32, U, close, lora_inputs, lora_ref, test_norm_and_its_gradients as check_norm


ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


# ------------------------------------------------------------------ precision
def _adapter(down, up, X, dY, dt, N, at=(0, 1)):
    """One adapter from nested lists; X and dY hold a few columns, put at `at` among N that are zero otherwise."""
    D, Up = torch.tensor([down]).to(dt).cuda(), torch.tensor([up]).to(dt).cuda()
    x, g = torch.tensor(X), torch.tensor(dY)
    Xn, Gn = torch.zeros(x.shape[0], N), torch.zeros(g.shape[0], N)
    for k, t in enumerate(at[:x.shape[1]]):
        Xn[:, t], Gn[:, t] = x[:, k], g[:, k]
    return Xn.to(dt).cuda(), D, Up, Gn.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("N,at", [(2, (0, 1)), (70, (3, 66))])
def test_gradients_keep_the_bits_of_fp32_operands(dt, N, at):
    """An fp32 dY and the fp32 intermediates H and P are not rounded to the tensor cores' 10 bits: what is left where two
    terms cancel is exact."""
    e, f = 2.0 ** -13, 2.0 ** -12
    # dU = (1 + e) h - h with h = 1: dY's low part.
    X, D, Up, G = _adapter([[1.0]], [[1.0]], [[1.0, 1.0]], [[1 + e, -1.0]], dt, N, at)
    H = T.lora(X, D, Up, hidden=True)[1]
    assert float(T.lora_backward(G, X, D, Up, H)[2]) == e
    # dU = h0 - h1 with h0 = 1 + f, h1 = 1: H's low part.
    X, D, Up, G = _adapter([[1.0, f]], [[1.0]], [[1.0, 1.0], [1.0, 0.0]], [[1.0, -1.0]], dt, N, at)
    H = T.lora(X, D, Up, hidden=True)[1]
    assert float(T.lora_backward(G, X, D, Up, H)[2]) == f
    # dD = p0 - p1 with p0 = 1 + f, p1 = 1: P's low part.
    X, D, Up, G = _adapter([[1.0]], [[1.0], [f]], [[1.0, -1.0]], [[1.0, 1.0], [1.0, 0.0]], dt, N, at)
    H = T.lora(X, D, Up, hidden=True)[1]
    assert float(T.lora_backward(G, X, D, Up, H)[1]) == f
    # p = (1 + e) - 1, dX = p: dY's low part in the product with up.
    X, D, Up, G = _adapter([[1.0]], [[1.0], [-1.0]], [[1.0, 0.0]], [[1 + e, 0.0], [1.0, 0.0]], dt, N, at)
    H = T.lora(X, D, Up, hidden=True)[1]
    assert float(T.lora_backward(G, X, D, Up, H)[0][0, at[0]]) == e


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("N", [1, 70])
def test_intermediate_keeps_its_bits_for_16_bit_results(dt, N):
    """S = down X (and P) is a sum, held in fp32's bits also where the result is 16-bit: what cancels there is exact."""
    e = 2.0 ** -20
    # P = (1 + 2^-9 + e, 1 + 2^-9), dX = their difference.
    X, D, Up, G = _adapter([[1.0], [-1.0]], [[1.0, 0.0], [0.0, 1.0]], [[0.0]], [[1 + 2.0 ** -9 + e], [1 + 2.0 ** -9]], dt, N)
    H = T.lora(X, D, Up, hidden=True)[1]
    assert float(T.lora_backward(G, X, D, Up, H)[0][0, 0]) == e
    # H the same, through the forward product, into a result of the factors' type.
    X, D, Up, _ = _adapter([[1.0, 2.0 ** -9, e], [1.0, 2.0 ** -9, 0.0]], [[1.0, -1.0]], [[1.0], [1.0], [1.0]], [[0.0]], dt, N)
    for hidden in (False, True):
        Y = T.lora(X, D, Up, None, None, torch.zeros(1, N, device="cuda", dtype=dt), hidden=hidden)
        assert float((Y[0] if hidden else Y)[0, 0]) == e


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 70])
def test_fp32_products_are_rounded_to_nearest(N):
    """fp32 operands in two TF32 parts.  Rounded to nearest a part leaves at most 2^-11, so that the product of both low parts,
    left out, is at most 2^-22, and each operand is held to 2^-23: a product is off by at most 2^-21 = 8 units of 2^-24.  The
    one step of 8 products adds three instructions that may cut 2 units each; the second product (up = 1: only S's own 2
    units) three more: 22 units.  Parts cut toward zero lose 28 of each product here."""
    x = 1 + 2.0 ** -10 - 2.0 ** -23
    X, D, Up = torch.full((8, N), x).cuda(), torch.full((1, 1, 8), x).cuda(), torch.ones(1, 1, 1).cuda()
    Y = T.lora(X, D, Up, hidden=True)[0].double().cpu()
    ref = 8 * x * x
    assert float((Y - ref).abs().max()) <= 22 * U * ref


@pytest.mark.gpu
@pytest.mark.parametrize("trans", [False, True])
def test_fp32_sums_over_the_rank_are_kept_outside_the_tensor_cores(trans):
    """2^24, then 31 steps that add 1.5 each: every addition rounded to nearest is off by at most half a step, 1, so the sum by
    31 at most; sums cut at every step never move from 2^24 and are 46.5 off."""
    R, N = 256, 5
    row = torch.zeros(R)
    row[8::8] = 1.5
    row[0] = 2.0 ** 24
    ones = torch.ones(R)
    if trans:  # dX = down^T P, P = up^T dY = 1
        D, Up = row.reshape(1, R, 1).cuda(), ones.reshape(1, 1, R).cuda()
        X, G = torch.zeros(1, N).cuda(), torch.ones(1, N).cuda()
        H = T.lora(X, D, Up, hidden=True)[1]
        got = T.lora_backward(G, X, D, Up, H)[0]
    else:
        D, Up = ones.reshape(1, R, 1).cuda(), row.reshape(1, 1, R).cuda()
        got = T.lora(torch.ones(1, N).cuda(), D, Up, hidden=True)[0]
    assert float((got.double().cpu() - (2.0 ** 24 + 46.5)).abs().max()) <= 31


# ------------------------------------------------------------------ infinities
def _same(got, ref, size):
    """Infinities by sign, NaN, and finite values within 2^-15 of the sum of their terms' magnitudes (two products in turn of at
    most 20 terms: 2 U (20 / 4 + 64) < 2^-16 each) and half a step of a 16-bit result."""
    step = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), (got, ref)
    inf = ref.isinf()
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf], ref[inf]), (got, ref)
    fin = ref.isfinite()
    assert bool(((got - ref).abs() <= 2.0 ** -15 * size + step * ref.abs())[fin].all())


def _product(a, b, own):
    """(a @ b over the columns `own`, the same of magnitudes), IEEE rules for infinities."""
    a, b = a[:, own], b[own]
    terms = a[:, :, None] * b[None]
    return terms.sum(1), torch.where(terms.isfinite(), terms.abs(), 0.0).sum(1)


INF = float("inf")
PLACES = [("X", (4, 3), INF), ("X", (0, 3), -INF), ("down", (1, 2, 3), INF), ("up", (2, 5, 0), -INF), ("up", (0, 1, 2), INF),
          ("dY", (5, 3), INF), ("dY", (2, 2), -INF)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("N", [6, 80])
@pytest.mark.parametrize("name,place,value", PLACES)
@pytest.mark.parametrize("g16", [False, True])
def test_infinities_are_those_of_the_formula(dt, N, name, place, value, g16):
    """One infinity among values that 16 bits and TF32 hold exactly (so that low parts are nothing): every result is the
    infinity, NaN or finite value of the formula, whichever kernel computes it."""
    M, K, R, L = 12, 10, 3, 4
    g = torch.Generator().manual_seed(5)
    pick = lambda *s: torch.tensor([0.5, 1.0, 2.0, 1.0, 4.0])[torch.randint(0, 5, s, generator=g)]  # noqa: E731
    t = {"X": pick(K, N), "down": pick(L, R, K), "up": pick(L, M, R), "dY": pick(M, N)}
    t["up"][:, 7] *= -1
    t["down"][:, :, 6] *= -1
    t[name][place] = value
    index = (torch.arange(N) % L).int()
    dev = {k: v.to(F32 if k == "dY" and not g16 else dt).cuda() for k, v in t.items()}
    X, down, up, dY = (t[k].double() for k in ("X", "down", "up", "dY"))
    Y, dX = torch.zeros(M, N).double(), torch.zeros(K, N).double()
    sY, sX, dD, dU = Y.clone(), dX.clone(), torch.zeros_like(down), torch.zeros_like(up)
    sD, sU = dD.clone(), dU.clone()
    for a in range(L):
        at = (index == a).nonzero().flatten()
        h, hs = _product(down[a], X[:, at], slice(None))
        p, ps = _product(up[a].T, dY[:, at], slice(None))
        Y[:, at] = _product(up[a], h, slice(None))[0]
        sY[:, at] = _product(up[a].abs(), hs, slice(None))[1]
        dX[:, at] = _product(down[a].T, p, slice(None))[0]
        sX[:, at] = _product(down[a].T.abs(), ps, slice(None))[1]
        dD[a], dU[a] = _product(p, X[:, at].T, slice(None))[0], _product(dY[:, at], h.T, slice(None))[0]
        sD[a], sU[a] = _product(ps, X[:, at].T.abs(), slice(None))[1], _product(dY[:, at].abs(), hs.T, slice(None))[1]
    args = (dev["X"], dev["down"], dev["up"], index.cuda())
    _same(T.lora(*args), Y, sY)
    got, H = T.lora(*args, hidden=True)
    _same(got, Y, sY)
    for got, ref, size in zip(T.lora_backward(dev["dY"], *args[:3], H, args[3]), (dX, dD, dU), (sX, sD, sU)):
        _same(got, ref, size)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [False, True])
def test_fp16_intermediate_beside_an_infinity_and_at_the_end_of_the_range(hidden):
    """H's parts are scaled by the column's largest finite value: a finite value past fp16's range beside an infinity stays
    finite, and so does one near the end of fp32's range."""
    def lora(*a):
        return T.lora(*a, hidden=True)[0] if hidden else T.lora(*a)

    down = torch.tensor([[[INF, 0.0], [0.0, 8.0]]]).half().cuda()  # h = (inf, 480000)
    up, X = torch.tensor([[[1.0, -1.0]]]).half().cuda(), torch.tensor([[1.0], [60000.0]]).half().cuda()
    assert float(lora(X, down, up)) == INF
    one = torch.ones(1, 1, 1).half().cuda()
    for e in (118, 127):
        assert float(lora(torch.ones(1, 1).half().cuda(), one, one, None, torch.tensor([2.0 ** e]).cuda())) == 2.0 ** e


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [False, True])
def test_fp32_values_at_the_end_of_the_range(hidden):
    """The largest values stay finite (both parts are cut there), beside ones that do not reach them: 2^-21 for each of two
    products and a cut, 2^-23, for each of three instructions: 2 (2^-21 + 3 2^-23) < 2^-19."""
    most = torch.finfo(F32).max
    X = torch.tensor([[most, -most, 3.4e38, 1.0]]).cuda()
    for down, up in ((1.0, 1.0), (0.25, 4.0), (-1.0, 1.0)):
        Y = T.lora(X, torch.full((1, 1, 1), down).cuda(), torch.full((1, 1, 1), up).cuda(), hidden=hidden)
        Y = (Y[0] if hidden else Y).double().cpu()
        ref = X.double().cpu() * down * up
        assert bool(((Y - ref).abs() <= 2.0 ** -19 * ref.abs()).all())


# ------------------------------------------------------------------ which kernels
@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,R,L", [(96, 72, 64, 16, 64), (130, 96, 200, 8, 40), (61, 35, 256, 5, 16), (40, 50, 65, 3, 33)])
@pytest.mark.parametrize("dt,ydt", [(F32, F32), (F16, F32), (BF16, F32), (BF16, BF16), (F16, F16), (F32, F16)])
def test_lora_many_adapters(M, K, N, R, L, dt, ydt):
    """Up to 64 adapters among a tile's columns, and up to 256 columns one by one."""
    X, down, up, index, scale, base = lora_inputs(M, K, N, R, L, dt, ydt, "each", seed=N)
    y, tol, _ = lora_ref(X, down, up, index, scale, base, ydt)
    close(T.lora(X, down, up, index, scale, base), y, tol)
    close(T.lora(X, down, up, index, scale, base, hidden=True)[0], y, tol)


def _allocations(f):
    f()
    n = [torch.cuda.memory_stats()["allocation.all.allocated"]]
    f()
    return torch.cuda.memory_stats()["allocation.all.allocated"] - n[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,ydt", [(F32, F32), (F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("M,K,N,R,L", [(300, 200, 1, 16, 3), (120, 70, 9, 5, 3), (96, 72, 64, 16, 64), (130, 96, 200, 8, 40),
                                       (90, 60, 300, 8, 3)])
def test_out_takes_the_same_kernels_and_keeps_nothing_unasked(M, K, N, R, L, dt, ydt):
    """A result in place, or in a window, has the bits of a new one; nothing is allocated where few columns go one by one."""
    X, down, up, index, scale, base = lora_inputs(M, K, N, R, L, dt, ydt, "each", seed=3)
    want = T.lora(X, down, up, index, scale, base)
    window = torch.full((M + 2, N + 5), 7.0, device="cuda").to(ydt)
    view = window[1:-1, 3:3 + N]
    assert torch.equal(T.lora(X, down, up, index, scale, base, out=view), want)
    view.fill_(7.0)
    assert bool((window == 7.0).all())
    C = base.clone()
    assert torch.equal(T.lora(X, down, up, index, scale, C, out=C), want)
    scratch = int(N == 300)  # the tiles' own, given back
    assert _allocations(lambda: T.lora(X, down, up, index, scale, C, out=C)) == scratch
    kept = base.clone()
    assert T.lora(X, down, up, index, scale, kept, out=kept, hidden=True)[1].numel() == dense.hidden_bytes(L, R, M, K, N, dt)


@pytest.mark.gpu
def test_adapted_product_without_gradients_keeps_nothing():
    """A @ X and its adapters, 64 tokens of 64 adapters: without gradients the bits of the product with lora in place, and no
    allocation beside the product's own; with gradients the same up to the order of sums, and H."""
    M, K, N, R, L = 192, 128, 64, 16, 64
    A = T.gen_uniform(M, K, 0.3, 0)
    csr = [torch.from_numpy(a) for a in (A.row_ptr, A.col, A.values())]
    X, down, up, index, scale, _ = lora_inputs(M, K, N, R, L, F16, F32, "each", seed=9)
    adapters = torch_op.LowRankAdapters(L, R, M, K, device="cuda", dtype=F16)
    with torch.no_grad():
        adapters.down.copy_(down)
        adapters.up.copy_(up)
    block = torch_op.AdaptedProduct(*csr, adapters)
    C = torch.ops.tcaspmm.spmm(*csr, X)
    want = T.lora(X, down, up, index, adapters.scale, C)
    with torch.no_grad():
        Y = block(X, index)
        assert torch.equal(Y, want)
        n = _allocations(lambda: torch.ops.tcaspmm.spmm(*csr, X))
        assert _allocations(lambda: block(X, index)) == n
    for p in adapters.parameters():  # nothing to train: nothing kept in grad mode either
        p.requires_grad_(False)
    assert _allocations(lambda: block(X, index)) == n
    for p in adapters.parameters():
        p.requires_grad_(True)
    Z = block(X, index)
    assert Z.requires_grad and torch.equal(Z, T.lora(X, down, up, index, adapters.scale, C, hidden=True)[0])
    dY = torch.randn(M, N, generator=torch.Generator().manual_seed(1)).cuda()
    got = torch.autograd.grad(Z, [adapters.down, adapters.up], dY)
    H = T.lora(X, down, up, index, adapters.scale, C, hidden=True)[1]
    for a, b in zip(got, T.lora_backward(dY, X, down, up, H, index, adapters.scale)[1:]):
        assert torch.equal(a, b)
    torch_op.clear_plan_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16, 20, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 333, 512, 513, 600, 1025, 1500, 2048, 2049, 3001,
                                  4096, 4097, 6000, 6001, 8192, 8193, 12001, 16384, 16385])
@pytest.mark.parametrize("dt,out,pdt", [(F32, F32, F32), (F16, F32, F16), (BF16, BF16, F32)])
def test_norm_of_every_row_plan(cols, dt, out, pdt):
    """Widths on both sides of each change of a row's threads and chunks, aligned and odd."""
    check_norm(5, cols, 1, dt, out, pdt)


# ------------------------------------------------------------------ autograd
def _fake_args():
    """X, weight, bias of a norm; X, down, up, index, scale, base of adapters: CUDA tensors without data."""
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    return (z(6, 5), z(5), z(5)), (z(6, 5), z(2, 3, 6), z(2, 4, 3), z(5, dtype=torch.int32), z(2), z(4, 5))


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A tangent would be dropped without a word: whichever input has one, the call raises."""
    with FakeTensorMode(), torch.set_grad_enabled(grad):
        norm, lora = _fake_args()
        csr = [torch.zeros(5, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(0)]
        for f, args, which in [(torch_op.layer_norm, norm, (0, 1, 2)), (torch_op.lora, lora, (0, 1, 2, 4, 5)),
                               (lambda *a: T.layer_norm(*a, stats=True), norm, (0, 1)),
                               (lambda *a: T.lora(*a, hidden=True), lora, (0, 2)),
                               (lambda *a: T.lora(*a, out=a[5].clone()), lora, (0, 1, 2, 5)),
                               (lambda *a: torch_op.spmm_lora(*csr, *a[:5]), lora, (0, 1, 2))]:
            f(*args)
            for k in which:
                with forward_ad.dual_level():
                    dual = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
                    with pytest.raises(NotImplementedError, match="forward"):
                        f(*args[:k], dual, *args[k + 1:])
        for f, args in ((torch_op.layer_norm, norm), (torch_op.lora, lora), (lambda *a: torch_op.spmm_lora(*csr, *a[:5]), lora)):
            with pytest.raises(NotImplementedError, match="forward"):
                torch.func.jvp(lambda x: f(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))


def test_out_is_seen_to_change():
    """A tensor written through out= gets a new version."""
    with FakeTensorMode():
        _, (X, down, up, index, scale, base) = _fake_args()
        C = base.clone()
        for k, hidden in enumerate((False, True, False)):
            assert C._version == k
            T.lora(X, down, up, index, scale, C, out=C, hidden=hidden)
        assert C._version == 3
        T.lora(X, down, up, index, scale, base, out=C)
        assert C._version == 4 and base._version == 0


@pytest.mark.gpu
def test_backward_refuses_what_out_overwrote():
    X, down, up, index, scale, base = lora_inputs(20, 12, 16, 4, 2, F32)
    C = base.requires_grad_(True).exp()  # its backward pass reads C
    with torch.no_grad():
        T.lora(X, down, up, index, scale, C, out=C)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        C.sum().backward()


def test_out_has_no_gradients():
    """As torch's own out= forms: an argument that requires a gradient is refused in grad mode."""
    with FakeTensorMode():
        _, args = _fake_args()
        for hidden in (False, True):
            for k in (0, 1, 2, 4, 5, 6):
                a = [t.clone() for t in (*args, args[5])]
                a[k].requires_grad_(True)
                with pytest.raises(RuntimeError, match="requires grad"):
                    T.lora(*a[:6], out=a[6], hidden=hidden)
                with torch.no_grad():
                    T.lora(*a[:6], out=a[6], hidden=hidden)


@pytest.mark.gpu
def test_registered_autograd():
    """The operators' registrations for autograd, by torch's own checks."""
    X, w, b = (t.requires_grad_(True) for t in (torch.randn(12, 16, device="cuda"), torch.ones(16, device="cuda"), torch.ones(16, device="cuda")))
    ops = torch.ops.tcaspmm
    check = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(ops.layer_norm.default, (X, w, b, 1e-5, 1, F32), test_utils=check)
    X, down, up, index, scale, base = lora_inputs(20, 12, 16, 4, 2, F32)
    leaves = [t.requires_grad_(True) for t in (X, down, up)]
    torch.library.opcheck(ops.lora.default, (*leaves, index, scale, base), test_utils=check)
    with torch.no_grad():
        torch.library.opcheck(ops.lora_into.default, (X.detach(), down.detach(), up.detach(), index, scale, base, base.clone()), test_utils=check)


# ------------------------------------------------------------------ without the torch operators
def _make(*args):
    return subprocess.run(["make", "-C", os.path.join(ROOT, "spmm_b200", "csrc"), *args], capture_output=True, text=True)


@pytest.mark.parametrize("python", ["no-such-python", "false"])
def test_make_without_torch(python):
    """The C library and the driver need no torch: where $(PYTHON) has none, only the torch operators are left out."""
    plan = _make("-n", "-B", f"PYTHON={python}")
    assert plan.returncode == 0, plan.stderr
    assert "libtcaspmm.so" in plan.stdout and "bin/test" in plan.stdout
    assert "torch_bind.cpp" not in plan.stdout and "torch_bind.cpp" in _make("-n", "-B", f"PYTHON={sys.executable}").stdout


def test_make_torch_says_what_is_missing(tmp_path):
    """Asked for by name, the torch operators are an error without torch."""
    got = _make(f"LIB={tmp_path}", "-o", f"{tmp_path}/libtcaspmm.so", "PYTHON=false", "torch")
    assert got.returncode != 0 and "no torch in false" in got.stderr


@pytest.mark.parametrize("broken", [False, True])
def test_import_without_the_torch_operators(tmp_path, broken):
    """Without libtcaspmm_torch.so, or with one that does not load, torch_op's sparse operators are there; the norm's and the
    adapters' first call raises."""
    path = tmp_path / "libtcaspmm_torch.so"
    if broken:
        path.write_bytes(b"not a library")
    code = (f"import spmm_b200.dense as d; d.TORCH_PATH = {str(path)!r}\n"
            "import torch, spmm_b200.torch_op as t\n"
            "assert torch.ops.tcaspmm.spmm and torch.ops.tcaspmm.spmm_fused and t.GCNAggregate\n"
            "for call in (lambda: t.layer_norm(torch.zeros(2, 2)), lambda: t.lora(*[torch.zeros(1, 1, 1)] * 3)):\n"
            "    try:\n        call()\n    except (ImportError, OSError) as e:\n        assert 'libtcaspmm_torch.so' in str(e)\n"
            "    else:\n        raise SystemExit('no error')\n")
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert got.returncode == 0, got.stdout + got.stderr
