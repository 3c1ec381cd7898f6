"""Layer norm and low-rank adapters around a sparse product: the cases their speed is measured on.

Layouts are those of the sparse product C = A X: X is K x N and C is M x N, row-major.  Of a pruned
weight, rows are features and columns are tokens; of a graph, rows are nodes and columns are features.
Layer norm therefore runs over rows' elements (dim 1: a node's features) or over columns' (dim 0: a
token's features), and adapters are chosen by column (a token belongs to one request).
"""
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # One small batch of node features through a norm: latency.
        {"name": "norm_rows_small", "op": "norm", "dim": 1, "rows": 64, "cols": 512, "x": "f32", "y": "f32", "train": False},
        # A GCN layer's output on a graph of 2^20 nodes with 128 features, trained.
        {"name": "norm_rows_gcn_train", "op": "norm", "dim": 1, "rows": 1 << 20, "cols": 128, "x": "f32", "y": "f32", "train": True},
        # Odd hidden width: fp32 aggregates normalised into the next layer's 16-bit features.
        {"name": "norm_rows_odd_cast", "op": "norm", "dim": 1, "rows": 100003, "cols": 233, "x": "f32", "y": "bf16", "train": False},
        # Wide rows, few of them, trained in 16 bits.
        {"name": "norm_rows_wide_train", "op": "norm", "dim": 1, "rows": 4096, "cols": 8192, "x": "bf16", "y": "bf16", "train": True},
        # Activations of a serving batch in front of a pruned FFN weight.
        {"name": "norm_cols_serve", "op": "norm", "dim": 0, "rows": 2048, "cols": 256, "x": "f16", "y": "f16", "train": False},
        # A training batch of tokens in front of a pruned FFN weight.
        {"name": "norm_cols_train", "op": "norm", "dim": 0, "rows": 4096, "cols": 8192, "x": "bf16", "y": "bf16", "train": True},
        # One token of one request: latency.
        {"name": "lora_one_token", "op": "lora", "M": 2048, "K": 512, "N": 1, "R": 16, "L": 8, "mix": "each", "x": "bf16", "y": "f32", "train": False},
        # A decoding batch, a request and an adapter for every token.
        {"name": "lora_decode", "op": "lora", "M": 4096, "K": 1024, "N": 64, "R": 16, "L": 64, "mix": "each", "x": "f16", "y": "f32", "train": False},
        # Prompts of several requests side by side, some without an adapter.
        {"name": "lora_prefill", "op": "lora", "M": 4096, "K": 1024, "N": 8192, "R": 64, "L": 6, "mix": "runs", "x": "bf16", "y": "f32", "train": False},
        # Odd sizes in fp32.
        {"name": "lora_odd_f32", "op": "lora", "M": 1000, "K": 515, "N": 333, "R": 12, "L": 5, "mix": "runs", "x": "f32", "y": "f32", "train": False},
        # Several adapters of one pruned weight trained side by side.
        {"name": "lora_train", "op": "lora", "M": 2048, "K": 2048, "N": 4096, "R": 32, "L": 3, "mix": "runs", "x": "bf16", "y": "f32", "train": True},
        # One adapter trained in fp32.
        {"name": "lora_train_f32", "op": "lora", "M": 512, "K": 2048, "N": 1024, "R": 8, "L": 1, "mix": "runs", "x": "f32", "y": "f32", "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; half of them are multiples of 8 where there is room."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if v >= 16 and rng.random() < 0.5:
        v -= v % 8
    return max(lo, min(hi, v))


def draw(rng):
    """A case of the same ranges: any direction, type and layout; sizes from one to the listed ones' largest."""
    x = rng.choice(["f32", "f16", "bf16"])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        dim = rng.choice([0, 1])
        if dim == 1:
            cols = _spread(rng, 8, 16384)
            rows = _spread(rng, 1, max(1, min(1 << 20, (1 << 25) // cols)))
        else:
            rows = _spread(rng, 32, 8192)
            cols = _spread(rng, 1, max(1, min(8192, (1 << 25) // rows)))
        y = rng.choice([x, x, "bf16", "f32"])
        return {"op": "norm", "dim": dim, "rows": rows, "cols": cols, "x": x, "y": y, "train": train}
    mix = "runs" if train else rng.choice(["runs", "each"])
    n = _spread(rng, 1, 256) if mix == "each" else _spread(rng, 16, 4096)
    return {"op": "lora", "M": _spread(rng, 64, 4096), "K": _spread(rng, 64, 4096), "N": n, "R": rng.choice([4, 8, 12, 16, 16, 32, 64, 128]),
            "L": _spread(rng, 1, 64 if mix == "each" else 6), "mix": mix, "x": x, "y": rng.choice(["f32", "f32", x]), "train": train}


def _index(case, seed):
    """The adapter of each column, -1 for none: runs of one request's tokens side by side, or a request for every column."""
    r = random.Random(seed)
    n, count = case["N"], case["L"]
    one = lambda: -1 if r.random() < 0.1 else r.randrange(count)  # noqa: E731
    if case["mix"] == "each":
        return [r.randrange(count)] + [one() for _ in range(n - 1)]
    runs = max(count, n // 700)
    ends = sorted(r.randrange(n + 1) for _ in range(runs - 1)) + [n]
    index = []
    for k, e in enumerate(ends):
        index += [k if k < count else one()] * (e - len(index))
    return index


def prepare(case, seed):
    """A program's tensors before the call, on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    xt, yt = TYPES[case["x"]], TYPES[case["y"]]
    s = dict(case)
    if case["op"] == "norm":
        rows, cols, dim = case["rows"], case["cols"], case["dim"]
        n = case["cols"] if dim == 1 else rows
        along = (1, n) if dim == 1 else (n, 1)
        # Features have scales and offsets of their own.
        s["X"] = rand(rows, cols).mul_(torch.exp(0.5 * rand(*along))).add_(0.5 * rand(*along)).to(xt)
        s["w"], s["b"] = 1 + 0.1 * rand(n), 0.1 * rand(n)
        leaves = ("X", "w", "b")
        out = (rows, cols)
    else:
        M, K, N, R, L = (case[k] for k in "MKNRL")
        s["X"] = rand(K, N).to(xt)
        s["down"] = (rand(L, R, K) / K ** 0.5).to(xt)
        s["up"] = (rand(L, M, R) / R ** 0.5).to(xt)
        s["index"] = torch.tensor(_index(case, seed), dtype=torch.int32, device="cuda")
        s["scale"] = 0.25 + torch.rand(L, device="cuda", generator=g)
        s["base"] = (2 * rand(M, N)).to(yt)
        leaves = ("X", "down", "up")
        out = (M, N)
    if case["train"]:
        s["dY"] = rand(*out).to(yt)
        for k in leaves:
            s[k].requires_grad_(True)
    return s


def run(state):
    s = state
    if own:
        return _own_norm(s) if s["op"] == "norm" else _own_lora(s)
    with torch.no_grad():
        return _plain_norm(s) if s["op"] == "norm" else _plain_lora(s)


def _own_norm(s):
    import spmm_b200
    from spmm_b200 import torch_op

    if not s["train"]:
        return spmm_b200.layer_norm(s["X"], s["w"], s["b"], EPS, s["dim"], TYPES[s["y"]])
    Y = torch_op.layer_norm(s["X"], s["w"], s["b"], EPS, s["dim"], TYPES[s["y"]])
    return [Y, *torch.autograd.grad(Y, [s["X"], s["w"], s["b"]], s["dY"])]


def _own_lora(s):
    import spmm_b200
    from spmm_b200 import torch_op

    if not s["train"]:
        return spmm_b200.lora(s["X"], s["down"], s["up"], s["index"], s["scale"], s["base"])
    Y = torch_op.lora(s["X"], s["down"], s["up"], s["index"], s["scale"], s["base"])
    return [Y, *torch.autograd.grad(Y, [s["X"], s["down"], s["up"]], s["dY"])]


def _plain_norm(s):
    d = s["dim"]
    n = s["X"].shape[d]
    x = s["X"].float()
    w, b = (s["w"], s["b"]) if d == 1 else (s["w"][:, None], s["b"][:, None])
    x = x - x.sum(d, keepdim=True) / n
    r = 1 / torch.sqrt((x * x).sum(d, keepdim=True) / n + EPS)
    xh = x * r
    Y = (xh * w + b).to(TYPES[s["y"]])
    if not s["train"]:
        return Y
    dy = s["dY"].float()
    g = dy * w
    dX = r * (g - g.sum(d, keepdim=True) / n - xh * ((g * xh).sum(d, keepdim=True) / n))
    return [Y, dX.to(s["X"].dtype), (dy * xh).sum(1 - d), dy.sum(1 - d)]


def _plain_lora(s):
    """All adapters' factors at once, as two products; every column keeps its own adapter's part."""
    L, R, K = s["down"].shape
    M, N = s["up"].shape[1], s["X"].shape[1]
    x, base = s["X"].float(), s["base"].float()
    down = s["down"].float().reshape(L * R, K)
    up = s["up"].float().permute(1, 0, 2).reshape(M, L * R)
    # part[a, t]: the adapter's scale where column t is its own, else 0.
    mine = s["index"][None, :] == torch.arange(L, device=x.device)[:, None]
    part = mine.float().mul(s["scale"][:, None]).repeat_interleave(R, 0)
    H = part * (down @ x)
    Y = (base + up @ H).to(s["base"].dtype)
    if not s["train"]:
        return Y
    dy = s["dY"].float()
    P = part * (up.T @ dy)
    dX = down.T @ P
    dD = (P @ x.T).reshape(L, R, K)
    dU = (dy @ H.T).reshape(M, L, R).permute(1, 0, 2).contiguous()
    t = s["X"].dtype
    return [Y, dX.to(t), dD.to(t), dU.to(t)]


def work(case):
    xs, ys = (4 if case[k] == "f32" else 2 for k in "xy")
    if case["op"] == "norm":
        e, n = case["rows"] * case["cols"], case["cols"] if case["dim"] == 1 else case["rows"]
        if case["train"]:
            return {"bytes": e * (2 * xs + 2 * ys) + 16 * n, "flops": 20 * e}
        return {"bytes": e * (xs + ys) + 8 * n, "flops": 8 * e}
    M, K, N, R = (case[k] for k in "MKNR")
    used = min(case["L"], N)
    rows = K * N * xs + 2 * M * N * ys + 4 * N
    factors = used * R * (K + M) * xs
    if case["train"]:
        # X, base, dY, index and factors in; Y, dX and the factors' gradients out.
        return {"bytes": rows + M * N * ys + K * N * xs + factors + case["L"] * R * (K + M) * xs, "flops": 6 * R * (K + M) * N}
    return {"bytes": rows + factors, "flops": 2 * R * (K + M) * N}


def exact(case, seed):
    """The same outputs in 64 bits, from the definitions: a norm by its mean and variance, adapters one by one."""
    s = prepare(case, seed)
    with torch.no_grad():
        X = s["X"].double()
        dY = s["dY"].double() if case["train"] else None
        if case["op"] == "norm":
            if case["dim"] == 0:
                X, dY = X.T, dY.T if dY is not None else None
            var, mean = torch.var_mean(X, 1, correction=0, keepdim=True)
            std = torch.sqrt(var + EPS)
            z = (X - mean) / std
            w, b = s["w"].double(), s["b"].double()
            Y = torch.addcmul(b, z, w)
            if dY is None:
                return Y.T if case["dim"] == 0 else Y
            dw, db = torch.einsum("ij,ij->j", dY, z), dY.sum(0)
            g = dY * w
            dX = (g - g.mean(1, keepdim=True) - z * (g * z).mean(1, keepdim=True)) / std
            return [Y.T, dX.T, dw, db] if case["dim"] == 0 else [Y, dX, dw, db]
        Y = s["base"].double()
        dX, dD, dU = torch.zeros_like(X), torch.zeros_like(s["down"]).double(), torch.zeros_like(s["up"]).double()
        for a in range(case["L"]):
            at = (s["index"] == a).nonzero().flatten()
            if not at.numel():
                continue
            D, U, k = s["down"][a].double(), s["up"][a].double(), float(s["scale"][a])
            x = X[:, at]
            h = D @ x
            Y[:, at] += k * (U @ h)
            if dY is not None:
                g = dY[:, at]
                p = U.T @ g
                dX[:, at] = k * (D.T @ p)
                dD[a] = k * (p @ x.T)
                dU[a] = k * (g @ h.T)
        return [Y, dX, dD, dU] if case["train"] else Y
