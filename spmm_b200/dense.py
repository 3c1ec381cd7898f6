"""Dense operators around a sparse product, over the C-ABI: layer norm and low-rank adapters.

These are the plain calls (no autograd), on the current stream of the tensors' device;
``spmm_b200.torch_op`` has the differentiable forms.  A matrix argument may be any 2-D CUDA
tensor of float32, float16 or bfloat16; one whose rows are not contiguous is copied first.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

from . import _check, _sig, dtype, lib

_vp, _i64 = C.c_void_p, C.c_int64
_TYPES: dict = {}


class _Adapters(C.Structure):
    _fields_ = [("down", _vp), ("up", _vp), ("index", _vp), ("scale", _vp), ("count", _i64), ("rank", _i64),
                ("M", _i64), ("K", _i64), ("dt", C.c_int), ("index_bytes", C.c_int)]


_sig("tcaspmm_layer_norm", [_vp, _i64, C.c_int, _vp, _i64, C.c_int, _vp, _vp, C.c_int, _vp, _vp, _i64, _i64, C.c_int,
                            C.c_double, _vp])
_sig("tcaspmm_layer_norm_backward_workspace", [_i64, _i64, C.c_int], C.c_size_t)
_sig("tcaspmm_layer_norm_backward", [_vp, _i64, C.c_int, _vp, _i64, C.c_int, _vp, _vp, _vp, C.c_int, _vp, _i64, _vp, _vp,
                                     _i64, _i64, C.c_int, _vp, C.c_size_t, _vp])
_sig("tcaspmm_lora", [C.POINTER(_Adapters), _vp, _i64, _i64, _vp, _i64, _vp, _i64, C.c_int, _vp, _vp])
_sig("tcaspmm_lora_backward", [C.POINTER(_Adapters), _vp, _i64, C.c_int, _vp, _i64, _i64, _vp, _vp, _i64, _vp, _i64, _vp,
                               _vp, _vp, _vp])


def _types() -> dict:
    if not _TYPES:
        import torch

        _TYPES.update({torch.float32: int(dtype.f32), torch.float16: int(dtype.f16), torch.bfloat16: int(dtype.bf16)})
    return _TYPES


def _code(t, name: str) -> int:
    c = _types().get(t.dtype)
    if c is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    return c


def _together(X, *others) -> None:
    """X and the (tensor or None, name) pairs lie on one CUDA device."""
    if not X.is_cuda:
        raise ValueError("X must be on a CUDA device")
    for t, name in others:
        if t is not None and t.device != X.device:
            raise ValueError(f"{name} is on {t.device}, not on {X.device}")


def _matrix(t, name: str):
    """(tensor with contiguous rows, leading dimension, type code)."""
    c = _code(t, name)
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, not {t.dim()}-D")
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, max(t.stride(0), cols), c


def _shape(t, name: str, shape: Tuple[int, ...]) -> None:
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")


class _Device:
    """The tensor's device made current for a launch, and its current stream."""

    __slots__ = ("device", "guard")

    def __init__(self, t):
        self.device = t.device

    def __enter__(self) -> int:
        import torch

        self.guard = None
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


# --------------------------------------------------------------- layer norm
def _norm_args(X, weight, bias, dim):
    if dim not in (0, 1, -1, -2):
        raise ValueError(f"dim must be 0 (columns) or 1 (rows), not {dim!r}")
    X, ldx, xt = _matrix(X, "X")
    dim = dim % 2
    n = X.shape[dim]
    if n == 0 and X.shape[1 - dim] > 0:
        raise ValueError("the normalised dimension is empty")
    pt = 0
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            pt = _code(t, name)
            _shape(t, name, (n,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one type, not {weight.dtype} and {bias.dtype}")
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    return X, ldx, xt, weight, bias, pt, dim


def layer_norm(X, weight=None, bias=None, eps: float = 1e-5, dim: int = 1, out_dtype=None, *, stats: bool = False):
    """Layer norm of each row of X (dim=1: a node's features) or of each column (dim=0: a token's features, the
    layout of a plan's B): weight * (x - mean) / sqrt(var + eps) + bias, stored as out_dtype (default: X's).

    weight and bias have one element per feature and one type (float32, float16 or bfloat16); None means 1 and 0.
    With stats, returns (Y, mean, rstd), the last two as layer_norm_backward takes them."""
    import torch

    X, ldx, xt, weight, bias, pt, dim = _norm_args(X, weight, bias, dim)
    out_dtype = X.dtype if out_dtype is None else out_dtype
    if out_dtype not in _types():
        raise ValueError(f"out_dtype must be float32, float16 or bfloat16, not {out_dtype}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, not {eps}")
    _together(X, (weight, "weight"), (bias, "bias"))
    rows, cols = X.shape
    Y = torch.empty((rows, cols), device=X.device, dtype=out_dtype)
    mean = rstd = None
    if stats:
        mean = torch.empty(X.shape[1 - dim], device=X.device, dtype=torch.float32)
        rstd = torch.empty_like(mean)
    with _Device(X) as stream:
        _check(lib.tcaspmm_layer_norm(X.data_ptr(), ldx, xt, Y.data_ptr(), cols, _types()[out_dtype],
                                      None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(),
                                      pt, mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None, rows, cols,
                                      dim, eps, stream))
    return (Y, mean, rstd) if stats else Y


def layer_norm_backward(dY, X, mean, rstd, weight=None, dim: int = 1, *, need_input: bool = True, need_weight: bool = True,
                        need_bias: bool = True, param_dtype=None):
    """(dX, dweight, dbias) of layer_norm from dY and the mean and rstd it returned; None for what is not needed.

    dX has X's type; dweight and dbias have weight's, or param_dtype (default float32) without one."""
    import torch

    X, ldx, xt, weight, _, pt, dim = _norm_args(X, weight, None, dim)
    dY, lddy, dyt = _matrix(dY, "dY")
    _shape(dY, "dY", tuple(X.shape))
    rows, cols = X.shape
    vecs, n = X.shape[1 - dim], X.shape[dim]
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _shape(t, name, (vecs,))
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name} must be the contiguous float32 tensor that layer_norm returned")
    if weight is None and param_dtype is not None:
        if param_dtype not in _types():
            raise ValueError(f"param_dtype must be float32, float16 or bfloat16, not {param_dtype}")
        pt = _types()[param_dtype]
    _together(X, (dY, "dY"), (mean, "mean"), (rstd, "rstd"), (weight, "weight"))
    pdt = weight.dtype if weight is not None else (param_dtype or torch.float32)
    dX = torch.empty((rows, cols), device=X.device, dtype=X.dtype) if need_input else None
    dw = torch.empty(n, device=X.device, dtype=pdt) if need_weight else None
    db = torch.empty(n, device=X.device, dtype=pdt) if need_bias else None
    with _Device(X) as stream:
        size = lib.tcaspmm_layer_norm_backward_workspace(rows, cols, dim) if need_weight or need_bias else 0
        ws = torch.empty(size, device=X.device, dtype=torch.uint8) if size else None
        _check(lib.tcaspmm_layer_norm_backward(
            dY.data_ptr(), lddy, dyt, X.data_ptr(), ldx, xt, mean.data_ptr(), rstd.data_ptr(),
            None if weight is None else weight.data_ptr(), pt, dX.data_ptr() if need_input else None, cols,
            dw.data_ptr() if need_weight else None, db.data_ptr() if need_bias else None, rows, cols, dim,
            ws.data_ptr() if size else None, size, stream))
    return dX, dw, db


# -------------------------------------------------------- low-rank adapters
def _adapters(X, down, up, index, scale):
    """Checked arguments: (X, ldx, adapters struct, tensors the struct points into)."""
    import torch

    X, ldx, xt = _matrix(X, "X")
    K, N = X.shape
    for t, name in ((down, "down"), (up, "up")):
        if t.dim() != 3:
            raise ValueError(f"{name} must be 3-D (adapters first), not {t.dim()}-D")
        if t.dtype != X.dtype:
            raise ValueError(f"{name} must have X's type {X.dtype}, not {t.dtype}")
    L, R, _ = down.shape
    M = up.shape[1]
    _shape(down, "down", (L, R, K))
    _shape(up, "up", (L, M, R))
    if not 1 <= R <= 256:
        raise ValueError(f"the rank must be between 1 and 256, not {R}")
    down, up = down.contiguous(), up.contiguous()
    if index is not None:
        _shape(index, "index", (N,))
        if index.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"index must be int32 or int64, not {index.dtype}")
        index = index.contiguous()
    if scale is not None:
        _shape(scale, "scale", (L,))
        if scale.dtype != torch.float32:
            raise ValueError(f"scale must be float32, not {scale.dtype}")
        scale = scale.contiguous()
    ad = _Adapters(down.data_ptr(), up.data_ptr(), None if index is None else index.data_ptr(),
                   None if scale is None else scale.data_ptr(), L, R, M, K, xt, 4 if index is None else index.element_size())
    return X, ldx, ad, (down, up, index, scale)


def lora(X, down, up, index=None, scale=None, base=None, *, out=None, hidden: bool = False):
    """base + scale[a] * up[a] @ (down[a] @ X[:, t]) for every column t, a = index[t]: the low-rank adapters of many
    requests beside a product C = A @ X (base = C, M x N, float32 or 16 bits; None = 0, float32 out).

    X: K x N; down: L x R x K and up: L x M x R, in X's type, R <= 256; index: int32 or int64, one per column, None =
    adapter 0 for all, a value outside [0, L) = no adapter (the column of base as it is); scale: float32, one per
    adapter, None = 1.  out: a tensor to write, base itself included.  With hidden, returns (Y, H) with the R x N
    float32 H = scale * down @ X as lora_backward takes it."""
    import torch

    X, ldx, ad, keep = _adapters(X, down, up, index, scale)
    M, N = ad.M, X.shape[1]
    ldb = 0
    out_dtype = torch.float32
    if base is not None:
        base, ldb, _ = _matrix(base, "base")
        _shape(base, "base", (M, N))
        out_dtype = base.dtype
    if out is not None:
        y, ldy, yt = _matrix(out, "out")
        _shape(out, "out", (M, N))
        if y is not out:
            raise ValueError("out must have contiguous rows")
        if base is not None and out.dtype != out_dtype:
            raise ValueError(f"out must have base's type {out_dtype}, not {out.dtype}")
    _together(X, (down, "down"), (up, "up"), (index, "index"), (scale, "scale"), (base, "base"), (out, "out"))
    if out is None:
        out = torch.empty((M, N), device=X.device, dtype=out_dtype)
        ldy, yt = N, _types()[out_dtype]
    H = torch.empty((ad.rank, N), device=X.device, dtype=torch.float32)
    with _Device(X) as stream:
        _check(lib.tcaspmm_lora(C.byref(ad), X.data_ptr(), ldx, N, None if base is None else base.data_ptr(), ldb,
                                out.data_ptr(), ldy, yt, H.data_ptr(), stream))
    return (out, H) if hidden else out


def lora_backward(dY, X, down, up, H, index=None, scale=None, base=None, *, need_input: bool = True, need_down: bool = True,
                  need_up: bool = True):
    """(dX, ddown, dup) of lora from dY and the H it returned, in X's type; None for what is not needed.

    base: a float32 K x N matrix that dX is added to (A^T @ dY), None = 0.  dY: float32, or X's type."""
    import torch

    X, ldx, ad, keep = _adapters(X, down, up, index, scale)
    K, N = X.shape
    dY, lddy, dyt = _matrix(dY, "dY")
    _shape(dY, "dY", (ad.M, N))
    if dY.dtype not in (torch.float32, X.dtype):
        raise ValueError(f"dY must be float32 or X's type {X.dtype}, not {dY.dtype}")
    if need_up:
        _shape(H, "H", (ad.rank, N))
        if H.dtype != torch.float32 or not H.is_contiguous():
            raise ValueError("H must be the contiguous float32 tensor that lora returned")
    ldb = 0
    if base is not None:
        if base.dtype != torch.float32:
            raise ValueError(f"base must be float32, not {base.dtype}")
        base, ldb, _ = _matrix(base, "base")
        _shape(base, "base", (K, N))
    _together(X, (dY, "dY"), (down, "down"), (up, "up"), (H, "H"), (index, "index"), (scale, "scale"), (base, "base"))
    dX = torch.empty((K, N), device=X.device, dtype=X.dtype) if need_input else None
    dD = torch.empty_like(keep[0]) if need_down else None
    dU = torch.empty_like(keep[1]) if need_up else None
    P = torch.empty((ad.rank, N), device=X.device, dtype=torch.float32) if need_input or need_down else None
    with _Device(X) as stream:
        _check(lib.tcaspmm_lora_backward(
            C.byref(ad), dY.data_ptr(), lddy, dyt, X.data_ptr(), ldx, N, H.data_ptr() if need_up else None,
            None if base is None else base.data_ptr(), ldb, dX.data_ptr() if need_input else None, N,
            dD.data_ptr() if need_down else None, dU.data_ptr() if need_up else None,
            None if P is None else P.data_ptr(), stream))
    return dX, dD, dU
