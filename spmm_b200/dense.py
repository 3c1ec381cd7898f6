"""Dense operators around a sparse product: layer norm and low-rank adapters.

``layer_norm`` and ``lora`` are differentiable torch operators (``torch.ops.tcaspmm.layer_norm`` and
``lora``, in C++ over the C-ABI: ``spmm_b200/lib/libtcaspmm_torch.so``); the other two are their
gradients as plain calls.  They launch on the current stream of the tensors' device.  A matrix argument
may be any 2-D CUDA tensor of float32, float16 or bfloat16; one whose rows are not contiguous is copied
first.  There is no CPU or PyTorch fallback: without a CUDA device the calls raise.
"""
from __future__ import annotations

import ctypes as C
import os

from . import LIB_DIR, _sig, as_dtype, lib

TORCH_PATH = os.path.join(LIB_DIR, "libtcaspmm_torch.so")
_vp, _i64 = C.c_void_p, C.c_int64


class _Adapters(C.Structure):
    _fields_ = [("down", _vp), ("up", _vp), ("index", _vp), ("scale", _vp), ("count", _i64), ("rank", _i64),
                ("M", _i64), ("K", _i64), ("dt", C.c_int), ("index_bytes", C.c_int)]


_sig("tcaspmm_layer_norm", [_vp, _i64, C.c_int, _vp, _i64, C.c_int, _vp, _vp, C.c_int, _vp, _vp, _i64, _i64, C.c_int,
                            C.c_double, _vp])
_sig("tcaspmm_layer_norm_backward_workspace", [_i64, _i64, C.c_int], C.c_size_t)
_sig("tcaspmm_layer_norm_backward", [_vp, _i64, C.c_int, _vp, _i64, C.c_int, _vp, _vp, _vp, C.c_int, _vp, _i64, _vp, _vp,
                                     _i64, _i64, C.c_int, _vp, C.c_size_t, _vp])
_sig("tcaspmm_lora_hidden_bytes", [_i64, _i64, _i64, _i64, _i64, C.c_int, C.c_int], C.c_size_t)
_sig("tcaspmm_lora", [C.POINTER(_Adapters), _vp, _i64, _i64, _vp, _i64, _vp, _i64, C.c_int, _vp, C.c_int, _vp])
_sig("tcaspmm_lora_backward", [C.POINTER(_Adapters), _vp, _i64, C.c_int, _vp, _i64, _i64, _vp, _vp, _i64, _vp, _i64, _vp,
                               _vp, _vp, _vp])

_OPS: dict = {}


def hidden_bytes(count: int, rank: int, M: int, K: int, N: int, dt) -> int:
    """Size of the buffer that lora returns with hidden."""
    return lib.tcaspmm_lora_hidden_bytes(count, rank, M, K, N, int(as_dtype(dt)), 1)


def _op(name: str):
    """The torch operator; the first call loads the library and registers the operators' shapes (for tracing)."""
    if not _OPS:
        import torch

        if not os.path.exists(TORCH_PATH):
            raise ImportError(f"{TORCH_PATH} is missing: build it with `make -C spmm_b200/csrc torch`")
        torch.ops.load_library(TORCH_PATH)
        _register_shapes()
        for k in ("layer_norm", "layer_norm_stats", "layer_norm_backward", "lora", "lora_hidden", "lora_into", "lora_backward"):
            _OPS[k] = getattr(torch.ops.tcaspmm, k).default
    return _OPS[name]


def _register_shapes() -> None:
    import torch

    fake = torch.library.register_fake

    def hidden(X, up):
        return X.new_empty(hidden_bytes(up.shape[0], up.shape[2], up.shape[1], X.shape[0], X.shape[1], X.dtype), dtype=torch.uint8)

    @fake("tcaspmm::layer_norm")
    def _(X, weight, bias, eps, dim, out_dtype):
        return torch.empty(X.shape, dtype=out_dtype, device=X.device)

    @fake("tcaspmm::layer_norm_stats")
    def _(X, weight, bias, eps, dim, out_dtype):
        vecs = X.new_empty(X.shape[1 - dim % 2], dtype=torch.float32)
        return torch.empty(X.shape, dtype=out_dtype, device=X.device), vecs, torch.empty_like(vecs)

    @fake("tcaspmm::layer_norm_backward")
    def _(dY, X, mean, rstd, weight, dim, param_dtype, need_input, need_weight, need_bias):
        n = X.shape[dim]
        return (X.new_empty(X.shape if need_input else 0), X.new_empty(n if need_weight else 0, dtype=param_dtype),
                X.new_empty(n if need_bias else 0, dtype=param_dtype))

    @fake("tcaspmm::lora")
    def _(X, down, up, index, scale, base):
        return X.new_empty((up.shape[1], X.shape[1]), dtype=torch.float32 if base is None else base.dtype)

    @fake("tcaspmm::lora_hidden")
    def _(X, down, up, index, scale, base):
        return X.new_empty((up.shape[1], X.shape[1]), dtype=torch.float32 if base is None else base.dtype), hidden(X, up)

    @fake("tcaspmm::lora_into")
    def _(X, down, up, index, scale, base, out, keep=True):
        return hidden(X, up) if keep else X.new_empty(0, dtype=torch.uint8)

    @fake("tcaspmm::lora_backward")
    def _(dY, X, down, up, H, index, scale, base, need_input, need_down, need_up):
        return (X.new_empty(X.shape if need_input else 0), X.new_empty(down.shape if need_down else 0),
                X.new_empty(up.shape if need_up else 0))


# --------------------------------------------------------------- layer norm
def layer_norm(X, weight=None, bias=None, eps: float = 1e-5, dim: int = 1, out_dtype=None, *, stats: bool = False):
    """Layer norm of each row of X (dim=1: a node's features) or of each column (dim=0: a token's features, the
    layout of a plan's B): weight * (x - mean) / sqrt(var + eps) + bias, stored as out_dtype (default: X's).

    weight and bias have one element per feature and one type (float32, float16 or bfloat16); None means 1 and 0.
    Differentiable in X, weight and bias.  With stats, returns (Y, mean, rstd), the last two as layer_norm_backward
    takes them (and no autograd)."""
    return _op("layer_norm_stats" if stats else "layer_norm")(X, weight, bias, eps, dim, X.dtype if out_dtype is None else out_dtype)


def layer_norm_backward(dY, X, mean, rstd, weight=None, dim: int = 1, *, need_input: bool = True, need_weight: bool = True,
                        need_bias: bool = True, param_dtype=None):
    """(dX, dweight, dbias) of layer_norm from dY and the mean and rstd it returned; None for what is not needed.

    dX has X's type; dweight and dbias have weight's, or param_dtype (default float32) without one."""
    import torch

    if param_dtype is None:
        param_dtype = torch.float32 if weight is None else weight.dtype
    got = _op("layer_norm_backward")(dY, X, mean, rstd, weight, dim, param_dtype, need_input, need_weight, need_bias)
    return tuple(t if n else None for t, n in zip(got, (need_input, need_weight, need_bias)))


# -------------------------------------------------------- low-rank adapters
def lora(X, down, up, index=None, scale=None, base=None, *, out=None, hidden: bool = False):
    """base + scale[a] * up[a] @ (down[a] @ X[:, t]) for every column t, a = index[t]: the low-rank adapters of many
    requests beside a product C = A @ X (base = C, M x N, float32 or 16 bits; None = 0, float32 out).

    X: K x N; down: L x R x K and up: L x M x R, in X's type, R <= 256; index: int32 or int64, one per column, None =
    adapter 0 for all, a value outside [0, L) = no adapter (the column of base as it is); scale: float32, one per
    adapter, None = 1.  Differentiable in X, down, up and base.  out: a tensor to write, base itself included.  With
    hidden, returns (Y, H) with scale * down @ X as lora_backward takes it (an opaque buffer).  (No autograd with out or
    hidden.)"""
    if out is not None:
        H = _op("lora_into")(X, down, up, index, scale, base, out, hidden)
        return (out, H) if hidden else out
    return _op("lora_hidden" if hidden else "lora")(X, down, up, index, scale, base)


def lora_backward(dY, X, down, up, H, index=None, scale=None, base=None, *, need_input: bool = True, need_down: bool = True,
                  need_up: bool = True):
    """(dX, ddown, dup) of lora from dY and the H it returned, in X's type; None for what is not needed.

    base: a float32 K x N matrix that dX is added to (A^T @ dY), None = 0.  dY: float32, or X's type."""
    got = _op("lora_backward")(dY, X, down, up, H, index, scale, base, need_input, need_down, need_up)
    return tuple(t if n else None for t, n in zip(got, (need_input, need_down, need_up)))
