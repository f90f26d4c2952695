"""Argument checks and the call shared by the operators at the ends of a model
(``embedding``, ``norm``, ``loss``): matrices of rows, token ids, the status word."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from cirrus_s_1a_b200 import _lib
from cirrus_s_1a_b200.kv8 import DTYPES, current_device, raw_stream


def matrix(t: torch.Tensor, name: str, device=None) -> tuple:
    """(rows, columns, elements between rows, type code) of a matrix with contiguous rows."""
    if t.dim() != 2 or not t.is_cuda:
        raise ValueError(f"{name} must be a matrix on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")
    R, D = t.shape
    if not 0 < D <= _lib.CB_ENDS_MAX_DIM or R > _lib.CB_ENDS_MAX_ROWS:
        raise ValueError(f"{name} must have 1 to {_lib.CB_ENDS_MAX_DIM} columns and at most {_lib.CB_ENDS_MAX_ROWS} rows")
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    ld, step = t.stride()
    if step != 1 and R and D > 1:
        raise ValueError(f"a row of {name} must be contiguous")
    return R, D, ld if R > 1 else D, code


def vocabulary(t: torch.Tensor, name: str, device=None) -> tuple:
    """``matrix`` of a table: rows at least their length apart, as many as ids may count."""
    V, D, ld, code = matrix(t, name, device)
    if not 0 < V <= _lib.CB_ENDS_MAX_VOCAB or ld < D:
        raise ValueError(f"{name} must have 1 to {_lib.CB_ENDS_MAX_VOCAB} rows, at least {D} elements apart")
    return V, D, ld, code


def upstream(g: torch.Tensor, D: int) -> tuple:
    """A gradient [rows, D] as the kernels read it, and the elements between its rows (0
    where one row was expanded); one whose rows are not contiguous is copied."""
    ld, step = g.stride()
    if step != 1 and D > 1:
        g = g.contiguous()
        ld = D
    return g, ld if g.shape[0] > 1 else D


def ids(t: torch.Tensor, name: str, device) -> int:
    """1 for int64 ids, 0 for int32."""
    wide = t.dtype == torch.int64
    if not (wide or t.dtype == torch.int32) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int64 or int32 ids on {device}")
    if t.numel() > _lib.CB_ENDS_MAX_ROWS:
        raise ValueError(f"at most {_lib.CB_ENDS_MAX_ROWS} {name}")
    return int(wide)


def status(t: torch.Tensor | None, device) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != (1,) or t.device != device:
        raise ValueError(f"status must be an int32 tensor [1] on {device}")
    return t.data_ptr()


def wants_grad(a: torch.Tensor, b: torch.Tensor | None = None) -> bool:
    """Whether results are to have a gradient; derivatives in forward mode are refused."""
    no_tangent(a, b)
    return (a.requires_grad or (b is not None and b.requires_grad)) and torch.is_grad_enabled()


def no_tangent(*tensors) -> None:
    if forward_ad._current_level < 0:  # outside of any dual level (0.4 us less a tensor than asking it)
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("this operator has no derivative in forward mode")


def once(*grads) -> None:
    """Called in a backward pass: what it returns has no derivative of its own."""
    if torch.is_grad_enabled():  # only under create_graph
        raise RuntimeError("the gradient of this operator is not differentiable (create_graph=True)")
    no_tangent(*grads)


def given(t: torch.Tensor | None, name: str, shape: tuple, dtype, device) -> None:
    """What a backward pass is handed or has kept has to be what goes with its other tensors:
    hooks on saved tensors may have given back another."""
    if t is not None and (t.shape != shape or t.dtype != dtype or t.device != device):
        raise ValueError(f"{name} must be {dtype} {list(shape)} on {device}, not {t.dtype} {list(t.shape)} on {t.device}")


_fns: dict = {}
_sizes: dict = {}


def call(device, name: str, *args) -> None:
    """One entry point on ``device``'s current stream."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.lib(), name)
    index = device.index
    if current_device() == index:
        rc = fn(*args, raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, raw_stream(index))
    if rc:
        _lib.check(rc, name)


def scratch(device, name: str, key: tuple, *args) -> torch.Tensor:
    """Scratch of a call, from the stream's (or the capture's) own memory; its size, which
    ``args`` give, is looked up by ``key``."""
    key = (name, device, key)
    n = _sizes.get(key)
    if n is None:
        with torch.cuda.device(device):
            n = getattr(_lib.lib(), name)(*args)
        if n == 0:
            raise _lib.CbError(f"{name}: shape not supported")
        if len(_sizes) >= 1024:  # a caller's rows may change with every call
            _sizes.clear()
        _sizes[key] = n
    return torch.empty(n, dtype=torch.uint8, device=device)
