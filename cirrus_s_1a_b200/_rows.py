"""Argument checks and the call shared by the operators at the ends of a model
(``embedding``, ``norm``, ``loss``): matrices of rows, token ids, the status word."""

from __future__ import annotations

import torch

from cirrus_s_1a_b200 import _lib
from cirrus_s_1a_b200.kv8 import _dtype, current_device, raw_stream


def matrix(t: torch.Tensor, name: str, device=None) -> tuple:
    """(rows, columns, elements between rows, type code) of a matrix with contiguous rows."""
    if t.dim() != 2 or not t.is_cuda:
        raise ValueError(f"{name} must be a matrix on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")
    R, D = t.shape
    if not 0 < D <= _lib.CB_ENDS_MAX_DIM or R > _lib.CB_ENDS_MAX_ROWS:
        raise ValueError(f"{name} must have 1 to {_lib.CB_ENDS_MAX_DIM} columns and at most {_lib.CB_ENDS_MAX_ROWS} rows")
    if R and D > 1 and t.stride(1) != 1:
        raise ValueError(f"a row of {name} must be contiguous")
    return R, D, t.stride(0) if R > 1 else D, _dtype(t, name)


def vocabulary(t: torch.Tensor, name: str, device=None) -> tuple:
    """``matrix`` of a table: rows at least their length apart, as many as ids may count."""
    V, D, ld, code = matrix(t, name, device)
    if not 0 < V <= _lib.CB_ENDS_MAX_VOCAB or ld < D:
        raise ValueError(f"{name} must have 1 to {_lib.CB_ENDS_MAX_VOCAB} rows, at least {D} elements apart")
    return V, D, ld, code


def upstream(g: torch.Tensor) -> torch.Tensor:
    """A gradient as the kernels read it: rows of any distance (0 where it was expanded), contiguous in themselves."""
    return g if g.stride(-1) == 1 or g.shape[-1] == 1 else g.contiguous()


def ids(t: torch.Tensor, name: str, device) -> int:
    """1 for int64 ids, 0 for int32."""
    if t.dtype not in (torch.int64, torch.int32) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int64 or int32 ids on {device}")
    if t.numel() > _lib.CB_ENDS_MAX_ROWS:
        raise ValueError(f"at most {_lib.CB_ENDS_MAX_ROWS} {name}")
    return int(t.dtype == torch.int64)


def status(t: torch.Tensor | None, device) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.shape != (1,) or t.device != device:
        raise ValueError(f"status must be an int32 tensor [1] on {device}")
    return t.data_ptr()


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def call(device, name: str, *args) -> None:
    """One entry point on ``device``'s current stream."""
    fn = getattr(_lib.lib(), name)
    if current_device() == device.index:
        rc = fn(*args, raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, raw_stream(device.index))
    if rc:
        _lib.check(rc, name)


def scratch(device, name: str, *shape) -> torch.Tensor:
    """Scratch of a call, from the stream's (or the capture's) own memory."""
    n = getattr(_lib.lib(), name)(*shape)
    if n == 0:
        raise _lib.CbError(f"{name}: shape not supported")
    return torch.empty(n, dtype=torch.uint8, device=device)
