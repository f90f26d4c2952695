"""RMSNorm of rows, and its gradient (``cb_rms_norm``, ``cb_rms_norm_grad``).

    y = rms_norm(x, weight, eps=1e-6)

The reference's ``RMSNorm`` (``cirrus/model/layers.py:33-44``); inside the decode path it
is fused into the products that follow.
"""

from __future__ import annotations

import torch

from cirrus_s_1a_b200 import _rows
from cirrus_s_1a_b200.kv8 import DTYPES


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` for the rows of ``x`` [rows, d] (float32,
    bfloat16 or float16, rows at any distance) and ``weight`` [d] (float32 or x's type),
    in x's type; gradients in x's and the weight's.  Runs on the current stream."""
    if _rows.wants_grad(x, weight):
        return _RMSNorm.apply(x, weight, float(eps))
    return _norm(x, weight, float(eps))


def _arguments(x, weight) -> tuple:
    """(rows, columns, elements between rows, both type codes)"""
    R, D, ld, code = _rows.matrix(x, "x")
    if weight.shape != (D,) or weight.device != x.device or not weight.is_contiguous() \
            or weight.dtype not in (torch.float32, x.dtype):
        raise ValueError(f"weight must be contiguous, float32 or {x.dtype}, [{D}] on {x.device}")
    return R, D, ld, code, DTYPES[weight.dtype]


def _norm(x, weight, eps):
    R, D, ld, code, w_code = _arguments(x, weight)
    dev = x.device
    y = torch.empty(R, D, dtype=x.dtype, device=dev)
    if R:
        _rows.call(dev, "cb_rms_norm", x.data_ptr(), code, ld, weight.data_ptr(), w_code, R, D, eps, y.data_ptr())
    return y


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return _norm(x, weight, eps)

    @staticmethod
    def backward(ctx, g):
        _rows.once(g)
        x, weight = ctx.saved_tensors
        # of the tensors as they come back: hooks may have moved them in between
        R, D, ld, code, w_code = _arguments(x, weight)
        dev = x.device
        _rows.given(g, "the result's gradient", (R, D), x.dtype, dev)
        if R == 0:
            return torch.zeros_like(x), torch.zeros_like(weight), None
        g, ldg = _rows.upstream(g, D)
        dx, dw = torch.empty(R, D, dtype=x.dtype, device=dev), torch.empty_like(weight)
        scratch = _rows.scratch(dev, "cb_rms_norm_grad_scratch_bytes", (R, D), R, D)
        _rows.call(dev, "cb_rms_norm_grad", x.data_ptr(), code, ld, g.data_ptr(), ldg, weight.data_ptr(), w_code, R, D,
                   ctx.eps, dx.data_ptr(), dw.data_ptr(), scratch.data_ptr(), scratch.numel())
        return dx, dw, None
