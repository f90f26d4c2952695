"""Embedding lookup with scaling, and its gradient (``cb_embedding``,
``cb_embedding_grad``).

    y = embedding(ids, table, scale=1.0)       # ids.shape + (d,), in the table's type
    y.backward(g)                              # table.grad: the same bits every time

The reference looks tokens up with ``nn.Embedding`` (``cirrus/model/model.py:124``),
tied to its head.
"""

from __future__ import annotations

import math

import torch

from cirrus_s_1a_b200 import _rows
from cirrus_s_1a_b200.kv8 import DTYPES


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * table[ids]`` for ``table`` [V, d] (float32, bfloat16 or float16; rows at
    least d apart), a finite ``scale`` and contiguous int64 or int32 ``ids`` of any shape; a
    negative id gives a zero row and no gradient.  ``status`` (int32 [1] on the table's
    device) receives 6 when an id is outside the table, which then counts as negative.  The
    table's gradient has its type, with sums in float32 in the order of the tokens.  Runs on
    the current stream."""
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, not {scale}")
    if _rows.wants_grad(table):
        return _Embedding.apply(ids, table, float(scale), status)
    return _lookup(ids, table, float(scale), status)


def _lookup(ids, table, scale, status):
    V, D, ld, code = _rows.vocabulary(table, "table")
    dev = table.device
    wide = _rows.ids(ids, "ids", dev)
    flag = _rows.status(status, dev)
    out = torch.empty(*ids.shape, D, dtype=table.dtype, device=dev)
    n = ids.numel()
    if n:
        _rows.call(dev, "cb_embedding", table.data_ptr(), code, ld, V, D, ids.data_ptr(), wide, n, scale, out.data_ptr(),
                   flag)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, status):
        ctx.save_for_backward(ids)
        ctx.args = scale, table.shape, table.dtype
        return _lookup(ids, table, scale, status)

    @staticmethod
    def backward(ctx, g):
        _rows.once(g)
        ids, = ctx.saved_tensors
        scale, (V, D), dtype = ctx.args
        n, dev = ids.numel(), g.device
        wide = _rows.ids(ids, "ids", dev)
        if n == 0:
            return None, torch.zeros(V, D, dtype=dtype, device=dev), None, None
        g, ldg = _rows.upstream(g.reshape(n, D), D)
        out = torch.empty(V, D, dtype=dtype, device=dev)
        scratch = _rows.scratch(dev, "cb_embedding_grad_scratch_bytes", (n, V, D), n, V, D)
        _rows.call(dev, "cb_embedding_grad", g.data_ptr(), DTYPES[dtype], ldg, ids.data_ptr(), wide, n, V, D, scale,
                   out.data_ptr(), scratch.data_ptr(), scratch.numel())
        return None, out, None, None
