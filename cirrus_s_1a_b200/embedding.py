"""Embedding lookup with scaling, and its gradient (``cb_embedding``,
``cb_embedding_grad``).

    y = embedding(ids, table, scale=1.0)       # ids.shape + (d,), in the table's type
    y.backward(g)                              # table.grad: the same bits every time

The reference looks tokens up with ``nn.Embedding`` (``cirrus/model/model.py:124``),
tied to its head.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from cirrus_s_1a_b200 import _rows


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * table[ids]`` for ``table`` [V, d] (float32, bfloat16 or float16; rows at
    least d apart) and contiguous int64 or int32 ``ids`` of any shape; a negative id gives
    a zero row and no gradient.  ``status`` (int32 [1] on the table's device) receives 6
    when an id is outside the table, which then counts as negative.  The table's gradient
    has its type, with sums in float32 in the order of the tokens.  Runs on the current
    stream."""
    _rows.vocabulary(table, "table")
    _rows.ids(ids, "ids", table.device)
    _rows.status(status, table.device)
    if _rows.wants_grad(table):
        return _Embedding.apply(ids, table, float(scale), status)
    return _lookup(ids, table, float(scale), status)


def _lookup(ids, table, scale, status):
    V, D, ld, code = _rows.vocabulary(table, "table")
    out = torch.empty(*ids.shape, D, dtype=table.dtype, device=table.device)
    if ids.numel():
        _rows.call(table.device, "cb_embedding", table.data_ptr(), code, ld, V, D, ids.data_ptr(),
                   _rows.ids(ids, "ids", table.device), ids.numel(), scale, out.data_ptr(),
                   _rows.status(status, table.device))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, status):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.shape, ctx.dtype = scale, table.shape, table.dtype
        return _lookup(ids, table, scale, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        ids, = ctx.saved_tensors
        V, D = ctx.shape
        n = ids.numel()
        if n == 0:
            return None, torch.zeros(V, D, dtype=ctx.dtype, device=ids.device), None, None
        g = g.reshape(n, D)
        g = _rows.upstream(g)
        out = torch.empty(V, D, dtype=ctx.dtype, device=ids.device)
        scratch = _rows.scratch(ids.device, "cb_embedding_grad_scratch_bytes", n, V, D)
        _, _, ldg, code = _rows.matrix(g, "the gradient")
        _rows.call(ids.device, "cb_embedding_grad", g.data_ptr(), code, ldg, ids.data_ptr(),
                   _rows.ids(ids, "ids", ids.device), n, V, D, ctx.scale, out.data_ptr(), scratch.data_ptr(),
                   scratch.numel())
        return None, out, None, None
