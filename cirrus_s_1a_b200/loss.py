"""Softmax cross entropy over the vocabulary from hidden rows, without keeping the
logits, and its gradient (``cb_linear_ce``, ``cb_linear_ce_grad``).

    r = linear_cross_entropy(hidden, weight, targets)      # hidden [N, d], weight [V, d]
    r.loss.backward()                                      # hidden.grad, weight.grad

Neither direction ever holds the [N, V] logits: the forward keeps each row's maximum and
sum, the backward takes the logits again for a piece of the vocabulary at a time.

The reference computes the same loss from its head's logits, in chunks
(``cirrus/model/model.py:176-228``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from cirrus_s_1a_b200 import _lib, _rows

REDUCTIONS = {"none": _lib.CB_REDUCE_NONE, "mean": _lib.CB_REDUCE_MEAN, "sum": _lib.CB_REDUCE_SUM}


class CrossEntropy(NamedTuple):
    loss: torch.Tensor  # float32: a scalar, or [N] with reduction "none" (0 where a row has no target)
    lse: torch.Tensor   # float32 [N]: log of each row's softmax sum (natural log)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, reduction: str = "mean",
                         status: torch.Tensor | None = None) -> CrossEntropy:
    """``logsumexp(x) - x[target]`` with ``x = hidden @ weight.T`` for ``hidden`` [N, d]
    and ``weight`` [V, d]: one type for both (float32, bfloat16 or float16), or float32
    against bfloat16.  ``targets`` int64 or int32 [N]; a negative one means the row has
    none.  ``reduction`` "mean" is over the rows that have a target (0 where none has).
    Both results are differentiable: ``r.loss + z * r.lse.square().mean()`` is a loss too.
    ``status`` (int32 [1] on the device) receives 6 when a target is outside the
    vocabulary, which then counts as none, and 8 when a bounded wait in a kernel gave up,
    which also makes the results that it would have gone into NaN.
    Runs on the current stream."""
    if _rows.wants_grad(hidden, weight):
        return CrossEntropy(*_LinearCE.apply(hidden, weight, targets, reduction, status))
    return CrossEntropy(*_forward(hidden, weight, targets, reduction, status, False)[:2])


def check_call(targets, reduction, status, device) -> tuple:
    """(1 for int64 targets, the reduction's code, the status word's address), or ValueError."""
    code = REDUCTIONS.get(reduction)
    if code is None:
        raise ValueError(f"unknown reduction {reduction!r}; choose from {sorted(REDUCTIONS)}")
    return _rows.ids(targets, "targets", device), code, _rows.status(status, device)


def _arguments(hidden, weight, targets, reduction, status) -> tuple:
    """The leading arguments of both entry points, and the status word's address."""
    N, D, ldh, h_code = _rows.matrix(hidden, "hidden")
    dev = hidden.device
    V, Dw, ldw, w_code = _rows.vocabulary(weight, "weight", dev)
    if Dw != D:
        raise ValueError(f"weight must have {D} columns as hidden, not {Dw}")
    if h_code != w_code and not (h_code == _lib.CB_F32 and w_code == _lib.CB_BF16):
        raise ValueError(f"hidden and weight must have one type, or float32 and bfloat16, not {hidden.dtype} and "
                         f"{weight.dtype}")
    if targets.shape != (N,):
        raise ValueError(f"targets must be [{N}]")
    wide, code, flag = check_call(targets, reduction, status, dev)
    return (hidden.data_ptr(), h_code, ldh, weight.data_ptr(), w_code, ldw, N, V, D, targets.data_ptr(), wide, code), flag


def _forward(hidden, weight, targets, reduction, status, rest) -> tuple:
    """(loss, lse, the number of targets and, with ``rest``, what rounding took off each lse)"""
    args, flag = _arguments(hidden, weight, targets, reduction, status)
    dev, N = hidden.device, args[6]
    lse = torch.empty(N, dtype=torch.float32, device=dev)
    if N == 0:
        return torch.zeros(() if reduction != "none" else 0, device=dev), lse, None
    loss = torch.empty(N if reduction == "none" else (), dtype=torch.float32, device=dev)
    if rest:
        args = (*args[:-1], args[-1] | _lib.CB_REDUCE_REST)
    n = 1 + N if rest else int(reduction != "none")
    count = torch.empty(n, dtype=torch.int32, device=dev) if n else None
    scratch = _scratch(dev, args, None, 0)
    _rows.call(dev, "cb_linear_ce", *args, loss.data_ptr(), lse.data_ptr(), _lib.ptr(count), scratch.data_ptr(),
               scratch.numel(), flag)
    return loss, lse, count


def _scratch(dev, args, dw, gradients) -> torch.Tensor:
    h, h_code, ldh, w, w_code, ldw, N, V, D = args[:9]
    at = None if dw is None else dw.data_ptr()
    # what the size goes by, beside the shape: which matrices can be read and written where they lie
    key = (h_code, w_code, N, V, D, ldh % 8, ldh >= D, ldw % 8, h % 16, w % 16, (at or 0) % 16, gradients)
    return _rows.scratch(dev, "cb_linear_ce_scratch_bytes", key, *args[:9], at, gradients)


class _LinearCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, reduction, status):
        loss, lse, count = _forward(hidden, weight, targets, reduction, status, True)
        ctx.save_for_backward(hidden, weight, targets, lse, count)
        ctx.reduction, ctx.status, ctx.like = reduction, status, (hidden.device, len(lse), weight.shape[0])
        ctx.set_materialize_grads(False)
        return loss, lse

    @staticmethod
    def backward(ctx, g_loss, g_lse):
        _rows.once(g_loss, g_lse)
        hidden, weight, targets, lse, count = ctx.saved_tensors
        want_h, want_w = ctx.needs_input_grad[:2]
        if g_loss is None and g_lse is None:
            return None, None, None, None, None
        # of the tensors as they come back: hooks may have moved them in between
        args, flag = _arguments(hidden, weight, targets, ctx.reduction, ctx.status)
        dev, (N, V, D) = hidden.device, args[6:9]
        if (dev, N, V) != ctx.like:  # which the gradients from above go with
            raise ValueError(f"the saved tensors must be of {ctx.like[1]} rows and {ctx.like[2]} of the vocabulary on "
                             f"{ctx.like[0]}, not {N} and {V} on {dev}")
        _rows.given(lse, "the saved lse", (N,), torch.float32, dev)
        _rows.given(count, "the saved number of targets", (1 + N,), torch.int32, dev)
        dh = torch.empty(N, D, dtype=hidden.dtype, device=dev) if want_h else None
        if N == 0:
            return dh, torch.zeros(V, D, dtype=weight.dtype, device=dev) if want_w else None, None, None, None
        dw = torch.empty(V, D, dtype=weight.dtype, device=dev) if want_w else None
        scratch = _scratch(dev, args, dw, want_h + 2 * want_w)
        lse, count = lse.contiguous(), count.contiguous()
        args = (*args[:-1], args[-1] | _lib.CB_REDUCE_REST)
        _rows.call(dev, "cb_linear_ce_grad", *args, lse.data_ptr(), count.data_ptr(), _lib.ptr(g_loss), _step(g_loss),
                   _lib.ptr(g_lse), _step(g_lse), _lib.ptr(dh), _lib.ptr(dw), scratch.data_ptr(), scratch.numel(),
                   flag)
        return dh, dw, None, None, None


def _step(g) -> int:
    """Elements between the rows of a gradient (0: one for all)."""
    return 0 if g is None or g.dim() == 0 else g.stride(0)
