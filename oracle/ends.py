"""The ends of a model in 64 bits: embedding, RMSNorm, cross entropy, and their
gradients, with the magnitudes that bounds on rounding go by.
TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``)."""

from __future__ import annotations

import torch


def embedding(ids, table, scale=1.0):
    V = table.shape[0]
    has = (ids >= 0) & (ids < V)
    rows = table.double()[ids.clamp(0, V - 1)] * scale
    return torch.where(has[..., None], rows, 0.0)


def embedding_grad(ids, g, V, scale=1.0):
    """(dtable, sum of magnitudes, tokens of each row)."""
    ids, g = ids.reshape(-1), g.double().reshape(ids.numel(), -1)
    d, mag, count = (torch.zeros(V, n, dtype=torch.float64) for n in (g.shape[1], g.shape[1], 1))
    for i, t in enumerate(ids.tolist()):
        if 0 <= t < V:
            d[t] += g[i] * scale
            mag[t] += g[i].abs() * abs(scale)
            count[t] += 1
    return d, mag, count


def rms_norm(x, w, eps):
    x = x.double()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()


def rms_norm_grad(x, w, eps, g):
    """(dx, dw, the magnitudes of the terms of each)."""
    x, w, g = x.double(), w.double(), g.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    gw = g * w
    dx = r * (gw - x * r * (gw * x * r).mean(-1, keepdim=True))
    mx = r * (gw.abs() + (x * r).abs() * (gw * x * r).abs().mean(-1, keepdim=True))
    return dx, (g * x * r).sum(0), mx, (g * x * r).abs().sum(0)


def cross_entropy(h, w, targets, reduction="mean", g_loss=None, g_lse=None):
    """A dict: loss, lse, dh, dw, and what their errors go by: ``size`` [N], the largest sum of
    magnitudes behind a logit of the row; ``terms`` [N, V], |a| p + |b| on the target."""
    h, w = h.double(), w.double()
    N, V = h.shape[0], w.shape[0]
    x = h @ w.T
    lse = torch.logsumexp(x, 1)
    has = (targets >= 0) & (targets < V)
    at = targets.clamp(0, V - 1).long()[:, None]
    rows = torch.where(has, lse - x.gather(1, at)[:, 0], 0.0)
    count = max(int(has.sum()), 1)
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / count}[reduction]
    b = torch.zeros(N, dtype=torch.float64) if g_loss is None else g_loss.double().expand(N)
    b = torch.where(has, b / (count if reduction == "mean" else 1), 0.0)
    a = b if g_lse is None else b + g_lse.double()
    p = torch.softmax(x, 1)
    hot = torch.zeros_like(x).scatter_(1, at, 1.0)
    G = a[:, None] * p - b[:, None] * hot
    dead = (a == 0) & (b == 0)
    G[dead] = 0.0
    hz = torch.where(dead[:, None], 0.0, h)
    return {"loss": loss, "lse": lse, "dh": G @ w, "dw": G.T @ hz, "rows": rows, "hz": hz, "count": count,
            "size": (h.abs() @ w.abs().T).amax(1), "terms": a.abs()[:, None] * p + b.abs()[:, None] * hot}
