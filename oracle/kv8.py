"""The 8-bit K/V cache and the log probabilities in 64 bits, on the CPU.

A cache is a dict of CPU tensors: ``k``, ``v`` [B, H, L, D] float64 values on the
codes' grid (code, before its scale), ``ks``, ``vs`` [B, H, L / 64] float64
scales, ``mass`` [B, H, L].  Formulas: ``include/cirrus_b200.h``.
"""

from __future__ import annotations

import math

import torch

BLOCK = 64
QMAX = {"e4m3": 448.0, "int8": 127.0}
E_MIN, E_MAX = -100, 120


def need_exponent(absmax: float, fmt: str) -> int:
    """The smallest e with absmax <= qmax * 2^e, clamped."""
    if absmax == 0.0:
        return E_MIN
    e = math.frexp(absmax / QMAX[fmt])[1] - 2
    while absmax > math.ldexp(QMAX[fmt], e):
        e += 1
    return min(max(e, E_MIN), E_MAX)


def encode(y: torch.Tensor, fmt: str) -> torch.Tensor:
    """float64 y = x / scale -> the nearest code, ties to even, as float64.
    Infinities saturate; NaN stays in E4M3 and becomes 0 in int8."""
    q = QMAX[fmt]
    z = y.clamp(-q, q)
    if fmt == "int8":
        return torch.where(y.isnan(), torch.zeros_like(y), z.round())
    _, x = torch.frexp(z)
    step = torch.ldexp(torch.ones_like(z), (x - 4).clamp(min=-9))
    return ((z / step).round() * step).clamp(-q, q)


def block_absmax(x: torch.Tensor) -> float:
    fine = x[torch.isfinite(x)]
    return float(fine.abs().max()) if fine.numel() else 0.0


def append(c: dict, fmt: str, k, v, pos: list, counts: list) -> None:
    """Tokens k, v float64 [B, T, H, D] into the cache, in place."""
    B, H, L, _ = c["k"].shape
    for b in range(B):
        if pos[b] < 0:
            continue
        end = min(pos[b] + counts[b], L)
        if end > pos[b]:
            c["mass"][b, :, pos[b]:end] = 0.0
        for new, codes, scales in ((k, c["k"], c["ks"]), (v, c["v"], c["vs"])):
            for blk in range(pos[b] // BLOCK, -(-end // BLOCK)):
                lo, hi = max(pos[b], blk * BLOCK), min(end, (blk + 1) * BLOCK)
                if lo >= hi:
                    continue
                for h in range(H):
                    x = new[b, lo - pos[b]:hi - pos[b], h]
                    e = need_exponent(block_absmax(x), fmt)
                    if lo > blk * BLOCK:
                        was = float(scales[b, h, blk])
                        e = max(e, int(math.log2(was)))
                        if math.ldexp(1.0, e) > was:
                            old = codes[b, h, blk * BLOCK:lo]
                            codes[b, h, blk * BLOCK:lo] = encode(old * (was / math.ldexp(1.0, e)), fmt)
                    scales[b, h, blk] = math.ldexp(1.0, e)
                    codes[b, h, lo:hi] = encode(x / math.ldexp(1.0, e), fmt)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return (codes.unflatten(-2, (-1, BLOCK)) * scales[..., None, None]).flatten(-3, -2)


def attend(c: dict, q, pos: list, counts: list, scale: float, add_mass: bool = False) -> tuple:
    """q float64 [B, T, Hq, D] -> (out, lse, size): ``size`` is the largest
    sum |q_i k_i| * scale of a visible pair of each row, which bounds the error of its scores."""
    B, T, Hq, D = q.shape
    H, L = c["k"].shape[1:3]
    G = Hq // H
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64)
    size = torch.zeros(B, T, Hq, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            n = min(max(pos[b] + counts[b], 0), L)
            if n == 0:
                continue
            k = values(c["k"][b, h], c["ks"][b, h])[:n]
            v = values(c["v"][b, h], c["vs"][b, h])[:n]
            for t in range(counts[b]):
                m = min(pos[b] + t + 1, n)
                if m <= 0:
                    continue
                for i in range(h * G, (h + 1) * G):
                    x = k[:m] @ q[b, t, i] * scale
                    lse[b, t, i] = torch.logsumexp(x, 0)
                    p = torch.exp(x - lse[b, t, i])
                    out[b, t, i] = p @ v[:m]
                    size[b, t, i] = (k[:m].abs() @ q[b, t, i].abs()).max() * abs(scale)
                    if add_mass:
                        c["mass"][b, h, :m] += p
    return out, lse, size


def evict(c: dict, fmt: str, pos: list, keep: int, recent: int) -> tuple:
    """In place; returns (kept [B, H, keep] with -1 past shorter sequences, new positions)."""
    B, H = c["k"].shape[:2]
    kept = torch.full((B, H, keep), -1, dtype=torch.int64)
    for b in range(B):
        for h in range(H):
            n = pos[b]
            if n <= keep:
                kept[b, h, :max(n, 0)] = torch.arange(max(n, 0))
                continue
            w = c["mass"][b, h].tolist()
            rank = sorted(range(n - recent), key=lambda j: (-w[j] if w[j] == w[j] else math.inf, w[j] != w[j], j))
            pick = torch.tensor(sorted(rank[:keep - recent]) + list(range(n - recent, n)))
            kept[b, h] = pick
            c["mass"][b, h, :keep] = c["mass"][b, h, pick].clone()
            for codes, scales in ((c["k"], c["ks"]), (c["v"], c["vs"])):
                x = values(codes[b, h], scales[b, h])[pick]
                for blk in range(-(-keep // BLOCK)):
                    part = x[blk * BLOCK:(blk + 1) * BLOCK]
                    s = math.ldexp(1.0, need_exponent(block_absmax(part), fmt))
                    scales[b, h, blk] = s
                    codes[b, h, blk * BLOCK:blk * BLOCK + part.shape[0]] = encode(part / s, fmt)
    return kept, [min(max(n, 0), keep) for n in pos]


def token_logprobs(x: torch.Tensor, tokens: list, top: int) -> tuple:
    """x float64 [R, V] -> (logprob, entropy, rank, top_logprob, top_token)."""
    d = x - x.amax(-1, keepdim=True)  # first: the sum's logarithm would be lost next to a logit of 1e38
    logp = d - d.exp().sum(-1, keepdim=True).log()
    entropy = torch.special.entr(logp.exp()).sum(-1)
    logprob = torch.tensor([0.0 if t < 0 else float(logp[r, t]) for r, t in enumerate(tokens)], dtype=torch.float64)
    rank = torch.tensor([-1 if t < 0 else int((x[r] > x[r, t]).sum()) for r, t in enumerate(tokens)])
    at = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return logprob, entropy, rank, logp.gather(1, at), at
