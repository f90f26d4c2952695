"""What the ends of a model are timed on: the embedding lookup, the RMSNorm and the
cross entropy over the vocabulary, each with its gradient.

``listed()`` gives the cases, ``draw`` more of the same ranges, ``prepare`` a case's
inputs, ``run`` one pass.  With ``own`` false a pass is the operator in plain torch
operations, held in 32 bits; with ``own`` true it is the call a user makes:
``linear_cross_entropy`` of ``cirrus_s_1a_b200.loss``, ``embedding`` of
``cirrus_s_1a_b200.embedding`` and ``rms_norm`` of ``cirrus_s_1a_b200.norm``, and
``torch.autograd.grad`` for the gradient.  ``exact`` restates each in 64 bits.

The cross entropy: x = h W^T for hidden rows h [N, d] and the vocabulary's rows
W [V, d]; lse_n = log sum_v exp x_nv; loss_n = lse_n - x_n,target(n), 0 where the
row has no target (a negative one); reduced to the mean over the rows that have one,
or kept per row.  The embedding: scale * table[ids], a zero row for a negative id.
The norm: x * rsqrt(mean(x^2) + eps) * weight.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the log likelihood of a verify step's 1 + 4 tokens over the benchmark's vocabulary: latency, and one read of W
        {"name": "loss 5 rows", "op": "loss", "N": 5, "V": 32000, "d": 768, "hidden": "bf16", "weight": "bf16",
         "grad": False, "reduce": "none", "masked": 0.0},
        # one 128-token chunk of the engine's float32 hidden states against its head (exact in bf16)
        {"name": "loss chunk of 128 f32", "op": "loss", "N": 128, "V": 32000, "d": 768, "hidden": "f32",
         "weight": "bf16", "grad": False, "reduce": "none", "masked": 0.0},
        # evaluation of a long text, no gradient
        {"name": "loss 16K rows", "op": "loss", "N": 16384, "V": 32000, "d": 768, "hidden": "bf16", "weight": "bf16",
         "grad": False, "reduce": "mean", "masked": 0.0},
        # a step of the draft head (8192 likely tokens) on an odd number of rows, a third of them without a target
        {"name": "loss+grad draft 1001", "op": "loss", "N": 1001, "V": 8192, "d": 768, "hidden": "f16",
         "weight": "f16", "grad": True, "reduce": "mean", "masked": 0.33},
        # a full training step's head: the largest
        {"name": "loss+grad 16K rows", "op": "loss", "N": 16384, "V": 32000, "d": 768, "hidden": "bf16",
         "weight": "bf16", "grad": True, "reduce": "mean", "masked": 0.0},
        # the larger preset in float32, prompts without targets, a gradient of its own for each row
        {"name": "loss+grad 4095 f32", "op": "loss", "N": 4095, "V": 32768, "d": 1024, "hidden": "f32",
         "weight": "f32", "grad": True, "reduce": "none", "masked": 0.25},
        # the lookup of a verify step's tokens
        {"name": "embed 5", "op": "embed", "N": 5, "V": 32000, "d": 768, "dtype": "bf16", "scale": 1.0, "grad": False,
         "padded": 0.0},
        # a training step's lookup and its gradient: tokens of a text, the frequent ones many times
        {"name": "embed+grad 16K", "op": "embed", "N": 16384, "V": 32000, "d": 768, "dtype": "bf16", "scale": 1.0,
         "grad": True, "padded": 0.0},
        # a large batch in float32, scaled by sqrt(d), with padding
        {"name": "embed+grad 131K f32", "op": "embed", "N": 131072, "V": 32768, "d": 1024, "dtype": "f32",
         "scale": 32.0, "grad": True, "padded": 0.1},
        # the final norm of a verify step
        {"name": "norm 5", "op": "norm", "N": 5, "d": 768, "dtype": "f32", "weight": "f32", "grad": False},
        # the final norm of a training step
        {"name": "norm+grad 16K", "op": "norm", "N": 16384, "d": 768, "dtype": "bf16", "weight": "f32", "grad": True},
        # an odd number of rows of the larger preset's width, in float32
        {"name": "norm+grad 65537 f32", "op": "norm", "N": 65537, "d": 1024, "dtype": "f32", "weight": "f32",
         "grad": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: (hidden, weight): one type for both, or float32 rows against a bf16 head
PAIRS = (("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"))


def draw(rng):
    op = rng.choice(("loss", "loss", "loss", "embed", "norm"))
    # the presets' widths, and any other
    d = rng.choice((64, 768, 1024, _log_int(rng, 16, 2048)))
    if op == "loss":
        V = rng.choice((512, 8192, 32000, 32768, _log_int(rng, 300, 200000)))
        hidden, weight = rng.choice(PAIRS)
        grad = rng.random() < 0.6
        cost = 16384 * 32000 * 768 // (5 if hidden == "f32" else 1)
        N = _log_int(rng, 1, max(1, min(16384, cost // (V * d))))
        return {"op": op, "N": N, "V": V, "d": d, "hidden": hidden, "weight": weight, "grad": grad,
                "reduce": rng.choice(("mean", "none")), "masked": rng.choice((0.0, 0.1, 0.5))}
    if op == "embed":
        N = _log_int(rng, 1, min(131072, 131072 * 1024 // d))
        return {"op": op, "N": N,
                "V": rng.choice((512, 32000, 32768, _log_int(rng, 100, min(200000, 131072 * 512 // d)))),
                "d": d, "dtype": rng.choice(tuple(TYPES)), "scale": rng.choice((1.0, math.sqrt(d))),
                "grad": rng.random() < 0.7, "padded": rng.choice((0.0, 0.2))}
    dtype = rng.choice(tuple(TYPES))
    return {"op": op, "N": _log_int(rng, 1, min(65536, 65536 * 1024 // d)), "d": d, "dtype": dtype,
            "weight": rng.choice(("f32", dtype)), "grad": rng.random() < 0.7}


# ----------------------------------------------------------------- inputs
def _frequencies(V):
    """How often the tokens of a text occur: the r-th most frequent one as 1 / (r + 2.7)."""
    p = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _text(N, V, g):
    below = _frequencies(V).cumsum(0).cuda()
    order = torch.randperm(V, generator=g, device="cuda")
    at = torch.searchsorted(below, torch.rand(N, generator=g, device="cuda", dtype=torch.float64))
    return order[at.clamp(max=V - 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    N, d = case["N"], case["d"]
    if case["op"] == "loss":
        V = case["V"]
        w = randn(V, d)
        targets = _text(N, V, g)
        # normed hidden rows of a trained model: towards the target's row, so that most of the probability lies on few
        # tokens (logits of a standard deviation near 2, the target's a few above)
        h = randn(N, d) + (8.0 * torch.rand(N, 1, generator=g, device="cuda") / math.sqrt(d)) * w[targets]
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        if case["masked"]:
            targets = targets.masked_fill(torch.rand(N, generator=g, device="cuda") < case["masked"], -1)
        s["h"] = h.to(TYPES[case["hidden"]])
        s["w"] = (w * (2.0 / math.sqrt(d))).to(TYPES[case["weight"]])
        s["targets"] = targets
        if case["grad"]:
            # what comes from above: 1 for the mean, or each row's own weight; in float16 as many times as there are
            # rows, the scale that a training loop puts on such a loss
            up = float(N) if case["hidden"] == "f16" else 1.0
            s["g"] = torch.full((), up, device="cuda") if case["reduce"] == "mean" else \
                torch.rand(N, generator=g, device="cuda") * (up / N)
        leaves = ("h", "w")
    elif case["op"] == "embed":
        V, t = case["V"], TYPES[case["dtype"]]
        ids = _text(N, V, g)
        if case["padded"]:
            ids = ids.masked_fill(torch.rand(N, generator=g, device="cuda") < case["padded"], -1)
        s |= {"ids": ids, "table": randn(V, d).mul_(0.02).to(t)}
        if case["grad"]:
            s["g"] = randn(N, d).to(t)
        leaves = ("table",)
    else:
        # a residual stream: rows of different sizes
        s["x"] = (randn(N, d) * torch.exp(randn(N, 1))).to(TYPES[case["dtype"]])
        s["weight_"] = (1 + 0.1 * randn(d)).to(TYPES[case["weight"]])
        if case["grad"]:
            s["g"] = randn(N, d).to(TYPES[case["dtype"]])
        leaves = ("x", "weight_")
    if own and case["grad"]:
        for n in leaves:
            s[n].requires_grad_(True)
    return s


# ------------------------------------------------------------------- runs
def run(s):
    if own:
        return _run_own(s)
    return {"loss": _loss, "embed": _embed, "norm": _norm}[s["op"]](s)


def _run_own(s):
    if s["op"] == "loss":
        from cirrus_s_1a_b200.loss import linear_cross_entropy

        r = linear_cross_entropy(s["h"], s["w"], s["targets"], reduction=s["reduce"])
        if not s["grad"]:
            return {"loss": r.loss, "lse": r.lse}
        dh, dw = torch.autograd.grad(r.loss, (s["h"], s["w"]), s["g"])
        return {"loss": r.loss.detach(), "lse": r.lse.detach(), "dh": dh, "dw": dw}
    if s["op"] == "embed":
        from cirrus_s_1a_b200.embedding import embedding

        y = embedding(s["ids"], s["table"], s["scale"])
        return {"y": y.detach(), "dtable": torch.autograd.grad(y, s["table"], s["g"])[0]} if s["grad"] else {"y": y}
    from cirrus_s_1a_b200.norm import rms_norm

    y = rms_norm(s["x"], s["weight_"], EPS)
    if not s["grad"]:
        return {"y": y}
    dx, dw = torch.autograd.grad(y, (s["x"], s["weight_"]), s["g"])
    return {"y": y.detach(), "dx": dx, "dweight": dw}


# --------------------------------------------------- plain forms, 32 bits
def _loss(s):
    h, w, t = s["h"].float(), s["w"].float(), s["targets"]
    x = h @ w.T
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = (m + z.log())[:, 0]
    has = t >= 0
    at = t.clamp(min=0)[:, None]
    loss = torch.where(has, (m - x.gather(1, at) + z.log())[:, 0], torch.zeros_like(lse))
    count = has.sum()
    out = {"loss": loss.sum() / count.clamp(min=1) if s["reduce"] == "mean" else loss, "lse": lse}
    if not s["grad"]:
        return out
    g = s["g"] / count.clamp(min=1) if s["reduce"] == "mean" else s["g"]
    g = torch.where(has, g, torch.zeros_like(g))
    p = e.mul_((g[:, None] / z))
    rows = torch.arange(s["N"], device="cuda")
    p[rows, at[:, 0]] -= g
    return out | {"dh": (p @ w).to(s["h"].dtype), "dw": (p.T @ h).to(s["w"].dtype)}


def _embed(s):
    ids, table = s["ids"], s["table"]
    has = (ids >= 0)[:, None]
    y = torch.where(has, table.float()[ids.clamp(min=0)] * s["scale"], torch.zeros((), device="cuda"))
    out = {"y": y.to(table.dtype)}
    if s["grad"]:
        # a frequent token's rows are a long sum, which the card adds up in any order
        d = torch.zeros(table.shape, dtype=torch.float64, device="cuda")
        d.index_add_(0, ids.clamp(min=0), torch.where(has, s["g"].double() * s["scale"], 0.0))
        out["dtable"] = d.to(table.dtype)
    return out


def _norm(s):
    x, w = s["x"].float(), s["weight_"].float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * r
    out = {"y": (xh * w).to(s["x"].dtype)}
    if s["grad"]:
        g = s["g"].float()
        gw = g * w
        out["dx"] = (r * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(s["x"].dtype)
        out["dweight"] = (g * xh).sum(0).to(s["weight_"].dtype)
    return out


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if torch.is_tensor(v) else v for k, v in s.items()}
    if case["op"] == "loss":
        h, w = s["h"].double(), s["w"].double()
        N, t = case["N"], s["targets"]
        valid = t >= 0
        n_valid = max(int(valid.sum()), 1)
        per_row = torch.zeros(N, dtype=torch.float64, device="cuda")
        lse = torch.zeros_like(per_row)
        dh = torch.zeros_like(h) if case["grad"] else None
        dw = torch.zeros_like(w) if case["grad"] else None
        for a in range(0, N, 1024):
            b = min(a + 1024, N)
            logits = torch.mm(h[a:b], w.t())
            lse[a:b] = torch.logsumexp(logits, 1)
            sel = torch.nonzero(valid[a:b])[:, 0]
            per_row[a:b][sel] = lse[a:b][sel] - logits[sel, t[a:b][sel]]
            if case["grad"]:
                up = s["g"].double().expand(N)[a:b] / (n_valid if case["reduce"] == "mean" else 1)
                q = torch.softmax(logits, 1)
                q[sel, t[a:b][sel]] -= 1.0
                q = q * (up * valid[a:b])[:, None]
                dh[a:b] = torch.mm(q, w)
                dw += torch.mm(q.t(), h[a:b])
        out = {"loss": per_row.sum() / n_valid if case["reduce"] == "mean" else per_row, "lse": lse}
        return out | {"dh": dh, "dw": dw} if case["grad"] else out
    if case["op"] == "embed":
        ids, table = s["ids"], s["table"].double()
        real = torch.nonzero(ids >= 0)[:, 0]
        y = torch.zeros(case["N"], case["d"], dtype=torch.float64, device="cuda")
        y[real] = table.index_select(0, ids[real]) * case["scale"]
        if not case["grad"]:
            return {"y": y}
        # rows of one token next to each other, and differences of running sums at the borders of their runs
        order = torch.argsort(ids[real], stable=True)
        keys, counts = torch.unique_consecutive(ids[real][order], return_counts=True)
        ends = counts.cumsum(0)
        d = torch.zeros_like(table)
        for c in range(0, case["d"], 256):
            total = torch.cumsum(s["g"][real][order][:, c:c + 256].double(), 0)
            total = torch.cat((torch.zeros_like(total[:1]), total))
            d[keys, c:c + 256] = (total[ends] - total[ends - counts]) * case["scale"]
        return {"y": y, "dtable": d}
    x, w = s["x"].double(), s["weight_"].double()
    rms = (x.pow(2).sum(1, keepdim=True) / case["d"] + EPS).sqrt()
    y = x / rms * w
    if not case["grad"]:
        return {"y": y}
    g = s["g"].double()
    inner = (g * w * x).sum(1, keepdim=True) / case["d"]
    return {"y": y, "dx": g * w / rms - x * inner / rms.pow(3), "dweight": (g * (x / rms)).sum(0)}


# ------------------------------------------------------------------- work
def work(case):
    N, d = case["N"], case["d"]
    if case["op"] == "loss":
        V, sh, sw = case["V"], SIZE[case["hidden"]], SIZE[case["weight"]]
        both = N * d * sh + V * d * sw
        if not case["grad"]:
            return {"bytes": both + 16 * N, "flops": 2 * N * V * d}
        # the gradient's rows are those with a target; the logits are counted once
        live = max(1, round(N * (1 - case["masked"])))
        return {"bytes": 2 * both + 20 * N, "flops": 2 * N * V * d + 4 * live * V * d}
    if case["op"] == "embed":
        V, size = case["V"], SIZE[case["dtype"]]
        n = N * (1 - case["padded"])
        rows = float((1 - (1 - _frequencies(V)).pow(n)).sum())  # different tokens among n of a text
        once = 8 * N + rows * d * size + N * d * size
        grad = n * d * size + V * d * size if case["grad"] else 0
        return {"bytes": int(once + grad), "flops": int((2 if case["grad"] else 1) * n * d)}
    size = SIZE[case["dtype"]]
    once = 2 * N * d * size + d * SIZE[case["weight"]]
    if not case["grad"]:
        return {"bytes": once, "flops": 4 * N * d}
    # x is read once, for the row and for its gradient
    return {"bytes": once + 2 * N * d * size + d * SIZE[case["weight"]], "flops": 12 * N * d}
