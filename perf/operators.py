"""What the 8-bit cache's operators and the log-probability operator are timed on.

``listed()`` gives the cases, ``draw`` more of the same ranges, ``prepare`` a
case's inputs, ``run`` one pass.  With ``own`` false a pass is the operator in
plain torch operations, held in 32 bits; with ``own`` true it is the call a user
makes: ``Kv8Cache.append`` / ``attend`` / ``evict`` of ``cirrus_s_1a_b200.kv8``
and ``token_logprobs`` of ``cirrus_s_1a_b200.logprobs``.  ``exact`` restates each
operator in 64 bits.

The cache: codes ``k``, ``v`` [batch, kv head, slot, dim] in 8 bits (E4M3 or
int8), and one scale, a power of two, for each block of 64 slots and head.  A
block's scale is the smallest 2^e with absmax <= qmax * 2^e (qmax 448 or 127); a
value is code * scale.  ``pos[b]`` slots are in use before a call.
"""

import math

import torch

own = False

BLOCK = 64
QMAX = {"e4m3": 448.0, "int8": 127.0}
E_MIN, E_MAX = -100, 120
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of one sequence joins a 32K context: a decode step's append, where latency is all
        {"name": "append 1x1 at 32K", "op": "append", "B": 1, "T": 1, "Hkv": 4, "D": 64, "past": 32700, "ragged": False,
         "fmt": "e4m3", "dtype": "f32"},
        # the prompts of sixteen sequences, of different lengths, written behind what they hold
        {"name": "append prompts 16x8192", "op": "append", "B": 16, "T": 8192, "Hkv": 2, "D": 128, "past": 1000,
         "ragged": True, "fmt": "int8", "dtype": "bf16"},
        # a decode step behind a 512-token prompt: the smallest call a user waits for
        {"name": "attend 1x1 at 512", "op": "attend", "B": 1, "T": 1, "Hq": 12, "Hkv": 4, "D": 64, "past": 511,
         "ragged": False, "fmt": "e4m3", "dtype": "f32", "weights": False},
        # a decode step of one sequence at 32K, the context the decode benchmark is quoted on
        {"name": "attend 1x1 at 32K", "op": "attend", "B": 1, "T": 1, "Hq": 12, "Hkv": 4, "D": 64, "past": 32767,
         "ragged": False, "fmt": "e4m3", "dtype": "bf16", "weights": False},
        # a verify step of 1 + 4 drafted tokens, sixteen sequences of up to 128K
        {"name": "attend 16x5 at 128K", "op": "attend", "B": 16, "T": 5, "Hq": 12, "Hkv": 4, "D": 64, "past": 131000,
         "ragged": True, "fmt": "int8", "dtype": "bf16", "weights": False},
        # a decode step of 64 sequences at 32K that also adds up each key's attention weight
        {"name": "attend+weights 64x1 at 32K", "op": "attend", "B": 64, "T": 1, "Hq": 6, "Hkv": 2, "D": 128,
         "past": 32000, "ragged": False, "fmt": "e4m3", "dtype": "f16", "weights": True},
        # a long prompt piece behind 28K tokens: bound by arithmetic
        {"name": "attend 1x4096 at 32K", "op": "attend", "B": 1, "T": 4096, "Hq": 12, "Hkv": 4, "D": 64, "past": 28600,
         "ragged": False, "fmt": "e4m3", "dtype": "bf16", "weights": False},
        # prompt pieces of an odd length, with the attention weights that eviction goes by
        {"name": "attend+weights 2x1000 at 8K", "op": "attend", "B": 2, "T": 1000, "Hq": 8, "Hkv": 2, "D": 128,
         "past": 7001, "ragged": True, "fmt": "int8", "dtype": "bf16", "weights": True},
        # one sequence's cache brought back to half after a chunk of 128 tokens
        {"name": "evict 1 of 16K", "op": "evict", "B": 1, "Hkv": 4, "D": 64, "n": 16512, "keep": 16384, "recent": 1024,
         "ragged": False, "fmt": "int8"},
        # many sequences brought down to half together
        {"name": "evict 32 of 64K", "op": "evict", "B": 32, "Hkv": 2, "D": 128, "n": 65536, "keep": 32768,
         "recent": 2048, "ragged": True, "fmt": "e4m3"},
        # the rows of a verify step of 1 + 4 tokens, with eight alternatives each
        {"name": "logprobs 5 rows", "op": "logprobs", "rows": 5, "V": 32000, "top": 8, "dtype": "f32"},
        # scoring a long text
        {"name": "logprobs 16K rows", "op": "logprobs", "rows": 16384, "V": 32000, "top": 20, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: (query heads, KV heads, head dim): the configurations' own, and one without shared heads, one with eight to a head
HEADS = ((12, 4, 64), (6, 2, 128), (8, 2, 128), (4, 2, 16), (4, 4, 32), (16, 2, 64))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "evict", "logprobs"))
    fmt = rng.choice(("e4m3", "int8"))
    Hq, Hkv, D = rng.choice(HEADS)
    ragged = rng.random() < 0.5
    if op == "append":
        T = rng.choice((1, rng.randint(2, 8), _log_int(rng, 9, 8192), _log_int(rng, 9, 8192)))
        past = rng.choice((0, _log_int(rng, 1, 32768)))
        most = max(1, min(64, 16 * 8192 * 256 // (Hkv * D * (T + past // 8 + 1))))
        return {"op": op, "B": _log_int(rng, 1, most), "T": T, "Hkv": Hkv, "D": D, "past": past, "ragged": ragged,
                "fmt": fmt, "dtype": rng.choice(tuple(TYPES))}
    if op == "attend":
        if rng.random() < 0.6:  # decode and verify steps
            T = rng.randint(1, 8)
            past = _log_int(rng, 1, 131072) - 1
            most = max(1, min(64, 16 * 131072 * 256 // ((past + T) * Hkv * D)))
            B = _log_int(rng, 1, most)
        else:  # prompt pieces
            T = _log_int(rng, 9, 4096)
            past = rng.choice((0, _log_int(rng, 1, 28000)))
            most = max(1, min(16, 4096 * 28600 * 12 * 64 // (T * (past + T) * Hq * D)))
            B = _log_int(rng, 1, most)
        return {"op": op, "B": B, "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "past": past, "ragged": ragged, "fmt": fmt,
                "dtype": rng.choice(tuple(TYPES)), "weights": rng.random() < 0.4}
    if op == "evict":
        n = _log_int(rng, 100, 65536)
        keep = max(1, int(n * rng.uniform(0.25, 0.99)))
        most = max(1, min(32, 32 * 65536 * 256 // (n * Hkv * D)))
        return {"op": op, "B": _log_int(rng, 1, most), "Hkv": Hkv, "D": D, "n": n, "keep": keep,
                "recent": rng.randint(0, keep), "ragged": ragged, "fmt": fmt}
    V = rng.choice((512, 8192, 32000, 32768, _log_int(rng, 300, 200000)))
    rows = _log_int(rng, 1, max(1, min(16384, 16384 * 32000 // V)))
    return {"op": op, "rows": rows, "V": V, "top": rng.randint(0, 20), "dtype": rng.choice(tuple(TYPES))}


# ----------------------------------------------------------------- inputs
def _lengths(case, g, top):
    """Slots in use of each sequence: ``top``, or lengths spread below it (the first at ``top``, one empty in four or more)."""
    B = case["B"]
    pos = torch.full((B,), top, dtype=torch.int32, device="cuda")
    if case["ragged"] and B > 1:
        r = torch.rand(B, generator=g, device="cuda")
        pos = (top * (0.25 + 0.75 * r)).to(torch.int32)
        pos[0] = top
        if B >= 4:
            pos[B // 2] = 0
    return pos


def _cache(case, g, slots):
    """A cache's tensors, filled as appends leave them: keys and values near N(0, 1), block scales a few octaves apart."""
    B, H, D = case["B"], case["Hkv"], case["D"]
    L = -(-slots // BLOCK) * BLOCK
    c = {}
    for name in ("k", "v"):
        codes = torch.empty(B, H, L, D, dtype=CODES[case["fmt"]], device="cuda")
        for b in range(B):
            x = torch.randn(H, L, D, generator=g, device="cuda")
            if case["fmt"] == "int8":
                codes[b] = x.mul_(32).round_().clamp_(-127, 127).to(torch.int8)
            else:
                codes[b] = x.mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn)
        c[name] = codes
        e = torch.randint(-7 if case["fmt"] == "e4m3" else -6, -4, (B, H, L // BLOCK), generator=g, device="cuda")
        c[name + "_scale"] = torch.exp2(e.float())
    c["mass"] = torch.rand(B, H, L, generator=g, device="cuda") ** 4
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "logprobs":
        R, V = case["rows"], case["V"]
        x = torch.empty(R, V, dtype=TYPES[case["dtype"]], device="cuda")
        for r in range(0, R, 4096):
            n = min(4096, R - r)
            # model logits: a few likely tokens over a broad floor, and some tokens that a grammar rules out
            x[r:r + n] = randn(n, V).mul_(2.5).to(x.dtype)
            x[r:r + n].masked_fill_(torch.rand(n, V, generator=g, device="cuda") < 0.01, -math.inf)
        tokens = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32)
        if R > 2:
            tokens[1] = -1  # a row without a token to score
        s |= {"logits": x, "tokens": tokens}
        return s
    if case["op"] == "append":
        B, T, H, D = case["B"], case["T"], case["Hkv"], case["D"]
        pos = _lengths(case, g, case["past"])
        s |= {"pos": pos, "counts": None}
        if case["ragged"]:
            s["counts"] = torch.randint(1, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        s |= _cache(case, g, case["past"] + T)
        # a projection's output holds keys and values side by side: strided views of it
        kv = randn(B, T, 2, H, D).to(TYPES[case["dtype"]])
        s |= {"k_new": kv[:, :, 0], "v_new": kv[:, :, 1]}
    elif case["op"] == "attend":
        B, T, D = case["B"], case["T"], case["D"]
        s |= _cache(case, g, case["past"] + T)
        s["pos"] = _lengths(case, g, case["past"])
        s["q"] = (1.5 * randn(B, T, case["Hq"], D)).to(TYPES[case["dtype"]])
    else:
        s |= _cache(case, g, case["n"])
        s["pos"] = _lengths(case, g, case["n"])
    if own:
        from cirrus_s_1a_b200.kv8 import Kv8Cache

        s["cache"] = Kv8Cache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"], s["mass"])
    return s


# ------------------------------------------------------------------- runs
def run(s):
    if own:
        return _run_own(s)
    return {"append": _append, "attend": _attend, "evict": _evict, "logprobs": _logprobs}[s["op"]](s)


def _state(s):
    return {n: s[n] for n in ("k", "v", "k_scale", "v_scale", "mass")}


def _run_own(s):
    if s["op"] == "logprobs":
        from cirrus_s_1a_b200.logprobs import token_logprobs

        r = token_logprobs(s["logits"], s["tokens"], top=s["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank, "top_logprob": r.top_logprob,
                "top_token": r.top_token}
    c = s["cache"]
    if s["op"] == "append":
        c.append(s["k_new"], s["v_new"], s["pos"], counts=s["counts"])
        return _state(s)
    if s["op"] == "attend":
        out, lse = c.attend(s["q"], s["pos"], add_mass=s["weights"])
        return {"out": out, "lse": lse} | ({"mass": s["mass"]} if s["weights"] else {})
    kept, pos = c.evict(s["pos"], s["keep"], s["recent"])
    return {"kept": kept, "pos": pos} | _state(s)


# --------------------------------------------------- plain forms, 32 bits
def _scale_of(absmax, fmt):
    """The smallest 2^e with absmax <= qmax * 2^e, as float32."""
    m, x = torch.frexp(absmax)
    top, shift = (0.875, 9) if fmt == "e4m3" else (127.0 / 128.0, 7)
    e = torch.where(m <= top, x - shift, x - shift + 1)
    e = torch.where(absmax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)
    return torch.ldexp(torch.ones_like(absmax), e)


def _encode(x, fmt):
    return (x.round() if fmt == "int8" else x).to(CODES[fmt])


def _append(s):
    B, T, H, D, fmt = s["B"], s["T"], s["Hkv"], s["D"], s["fmt"]
    L = s["k"].shape[2]
    pos = s["pos"].long()
    n = pos + (T if s["counts"] is None else s["counts"].long())
    slot = torch.arange(L, device="cuda")
    new = (slot >= pos[:, None]) & (slot < n[:, None])
    t = (slot - pos[:, None]).clamp(0, T - 1)
    old = slot < pos[:, None]
    for name in ("k", "v"):
        x = torch.gather(s[name + "_new"].float(), 1, t[:, :, None, None].expand(B, L, H, D)).transpose(1, 2)
        x = torch.where(new[:, None, :, None], x, torch.zeros_like(x))
        held = (s[name].float().view(B, H, L // BLOCK, BLOCK, D) * s[name + "_scale"][..., None, None]).view(B, H, L, D)
        need = _scale_of(x.abs().reshape(B, H, L // BLOCK, BLOCK * D).amax(-1), fmt)
        touched = new.view(B, 1, L // BLOCK, BLOCK).any(-1)
        begun = old.view(B, 1, L // BLOCK, BLOCK).any(-1)
        scale = torch.where(begun, torch.maximum(s[name + "_scale"], need), need)
        scale = torch.where(touched, scale, s[name + "_scale"])
        x = torch.where(new[:, None, :, None], x, held).view(B, H, L // BLOCK, BLOCK, D) / scale[..., None, None]
        put = ((new | old) & touched[:, 0].repeat_interleave(BLOCK, 1))[:, None, :, None]
        raw = _encode(x, fmt).view(B, H, L, D)
        s[name].copy_(torch.where(put, raw.view(torch.uint8), s[name].view(torch.uint8)).view(CODES[fmt]))
        s[name + "_scale"].copy_(scale)
    s["mass"].masked_fill_(new[:, None], 0.0)
    return _state(s)


def _attend(s):
    B, T, Hq, H, D = s["B"], s["T"], s["Hq"], s["Hkv"], s["D"]
    G, L = Hq // H, s["k"].shape[2]
    sight = s["pos"][:, None].long() + torch.arange(T, device="cuda")  # the last slot each row sees
    out = torch.empty(B, T, Hq, D, dtype=s["q"].dtype, device="cuda")
    lse = torch.empty(B, T, Hq, device="cuda")
    slot = torch.arange(L, device="cuda")
    step = max(1, int(2e9 // max(1, H * G * T * L)))
    for b0 in range(0, B, step):
        b = slice(b0, min(B, b0 + step))
        nb = b.stop - b.start
        q = s["q"][b].float().view(nb, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(nb, H, G * T, D)
        k = (s["k"][b].float().view(nb, H, -1, BLOCK, D) * s["k_scale"][b][..., None, None]).view(nb, H, L, D)
        x = (q * D ** -0.5) @ k.transpose(2, 3)
        x = x.view(nb, H, G, T, L).masked_fill_(slot > sight[b][:, None, None, :, None], -math.inf)
        top = x.amax(-1, keepdim=True)
        p = x.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        lse[b] = (top + total.log()).view(nb, Hq, T).transpose(1, 2)
        p.div_(total)
        if s["weights"]:
            s["mass"][b] += p.sum((2, 3))
        v = (s["v"][b].float().view(nb, H, -1, BLOCK, D) * s["v_scale"][b][..., None, None]).view(nb, H, L, D)
        o = (p.view(nb, H, G * T, L) @ v).view(nb, H, G, T, D)
        out[b] = o.permute(0, 3, 1, 2, 4).reshape(nb, T, Hq, D).to(out.dtype)
    return {"out": out, "lse": lse} | ({"mass": s["mass"]} if s["weights"] else {})


def _evict(s):
    B, H, D, fmt, keep, recent = s["B"], s["Hkv"], s["D"], s["fmt"], s["keep"], s["recent"]
    L = s["k"].shape[2]
    n = s["pos"].long()
    slot = torch.arange(L, device="cuda")
    # ranks: the recent slots first, then the older ones by weight (ties to the lowest slot), then what is not in use
    rank = torch.where(slot >= (n - recent)[:, None, None], math.inf, s["mass"])
    rank = torch.where(slot >= n[:, None, None], -math.inf, rank)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    over = n > keep
    kept = torch.where(over[:, None, None], kept, torch.arange(keep, device="cuda"))
    nb = -(-keep // BLOCK)
    at = torch.nn.functional.pad(kept, (0, nb * BLOCK - keep))
    live = (torch.arange(nb * BLOCK, device="cuda") < keep) & over[:, None, None]
    for name in ("k", "v"):
        x = (s[name].float().view(B, H, L // BLOCK, BLOCK, D) * s[name + "_scale"][..., None, None]).view(B, H, L, D)
        x = torch.gather(x, 2, at[..., None].expand(B, H, nb * BLOCK, D)) * live[..., None]
        scale = _scale_of(x.abs().view(B, H, nb, BLOCK * D).amax(-1), fmt)
        raw = _encode(x.view(B, H, nb, BLOCK, D) / scale[..., None, None], fmt).view(B, H, -1, D).view(torch.uint8)
        whole = s[name].view(torch.uint8)
        whole[:, :, :nb * BLOCK] = torch.where(live[..., None], raw, whole[:, :, :nb * BLOCK])
        s[name + "_scale"][:, :, :nb] = torch.where(over[:, None, None], scale, s[name + "_scale"][:, :, :nb])
    s["mass"][:, :, :keep] = torch.gather(s["mass"], 2, kept)
    kept = torch.where(kept < n[:, None, None], kept, -1).to(torch.int32)
    return {"kept": kept, "pos": n.clamp(max=keep).to(torch.int32)} | _state(s)


def _logprobs(s):
    R, V, top = s["rows"], s["V"], s["top"]
    got = {"logprob": torch.empty(R, device="cuda"), "entropy": torch.empty(R, device="cuda"),
           "rank": torch.empty(R, dtype=torch.int32, device="cuda"),
           "top_logprob": torch.empty(R, top, device="cuda"),
           "top_token": torch.empty(R, top, dtype=torch.int32, device="cuda")}
    step = max(1, (1 << 28) // V)
    for r0 in range(0, R, step):
        r = slice(r0, min(R, r0 + step))
        x = s["logits"][r].float()
        d = x - x.amax(-1, keepdim=True)
        p = d.exp()
        total = p.sum(-1, keepdim=True)
        logp = d - total.log()
        tok = s["tokens"][r].long()
        at = tok.clamp(min=0)[:, None]
        got["logprob"][r] = torch.where(tok >= 0, logp.gather(1, at)[:, 0], 0.0)
        got["rank"][r] = torch.where(tok >= 0, (x > x.gather(1, at)).sum(-1), -1).to(torch.int32)
        got["entropy"][r] = -(p / total * torch.where(p > 0, logp, 0.0)).sum(-1)
        if top:
            # ties go to the lowest token: a stable sort
            at = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]
            got["top_logprob"][r] = logp.gather(1, at)
            got["top_token"][r] = at.to(torch.int32)
    return got


# ------------------------------------------------------- 64 bits, from the definitions
def _value(codes, scale):
    return codes.to(torch.float64).unflatten(-2, (-1, BLOCK)) * scale.to(torch.float64)[..., None, None]


def _round64(y, fmt):
    """y (float64, within range) to the nearest value of the format, ties to even."""
    if fmt == "int8":
        return torch.round(y)
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.pow(torch.full_like(y, 2.0), e - 3)
    return torch.round(y / step) * step


def _pow2_64(absmax, fmt):
    e = torch.ceil(torch.log2(absmax.clamp(min=1e-300) / QMAX[fmt]))
    for d in (1, 0):  # log2 may be one off at a power of two
        lower = e - 1
        e = torch.where(absmax <= QMAX[fmt] * torch.pow(torch.full_like(e, 2.0), lower), lower, e)
        e = torch.where(absmax > QMAX[fmt] * torch.pow(torch.full_like(e, 2.0), e), e + d, e)
    e = torch.where(absmax > 0, e, torch.full_like(e, float(E_MIN))).clamp(E_MIN, E_MAX)
    return torch.pow(torch.full_like(e, 2.0), e)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict,
            "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_append(s):
    fmt, T = s["fmt"], s["T"]
    got = {"mass": s["mass"].double()}
    pos = s["pos"].tolist()
    counts = [T] * s["B"] if s["counts"] is None else s["counts"].tolist()
    for name in ("k", "v"):
        codes, scales = s[name].double(), s[name + "_scale"].double()
        for b in range(s["B"]):
            n0, n1 = pos[b], pos[b] + counts[b]
            got["mass"][b, :, n0:n1] = 0
            b0, b1 = n0 // BLOCK, -(-n1 // BLOCK)
            x = s[name + "_new"][b, :counts[b]].double().transpose(0, 1)
            full = torch.zeros(s["Hkv"], (b1 - b0) * BLOCK, s["D"], dtype=torch.float64, device="cuda")
            full[:, n0 - b0 * BLOCK:n1 - b0 * BLOCK] = x
            scale = _pow2_64(full.abs().unflatten(1, (-1, BLOCK)).amax((2, 3)), fmt)
            first = n0 - b0 * BLOCK
            if first:
                full[:, :first] = codes[b, :, b0 * BLOCK:n0] * scales[b, :, b0, None, None]
                scale[:, 0] = torch.maximum(scale[:, 0], scales[b, :, b0])
            rounded = _round64(full.unflatten(1, (-1, BLOCK)) / scale[..., None, None], fmt).flatten(1, 2)
            codes[b, :, b0 * BLOCK:n1] = rounded[:, :n1 - b0 * BLOCK]
            scales[b, :, b0:b1] = scale
        got[name], got[name + "_scale"] = (codes if fmt == "e4m3" else None), scales
    return got


def _exact_attend(s):
    B, T, Hq, H, D = s["B"], s["T"], s["Hq"], s["Hkv"], s["D"]
    G = Hq // H
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, T, Hq, dtype=torch.float64, device="cuda")
    mass = s["mass"].double()
    pos = s["pos"].tolist()
    for b in range(B):
        n = pos[b] + T
        below = torch.arange(n, device="cuda") <= pos[b] + torch.arange(T, device="cuda")[:, None]
        for h in range(H):
            k = _value(s["k"][b, h], s["k_scale"][b, h]).flatten(0, 1)[:n]
            v = _value(s["v"][b, h], s["v_scale"][b, h]).flatten(0, 1)[:n]
            for g in range(G):
                x = s["q"][b, :, h * G + g].double() @ k.t() / math.sqrt(D)
                x = torch.where(below, x, -math.inf)
                total = torch.logsumexp(x, -1)
                p = torch.exp(x - total[:, None])
                lse[b, :, h * G + g] = total
                out[b, :, h * G + g] = p @ v
                mass[b, h, :n] += p.sum(0)
    return {"out": out, "lse": lse} | ({"mass": mass} if s["weights"] else {})


def _exact_evict(s):
    fmt, keep, recent = s["fmt"], s["keep"], s["recent"]
    got = {"kept": None, "pos": None, "mass": s["mass"].double()}
    pos, w = s["pos"].tolist(), s["mass"].double().cpu().numpy()
    chosen = {}
    for b in range(s["B"]):
        for h in range(s["Hkv"]):
            if pos[b] <= keep:
                continue
            old = pos[b] - recent
            order = (-w[b, h, :old]).argsort(kind="stable")[:keep - recent]
            pick = torch.from_numpy(order).sort().values.to("cuda")
            chosen[b, h] = torch.cat([pick, torch.arange(old, pos[b], device="cuda")])
    for name in ("k", "v"):
        codes, scales = s[name].double() if fmt == "e4m3" else None, s[name + "_scale"].double()
        for (b, h), pick in chosen.items():
            x = _value(s[name][b, h], s[name + "_scale"][b, h]).flatten(0, 1)[pick]
            x = torch.cat([x, x.new_zeros(-keep % BLOCK, x.shape[1])]).unflatten(0, (-1, BLOCK))
            scale = _pow2_64(x.abs().amax((1, 2)), fmt)
            if codes is not None:
                codes[b, h, :keep] = _round64(x / scale[:, None, None], fmt).flatten(0, 1)[:keep]
            scales[b, h, :scale.numel()] = scale
        got[name], got[name + "_scale"] = codes, scales
    for (b, h), pick in chosen.items():
        got["mass"][b, h, :keep] = s["mass"][b, h, pick].double()
    return got


def _exact_logprobs(s):
    R, top = s["rows"], s["top"]
    f64 = dict(dtype=torch.float64, device="cuda")
    got = {"logprob": torch.zeros(R, **f64), "entropy": torch.zeros(R, **f64), "rank": None,
           "top_logprob": torch.zeros(R, top, **f64), "top_token": None}
    for r0 in range(0, R, 1024):
        r = slice(r0, min(R, r0 + 1024))
        x = s["logits"][r].double()
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        tok = s["tokens"][r].long()
        one = logp[torch.arange(x.shape[0], device="cuda"), tok.clamp(min=0)]
        got["logprob"][r] = torch.where(tok < 0, 0.0, one)
        got["entropy"][r] = torch.special.entr(logp.exp()).sum(-1)
        if top:
            got["top_logprob"][r] = logp.topk(top, -1).values
    return got


# ------------------------------------------------------------------ floors
def _pairs(case):
    """Visible (row, slot) pairs of one query head, and slots read, over the batch (ragged lengths at their mean)."""
    B, T, past = case["B"], case["T"], case["past"]
    if case["ragged"] and B > 1:
        rest = (B - 2 if B >= 4 else B - 1) * 0.625 * past
        total = past + rest
    else:
        total = B * past
    return T * total + B * T * (T + 1) / 2, total + B * T


def work(case):
    if case["op"] == "logprobs":
        R, V, top = case["rows"], case["V"], case["top"]
        return {"bytes": R * V * SIZE[case["dtype"]] + R * (16 + 8 * top), "flops": 5 * R * V}
    B, H, D = case["B"], case["Hkv"], case["D"]
    if case["op"] == "append":
        tokens = B * case["T"] * (0.5 if case["ragged"] else 1)
        return {"bytes": 2 * tokens * H * D * (SIZE[case["dtype"]] + 1) + 4 * tokens * H, "flops": 4 * tokens * H * D}
    if case["op"] == "attend":
        pairs, slots = _pairs(case)
        rows = B * case["T"] * case["Hq"]
        size = 2 * slots * H * D * (1 + 4 / (BLOCK * D)) + 2 * rows * D * SIZE[case["dtype"]] + 4 * rows
        return {"bytes": size + (8 * slots * H if case["weights"] else 0), "flops": 4 * pairs * case["Hq"] * D}
    n, keep = case["n"], case["keep"]
    share = 1.0
    if case["ragged"] and B > 1:  # sequences longer than keep, of lengths spread over the upper three quarters
        rest = (B - 2 if B >= 4 else B - 1) / B
        share = 1 / B + rest * min(1.0, max(0.0, (n - keep) / (0.75 * n)))
    tokens = share * B * H * keep
    return {"bytes": 4 * share * B * H * n + tokens * (2 * 2 * D + 8 + 4), "flops": 2 * tokens * D}
