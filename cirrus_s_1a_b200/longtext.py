"""Scoring a long text from a bounded 8-bit cache: the log probability of every
token, with entropy and rank, while the shared K/V stays within a fixed number of
slots.

    cache = engine.new_cache(batch=1, max_ctx=4096 + 128, kv8="e4m3", add_mass=True)
    scores = score_text(engine, tokens, cache, keep=4096, recent=1024)

Each chunk of tokens runs through the model (``cb_forward_kv8``: append, attention
over the 8-bit cache, attention weights added up), its logits give the scores of
the tokens that follow (``token_logprobs``), and slots beyond ``keep`` are evicted
by their weight (``Kv8Cache.evict``).  A bf16 cache (``engine.new_cache()``) works
the same way without eviction, so the two scores of one text say what the 8 bits
and the bound cost.

Where only the mean counts, ``mean_loss`` gives it from the hidden states, without the
logits of a chunk.

    python -m cirrus_s_1a_b200.longtext --tokens 8192 --keep 2048

runs a model of random weights both ways and prints the comparison; ``--mean-only`` takes the
mean alone.

The reference scores a text through its training loss (``cirrus/model/model.py:176-228``).
"""

from __future__ import annotations

import argparse
import time
from dataclasses import replace

import torch

from cirrus_s_1a_b200 import _lib
from cirrus_s_1a_b200._lib import CB_PREFILL_CHUNK
from cirrus_s_1a_b200.logprobs import TokenLogprobs, token_logprobs


@torch.no_grad()
def score_text(engine, tokens: torch.Tensor, cache, keep: int | None = None, recent: int = 0, top: int = 0,
               chunk: int = CB_PREFILL_CHUNK) -> TokenLogprobs:
    """Scores ``tokens`` (int64 [B, N]) behind what ``cache`` holds: entry [b, t] is
    about token t + 1 given the tokens up to t (N - 1 of them; the arrays of
    ``TokenLogprobs`` with a leading [B, N - 1]).  ``keep`` (8-bit caches): after each
    chunk sequences are brought down to ``keep`` slots, the ``recent`` last among them.
    Reads the device status at the end (and synchronises): a token outside the vocabulary,
    a full cache or a wait that gave up is an error, with the status cleared."""
    B, N = tokens.shape
    if N < 2:
        raise ValueError("scoring needs at least two tokens")
    _check_eviction(cache, keep)
    ids = tokens.to(engine.device, torch.int64)
    vocab = engine.cfg.vocab_size
    follow = ids[:, 1:]
    follow = torch.where((follow >= 0) & (follow < vocab), follow, vocab).to(torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device=engine.device)
    parts, lengths = [], set()
    for t in range(0, N - 1, chunk):
        n = min(chunk, N - 1 - t)
        out = engine(ids[:, t:t + n], cache=cache)
        parts.append(token_logprobs(out.logits.flatten(0, 1), follow[:, t:t + n].reshape(-1).contiguous(), top,
                                    status))
        lengths.add(n)
        if keep is not None:
            cache.evict(keep, recent)
    _check_status(engine, cache, status, lengths, "score_text")
    return TokenLogprobs(*(torch.cat([x.unflatten(0, (B, -1)) for x in xs], 1) for xs in zip(*parts)))


@torch.no_grad()
def mean_loss(engine, tokens: torch.Tensor, cache, keep: int | None = None, recent: int = 0,
              chunk: int = CB_PREFILL_CHUNK) -> torch.Tensor:
    """The mean of -log p over what ``score_text`` scores, as a float32 scalar on the device
    (``CirrusB200.loss`` for each chunk); ``keep`` and errors as there."""
    B, N = tokens.shape
    if N < 2:
        raise ValueError("scoring needs at least two tokens")
    _check_eviction(cache, keep)
    ids = tokens.to(engine.device, torch.int64)
    status = torch.zeros(1, dtype=torch.int32, device=engine.device)
    total, lengths = torch.zeros((), dtype=torch.float64, device=engine.device), set()
    for t in range(0, N - 1, chunk):
        n = min(chunk, N - 1 - t)
        # (a token below 0 is one outside the vocabulary, as it is for the model)
        follow = ids[:, t + 1:t + 1 + n]
        follow = torch.where(follow < 0, engine.cfg.vocab_size, follow)
        total += engine.loss(ids[:, t:t + n], follow, cache, reduction="sum", status=status).loss
        lengths.add(n)
        if keep is not None:
            cache.evict(keep, recent)
    _check_status(engine, cache, status, lengths, "mean_loss")
    return (total / (B * (N - 1))).float()


def _check_eviction(cache, keep) -> None:
    if keep is not None and cache.kv8 is None:
        raise ValueError("keep needs an 8-bit shared cache (kv8=...)")
    if keep is not None and not cache.add_mass:
        raise ValueError("eviction goes by attention weights: a cache with add_mass=True")


def _check_status(engine, cache, status, lengths, what) -> None:
    rc = int(status) or next((r for r in (engine.read_status(cache, n) for n in lengths) if r), 0)
    for n in lengths if rc else ():
        engine.clear_status(cache, n)
    _lib.check(rc, what)


def main() -> None:
    from cirrus_s_1a_b200 import synthetic
    from cirrus_s_1a_b200.config import baseline_config
    from cirrus_s_1a_b200.engine import CirrusB200

    ap = argparse.ArgumentParser(description="score a synthetic text from a bf16 and from a bounded 8-bit cache")
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--keep", type=int, default=2048, help="slots of the 8-bit cache after each chunk")
    ap.add_argument("--recent", type=int, default=512, help="of them the last ones")
    ap.add_argument("--fmt", choices=("e4m3", "int8"), default="e4m3")
    ap.add_argument("--mean-only", action="store_true", help="the mean alone, without the logits")
    a = ap.parse_args()
    cfg = replace(baseline_config(), sparse_topk=None)
    engine = CirrusB200(cfg, synthetic.random_state_dict(cfg, seed=0), max_ctx=a.tokens + CB_PREFILL_CHUNK)
    text = torch.tensor([synthetic.random_prompt(a.tokens, cfg.vocab_size, seed=1)])
    caches = (("bf16", engine.new_cache(), None),
              (a.fmt, engine.new_cache(max_ctx=a.tokens + CB_PREFILL_CHUNK, kv8=a.fmt), None),
              (f"{a.fmt}, {a.keep} slots", engine.new_cache(max_ctx=a.keep + CB_PREFILL_CHUNK, kv8=a.fmt, add_mass=True),
               a.keep))
    first = None
    score = mean_loss if a.mean_only else score_text
    for name, cache, keep in caches:
        score(engine, text[:, :2 * CB_PREFILL_CHUNK], cache.clone(), keep=keep, recent=min(a.recent, keep or 0))
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        s = score(engine, text, cache, keep=keep, recent=min(a.recent, keep or 0))
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        if a.mean_only:
            print(f"{name:>18}: mean log p {-s:.5f}, {(a.tokens - 1) / dt:.0f} tokens/s")
            continue
        nbytes = cache.kv8.nbytes if cache.kv8 else 2 * cache.kv_k.numel() * 2
        first = s.logprob if first is None else first
        print(f"{name:>18}: mean log p {s.logprob.mean():.5f}, entropy {s.entropy.mean():.5f}, "
              f"largest difference to bf16 {(s.logprob - first).abs().max():.4f}, cache {nbytes / 2 ** 20:.1f} MiB, "
              f"{(a.tokens - 1) / dt:.0f} tokens/s")


if __name__ == "__main__":
    main()
