"""Log probabilities of given tokens, with entropy, rank and top alternatives
(``cb_token_logprobs``), from the logits that a forward leaves on the device.

    r = token_logprobs(out.logits[0], tokens, top=5)
    r.logprob, r.entropy, r.rank, r.top_logprob, r.top_token

The reference computes the same log probabilities inside its loss
(``cirrus/model/model.py:176-228``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from cirrus_s_1a_b200 import _lib
from cirrus_s_1a_b200.kv8 import _dtype, raw_stream


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor      # float32 [rows]: log p(token); 0 where the row has none
    entropy: torch.Tensor      # float32 [rows]: -sum p log p
    rank: torch.Tensor         # int32 [rows]: how many tokens are likelier; -1 where the row has none
    top_logprob: torch.Tensor  # float32 [rows, top], descending
    top_token: torch.Tensor    # int32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   status: torch.Tensor | None = None) -> TokenLogprobs:
    """``logits`` [rows, vocab] (float32, bfloat16 or float16; rows at least ``vocab`` apart,
    or one row expanded), ``tokens`` int32 [rows] (negative: no token).  ``status`` (int32
    [1] on the logits' device) receives 6 when a token is outside the vocabulary.  Runs on
    the current stream."""
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits must be [rows, vocab] on a CUDA device")
    R, V = logits.shape
    if R and V > 1 and logits.stride(1) != 1:
        raise ValueError("a row of logits must be contiguous")
    if R > 1 and logits.stride(0) < V and logits.stride(0) != 0:
        raise ValueError(f"rows of logits must be at least {V} apart (or one row expanded)")
    if status is not None and (status.dtype != torch.int32 or status.shape != (1,) or status.device != logits.device):
        raise ValueError(f"status must be an int32 tensor [1] on {logits.device}")
    if tokens.dtype != torch.int32 or tokens.shape != (R,) or tokens.device != logits.device \
            or not tokens.is_contiguous():
        raise ValueError(f"tokens must be a contiguous int32 tensor [{R}] on {logits.device}")
    if not 0 <= top <= min(_lib.CB_LOGPROB_MAX_TOP, V):
        raise ValueError(f"top must be between 0 and {min(_lib.CB_LOGPROB_MAX_TOP, V)}")
    dtype = _dtype(logits, "logits")
    dev = logits.device
    r = TokenLogprobs(torch.empty(R, dtype=torch.float32, device=dev), torch.empty(R, dtype=torch.float32, device=dev),
                      torch.empty(R, dtype=torch.int32, device=dev),
                      torch.empty(R, top, dtype=torch.float32, device=dev),
                      torch.empty(R, top, dtype=torch.int32, device=dev))
    if R:
        L = _lib.lib()
        ld = logits.stride(0) if R > 1 else V
        args = (logits.data_ptr(), dtype, ld, R, V, tokens.data_ptr(), top, r.logprob.data_ptr(), r.entropy.data_ptr(),
                r.rank.data_ptr(), r.top_logprob.data_ptr(), r.top_token.data_ptr(), _lib.ptr(status),
                raw_stream(dev.index))
        if torch.cuda.current_device() == dev.index:
            rc = L.cb_token_logprobs(*args)
        else:
            with torch.cuda.device(dev):
                rc = L.cb_token_logprobs(*args)
        _lib.check(rc, "cb_token_logprobs")
    return r
