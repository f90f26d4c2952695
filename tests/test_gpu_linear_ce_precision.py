"""What the cross entropy's results are off by, where a bound on single roundings tells."""

import math

import pytest
import torch

from oracle import ends
from test_gpu_linear_ce import call, half_step, inputs, smallest

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("pair", ["bf16", "f16"])
@pytest.mark.parametrize("N,V,d", [(1, 300, 64), (3, 2000, 768), (5, 33, 7), (40, 4100, 72), (128, 1000, 200)])
def test_gradients_of_few_16_bit_rows_are_rounded_once(pair, N, V, d):
    """Of up to 128 rows G is held in two parts of 16 bits: what is left out is the square of a
    half step (the second part is a half step of the first's remainder).  So beside the logits',
    lse's and sums' errors (as in ``test_gpu_linear_ce.bounds``) the result's own rounding is
    all; one part alone adds up to another half step of the terms."""
    h, w, t = inputs(N, V, d, (pair, pair), seed=N + V)
    up = torch.linspace(0.5, 1, N) * (1.0 if pair == "bf16" else 16.0)
    got = call(h.to(DEV), w.to(DEV), t.to(DEV), "none", up)
    r = ends.cross_entropy(h, w, t, "none", up)
    u = half_step(h.dtype) ** 2
    x = r["size"] * ((d / 8 + 8) * 2.0 ** -23 + 2.0 ** -22)
    lse = x + 2.0 ** -20 + r["lse"].abs() * 2.0 ** -23
    dG = r["terms"] * (u + 2.0 ** -20 + x[:, None] + lse[:, None])
    if pair == "f16":
        dG = dG + r["terms"].sum(1, keepdim=True) * 2.0 ** -37
    k = lambda K: (K / 8 + 8) * 2.0 ** -23  # noqa: E731
    for n, tol in (("dh", (dG + r["terms"] * k(V)) @ w.double().abs()), ("dw", (dG + r["terms"] * k(N)).T @ r["hz"].abs())):
        err = (got[n].cpu().double() - r[n]).abs()
        tol = tol * 1.01 + r[n].abs() * half_step(h.dtype) * (1 + half_step(h.dtype)) + smallest(h.dtype)
        assert (err <= tol).all(), (n, float((err / tol).max()))
