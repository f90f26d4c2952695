"""The cross entropy's gradient where G takes more than one piece of the vocabulary (256 MiB
of G a piece): targets in every piece, a last piece that is smaller and dealt otherwise, dW
written in place and through scratch, whole and split along the rows.  The 64-bit values are
taken on the device."""

import pytest
import torch

from oracle import ends
from test_gpu_linear_ce import DEV, bounds, call, inputs

pytestmark = pytest.mark.gpu


def check_on_device(h, w, t, reduction="mean", g_loss=None, g_lse=None):
    if g_loss is None:
        g_loss = torch.ones(()) if reduction != "none" else torch.full((len(t),), 1.0 / len(t))
    h, w, t = h.to(DEV), w.to(DEV), t.to(DEV)
    g_loss, g_lse = g_loss.to(DEV), None if g_lse is None else g_lse.to(DEV)
    got = call(h, w, t, reduction, g_loss, g_lse)
    with torch.device(DEV):
        r = ends.cross_entropy(h, w, t, reduction, g_loss, g_lse)
        b = bounds(r, h, w, reduction)
    for n in ("loss", "lse", "dh", "dw"):
        err = (got[n].detach().double() - r[n]).abs()
        assert torch.isfinite(got[n]).all(), n
        assert (err <= b[n]).all(), (n, float((err / b[n].clamp(min=1e-300)).max()), float(err.max()))
    return got


#: (pair, N, V, d), with pieces x splits of dW on 148 SMs: 16896 + 16437; 23552 x 2 + 22897 (d odd: dW
#: through scratch); 16896 + 16437; 11008 x 2 + 10985; 16896 + 16437; 8448 x 3 + 7989, two splits;
#: 16640 + 16360; 10240 x 6 + 8561, four splits and then two; 16896 + 16437; 4864 x 6 + 3817, four and two
SHAPES = [(("bf16", "bf16"), 4300, 33333, 24), (("bf16", "bf16"), 4300, 70001, 25), (("f16", "f16"), 4300, 33333, 266),
          (("f16", "f16"), 9000, 33001, 24), (("f32", "f32"), 1500, 33333, 24), (("f32", "f32"), 4300, 33333, 25),
          (("f32", "f32"), 2100, 33000, 264), (("f32", "bf16"), 4300, 70001, 24), (("f32", "bf16"), 1500, 33333, 266),
          (("f32", "bf16"), 9000, 33001, 264)]


@pytest.mark.parametrize("pair,N,V,d", SHAPES)
def test_pieces_match_oracle(pair, N, V, d):
    h, w, t = inputs(N, V, d, pair, seed=N + V + d)
    t[-3:] = torch.tensor([V - 1, 0, V // 2])
    check_on_device(h, w, t)


@pytest.mark.parametrize("pair", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
def test_pieces_with_a_gradient_for_each_row_and_lse(pair):
    h, w, t = inputs(4300, 33333, 40, pair, seed=31)
    g = torch.Generator().manual_seed(32)
    check_on_device(h, w, t, "none", torch.randn(4300, generator=g), 0.1 * torch.randn(4300, generator=g))


@pytest.mark.parametrize("pair", [("f32", "f32"), ("f32", "bf16")])
def test_pieces_in_three_parts(pair):
    """A vocabulary row out of the two-part form's range."""
    h, w, t = inputs(2100, 33000, 40, pair, seed=33)
    w[20000] *= 1e-9
    check_on_device(h, w, t, "sum", torch.full((), 1e-3))


@pytest.mark.parametrize("pair", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
def test_pieces_have_the_same_bits_whatever_memory_held(pair):
    h, w, t = (x.to(DEV) for x in inputs(4300, 33333, 25, pair, seed=34))
    first = call(h, w, t, "mean", torch.ones(()))
    for fill in (float("nan"), 3e38):
        torch.full((1 << 28,), fill, device=DEV)  # 1 GiB, freed at once: what the next call's scratch holds
        again = call(h, w, t, "mean", torch.ones(()))
        for n in first:
            assert torch.equal(first[n], again[n]), n
