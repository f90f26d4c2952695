"""Failure detection of the cross entropy's products: a bounded wait that gives up.

The host shortens the limit and has one pair of CTAs bring nothing in
(``cb_linear_ce_set_wait_limit``), so that the pair's waits run out.  The kernel returns, the
context stays usable, the status word says so, and what would have come from the pair is NaN:
a caller without a status word sees it too."""

import pytest
import torch

from cirrus_s_1a_b200 import _lib
from test_gpu_linear_ce import DEV, PAIRS, call, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture
def stall():
    """stall(pair) from here on; off again at the end."""
    def set_to(pair):
        assert _lib.lib().cb_linear_ce_set_wait_limit(1_000_000 if pair else 0, pair) == 0

    yield set_to
    set_to(0)


def agree(got, want, names):
    """Equal where not NaN, and NaN somewhere."""
    for n in names:
        bad = got[n].isnan()
        assert bad.any(), n
        assert torch.equal(got[n][~bad], want[n][~bad]), n


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("N", [5, 300, 1100])  # as columns of the tiles, as rows, float32 in f16 parts
def test_a_wait_that_gives_up_gives_nan(pair, N, stall):
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    h, w, t = (x.to(DEV) for x in inputs(N, 3000, 72, pair, seed=N, masked=0.0))
    up = torch.ones(N)
    want = call(h, w, t, "none", up)
    mean = linear_cross_entropy(h, w, t).loss
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    stall(1)
    r = linear_cross_entropy(h, w, t, "none", status)
    assert int(status) == 8
    agree({"loss": r.loss, "lse": r.lse}, want, ("loss", "lse"))
    assert linear_cross_entropy(h, w, t).loss.isnan()  # no status word
    stall(0)
    hd, wd = h.detach().requires_grad_(), w.detach().requires_grad_()
    status.zero_()
    r = linear_cross_entropy(hd, wd, t, "none", status)
    stall(1)
    dh, dw = torch.autograd.grad(r.loss, (hd, wd), up.to(DEV))
    assert int(status) == 8
    agree({"dh": dh, "dw": dw}, want, ("dh", "dw"))
    stall(0)
    again = call(h, w, t, "none", up, status=status.zero_())
    assert int(status) == 0 and torch.equal(linear_cross_entropy(h, w, t).loss, mean)
    for n in want:
        assert torch.equal(again[n], want[n]), n
