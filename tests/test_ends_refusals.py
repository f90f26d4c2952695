"""CPU tests of what the operators at the ends of a model refuse, beside ``test_ends_host``."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from cirrus_s_1a_b200 import _rows
from test_host import built_lib  # noqa: F401


def test_wait_limit_refuses_a_negative_pair(built_lib):  # noqa: F811
    L = built_lib
    assert L.cb_linear_ce_set_wait_limit(0, -1) == 1 and L.cb_linear_ce_set_wait_limit(1000, 3) == 0
    assert L.cb_linear_ce_set_wait_limit(0, 0) == 0


def test_forward_mode_is_refused():
    """A tangent would be lost: no autograd function is entered where nothing requires grad."""
    from cirrus_s_1a_b200.embedding import embedding
    from cirrus_s_1a_b200.loss import linear_cross_entropy
    from cirrus_s_1a_b200.norm import rms_norm

    x, t, w = torch.ones(4, 8), torch.zeros(4, dtype=torch.int64), torch.ones(8)
    with fw.dual_level():
        dual, dual_w = fw.make_dual(x, torch.ones(4, 8)), fw.make_dual(w, torch.ones(8))
        for call in (lambda: embedding(t, dual), lambda: rms_norm(dual, w), lambda: rms_norm(x, dual_w),
                     lambda: linear_cross_entropy(dual, x, t), lambda: linear_cross_entropy(x, dual, t)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
    with pytest.raises(RuntimeError, match="forward mode"):
        torch.func.jvp(lambda a: rms_norm(a, w), (x,), (x,))
    assert _rows.wants_grad(x) is False and _rows.wants_grad(x, w.requires_grad_()) is True


def test_embedding_refuses_a_scale_that_is_not_finite(built_lib):  # noqa: F811
    """Zero rows of ids without a token would not be zero."""
    L = built_lib
    before = L.cb_launch_count()
    for scale in (math.inf, -math.inf, math.nan, 1e39):
        assert L.cb_embedding(256, 0, 8, 4, 8, 256, 1, 3, scale, 256, None, None) == 1
        assert L.cb_embedding_grad(256, 0, 8, 256, 1, 3, 4, 8, scale, 256, 256, 1 << 40, None) == 1
    assert L.cb_launch_count() == before
    from cirrus_s_1a_b200.embedding import embedding

    with pytest.raises(ValueError, match="scale"):
        embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), math.nan)


def test_what_rounding_takes_off_lse_has_its_room(built_lib):  # noqa: F811
    """CB_REDUCE_REST (4) writes behind the count: without one it is refused, in any reduction."""
    L = built_lib
    before = L.cb_launch_count()
    for reduction in (0, 1, 2):
        assert L.cb_linear_ce(256, 1, 8, 256, 1, 8, 3, 4, 8, 256, 1, reduction | 4, 256, 256, None, 256, 1 << 40, None,
                              None) == 1
        assert L.cb_linear_ce_grad(256, 1, 8, 256, 1, 8, 3, 4, 8, 256, 1, reduction | 4, 256, None, 256, 1, None, 0, 256,
                                   256, 256, 1 << 40, None, None) == 1
    for reduction in (3, 7, 8, -1):
        assert L.cb_linear_ce(256, 1, 8, 256, 1, 8, 3, 4, 8, 256, 1, reduction, 256, 256, 256, 256, 1 << 40, None, None) == 1
    assert L.cb_launch_count() == before
