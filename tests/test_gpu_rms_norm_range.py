"""RMSNorm at the end of float32's range: a row's squares are added up in float32, so its 2-norm,
not its largest value, is what has to stay below 2^64."""

import pytest
import torch

from test_gpu_rms_norm import case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pair", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("R,d", [(3, 64), (700, 96), (5, 1024), (20, 1025), (700, 4096), (3, 8200), (3, 65536)])
def test_rows_of_a_norm_just_below_the_limit(pair, R, d):
    x, w, g = case(R, d, pair, seed=R)
    x = x.double()
    x = (x * (0.9 * 2.0 ** 64 / x.norm(dim=1, keepdim=True))).to(g.dtype)
    check(x, w, g)
