"""RMSNorm and its gradient (cb_rms_norm, cb_rms_norm_grad) against the 64-bit oracle."""

import math

import pytest
import torch

from oracle import ends

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def run(x, w, g, eps=EPS):
    from cirrus_s_1a_b200.norm import rms_norm

    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = rms_norm(x, w, eps)
    return (y.detach(), *torch.autograd.grad(y, (x, w), g))


def check(x, w, g, eps=EPS, dev=None):
    """A row's sums have at most d / 32 + 16 roundings in a row, each of 2^-24 of a sum of
    magnitudes; half of that reaches the root, a few more roundings the result.  The
    weight's gradient adds up over rows in groups: at most rows / 64 + 64 in a row."""
    R, d = x.shape
    got = run(*((x.to(DEV), w.to(DEV), g.to(DEV)) if dev is None else dev), eps)
    e = (d / 32 + 24) * 2.0 ** -24
    ux, uw = torch.finfo(x.dtype).eps / 2, torch.finfo(w.dtype).eps / 2
    low = lambda t: torch.finfo(t).smallest_normal * torch.finfo(t).eps  # noqa: E731
    y = ends.rms_norm(x, w, eps)
    dx, dw, mx, mw = ends.rms_norm_grad(x, w, eps, g)
    for name, a, b, tol in (("y", got[0], y, y.abs() * (ux + e) + low(x.dtype)),
                            ("dx", got[1], dx, 3 * e * mx + dx.abs() * ux + low(x.dtype)),
                            ("dw", got[2], dw, mw * (e + (R / 64 + 64) * 2.0 ** -24) + dw.abs() * uw + low(w.dtype))):
        err = (a.cpu().double() - b).abs()
        assert (err <= tol * 1.001).all(), (name, float((err / tol).max()))
    return got


def case(R, d, pair, seed=0):
    g0 = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, d, generator=g0) * torch.exp(torch.randn(R, 1, generator=g0))).to(TYPES[pair[0]])
    w = (1 + 0.1 * torch.randn(d, generator=g0)).to(TYPES[pair[1]])
    return x, w, torch.randn(R, d, generator=g0).to(TYPES[pair[0]])


PAIRS = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")]


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("R,d", [(1, 1), (1, 8), (2, 7), (3, 64), (5, 768), (33, 1000), (65, 257), (130, 1024), (700, 96),
                                 (9, 2048), (7, 2056), (3, 5000), (2000, 16), (4, 20000)])
def test_matches_oracle(pair, R, d):
    check(*case(R, d, pair, seed=R + d))


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("R,d", [(1, 33), (16, 127), (1500, 127), (17, 129), (600, 255), (1200, 257), (40, 511), (1001, 512),
                                 (2500, 513), (50, 769), (1, 1023), (20, 1025), (2500, 1031), (9, 2047), (700, 4095),
                                 (5, 4097)])
def test_rows_of_single_elements(pair, R, d):
    """Widths at both ends of each number of elements a thread, and past the last."""
    check(*case(R, d, pair, seed=R + d))


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("R,d", [(1, 2056), (700, 4096), (3, 4104), (40, 6152), (601, 8192), (5, 8200), (3, 65536)])
def test_long_rows(pair, R, d):
    check(*case(R, d, pair, seed=R + d))


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("R,d", [(1500, 8), (1200, 264), (1000, 512), (999, 768), (1300, 1024), (1300, 1032), (1000, 2048)])
def test_many_rows(pair, R, d):
    """Rows enough for a warp each, at the ends of each number of pieces a lane."""
    check(*case(R, d, pair, seed=R + d))


@pytest.mark.parametrize("pair", PAIRS)
def test_strides_and_alignment(pair):
    X, W, G = case(50, 300, pair, seed=1)
    Xd, Wd, Gd = X.to(DEV), W.to(DEV), G.to(DEV)
    for a, d, step in ((0, 300, 1), (1, 64, 2), (3, 77, 1), (8, 128, 2), (16, 256, 1), (5, 1, 1)):
        s = (slice(None, None, step), slice(a, a + d))
        check(X[s], W[a:a + d].clone(), G[s], dev=(Xd[s], Wd[a:a + d].clone(), Gd[s]))
        check(X[s], W[a:a + d], G[s], dev=(Xd[s], Wd[a:a + d], Gd[s]))
    one = torch.ones(1, 1, dtype=X.dtype).expand(50, 300)
    check(X, W, one, dev=(Xd, Wd, one.to(DEV)))
    row = X[4:5].expand(50, 300)
    check(row, W, G, dev=(Xd[4:5].expand(50, 300), Wd, Gd))


@pytest.mark.parametrize("pair", PAIRS)
def test_rows_of_zeros_and_rows_that_are_not_finite(pair):
    x, w, g = case(40, 136, pair, seed=2)
    x[3] = 0.0
    ref = check(x, w, g)
    x[7, 5], x[11] = math.nan, math.inf
    got = run(x.to(DEV), w.to(DEV), g.to(DEV))
    fine = torch.ones(40, dtype=torch.bool)
    fine[[7, 11]] = False
    for a, b in zip(got[:2], ref[:2]):
        assert torch.equal(a.cpu()[fine], b.cpu()[fine])
        assert a.cpu()[7].isnan().all() and a.cpu()[11].isnan().all()


def test_gradient_against_differences():
    x, w, g = case(6, 40, ("f32", "f32"), seed=3)
    _, dx, dw = run(x.to(DEV), w.to(DEV), g.to(DEV))
    g0 = torch.Generator().manual_seed(4)
    for got, i in ((dx, 0), (dw, 1)):
        at = [x.double(), w.double()]
        u = torch.randn(at[i].shape, generator=g0, dtype=torch.float64)
        f = []
        for s in (1e-5, -1e-5):
            moved = list(at)
            moved[i] = at[i] + s * u
            f.append((ends.rms_norm(*moved, EPS) * g.double()).sum())
        assert abs(float((got.cpu().double() * u).sum() - (f[0] - f[1]) / 2e-5)) < 1e-3


@pytest.mark.parametrize("R,d", [(3000, 768), (500, 77)])
def test_same_bits_streams_and_graphs(R, d):
    x, w, g = (t.to(DEV) for t in case(R, d, ("bf16", "f32"), seed=5))
    first = run(x, w, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(x, w, g)
    again = run(x, w, g)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, other, again))
    buf = [t.clone() for t in (x, w, g)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(*buf)
    for seed in (6, 7):
        new = [t.to(DEV) for t in case(R, d, ("bf16", "f32"), seed=seed)]
        for b, t in zip(buf, new):
            b.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, run(*new)))


def test_refusals_and_no_rows():
    from cirrus_s_1a_b200.norm import rms_norm

    x, w, _ = (t.to(DEV) for t in case(6, 16, ("bf16", "f32")))
    for bad in ((x[0], w), (x, w[:8]), (x, w.half()), (x, w.cpu()), (x.double(), w.double()), (x.T, w[:6]),
                (x, torch.ones(32, device=DEV)[::2])):
        with pytest.raises(ValueError):
            rms_norm(*bad)
    assert rms_norm(x[:0], w).shape == (0, 16)
