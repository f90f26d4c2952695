"""Cross entropy over the vocabulary without the logits, and its gradient
(cb_linear_ce, cb_linear_ce_grad), against the 64-bit oracle."""

import math

import pytest
import torch

from oracle import ends

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAIRS = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def inputs(N, V, d, pair, seed=0, masked=0.2, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(N, d, generator=g).to(TYPES[pair[0]])
    w = (gain * torch.randn(V, d, generator=g) / math.sqrt(d)).to(TYPES[pair[1]])
    t = torch.randint(0, V, (N,), generator=g)
    t[torch.rand(N, generator=g) < masked] = -1
    return h, w, t


def bounds(r, h, w, reduction):
    """Bounds on the errors of one call, from the magnitudes that the oracle gives.

    A logit: products of 16-bit values are exact, of float32 ones carried to 2^-22; the sum is
    rounded (or cut) at most once per 8 products and 8 times at the ends, by 2^-23 of a partial
    sum that ``size`` bounds.  The row's sum of exponentials: 2^-20, as for log probabilities
    (its vocabulary is summed in pieces of at most 2^10 additions).  A mean or sum adds the
    rows' errors and one rounding of the result.  G: the logit's and lse's errors, 2^-20 for
    the exponential and the factors, half a step of its 16-bit type (2^-22 in float32), and
    what lies below float16's range: the factor is scaled so that this is 2^-37 of it.  A
    product over K terms: (K / 8 + 8) roundings of 2^-23 of the sum of magnitudes."""
    d, (N, V) = h.shape[1], r["terms"].shape
    x = r["size"] * ((d / 8 + 8) * 2.0 ** -23 + 2.0 ** -22)
    lse = x + 2.0 ** -20 + r["lse"].abs() * 2.0 ** -23
    rows = torch.where(r["rows"] != 0, 2 * x + 2.0 ** -20 + r["rows"].abs() * 2.0 ** -22, 0.0)
    loss = {"none": rows, "sum": rows.sum() + r["loss"].abs() * 2.0 ** -23,
            "mean": rows.sum() / r["count"] + r["loss"].abs() * 2.0 ** -23}[reduction]
    u = 2.0 ** -22 if h.dtype == torch.float32 else half_step(h.dtype)
    dG = r["terms"] * (u + 2.0 ** -20 + x[:, None] + lse[:, None])
    if h.dtype == torch.float16:
        dG = dG + r["terms"].sum(1, keepdim=True) * 2.0 ** -37
    k = lambda K: (K / 8 + 8) * 2.0 ** -23  # noqa: E731
    aw, ah = w.double().abs(), r["hz"].abs()
    dh = (dG + r["terms"] * k(V)) @ aw
    dw = (dG + r["terms"] * k(N)).T @ ah
    dh = dh * 1.01 + r["dh"].abs() * half_step(h.dtype) + smallest(h.dtype)
    dw = dw * 1.01 + r["dw"].abs() * half_step(w.dtype) + smallest(w.dtype)
    return {"loss": loss, "lse": lse, "dh": dh, "dw": dw}


def compare(got, r, h, w, reduction, names=("loss", "lse", "dh", "dw")):
    b = bounds(r, h, w, reduction)
    for n in names:
        err = (got[n].detach().cpu().double() - r[n]).abs()
        assert torch.isfinite(got[n]).all(), n
        assert (err <= b[n]).all(), (n, float((err / b[n].clamp(min=1e-300)).max()), float(err.max()))


def call(h, w, t, reduction="mean", g_loss=None, g_lse=None, want=(True, True), status=None):
    """One forward and backward on the device: a dict of results."""
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    h, w = h.detach().requires_grad_(want[0]), w.detach().requires_grad_(want[1])
    r = linear_cross_entropy(h, w, t, reduction=reduction, status=status)
    outs, ups = zip(*[(o, g.to(DEV)) for o, g in ((r.loss, g_loss), (r.lse, g_lse)) if g is not None])
    grads = iter(torch.autograd.grad(outs, [x for x, use in ((h, want[0]), (w, want[1])) if use], ups))
    return {"loss": r.loss, "lse": r.lse, "dh": next(grads) if want[0] else None, "dw": next(grads) if want[1] else None}


def check(h, w, t, reduction="mean", g_loss=None, g_lse=None, dev=None):
    if g_loss is None and g_lse is None:
        g_loss = torch.ones(()) if reduction != "none" else torch.full((len(t),), 1.0 / len(t))
    hd, wd = (h.to(DEV), w.to(DEV)) if dev is None else dev
    got = call(hd, wd, t.to(DEV), reduction, g_loss, g_lse)
    compare(got, ends.cross_entropy(h, w, t, reduction, g_loss, g_lse), h, w, reduction)
    return got


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("N,V,d", [(1, 1, 1), (1, 2, 8), (3, 5, 7), (2, 129, 64), (5, 300, 64), (33, 513, 72),
                                   (128, 256, 64), (130, 1000, 40), (257, 777, 129), (64, 4100, 768), (300, 2000, 200),
                                   (513, 515, 320), (1025, 64, 16)])
def test_matches_oracle(pair, N, V, d):
    h, w, t = inputs(N, V, d, pair, seed=N + V + d)
    check(h, w, t)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("N,V,d", [(17, 15001, 72), (32, 19200, 40), (33, 40000, 24), (64, 20000, 300), (65, 15001, 64)])
def test_some_rows_over_a_large_vocabulary(pair, N, V, d):
    """Few rows as columns of tiles of the vocabulary, one, two and three tiles a CTA, and the
    first number of rows that is not."""
    h, w, t = inputs(N, V, d, pair, seed=N)
    check(h, w, t, "none")


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("N,V", [(3, 40), (270, 5)])
def test_widest_rows(pair, N, V):
    h, w, t = inputs(N, V, 65536, pair, seed=N)
    check(h, w, t, "sum")


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reductions_and_gradients_from_above(pair, reduction):
    h, w, t = inputs(70, 333, 96, pair, seed=3)
    g = torch.Generator().manual_seed(4)
    one = torch.randn((70,) if reduction == "none" else (), generator=g)
    z = torch.randn(70, generator=g) * 0.1
    check(h, w, t, reduction, one)
    check(h, w, t, reduction, one, z)
    check(h, w, t, reduction, None, z)  # lse alone
    # rows of very different weight keep their own precision in dh, and add up in dw
    if reduction == "none":
        check(h, w, t, "none", one * torch.exp2(torch.randint(-18, 12, (70,), generator=g).float()))


@pytest.mark.parametrize("pair", PAIRS)
def test_forward_alone_and_one_gradient_alone(pair):
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    h, w, t = inputs(45, 400, 80, pair, seed=5)
    both = check(h, w, t)
    plain = linear_cross_entropy(h.to(DEV), w.to(DEV), t.to(DEV))
    assert plain.loss.grad_fn is None and torch.equal(plain.loss, both["loss"]) and torch.equal(plain.lse, both["lse"])
    for want in ((True, False), (False, True)):
        one = call(h.to(DEV), w.to(DEV), t.to(DEV), "mean", torch.ones(()), want=want)
        for n in ("dh", "dw"):
            assert one[n] is None or torch.equal(one[n], both[n])


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_rows_without_a_target(pair, reduction):
    """No target anywhere: 0 and zero gradients.  A row without one may hold anything."""
    h, w, t = inputs(40, 210, 64, pair, seed=6)
    up = torch.ones(40 if reduction == "none" else ())
    none = call(h.to(DEV), w.to(DEV), torch.full_like(t, -1).to(DEV), reduction, up)
    assert none["loss"].eq(0).all() and none["dh"].eq(0).all() and none["dw"].eq(0).all()
    assert torch.isfinite(none["lse"]).all()
    t[::3] = -100
    ref = check(h, w, t, reduction, up)
    bad = h.clone()
    bad[0], bad[3], bad[6], bad[9] = math.nan, math.inf, -math.inf, torch.finfo(h.dtype).min
    got = call(bad.to(DEV), w.to(DEV), t.to(DEV), reduction, up)
    for n in ("loss", "dh", "dw"):
        assert torch.equal(got[n], ref[n]), n
    keep = torch.ones(40, dtype=torch.bool)
    keep[[0, 3, 6, 9]] = False
    assert torch.equal(got["lse"][keep.to(DEV)], ref["lse"][keep.to(DEV)])


@pytest.mark.parametrize("pair", PAIRS)
def test_a_row_that_is_not_finite_spoils_itself_and_the_weights_only(pair):
    h, w, t = inputs(40, 210, 64, pair, seed=7, masked=0.0)
    up = torch.ones(40)
    ref = check(h, w, t, "none", up)
    bad = h.clone()
    bad[5, 3], bad[33] = math.nan, math.inf
    got = call(bad.to(DEV), w.to(DEV), t.to(DEV), "none", up)
    others = torch.ones(40, dtype=torch.bool)
    others[[5, 33]] = False
    for n in ("loss", "lse", "dh"):
        assert torch.equal(got[n].cpu()[others], ref[n].cpu()[others])
        assert got[n].cpu()[~others].isnan().all()
    assert got["dw"].isnan().all()
    # a vocabulary row that is NaN is part of every row's sum
    badw = w.clone()
    badw[100] = math.nan
    got = call(h.to(DEV), badw.to(DEV), t.to(DEV), "none", up)
    assert got["loss"].isnan().all() and got["lse"].isnan().all()


@pytest.mark.parametrize("pair", PAIRS)
def test_target_outside_the_vocabulary(pair):
    h, w, t = inputs(20, 77, 32, pair, seed=8)
    bad = t.clone()
    bad[4], bad[11] = 77, 2 ** 40
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = call(h.to(DEV), w.to(DEV), bad.to(DEV), "mean", torch.ones(()), status=status)
    assert int(status) == 6
    t[4] = t[11] = -1
    ref = check(h, w, t)
    for n in got:
        assert torch.equal(got[n], ref[n])
    status.zero_()
    got = call(h.to(DEV), w.to(DEV), t.int().to(DEV), "mean", torch.ones(()), status=status)
    assert int(status) == 0
    for n in got:
        assert torch.equal(got[n], ref[n])


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("centre", [0.0, 40.0, -40.0])
def test_peaked_and_far_rows(pair, centre):
    """Logits of thousands, equal rows, rows whose target has no probability left."""
    h, w, t = inputs(36, 300, 64, pair, seed=9, masked=0.1)
    h[1] = 0.0
    h[2:8] *= 300
    h[8:12] = (w[t[8:12].clamp(min=0)].float() * 100).to(h.dtype)
    w[:, 0] += centre
    h[12:20, 0] = 50.0
    w[200] = w[100]
    check(h, w, t, "none", torch.linspace(0.1, 1, 36))


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("N", [1, 5, 16, 17, 45, 129, 300, 1100])
@pytest.mark.parametrize("parts", ["two", "three"])
def test_both_directions_take_a_logit_alike(pair, N, parts):
    """A word that has all the probability, with a logit of 2000 and more: loss and gradients
    are exactly 0, for every other exponential is, unless the backward pass's logit differs by
    a bit from the one that lse is.  (Another word's logit is below 3 * 26 * 8 + 30 = 660 in
    magnitude, with 8 deviations and all that the rows add.)"""
    g = torch.Generator().manual_seed(N)
    V, d = 270, 700
    w = torch.randn(V, d, generator=g)
    w[3, 5] = 1.0 if parts == "two" else 300.0
    w = w.to(TYPES[pair[1]])
    t = torch.randint(4, V, (N,), generator=g)
    h = 3 * w[t].float() * (1 + torch.rand(N, 1, generator=g)) + 0.01 * torch.randn(N, d, generator=g)
    h[:, 5] = 0.0
    h = h.to(TYPES[pair[0]])
    got = call(h.to(DEV), w.to(DEV), t.to(DEV), "none", torch.linspace(0.5, 2, N))
    for n in ("loss", "dh", "dw"):
        assert got[n].eq(0).all(), (n, float(got[n].abs().max()))
    x = (h.double() * w.double()[t]).sum(1)
    assert (got["lse"].cpu().double() - x).abs().le(x * ((d / 8 + 8) * 2.0 ** -23 + 2.0 ** -22)).all()


@pytest.mark.parametrize("N", [1, 3, 40, 1030])
@pytest.mark.parametrize("pair", PAIRS)
def test_a_vocabulary_of_one(pair, N):
    h, w, t = inputs(N, 1, 1500, pair, seed=N, masked=0.0, gain=30.0)
    got = call(h.to(DEV), w.to(DEV), t.to(DEV), "sum", torch.ones(()))
    assert all(got[n].eq(0).all() for n in ("loss", "dh", "dw"))


@pytest.mark.parametrize("weight", ["f32", "bf16"])
def test_rows_of_very_different_size(weight):
    """Rows of 2^-8 to 2^9 with weights to match, whose logits are ordinary ones: every row has
    its part in dw."""
    h, w, t = inputs(1100, 200, 72, ("f32", weight), seed=23, gain=2.0 ** -6)
    h *= torch.exp2(torch.arange(1100) % 18 - 8.0)[:, None]
    check(h, w, t, "none", torch.linspace(0.2, 1, 1100))
    check(h, w, t, "none", torch.linspace(0.2, 1, 1100) * torch.exp2(8 - torch.arange(1100) % 18))


def test_float32_of_any_size():
    """No common scale: tiny rows keep their bits beside huge ones."""
    h, w, t = inputs(32, 200, 64, ("f32", "f32"), seed=10, masked=0.0)
    h[::4] *= 2.0 ** 30
    w[::5] *= 2.0 ** -30
    h[1::4] *= 2.0 ** -20
    check(h, w, t, "none", torch.ones(32))


@pytest.mark.parametrize("weight", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["fits", "large row", "small row", "large vocabulary row", "small vocabulary row"])
def test_float32_in_two_parts_or_three(weight, what):
    """Rows enough for the two-part form against either weight; values just in its range, and
    one row or vocabulary row out of it."""
    h, w, t = inputs(1100, 200, 72, ("f32", weight), seed=21)
    h[7] *= 250 / h[7].abs().max()
    w[9] *= 2.0 ** -9 / w[9].abs().max()
    if what == "large row":
        h[50] *= 3e4
    elif what == "small row":
        h[50] *= 1e-9
    elif what == "large vocabulary row":
        w[60] *= 1e4
    elif what == "small vocabulary row":
        w[60] *= 1e-9
    check(h, w, t, "none", torch.linspace(0.2, 1, 1100))
    check(h, w, t, "mean")


@pytest.mark.parametrize("pair", PAIRS)
def test_strides_and_alignment(pair):
    g = torch.Generator().manual_seed(11)
    H = torch.randn(41, 150, generator=g).to(TYPES[pair[0]])
    W = (torch.randn(2 * 203, 150, generator=g) / 8).to(TYPES[pair[1]])
    t = torch.randint(0, 203, (41,), generator=g)
    Hd, Wd = H.to(DEV), W.to(DEV)
    for a, d, step in ((0, 150, 1), (1, 64, 2), (3, 77, 1), (8, 128, 2), (5, 1, 1), (2, 6, 2)):
        n = len(range(0, 41, step))
        check(H[::step, a:a + d], W[::2, a:a + d], t[:n], dev=(Hd[::step, a:a + d], Wd[::2, a:a + d]))
    row = H[7:8].expand(9, 150)
    got = call(Hd[7:8].expand(9, 150), Wd[:203], t[:9].to(DEV), "none", torch.ones(9))
    compare(got, ends.cross_entropy(row, W[:203], t[:9], "none", torch.ones(9)), row, W[:203], "none")


def test_expanded_gradients_from_above():
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    h, w, t = inputs(50, 150, 64, ("bf16", "bf16"), seed=12)
    hd, wd = h.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    r = linear_cross_entropy(hd, wd, t.to(DEV), reduction="none")
    (r.loss.sum() + 0.5 * r.lse.sum()).backward()  # both come as one number expanded over the rows
    ref = ends.cross_entropy(h, w, t, "none", torch.ones(50), torch.full((50,), 0.5))
    compare({"dh": hd.grad, "dw": wd.grad}, ref, h, w, "none", ("dh", "dw"))


@pytest.mark.parametrize("pair", PAIRS)
def test_gradient_against_differences(pair):
    """Central differences of the oracle's 64-bit loss, whose own error is of the order of step^2."""
    h, w, t = inputs(12, 90, 24, pair, seed=13)
    got = call(h.to(DEV), w.to(DEV), t.to(DEV), "mean", torch.ones(()))
    ref = ends.cross_entropy(h, w, t, "mean", torch.ones(()))
    tol = bounds(ref, h, w, "mean")
    g = torch.Generator().manual_seed(14)
    step = 1e-5
    for name, i in (("dh", 0), ("dw", 1)):
        for _ in range(4):
            at = [h.double(), w.double()]
            u = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
            f = []
            for s in (step, -step):
                moved = list(at)
                moved[i] = at[i] + s * u
                f.append(ends.cross_entropy(*moved, t)["loss"])
            slope = (f[0] - f[1]) / (2 * step)
            # third derivatives of the loss are below |u|^3 max|w|^3 here: 1e-10 times a few thousands
            assert abs(float((got[name].cpu().double() * u).sum() - slope)) <= float((tol[name] * u.abs()).sum()) + 1e-6


@pytest.mark.parametrize("pair", PAIRS)
def test_same_bits_every_time_and_on_another_stream(pair):
    h, w, t = inputs(700, 2500, 128, pair, seed=15)
    hd, wd, td = h.to(DEV), w.to(DEV), t.to(DEV)
    first = call(hd, wd, td, "mean", torch.ones(()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(hd, wd, td, "mean", torch.ones(()))
    again = call(hd, wd, td, "mean", torch.ones(()))  # while the other may still run
    torch.cuda.synchronize()
    for n in first:
        assert torch.equal(first[n], other[n]) and torch.equal(first[n], again[n]), n


@pytest.mark.parametrize("pair", PAIRS)
def test_captured_step(pair):
    """Forward and backward in a graph, replayed on other values; two graphs, replayed in turn."""
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    sets = [inputs(90, 600, 64, pair, seed=s) for s in (16, 17, 18)]
    graphs = []
    for k in range(2):
        buf = [x.to(DEV) for x in sets[k]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())

        def step():
            h, w = buf[0].detach().requires_grad_(), buf[1].detach().requires_grad_()
            r = linear_cross_entropy(h, w, buf[2])
            return (r.loss.detach(), r.lse.detach(), *torch.autograd.grad(r.loss, (h, w)))

        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, buf, outs))
    for use in (2, 0, 1):
        for graph, buf, _ in graphs:
            for b, x in zip(buf, sets[use]):
                b.copy_(x)
            graph.replay()
        h, w, t = sets[use]
        ref = ends.cross_entropy(h, w, t, "mean", torch.ones(()))
        for _, _, outs in graphs:
            compare(dict(zip(("loss", "lse", "dh", "dw"), outs)), ref, h, w, "mean")


def test_no_rows():
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    w = torch.randn(30, 16, device=DEV, requires_grad=True)
    h = torch.empty(0, 16, device=DEV, requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device=DEV)
    r = linear_cross_entropy(h, w, t)
    assert r.loss.item() == 0 and r.lse.shape == (0,)
    r.loss.backward()
    assert h.grad.shape == (0, 16) and w.grad.eq(0).all()


def test_rows_past_32_bits():
    """Hidden rows of a buffer of more than 2^32 elements."""
    h, w, t = inputs(4100, 64, 32, ("bf16", "bf16"), seed=19)
    far = torch.empty(4100 << 20, dtype=torch.bfloat16, device=DEV).view(4100, 1 << 20)[:, 40:72]
    far.copy_(h)
    check(h, w, t, dev=(far, w.to(DEV)))


def test_large_against_chunks_of_the_oracle():
    """The benchmark's vocabulary and more rows than a tile, some rows of the gradient checked."""
    h, w, t = inputs(600, 32000, 768, ("bf16", "bf16"), seed=20)
    check(h, w, t)


def test_refusals():
    from cirrus_s_1a_b200.loss import linear_cross_entropy

    h, w, t = (x.to(DEV) for x in inputs(6, 20, 16, ("f32", "f32")))
    for bad in ((h[0], w, t), (h, w[:, :8], t), (h, w.half(), t), (h.bfloat16(), w, t), (h.double(), w.double(), t),
                (h, w, t[:5]), (h, w, t.float()), (h, w, t.cpu()), (h, w.cpu(), t), (h.cpu(), w.cpu(), t.cpu()),
                (h, w[:0], t), (h.T.contiguous().T, w, t), (h, w[:1].expand(20, 16), t), (h, w, t[::2].repeat(2)[::2])):
        with pytest.raises(ValueError):
            linear_cross_entropy(*bad)
    with pytest.raises(ValueError):
        linear_cross_entropy(h, w, t, reduction="median")
    with pytest.raises(ValueError):
        linear_cross_entropy(h, w, t, status=torch.zeros(1, device=DEV))
