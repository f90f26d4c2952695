"""CPU tests of the operators at the ends of a model: the C entry points and the Python
functions refuse bad arguments before any CUDA call, and the 64-bit oracle agrees with
torch's own autograd."""

import pytest
import torch

from oracle import ends
from test_host import built_lib  # noqa: F401

BIG = 1 << 40


def test_entry_points_refuse_bad_arguments_without_launching(built_lib):  # noqa: F811
    L = built_lib
    before = L.cb_launch_count()
    emb = lambda t=256, dtype=0, ld=8, V=4, d=8, ids=256, n=3, out=256: L.cb_embedding(  # noqa: E731
        t, dtype, ld, V, d, ids, 1, n, 1.0, out, None, None)
    assert emb(t=None) == 1 and emb(dtype=3) == 1 and emb(ld=7) == 1 and emb(V=0) == 1 and emb(d=0) == 1
    assert emb(ids=None) == 1 and emb(ids=260) == 1 and emb(n=0) == 1 and emb(out=None) == 1 and emb(t=258) == 1
    assert emb(n=(1 << 24) + 1) == 2 and emb(V=(1 << 20) + 1) == 2 and emb(d=65537, ld=65537) == 2
    eg = lambda g=256, dtype=0, ldg=8, ids=256, n=3, V=4, d=8, out=256, scratch=256, nb=BIG: L.cb_embedding_grad(  # noqa: E731
        g, dtype, ldg, ids, 1, n, V, d, 1.0, out, scratch, nb, None)
    assert eg(g=None) == 1 and eg(dtype=-1) == 1 and eg(ldg=-1) == 1 and eg(ids=None) == 1 and eg(n=0) == 1
    assert eg(out=None) == 1 and eg(scratch=None) == 1 and eg(scratch=264) == 1 and eg(nb=0) == 4 and eg(n=1 << 25) == 2
    assert L.cb_embedding_grad_scratch_bytes(0, 4, 8) == 0 and L.cb_embedding_grad_scratch_bytes(5, 4, 8) > 0
    nrm = lambda x=256, dtype=1, ld=8, w=256, wd=0, rows=3, d=8, y=256: L.cb_rms_norm(  # noqa: E731
        x, dtype, ld, w, wd, rows, d, 1e-6, y, None)
    assert nrm(x=None) == 1 and nrm(dtype=9) == 1 and nrm(w=None) == 1 and nrm(wd=2) == 1 and nrm(rows=0) == 1
    assert nrm(d=0) == 1 and nrm(y=None) == 1 and nrm(x=257) == 1 and nrm(w=258) == 1 and nrm(d=65537) == 2
    ng = lambda g=256, ldg=8, dx=256, dw=256, scratch=256, nb=BIG: L.cb_rms_norm_grad(  # noqa: E731
        256, 1, 8, g, ldg, 256, 0, 3, 8, 1e-6, dx, dw, scratch, nb, None)
    assert ng(g=None) == 1 and ng(ldg=-1) == 1 and ng(dx=None) == 1 and ng(dw=None) == 1 and ng(scratch=None) == 1
    assert ng(nb=0) == 4 and ng(scratch=8) == 1 and L.cb_rms_norm_grad_scratch_bytes(3, 0) == 0
    ce = lambda h=256, hd=1, ldh=8, w=256, wd=1, ldw=8, N=3, V=4, d=8, t=256, red=0, loss=256, lse=256, count=256, s=256, nb=BIG: (  # noqa: E731,E501
        L.cb_linear_ce(h, hd, ldh, w, wd, ldw, N, V, d, t, 1, red, loss, lse, count, s, nb, None, None))
    assert ce(h=None) == 1 and ce(w=None) == 1 and ce(t=None) == 1 and ce(hd=3) == 1 and ce(hd=1, wd=2) == 1
    assert ce(hd=1, wd=0) == 1 and ce(hd=0, wd=2) == 1 and ce(N=0) == 1 and ce(V=0) == 1 and ce(d=0) == 1
    assert ce(ldh=-1) == 1 and ce(ldw=7) == 1 and ce(t=260) == 1 and ce(red=3) == 1 and ce(loss=None) == 1
    assert ce(lse=None) == 1 and ce(red=1, count=None) == 1 and ce(s=None) == 1 and ce(s=264) == 1 and ce(nb=0) == 4
    assert ce(N=(1 << 24) + 1) == 2 and ce(V=(1 << 20) + 1) == 2 and ce(d=65537, ldw=65537) == 2
    cg = lambda red=0, lse=256, count=256, gl=256, s1=1, dh=256, dw=256, s=256, nb=BIG: L.cb_linear_ce_grad(  # noqa: E731
        256, 1, 8, 256, 1, 8, 3, 4, 8, 256, 1, red, lse, count, gl, s1, None, 0, dh, dw, s, nb, None, None)
    assert cg(lse=None) == 1 and cg(red=1, count=None) == 1 and cg(s1=-1) == 1 and cg(dh=None, dw=None) == 1
    assert cg(dh=257) == 1 and cg(dw=257) == 1 and cg(s=None) == 1 and cg(nb=0) == 4
    need = lambda hd, back: L.cb_linear_ce_scratch_bytes(256, hd, 8, 256, 1, 8, 3, 4, 8, 256, back)  # noqa: E731
    assert need(7, 0) == 0 and need(1, 0) > 0 and need(1, 1) > 0 and need(0, 1) > need(1, 1)
    assert L.cb_launch_count() == before


def test_tensors_that_are_not_on_a_gpu_are_refused():
    from cirrus_s_1a_b200.embedding import embedding
    from cirrus_s_1a_b200.loss import linear_cross_entropy
    from cirrus_s_1a_b200.norm import rms_norm

    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for bad in (lambda: linear_cross_entropy(x, x, t), lambda: embedding(t, x), lambda: rms_norm(x, x[0])):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_oracle_cross_entropy_agrees_with_autograd(reduction):
    g = torch.Generator().manual_seed(0)
    h = torch.randn(9, 12, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(20, 12, generator=g, dtype=torch.float64, requires_grad=True)
    t = torch.randint(0, 20, (9,), generator=g)
    t[2] = -1
    x = h @ w.T
    loss = torch.nn.functional.cross_entropy(x, t, ignore_index=-1, reduction=reduction)
    lse = torch.logsumexp(x, 1)
    up = torch.randn(loss.shape, generator=g, dtype=torch.float64)
    z = torch.randn(9, generator=g, dtype=torch.float64)
    dh, dw = torch.autograd.grad((loss, lse), (h, w), (up, z))
    r = ends.cross_entropy(h.detach(), w.detach(), t, reduction, up, z)
    for got, want in ((r["loss"], loss), (r["lse"], lse), (r["dh"], dh), (r["dw"], dw)):
        torch.testing.assert_close(got, want.detach(), rtol=1e-12, atol=1e-12)


def test_oracle_embedding_and_norm_agree_with_autograd():
    g = torch.Generator().manual_seed(1)
    table = torch.randn(7, 5, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([3, 1, 3, 0, 6, 3])
    up = torch.randn(6, 5, generator=g, dtype=torch.float64)
    y = torch.nn.functional.embedding(ids, table) * 2.5
    torch.testing.assert_close(ends.embedding(ids, table.detach(), 2.5), y.detach())
    torch.testing.assert_close(ends.embedding_grad(ids, up, 7, 2.5)[0], torch.autograd.grad(y, table, up)[0])
    x = torch.randn(6, 5, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(5, generator=g, dtype=torch.float64, requires_grad=True)
    y = torch.nn.functional.rms_norm(x, (5,), w, 1e-6)
    torch.testing.assert_close(ends.rms_norm(x.detach(), w.detach(), 1e-6), y.detach())
    for got, want in zip(ends.rms_norm_grad(x.detach(), w.detach(), 1e-6, up), torch.autograd.grad(y, (x, w), up)):
        torch.testing.assert_close(got, want)
