"""Embedding lookup with scaling and its gradient (cb_embedding, cb_embedding_grad)
against the 64-bit oracle."""

import math

import pytest
import torch

from oracle import ends

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def run(ids, table, scale, g):
    from cirrus_s_1a_b200.embedding import embedding

    table = table.detach().requires_grad_()
    y = embedding(ids, table, scale)
    return y.detach(), torch.autograd.grad(y, table, g)[0]


def check(ids, table, g, scale=1.0, dev=None):
    """A product is rounded in float32 and then to the type; a sum of n terms has at most n
    roundings of 2^-24 of the sum of their magnitudes, one more for the scale, one to the type."""
    V = table.shape[0]
    got_y, got_d = run(*((ids.to(DEV), table.to(DEV), scale, g.to(DEV)) if dev is None else dev))
    u, low = torch.finfo(table.dtype).eps / 2, torch.finfo(table.dtype).smallest_normal * torch.finfo(table.dtype).eps
    want = ends.embedding(ids, table, scale)
    assert ((got_y.cpu().double() - want).abs() <= want.abs() * (u + 2.0 ** -24) * 1.001 + low).all()
    d, mag, n = ends.embedding_grad(ids, g, V, scale)
    err = (got_d.cpu().double() - d).abs()
    assert (err <= mag * (n + 1) * 2.0 ** -24 * 1.001 + d.abs() * u + low).all()
    assert got_d.cpu()[n[:, 0] == 0].eq(0).all()
    return got_y, got_d


def case(n, V, d, dtype, seed=0, padded=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = (V * torch.rand(n, generator=g) ** 3).long().clamp(max=V - 1)
    ids[torch.rand(n, generator=g) < padded] = -1
    return ids, torch.randn(V, d, generator=g).to(TYPES[dtype]), torch.randn(n, d, generator=g).to(TYPES[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 5, 3), (2, 1, 8), (7, 300, 16), (33, 4, 5), (65, 1000, 24), (100, 37, 64),
                                   (1000, 20, 129), (1025, 70000, 8), (3000, 511, 40), (5000, 2, 96), (2048, 2048, 768),
                                   (17000, 300, 32)])
def test_matches_oracle(dtype, n, V, d):
    ids, table, g = case(n, V, d, dtype, seed=n + V + d)
    check(ids, table, g, scale=1.0)
    check(ids, table, g, scale=math.sqrt(d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [2, 6, 12, 70, 100, 258, 516, 771])
def test_widths_of_smaller_pieces(dtype, d):
    """Rows whose pieces are 8 or 4 bytes or one element."""
    ids, table, g = case(700, 60, d, dtype, seed=d)
    check(ids, table, g, scale=1.5)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_token_many_times_and_none_at_all(dtype):
    ids, table, g = case(4097, 50, 72, dtype, seed=1, padded=0.0)
    check(torch.full_like(ids, 49), table, g)
    check(torch.full_like(ids, 0), table, g, scale=-2.0)
    y, d = check(torch.full_like(ids, -1), table, g)
    assert y.eq(0).all() and d.eq(0).all()
    check(torch.arange(4097) % 50, table, g)
    check(torch.arange(4097) // 100, table, g)


def test_padding_may_hold_anything():
    """The gradient of a row without a token is not read into any sum; what is not finite stays in its own row."""
    ids, table, g = case(300, 40, 33, "f32", seed=2, padded=0.0)
    ids[::7] = -1
    ids[100] = 11
    ref = run(ids.to(DEV), table.to(DEV), 1.0, torch.where(ids[:, None] < 0, 0.0, g).to(DEV))
    g[::7] = math.nan
    got = run(ids.to(DEV), table.to(DEV), 1.0, g.to(DEV))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    g[100, 5] = math.inf
    d = run(ids.to(DEV), table.to(DEV), 1.0, g.to(DEV))[1]
    assert torch.isinf(d[11, 5])
    d[11, 5] = ref[1][11, 5]
    assert torch.equal(d, ref[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_shapes_and_int32(dtype):
    g0 = torch.Generator().manual_seed(3)
    T = torch.randn(90, 100, generator=g0).to(TYPES[dtype])
    G = torch.randn(60, 130, generator=g0).to(TYPES[dtype])
    ids = torch.randint(-1, 45, (60,), generator=g0)
    Td, Gd = T.to(DEV), G.to(DEV)
    for a, d in ((0, 100), (1, 64), (3, 33), (8, 32), (4, 1)):
        check(ids, T[::2, a:a + d], G[:, a:a + d], dev=(ids.to(DEV), Td[::2, a:a + d], 1.0, Gd[:, a:a + d]))
    check(ids.int(), T, G[:, :100], dev=(ids.int().to(DEV), Td, 1.0, Gd[:, :100]))
    one = torch.ones(1, 1, dtype=T.dtype).expand(60, 100)  # the gradient of a sum: one number for all
    check(ids, T, one, dev=(ids.to(DEV), Td, 1.0, one.to(DEV)))
    row = G[:1, :100].expand(60, 100)
    check(ids, T, row, dev=(ids.to(DEV), Td, 1.0, Gd[:1, :100].expand(60, 100)))
    from cirrus_s_1a_b200.embedding import embedding

    y = embedding(ids.view(3, 4, 5).to(DEV), Td)
    assert y.shape == (3, 4, 5, 100) and torch.equal(y.view(60, 100), embedding(ids.to(DEV), Td))


def test_id_outside_the_table():
    from cirrus_s_1a_b200.embedding import embedding

    ids, table, g = case(64, 30, 16, "bf16", seed=4)
    ref = run(ids.masked_fill(torch.arange(64) % 9 == 0, -1).to(DEV), table.to(DEV), 1.0, g.to(DEV))
    bad = ids.masked_fill(torch.arange(64) % 9 == 0, 30)
    bad[0] = 2 ** 50
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    embedding(bad.to(DEV), table.to(DEV), status=status)
    assert int(status) == 6
    got = run(bad.to(DEV), table.to(DEV), 1.0, g.to(DEV))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert embedding(torch.empty(0, 3, dtype=torch.int64, device=DEV), table.to(DEV)).shape == (0, 3, 16)


@pytest.mark.parametrize("n", [700, 20000])
def test_same_bits_streams_and_graphs(n):
    ids, table, g = (x.to(DEV) for x in case(n, 900, 128, "bf16", seed=5))
    first = run(ids, table, 1.0, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(ids, table, 1.0, g)
    again = run(ids, table, 1.0, g)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, other, again))
    more = [tuple(x.to(DEV) for x in case(n, 900, 128, "bf16", seed=s)) for s in (6, 7)]
    graphs = []
    for _ in range(2):
        buf = [x.clone() for x in (ids, table, g)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run(buf[0], buf[1], 1.0, buf[2])
        graphs.append((graph, buf, outs))
    for which in ((0, 1), (1, 0)):
        for (graph, buf, _), k in zip(graphs, which):
            for b, x in zip(buf, more[k]):
                b.copy_(x)
            graph.replay()
        for (_, _, outs), k in zip(graphs, which):
            want = run(more[k][0], more[k][1], 1.0, more[k][2])
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_many_tokens():
    """More tokens than one sort holds: the sums of the parts are joined in order."""
    g0 = torch.Generator().manual_seed(8)
    n, V, d = 300_000, 1000, 8
    ids = (V * torch.rand(n, generator=g0) ** 4).long()
    g = torch.randn(n, d, generator=g0)
    table = torch.randn(V, d, generator=g0)
    _, got = run(ids.to(DEV), table.to(DEV), 1.0, g.to(DEV))
    want = torch.zeros(V, d, dtype=torch.float64).index_add_(0, ids, g.double())
    mag = torch.zeros(V, d, dtype=torch.float64).index_add_(0, ids, g.double().abs())
    n_of = torch.bincount(ids, minlength=V)[:, None]
    assert ((got.cpu().double() - want).abs() <= mag * (n_of + 1) * 2.0 ** -24 * 1.001 + want.abs() * 2.0 ** -24).all()


def test_refusals():
    from cirrus_s_1a_b200.embedding import embedding

    ids, table, _ = (x.to(DEV) for x in case(10, 20, 16, "f32"))
    for bad in ((ids.float(), table), (ids, table.double()), (ids, table[0]), (ids, table.cpu()), (ids.cpu(), table),
                (ids, table.T), (ids, table[:0]), (ids, table[:1].expand(20, 16)), (ids.view(5, 2).T, table)):
        with pytest.raises(ValueError):
            embedding(*bad)
    with pytest.raises(ValueError):
        embedding(ids, table, status=torch.zeros(2, dtype=torch.int32, device=DEV))
