"""Log probabilities of given tokens, entropy, rank and top alternatives
(cb_token_logprobs) against the 64-bit oracle."""

import math

import pytest
import torch

from oracle import kv8 as ok

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def check(x, tokens, top, dev=None):
    """Bounds: the row's sum has a relative error of at most 2^-20 (exp's two units
    and the rounding of up to 2^10 additions in a row), which is an absolute one of
    its logarithm; x - m is rounded once.  The entropy's sum carries the same 2^-20
    per term, and its terms add up to the entropy itself plus log l."""
    from cirrus_s_1a_b200.logprobs import token_logprobs

    dev = x.to(DEV) if dev is None else dev
    r = token_logprobs(dev, torch.tensor(tokens, dtype=torch.int32, device=DEV), top)
    lp, ent, rank, tlp, tt = ok.token_logprobs(x.double(), tokens, top)
    assert torch.equal(r.rank.cpu().long(), rank)
    assert torch.equal(r.top_token.cpu().long(), tt)
    for got, want in ((r.logprob, lp), (r.top_logprob, tlp)):
        got = got.cpu().double()
        # float32 has no value past its range: the nearest there is infinity
        want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine], want[~fine])
        assert (got - want)[fine].abs().le(2.0 ** -20 + want[fine].abs() * 2.0 ** -22).all()
    assert (r.entropy.cpu().double() - ent).abs().le(2.0 ** -19 * (1 + 2 * ent)).all()
    return r


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (3, 2, 2), (5, 31, 20), (2, 512, 32), (7, 1000, 0), (4, 8191, 5),
                                        (3, 32000, 20), (2, 50001, 32), (1, 200003, 7), (300, 515, 3)])
def test_matches_oracle(dtype, rows, V, top):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(rows, V, generator=g) * 3).to(TYPES[dtype])
    tokens = torch.randint(0, V, (rows,), generator=g).tolist()
    if rows > 2:
        tokens[1] = -1
    check(x, tokens, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [32000, 777])
def test_ties_masks_and_extremes(dtype, V):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(9, V, generator=g)
    x[0] = 1.25  # all alike
    x[1] = (x[1] * 2).round()  # many ties
    x[2] = -math.inf
    x[2, V - 3] = 5.0  # one token left
    x[3, ::2] = -math.inf
    x[4] = x[4] * 100  # peaked
    x[5] = 3e38
    x[5, 7] = -3e38
    x[6] = torch.finfo(torch.float32).min
    x[6, 11] = 0.0  # masked by the type's lowest value
    x[7] = x[7].sort().values  # ascending: each element beats all before it
    x[8] = x[8].sort(descending=True).values
    x = x.to(TYPES[dtype]).clamp(min=torch.finfo(TYPES[dtype]).min) if dtype == "bf16" else x
    x[2] = -math.inf
    x[2, V - 3] = 5.0
    x[3, ::2] = -math.inf
    tokens = [3, 5, V - 3, 1, int(x[4].argmax()), 7, 11, 0, V - 1]
    check(x, tokens, 20)
    check(x, [V - 1, 0, 0, 0, 0, 0, 0, V - 1, 0], 32)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [32000, 777])
def test_rows_far_from_zero(dtype, V):
    """Masks by a finite value of any size, rows that hold nothing else, and logits around
    2^20 and up to the ends of the range (the bounds of ``check`` hold over all of it)."""
    g = torch.Generator().manual_seed(V + 1)
    few = torch.rand(V, generator=g) < 0.02
    few[V // 2] = True
    rows = []
    for mask in (-1e4, -1e9, -1e10, -1e20, -1e30, -3.3e38):
        rows += [torch.where(few, torch.randn(V, generator=g) * 3, mask), torch.full((V,), mask)]
    for peak in (2e9, 1e10, 1e30, 3.3e38):
        one = torch.zeros(V)
        one[V // 3] = peak
        rows += [one, torch.full((V,), peak)]
    for centre in (2.0 ** 10, -(2.0 ** 10), 2.0 ** 20, -(2.0 ** 20), 2.0 ** 24, -(2.0 ** 24)):
        rows.append(centre + (torch.randn(V, generator=g) * 3).round())
    x = torch.stack(rows)
    top = torch.finfo(TYPES[dtype]).max
    x = x.clamp(-top, top).to(TYPES[dtype])
    tokens = [int(r.argmax()) if i % 2 else (V // 2 + i) % V for i, r in enumerate(x)]
    check(x, tokens, 20)
    check(x, tokens[::-1], 0)


def test_rows_of_any_stride_and_alignment():
    g = torch.Generator().manual_seed(1)
    for dtype in TYPES.values():
        big = torch.randn(6, 1013, generator=g).to(dtype)
        dev = big.to(DEV)
        for a, n in ((0, 1013), (1, 1000), (3, 517), (5, 64)):
            check(big[:, a:a + n], [0, n - 1, 5, -1, 2, 9], 9, dev=dev[:, a:a + n])
            check(big[::2, a:a + n], [0, n - 1, 5], 9, dev=dev[::2, a:a + n])


def test_offsets_past_32_bits():
    R, V = 70000, 32000  # 2.24e9 logits
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(2)
    tail = (torch.randn(3, V, generator=g) * 2).bfloat16()
    x[R - 3:] = tail.to(DEV)
    from cirrus_s_1a_b200.logprobs import token_logprobs

    r = token_logprobs(x, torch.full((R,), 17, dtype=torch.int32, device=DEV), 4)
    lp, ent, rank, tlp, tt = ok.token_logprobs(tail.double(), [17] * 3, 4)
    assert torch.equal(r.rank[R - 3:].cpu().long(), rank) and torch.equal(r.top_token[R - 3:].cpu().long(), tt)
    assert (r.logprob[R - 3:].cpu().double() - lp).abs().max() < 1e-5
    assert (r.logprob[:R - 3] + math.log(V)).abs().max() < 1e-5
    assert r.top_token[0].tolist() == [0, 1, 2, 3]


def test_nan_rows_stay_in_their_row():
    from cirrus_s_1a_b200.logprobs import token_logprobs

    x = torch.randn(3, 700, generator=torch.Generator().manual_seed(6))
    y = x.clone()
    y[1, 300] = math.nan
    tokens = torch.tensor([4, 4, 4], dtype=torch.int32, device=DEV)
    a, b = token_logprobs(x.to(DEV), tokens, 3), token_logprobs(y.to(DEV), tokens, 3)
    for p, q in zip(a, b):
        assert torch.equal(p[[0, 2]], q[[0, 2]])
    assert bool(b.logprob[1].isnan()) and bool(b.entropy[1].isnan())


def test_tokens_outside_the_vocabulary_are_reported():
    from cirrus_s_1a_b200.logprobs import token_logprobs

    x = torch.randn(3, 100, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    r = token_logprobs(x, torch.tensor([5, 100, -7], dtype=torch.int32, device=DEV), 2, status)
    assert int(status) == 6
    assert r.logprob[1:].tolist() == [0.0, 0.0] and r.rank[1:].tolist() == [-1, -1]
    assert float(r.logprob[0]) < 0


def test_refusals():
    from cirrus_s_1a_b200.logprobs import token_logprobs

    x = torch.randn(3, 100, device=DEV)
    t = torch.zeros(3, dtype=torch.int32, device=DEV)
    for bad in (x[0], x.cpu(), x.double(), x.t()[:3, :3]):
        with pytest.raises(ValueError):
            token_logprobs(bad, t)
    for bad in (t.long(), t[:2], t.cpu()):
        with pytest.raises(ValueError):
            token_logprobs(x, bad)
    for top in (-1, 33, 101):
        with pytest.raises(ValueError):
            token_logprobs(x, t, top)
    empty = token_logprobs(x[:0], t[:0], 2)
    assert empty.logprob.shape == (0,) and empty.top_token.shape == (0, 2)


def test_the_status_is_checked():
    from cirrus_s_1a_b200.logprobs import token_logprobs

    x = torch.randn(3, 100, device=DEV)
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for bad in (status.cpu(), status.long(), status[:0], torch.zeros(2, dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError):
            token_logprobs(x, t, 2, bad)
    token_logprobs(x, t, 2, status)


def test_rows_expanded_from_one():
    from cirrus_s_1a_b200.logprobs import token_logprobs

    x = torch.randn(3, 100, device=DEV)
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        token_logprobs(x.flatten().as_strided((3, 100), (50, 1)), t)  # rows over one another
    one = x[:1].expand(3, 100)  # one row for several tokens
    a, b = token_logprobs(one, t, 4), token_logprobs(one.contiguous(), t, 4)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
