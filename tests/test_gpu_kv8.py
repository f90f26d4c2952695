"""The 8-bit K/V cache (cb_kv8_append, cb_kv8_attend, cb_kv8_evict) against the
64-bit oracle.

Codes, scales and kept slots are compared exactly: a scale is a power of two, so
nothing but the final rounding to a code is inexact, and that rounding is the
same in any width.  Attention's bounds are derived below from the inputs."""

import math

import pytest
import torch

from oracle import kv8 as ok

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
#: half a unit in the last place of the output type, relative
HALF_ULP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def to_oracle(cache):
    f = lambda t: t.float().cpu().double()  # noqa: E731
    return {"k": f(cache.k), "v": f(cache.v), "ks": f(cache.k_scale), "vs": f(cache.v_scale),
            "mass": f(cache.mass) if cache.mass is not None else None}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def same(got, want):
    got, want = got.float().cpu().double(), want.double()
    assert torch.equal(torch.nan_to_num(got, nan=1e30), torch.nan_to_num(want, nan=1e30))


def check_state(cache, c):
    for t, n in ((cache.k, "k"), (cache.v, "v"), (cache.k_scale, "ks"), (cache.v_scale, "vs"), (cache.mass, "mass")):
        same(t, c[n])


def filled(B, H, D, L, fmt, seed=0, spread=2):
    """A cache full of codes, with block scales a few octaves apart and some mass."""
    from cirrus_s_1a_b200.kv8 import Kv8Cache

    g = torch.Generator().manual_seed(seed)
    c = Kv8Cache(B, H, D, L, fmt, device=DEV)
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = torch.randn(codes.shape, generator=g)
        x = (x * 30).round().clamp(-127, 127) if fmt == "int8" else (x * 100).clamp(-448, 448)
        codes.copy_(x.to(codes.dtype))
        scale.copy_(torch.exp2(torch.randint(-6 - spread, -5 + spread, scale.shape, generator=g).float()))
    c.mass.copy_(torch.rand(c.mass.shape, generator=g))
    return c


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_append_matches_oracle_over_a_sequence_of_calls(fmt, dtype, D):
    B, H = 3, 2
    cache = filled(B, H, D, 320, fmt)
    c = to_oracle(cache)
    g = torch.Generator().manual_seed(D)
    pos = [0, 37, 63]
    for step, T in enumerate((1, 64, 5, 1, 130, 2)):
        kv = (torch.randn(B, T, 2, H, D, generator=g) * 2.0 ** (step - 2)).to(TYPES[dtype])
        counts = [T, max(T - 3, 0), T] if step % 2 else None
        dev = kv.to(DEV)
        cache.append(dev[:, :, 0], dev[:, :, 1], ints(pos), None if counts is None else ints(counts))
        n = counts or [T] * B
        ok.append(c, fmt, kv[:, :, 0].double(), kv[:, :, 1].double(), pos, n)
        pos = [p + m for p, m in zip(pos, n)]
        check_state(cache, c)
    assert cache.read_status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_values_at_the_ends_of_the_range(fmt):
    """Zeros, subnormals, the largest floats, ties between codes, infinities and NaN."""
    top = ok.QMAX[fmt]
    x = torch.zeros(1, 64 * 6, 1, 16)
    x[0, 64:128] = 1e-40  # below 2^-100 * 0.5: all codes 0
    x[0, 128, 0, 0] = 3.4028234e38
    x[0, 129, 0, 1] = -1e30
    tie = (torch.arange(64 * 16) * 0.5 - 200).view(64, 1, 16).clamp(-top, top)
    x[0, 192:256] = tie
    x[0, 256:320] = torch.randn(64, 1, 16, generator=torch.Generator().manual_seed(1))
    x[0, 256, 0, 0], x[0, 257, 0, 0], x[0, 258, 0, 0] = math.inf, -math.inf, math.nan
    x[0, 320:384] = math.inf  # nothing finite
    cache = filled(1, 1, 16, 384, fmt)
    c = to_oracle(cache)
    dev = x.to(DEV)
    cache.append(dev, dev, ints([0]))
    ok.append(c, fmt, x.double(), x.double(), [0], [384])
    check_state(cache, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_of_misaligned_and_transposed_inputs(dtype):
    B, T, H, D = 2, 70, 3, 64
    g = torch.Generator().manual_seed(5)
    cache = filled(B, H, D, 192, "int8")
    c = to_oracle(cache)
    flat = torch.randn(1 + B * T * H * D, generator=g).to(TYPES[dtype]).to(DEV)
    k = flat[1:].view(B, H, T, D).transpose(1, 2)  # odd start, head-major
    v = flat[1:].view(T, B, H, D).transpose(0, 1)
    cache.append(k, v, ints([11, 64]))
    ok.append(c, "int8", k.cpu().double(), v.cpu().double(), [11, 64], [T, T])
    check_state(cache, c)


def test_append_past_the_end_drops_and_reports():
    cache = filled(2, 1, 32, 128, "e4m3")
    c = to_oracle(cache)
    x = torch.randn(2, 10, 1, 32)
    cache.append(x.to(DEV), x.to(DEV), ints([122, -1]))
    ok.append(c, "e4m3", x.double(), x.double(), [122, -1], [10, 10])
    check_state(cache, c)
    assert cache.read_status() == 5
    cache.clear_status()
    cache.append(x.to(DEV), x.to(DEV), ints([118, 0]))
    assert cache.read_status() == 0


# ----------------------------------------------------------------- attend
def check_attend(cache, q, pos, counts=None, dtype="bf16", add_mass=False, scale=None, longest=None, hold=None):
    """Bounds.  The codes and 16-bit queries meet exactly, so a score's error is
    that of D float32 additions: at most D * 2^-22 * sum |q k| (tensor cores may
    truncate: twice 2^-23), plus 2^-21 of it where a float32 query is carried in 22
    bits; call it d.  A probability is off by a factor exp(2 d) and the hardware
    exp2's and the sums' 2^-20; f16 probabilities add 2^-11 each and at least 2^-25
    against the row's largest.  The output adds its own rounding."""
    D = q.shape[-1]
    B, T = q.shape[:2]
    n = counts or [T] * B
    scale = D ** -0.5 if scale is None else scale
    c = hold or to_oracle(cache)
    before = c["mass"].clone() if add_mass else None
    out, lse = cache.attend(q.to(DEV), ints(pos), None if counts is None else ints(counts), scale=scale,
                            add_mass=add_mass, longest=longest)
    want, wlse, size = ok.attend(c, q.double(), pos, n, scale, add_mass)
    assert out.dtype == TYPES[dtype] and lse.dtype == torch.float32
    d = size * (D * 2.0 ** -22 + 2.0 ** -21)
    finite = torch.isfinite(wlse)
    assert torch.equal(torch.isfinite(lse.cpu()), finite)
    assert (lse.cpu().double() - wlse)[finite].abs().le((d + 2.0 ** -20 * (1 + wlse.abs()))[finite]).all()
    vmax = ok.values(torch.nan_to_num(c["v"]), c["vs"]).abs().max()
    most = max(p + m for p, m in zip(pos, n))
    rel = 2 * d + 2.0 ** -20 + (0 if dtype == "f32" else 2.0 ** -11 + max(most, 1) * 2.0 ** -25)
    bound = want.abs() * HALF_ULP[dtype] + vmax * rel[..., None] + 1e-30
    err = (out.cpu().double() - want).abs()
    assert err.le(bound).all(), float((err / bound).max())
    if add_mass:
        added = c["mass"] - before
        off = (cache.mass.cpu().double() - c["mass"]).abs()
        assert off.le(added * (2 * float(d.max()) + 2.0 ** -19) + c["mass"] * 2.0 ** -22).all()
    return out, lse


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Hq,H,D", [(4, 2, 16), (4, 4, 32), (12, 4, 64), (6, 2, 128), (16, 2, 64), (5, 1, 128)])
def test_attend_decode_and_verify(fmt, dtype, Hq, H, D):
    g = torch.Generator().manual_seed(Hq * D)
    cache = filled(3, H, D, 832, fmt, seed=D)
    for T, pos in ((1, [0, 63, 64]), (5, [700, 129, -1]), (8, [823, 1, 256])):
        q = (1.5 * torch.randn(3, T, Hq, D, generator=g)).to(TYPES[dtype])
        check_attend(cache, q, pos, dtype=dtype, add_mass=T == 5)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Hq,H,D,T,pos", [(12, 4, 64, 150, [0, 77]), (8, 2, 128, 97, [300, 0]), (4, 2, 16, 40, [5, 9]),
                                          (3, 1, 64, 257, [0, 511]), (1, 1, 128, 129, [64, 130])])
def test_attend_prompts(fmt, dtype, Hq, H, D, T, pos):
    g = torch.Generator().manual_seed(T)
    cache = filled(2, H, D, 832, fmt, seed=T)
    q = (1.5 * torch.randn(2, T, Hq, D, generator=g)).to(TYPES[dtype])
    check_attend(cache, q, pos, dtype=dtype, add_mass=True)
    check_attend(cache, q, pos, counts=[T - 9, 0], dtype=dtype, add_mass=True)


@pytest.mark.parametrize("D,dtype", [(16, "bf16"), (32, "f32")])
def test_long_prompts_of_many_sequences(D, dtype):
    """More query rows over all heads than the scratch has counters for.  Against a call for
    each sequence: the same scores, joined in other parts."""
    from cirrus_s_1a_b200.kv8 import Kv8Cache

    B, T = 33, 4096
    big = filled(B, 2, D, T + 64, "int8")
    q = torch.randn(B, T, 4, D, generator=torch.Generator().manual_seed(D)).to(TYPES[dtype]).to(DEV)
    pos = ints([b % 7 for b in range(B)])
    before = big.mass.clone()
    out, lse = big.attend(q, pos, add_mass=True)
    again, _ = big.attend(q, pos)
    assert torch.equal(out, again)
    for b in (0, 17, 32):
        one = Kv8Cache.from_tensors(*(t[b:b + 1].contiguous() for t in (big.k, big.v, big.k_scale, big.v_scale, before)))
        o, s = one.attend(q[b:b + 1].contiguous(), ints([b % 7]), add_mass=True)
        near = 127 * float(big.v_scale.max()) * (2.0 ** -7 if dtype == "bf16" else 2.0 ** -17)
        assert (o[0].float() - out[b].float()).abs().max() <= near
        assert (s[0] - lse[b]).abs().max() < 2.0 ** -16
        assert (one.mass[0] - big.mass[b]).abs().max() <= 2.0 ** -15 * one.mass.abs().max()


def test_rows_that_see_nothing_give_zero_and_minus_infinity():
    cache = filled(4, 2, 64, 128, "e4m3")
    q = torch.randn(4, 3, 6, 64).bfloat16()
    out, lse = check_attend(cache, q, [-3, -1, 0, 20], counts=[3, 3, 0, 2])
    assert torch.equal(out[0].float().cpu(), torch.zeros(3, 6, 64)) and bool((lse[0] == -math.inf).all())
    assert bool((out[3, 2] == 0).all()) and bool((out[2] == 0).all())


@pytest.mark.parametrize("T", [1, 150])
@pytest.mark.parametrize("D", [64, 128])
def test_unused_slots_may_hold_nan(T, D):
    """Codes, scales and mass past the sequence's end reach no result."""
    cache = filled(1, 2, D, 512, "e4m3")
    n = 203 + T
    hold = to_oracle(cache)
    cache.k.view(torch.uint8)[:, :, n:] = 0x7F
    cache.v.view(torch.uint8)[:, :, n:] = 0xFF
    cache.k_scale[:, :, -(-n // 64):] = math.nan
    cache.v_scale[:, :, -(-n // 64):] = math.inf
    q = torch.randn(1, T, 6, D, generator=torch.Generator().manual_seed(3)).bfloat16()
    out, lse = check_attend(cache, q, [203], hold=hold)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    mass = cache.mass.clone()
    cache.attend(q.to(DEV), ints([203]), add_mass=True)
    assert torch.equal(mass[:, :, n:], cache.mass[:, :, n:])


@pytest.mark.parametrize("T", [1, 140])
def test_block_scales_twenty_octaves_apart(T):
    """Neither a block of tiny values nor one of huge ones costs the others their precision."""
    cache = filled(1, 1, 64, 512, "int8")
    cache.k_scale[0, 0] = torch.exp2(torch.tensor([-7., -27., -8., -7., -9., -7., -17., -7.]))
    cache.v_scale[0, 0] = torch.exp2(torch.tensor([-7., 13., -7., -7., -27., -7., -7., 3.]))
    q = torch.randn(1, T, 3, 64, generator=torch.Generator().manual_seed(9)).half()
    check_attend(cache, q, [300], dtype="f16")
    # only the small blocks are visible to the first rows: their error is bounded by their own values
    cache.v_scale[0, 0] = torch.exp2(torch.tensor([-27., -27., -27., -27., -27., -27., -27., 13.]))
    out, _ = cache.attend(q.float().to(DEV), ints([300]))
    want, _, _ = ok.attend(to_oracle(cache), q.double(), [300], [T], 0.125)
    rows = min(T, 448 - 300)
    assert (out[:, :rows].cpu().double() - want[:, :rows]).abs().max() <= 127 * 2.0 ** -27 * 2.0 ** -10


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 1), (64, 140), (128, 1), (128, 140), (16, 6)])
@pytest.mark.parametrize("e", [1, 10, 30, 110])
def test_value_blocks_of_zeros_beside_large_ones(fmt, dtype, D, T, e):
    """A block of zero values has the scale 2^-100: its keys weigh as much as any others',
    wherever it lies, and so do those of a block whose values are as small as that."""
    cache = filled(1, 2, D, 704, fmt, seed=e)
    for h, zero in ((0, (0, 4)), (1, (3, 7, 8))):
        cache.v_scale[0, h] = torch.exp2(torch.randint(e - 2, e + 1, (11,), generator=torch.Generator().manual_seed(h)))
        for blk in zero:
            cache.v_scale[0, h, blk] = 2.0 ** -100
            if blk != 7:
                cache.v.view(torch.uint8)[0, h, 64 * blk:64 * blk + 64] = 0
    q = (1.5 * torch.randn(1, T, 6, D, generator=torch.Generator().manual_seed(T))).to(TYPES[dtype])
    check_attend(cache, q, [700 - T], dtype=dtype, add_mass=True)
    # only keys of zero values, then one block of others
    check_attend(cache, q, [max(63 - T, 0)], dtype=dtype, add_mass=True)


@pytest.mark.parametrize("n", [64, 128, 32768])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_float32_keeps_small_probabilities(D, n):
    """One key weighs 2^13 times as much as each of the others but its value is 0: head and tail
    carry every probability to 2^-22 of itself, the exponential and the sums add 2^-20, truncated
    products of 64 keys as much again: less than 2^-18 in all.  (The scores are exact.)"""
    cache = filled(1, 1, D, n, "int8")
    cache.k.zero_()
    cache.k[0, 0, 50, 0] = 1
    cache.k_scale.fill_(1.0)
    v = torch.arange(D).remainder(127) + 1
    cache.v.copy_(v.to(torch.int8).expand(1, 1, n, D))
    cache.v[0, 0, 50] = 0
    cache.v_scale.fill_(1.0)
    for score in (9.125, 8.875, 9.25):
        q = torch.zeros(1, 1, 1, D)
        q[..., 0] = score
        out, lse = cache.attend(q.to(DEV), ints([n - 1]), scale=1.0)
        small = (n - 1) * math.exp(-score)
        want = v.double() * small / (1 + small)
        assert (out[0, 0, 0].cpu().double() / want - 1).abs().max() < 2.0 ** -18


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("T", [1, 130])
def test_values_of_equal_keys_come_out_whatever_the_scores(D, T):
    """Keys and values all alike: the output is the value.  Probabilities carry 2^-22, exponentials
    and sums 2^-20, and up to 18 products of 16 keys a truncation of 2^-23 each: less than 2^-18.
    (A score of 4095 has its last bit at 2^-12, but it is the same for all keys.)"""
    cache = filled(1, 1, D, 192, "int8")
    cache.k.fill_(1)
    cache.v.fill_(93)
    cache.k_scale.fill_(1.0)
    for e in (-20, -6, 0, 9):
        cache.v_scale.fill_(2.0 ** e)
        for score in (0.0, 11.0, 2848.5, 2849.125, 2849.75, 2850.5, -2834.5, -2835.125, -2836.25, 90000.0):
            q = torch.full((1, T, 1, D), score / D)
            out, lse = cache.attend(q.to(DEV), ints([130 - T]), scale=1.0)
            assert (out.cpu().double() / (93 * 2.0 ** e) - 1).abs().max() < 2.0 ** -18, (e, score)


@pytest.mark.parametrize("T", [1, 130])
def test_peaked_and_extreme_scores(T):
    """Scores of thousands (one key takes all), queries of 1e-30 (all keys alike) and zeros."""
    cache = filled(1, 1, 64, 320, "e4m3")
    q = torch.randn(1, T, 3, 64, generator=torch.Generator().manual_seed(2))
    check_attend(cache, (q * 1000).bfloat16(), [190 - T])
    check_attend(cache, (q * 1e-30).bfloat16(), [190 - T])
    check_attend(cache, torch.zeros(1, T, 3, 64).bfloat16(), [190 - T])
    check_attend(cache, q, [190 - T], dtype="f32", scale=0.7, longest=190)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 1), (64, 130), (128, 5), (128, 130), (16, 3)])
def test_scores_of_any_size(D, T, dtype):
    """Queries up to the end of the range.  A key thousands ahead of the others takes the row:
    its value comes out to the type's rounding and the 2^-20 of probabilities and sums, and
    it takes each row's weight (to the 2 d of ``check_attend``, d the error of such a score).
    Where float32 scores are too coarse to say which key does, outputs stay within the
    values seen and weights within the number of rows."""
    cache = filled(1, 1, D, 320, "e4m3")
    cache.k.view(torch.uint8)[0, 0, :, 0] = 0x38  # 1
    cache.k.view(torch.uint8)[0, 0, 20, 0] = 0x7E  # 448
    cache.k_scale.fill_(2.0 ** -6)
    cache.mass.zero_()
    for size in (1e3, 1e6, 1e8, 1e9, 1e12, 1e30, 1e34):
        q = torch.zeros(1, T, 3, D)
        q[..., 0] = size
        q = q.to(TYPES[dtype])
        out, lse = cache.attend(q.to(DEV), ints([180 - T]), scale=0.5, add_mass=True)
        score = float(q[0, 0, 0, 0].double()) * 7 * 0.5
        want = cache.v[0, 0, 20].float() * cache.v_scale[0, 0, 0]
        assert ((out.float() - want).abs() <= want.abs() * (2.0 ** -8 if dtype == "bf16" else 2.0 ** -19)).all(), size
        assert (lse.double() / score - 1).abs().max() < 2.0 ** -20
        d = score * (D * 2.0 ** -22 + 2.0 ** -21)
        assert 3 * T * (1 - 2 * d - 2.0 ** -19) <= float(cache.mass[0, 0, 20]) <= 3 * T * (1 + 2.0 ** -19)
        assert not cache.mass[0, 0, :20].any() and not cache.mass[0, 0, 21:].any()
        cache.mass.zero_()
    g = torch.Generator().manual_seed(1)
    top = (cache.v.float() * cache.v_scale.repeat_interleave(64, -1)[..., None]).abs().max()
    for size in (1e6, 1e9, 1e20, 1e34):
        q = (torch.randn(1, T, 3, D, generator=g) * size).to(TYPES[dtype]).to(DEV)
        out, lse = cache.attend(q, ints([180 - T]), add_mass=True)
        assert bool(torch.isfinite(lse).all()) and bool((out.abs() <= top * 1.01).all())
        assert bool((cache.mass >= 0).all()) and bool((cache.mass <= 3 * T * 1.01).all())
        cache.mass.zero_()


def test_nan_in_a_visible_key_reaches_its_rows_only():
    cache = filled(1, 1, 64, 128, "e4m3")
    cache.k.view(torch.uint8)[0, 0, 70, 5] = 0x7F
    q = torch.randn(1, 4, 2, 64).bfloat16().to(DEV)
    out, lse = cache.attend(q, ints([68]))
    assert bool(torch.isfinite(out[0, :2]).all()) and bool(out[0, 2:].isnan().all()) and bool(lse[0, 2:].isnan().all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 4), (64, 140), (128, 140), (128, 1), (16, 5)])
def test_nan_in_a_value_reaches_the_rows_that_see_it_only(D, T, dtype):
    """A NaN value in a slot that later rows see and earlier ones do not (0 * NaN is not 0)."""
    cache = filled(1, 1, D, 512, "e4m3")
    q = torch.randn(1, T, 3, D, generator=torch.Generator().manual_seed(8)).to(TYPES[dtype]).to(DEV)
    clean, clean_lse = cache.attend(q, ints([200]))
    at = T // 2
    cache.v.view(torch.uint8)[0, 0, 200 + at, 3] = 0xFF
    cache.v.view(torch.uint8)[0, 0, 200 + T] = 0x7F  # no row sees this one
    out, lse = cache.attend(q, ints([200]))
    assert torch.equal(out[0, :at], clean[0, :at]) and torch.equal(lse[0, :at], clean_lse[0, :at])
    assert bool(out[0, at:, :, 3].isnan().all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 1), (64, 2), (64, 4), (64, 140), (128, 140), (128, 1), (128, 5), (16, 5), (32, 60)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_query_that_is_not_finite_gives_nan(D, T, dtype, bad):
    """Not the 0 and -infinity of a row that sees nothing.  The other rows, and the
    weights of slots that the row does not see, are as they would be without it, up to
    the roundings of two runs whose maxima rise at other keys: 2^-20 in the sums, and in
    bf16 outputs that of the probabilities and of the output."""
    cache = filled(1, 1, D, 512, "int8")
    mass = cache.mass.clone()
    q = torch.randn(1, T, 3, D, generator=torch.Generator().manual_seed(8)).to(TYPES[dtype]).to(DEV)
    clean, clean_lse = cache.attend(q, ints([200]), add_mass=True)
    clean_mass = cache.mass.clone()
    at = T // 2
    q[0, at, 1, D - 3] = bad
    cache.mass.copy_(mass)
    out, lse = cache.attend(q, ints([200]), add_mass=True)
    rest = torch.ones(T, 3, dtype=torch.bool)
    rest[at, 1] = False
    assert bool(out[0, at, 1].isnan().all()) and bool(lse[0, at, 1].isnan())
    near = 127 * float(cache.v_scale.max()) * (2.0 ** -7 if dtype == "bf16" else 2.0 ** -18)
    assert (out[0][rest].float() - clean[0][rest].float()).abs().amax().le(near) 
    assert torch.allclose(lse[0][rest], clean_lse[0][rest], rtol=2.0 ** -19, atol=2.0 ** -19)
    assert bool(cache.mass[0, 0, :201 + at].isnan().all())
    assert torch.allclose(cache.mass[0, 0, 201 + at:], clean_mass[0, 0, 201 + at:], rtol=2.0 ** -17, atol=0)


@pytest.mark.parametrize("D,T", [(64, 1), (64, 4), (64, 140), (128, 140), (128, 1), (16, 5)])
def test_a_row_that_sees_nan_keys_alone_gives_nan(D, T):
    cache = filled(1, 1, D, 512, "e4m3")
    cache.k.view(torch.uint8)[0, 0, 0, 5] = 0x7F
    q = torch.randn(1, T, 3, D, generator=torch.Generator().manual_seed(8)).bfloat16().to(DEV)
    out, lse = cache.attend(q, ints([0]), add_mass=True)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())  # every row sees slot 0
    assert bool(cache.mass[0, 0, :T].isnan().all()) and bool(torch.isfinite(cache.mass[0, 0, T:]).all())
    cache = filled(1, 1, D, 512, "e4m3")
    cache.k.view(torch.uint8)[0, 0, :64, 5] = 0x7F  # a whole block, beside finite ones
    out, lse = cache.attend(q, ints([300]))
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,T", [(64, 4), (64, 140), (128, 140), (128, 1), (128, 9), (16, 5), (32, 50)])
def test_a_nan_value_stays_in_its_dimension(D, T, dtype):
    """In a block that every row sees and in one that some rows see in part: the other
    dims, the sums and the weights do not change."""
    cache = filled(1, 1, D, 512, "e4m3")
    mass = cache.mass.clone()
    q = torch.randn(1, T, 3, D, generator=torch.Generator().manual_seed(8)).to(TYPES[dtype]).to(DEV)
    clean, clean_lse = cache.attend(q, ints([200]), add_mass=True)
    clean_mass = cache.mass.clone()
    at = T // 2
    for slot, first in ((200 + at, at), (7, 0)):
        codes = cache.v.view(torch.uint8)
        was = codes[0, 0, slot].clone()
        codes[0, 0, slot, 3], codes[0, 0, slot, D - 1] = 0xFF, 0x7F
        cache.mass.copy_(mass)
        out, lse = cache.attend(q, ints([200]), add_mass=True)
        codes[0, 0, slot] = was
        assert torch.equal(lse, clean_lse) and torch.equal(cache.mass, clean_mass)
        assert bool(out[0, first:, :, [3, D - 1]].isnan().all())
        out[0, first:, :, [3, D - 1]] = clean[0, first:, :, [3, D - 1]]
        assert torch.equal(out, clean)


def test_query_strides_and_other_streams():
    cache = filled(2, 2, 64, 256, "int8")
    proj = torch.randn(2, 7, 6 * 64 + 13, generator=torch.Generator().manual_seed(4)).to(DEV)
    q = proj[..., 13:].unflatten(-1, (6, 64))  # rows of an odd stride, misaligned
    pos = ints([100, 3])
    a, la = cache.attend(q, pos)
    b, lb = cache.attend(q.contiguous(), pos)
    assert torch.equal(a, b) and torch.equal(la, lb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d, ld = cache.attend(q, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, d) and torch.equal(la, ld)


@pytest.mark.parametrize("T", [1, 200])
def test_results_repeat_and_replay_in_a_graph(T):
    cache = filled(2, 2, 64, 1024, "e4m3")
    q = torch.randn(2, T, 6, 64).bfloat16().to(DEV)
    pos = ints([800, 333])
    cache.mass.zero_()
    a, la = cache.attend(q, pos, add_mass=True)
    mass = cache.mass.clone()
    cache.mass.zero_()
    b, lb = cache.attend(q, pos, add_mass=True)
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(mass, cache.mass)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(q, pos)
        with torch.cuda.graph(graph, stream=side):
            d, _ = cache.attend(q, pos)
    torch.cuda.current_stream().wait_stream(side)
    pos.copy_(ints([500, 1]))
    graph.replay()
    e, _ = cache.attend(q, pos)
    assert torch.equal(d, e)


def test_a_graph_keeps_its_scratch():
    """A longer call on the capture's stream replaces the stream's buffer, not the graph's."""
    cache = filled(2, 2, 64, 1024, "e4m3")
    q = torch.randn(2, 1, 6, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    long = torch.randn(2, 500, 6, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    pos = ints([400, 333])
    want, wlse = cache.attend(q, pos)
    wlong, _ = cache.attend(long, pos)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(q, pos)
        with torch.cuda.graph(graph, stream=side):
            out, lse = cache.attend(q, pos)
        got, _ = cache.attend(long, pos)
        held = [torch.full((1 << 20,), 7, dtype=torch.uint8, device=DEV) for _ in range(64)]  # where it may have been
        for _ in range(3):
            graph.replay()
        again, _ = cache.attend(long, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    assert torch.equal(got, wlong) and torch.equal(again, wlong)
    assert all(bool((h == 7).all()) for h in held)


def test_graphs_captured_without_a_call_before_replay_in_any_order():
    cache = filled(2, 2, 64, 1024, "e4m3")
    pos = ints([400, 333])
    qs = [torch.randn(2, T, 6, 64, generator=torch.Generator().manual_seed(T)).bfloat16().to(DEV) for T in (1, 5, 130)]
    want = [cache.attend(q, pos) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, got = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            got.append(cache.attend(q, pos))
    with torch.cuda.stream(side):
        eager = cache.attend(qs[0], pos)  # between the captures and their first replay
        for i in (2, 1, 0, 1, 2):
            graphs[i].replay()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(eager[0], want[0][0])
    for (a, la), (b, lb) in zip(got, want):
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_lengths_that_change_with_every_token_keep_no_entry_each():
    cache = filled(1, 1, 16, 1024, "int8")
    q = torch.randn(1, 1, 1, 16).to(DEV)
    for n in range(600):
        cache.attend(q, ints([n]), longest=n + 1)
    assert len(cache._sizes) <= 256 and len(cache._scratch) == 1


def test_offsets_past_32_bits():
    """The last sequence of a cache whose codes pass 2^31 bytes."""
    from cirrus_s_1a_b200.kv8 import Kv8Cache

    B, H, D, L = 65, 2, 128, 131072
    big = Kv8Cache(B, H, D, L, "int8", device=DEV, mass=False)
    small = filled(1, H, D, 320, "int8")
    for name in ("k", "v"):
        getattr(big, name)[B - 1, :, :320] = getattr(small, name)[0]
        getattr(big, name + "_scale")[B - 1, :, :5] = getattr(small, name + "_scale")[0]
    for T in (1, 140):
        q = torch.randn(B, T, 4, D).bfloat16().to(DEV)
        pos = torch.full((B,), -T, dtype=torch.int32, device=DEV)
        pos[B - 1] = 150
        out, lse = big.attend(q, pos)
        want, wlse = small.attend(q[B - 1:].contiguous(), ints([150]))
        assert (out[B - 1].float() - want[0].float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
        assert (lse[B - 1] - wlse[0]).abs().max() < 1e-4
        assert bool((out[:B - 1] == 0).all())
    x = torch.randn(B, 3, H, D).to(DEV)
    big.append(x, x, ints([-1] * (B - 1) + [L - 3]))
    got = big.k[B - 1, :, L - 3:].float() * big.k_scale[B - 1, :, -1, None, None]
    assert (got - x[B - 1].transpose(0, 1)).abs().max() <= 0.5 * float(big.k_scale[B - 1, :, -1].max())


# ------------------------------------------------------------------ evict
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("keep,recent", [(300, 100), (64, 0), (129, 129), (1, 0), (1, 1), (511, 3)])
def test_evict_matches_oracle(fmt, D, keep, recent):
    B, H = 4, 2
    cache = filled(B, H, D, 512, fmt, seed=keep)
    cache.mass[0, 0, :200] = cache.mass[0, 0, 0].clone()  # ties
    cache.mass[0, 1, 5:90:7] = math.nan
    cache.mass[2] = 0.0  # nothing but ties
    cache.mass[3, 0, ::3] = -0.0
    cache.mass[3, 1, ::5] = math.inf
    pos = [512, keep, 300, 511]
    c = to_oracle(cache)
    kept, new = cache.evict(ints(pos), keep, recent)
    wkept, wnew = ok.evict(c, fmt, pos, keep, recent)
    assert torch.equal(kept.cpu().long(), wkept)
    assert new.tolist() == wnew
    check_state(cache, c)


def test_evict_of_long_and_empty_sequences():
    cache = filled(3, 1, 32, 20480, "e4m3")
    cache.mass.copy_((cache.mass * 50).floor())  # many ties over a long sequence
    c = to_oracle(cache)
    pos = [20480, 0, 17001]
    kept, new = cache.evict(ints(pos), 10001, 777)
    wkept, wnew = ok.evict(c, "e4m3", pos, 10001, 777)
    assert torch.equal(kept.cpu().long(), wkept) and new.tolist() == wnew
    check_state(cache, c)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_bounded_cache_through_its_life(fmt):
    """Append, attend with weights, evict, again and again, against the oracle's same steps."""
    from cirrus_s_1a_b200.kv8 import Kv8Cache

    B, H, G, D = 2, 2, 3, 64
    cache = Kv8Cache(B, H, D, 256, fmt, device=DEV)
    c = to_oracle(cache)
    g = torch.Generator().manual_seed(11)
    pos = [0, 0]
    for T in (90, 100, 1, 1, 40, 66, 8, 90):
        x = torch.randn(B, T, 2 * H + H * G, D, generator=g)
        k, v, q = x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:].bfloat16()
        dev = x.to(DEV)
        cache.append(dev[:, :, :H], dev[:, :, H:2 * H], ints(pos))
        ok.append(c, fmt, k.double(), v.double(), pos, [T] * B)
        same(cache.k, c["k"])
        check_attend(cache, q, pos, add_mass=True)
        c = to_oracle(cache)  # go on from the device's mass: ranks of near ties follow its rounding
        pos = [p + T for p in pos]
        _, new = cache.evict(ints(pos), 160, 32)
        _, pos = ok.evict(c, fmt, pos, 160, 32)
        assert new.tolist() == pos
        check_state(cache, c)


# --------------------------------------------------------------- refusals
def test_refusals():
    from cirrus_s_1a_b200 import _lib
    from cirrus_s_1a_b200.kv8 import Kv8Cache

    with pytest.raises(ValueError):
        Kv8Cache(1, 1, 64, 64, "fp4", device=DEV)
    with pytest.raises(ValueError):
        Kv8Cache(1, 1, 48, 64, device=DEV)
    with pytest.raises(ValueError):
        Kv8Cache(0, 1, 64, 64, device=DEV)
    c = Kv8Cache(2, 2, 64, 100, device=DEV)
    assert c.max_len == 128
    pos = ints([0, 0])
    x = torch.zeros(2, 3, 2, 64, device=DEV)
    for bad in (x[:1], x[..., :32], x.cpu(), x.double(), torch.zeros(2, 0, 2, 64, device=DEV),
                torch.zeros(2, 3, 2, 128, device=DEV)[..., ::2]):
        with pytest.raises(ValueError):
            c.append(bad, bad, pos)
    with pytest.raises(ValueError):
        c.append(x, x[:, :2], pos)
    with pytest.raises(ValueError):
        c.append(x, x.half(), pos)
    with pytest.raises(_lib.CbError):
        c.append(torch.zeros(2, 129, 2, 64, device=DEV), torch.zeros(2, 129, 2, 64, device=DEV), pos)
    for bad in (pos.long(), pos[:1], pos.cpu()):
        with pytest.raises(ValueError):
            c.append(x, x, bad)
    with pytest.raises(ValueError):
        c.attend(torch.zeros(2, 1, 3, 64, device=DEV), pos)
    with pytest.raises(ValueError):
        c.attend(x, pos, out=torch.empty(2, 3, 2, 64, device=DEV, dtype=torch.bfloat16))
    for keep, recent in ((0, 0), (129, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            c.evict(pos, keep, recent)
    bare = Kv8Cache(2, 2, 64, 64, device=DEV, mass=False)
    with pytest.raises(ValueError):
        bare.evict(pos, 4, 0)
    with pytest.raises(ValueError):
        bare.attend(x, pos, add_mass=True)
    with pytest.raises(ValueError):
        Kv8Cache.from_tensors(c.k, c.v, c.k_scale[..., :1], c.v_scale)
    with pytest.raises(ValueError):
        Kv8Cache.from_tensors(c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)
