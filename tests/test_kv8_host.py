"""CPU tests of the 8-bit cache and the log probabilities: the C entry points
refuse bad arguments before any CUDA call, the ctypes struct matches the C
layout, and the 64-bit oracle's codec agrees with independent statements of it."""

import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from conftest import ROOT
from oracle import kv8 as ok
from test_host import built_lib  # noqa: F401


def desc(**kw):
    from cirrus_s_1a_b200._lib import CbKv8

    a = dict(batch=1, n_kv_heads=2, head_dim=64, max_len=128, format=0, k=256, v=512, k_scale=256, v_scale=256, mass=256)
    a.update(kw)
    return C.byref(CbKv8(*a.values()))


def test_entry_points_refuse_bad_arguments_without_launching(built_lib):  # noqa: F811
    L = built_lib
    s3 = (C.c_int64 * 3)(1, 1, 1)
    before = L.cb_launch_count()
    app = lambda c, k=256, dtype=0, T=1, pos=256: L.cb_kv8_append(c, k, 256, dtype, s3, s3, T, pos, None, None, None)  # noqa: E731
    assert app(None) == 1 and app(desc(), k=None) == 1 and app(desc(), dtype=3) == 1 and app(desc(), T=0) == 1
    assert app(desc(), pos=None) == 1 and app(desc(k=None)) == 1 and app(desc(batch=0)) == 1
    assert app(desc(head_dim=48)) == 2 and app(desc(max_len=100)) == 2 and app(desc(format=2)) == 1
    assert app(desc(k=260)) == 1  # codes are read 16 bytes at a time
    assert app(desc(batch=65536)) == 2
    assert app(desc(), T=129) == 1  # more tokens than slots
    big = 1 << 40
    att = lambda c, hq=2, T=1, longest=128, mass=0, scratch=256, n=big, dtype=1: L.cb_kv8_attend(  # noqa: E731
        c, 256, dtype, s3, hq, T, 256, None, longest, 1.0, mass, 256, 256, scratch, n, None, None)
    assert att(None) == 1 and att(desc(), hq=3) == 2 and att(desc(), T=0) == 1 and att(desc(), longest=0) == 1
    assert att(desc(), scratch=None) == 1 and att(desc(), n=0) == 4 and att(desc(mass=None), mass=1) == 1
    assert att(desc(), dtype=7) == 1 and att(desc(head_dim=100)) == 2
    assert att(desc(), scratch=264) == 1
    need = lambda c, dtype, hq, T, n: L.cb_kv8_attend_scratch_bytes(c, dtype, hq, T, n, 0)  # noqa: E731
    assert need(desc(), 1, 2, 1, 128) > 0 and L.cb_kv8_attend_scratch_bytes(desc(), 1, 2, 1, 128, 1) > need(desc(), 1, 2, 1, 128)
    assert need(desc(), 1, 3, 1, 128) == 0 and need(None, 1, 2, 1, 1) == 0 and need(desc(), 5, 2, 1, 1) == 0
    ev = lambda c, keep=4, recent=2, pos=256, new=512: L.cb_kv8_evict(c, pos, keep, recent, 256, new, None)  # noqa: E731
    assert ev(None) == 1 and ev(desc(mass=None)) == 1 and ev(desc(), keep=0) == 1 and ev(desc(), recent=5) == 1
    assert ev(desc(), keep=129, recent=0) == 1 and ev(desc(), new=256) == 1 and ev(desc(), recent=-1) == 1
    lp = lambda x=256, dtype=0, ld=100, rows=1, V=100, tok=256, top=0, tp=256: L.cb_token_logprobs(  # noqa: E731
        x, dtype, ld, rows, V, tok, top, 256, 256, 256, tp, tp, None, None)
    assert lp(x=None) == 1 and lp(dtype=4) == 1 and lp(ld=99) == 1 and lp(rows=0) == 1 and lp(V=0) == 1
    assert lp(tok=None) == 1 and lp(top=101) == 1 and lp(top=2, tp=None) == 1 and lp(top=33) == 2
    assert lp(V=(1 << 20) + 1, ld=1 << 21) == 2
    assert L.cb_launch_count() == before


def test_struct_matches_the_c_layout(built_lib, tmp_path):  # noqa: F811
    from cirrus_s_1a_b200._lib import CbKv8

    src = tmp_path / "o.c"
    names = [n for n, _ in CbKv8._fields_]
    src.write_text('#include <stdio.h>\n#include "cirrus_b200.h"\nint main(void){printf("%zu", sizeof(CbKv8));'
                   + "".join(f'printf(" %zu", offsetof(CbKv8, {n}));' for n in names) + "return 0;}")
    exe = tmp_path / "o"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    assert got == [C.sizeof(CbKv8)] + [getattr(CbKv8, n).offset for n in names]


def test_classes_refuse_without_a_gpu():
    from cirrus_s_1a_b200 import _lib
    from cirrus_s_1a_b200.kv8 import Kv8Cache
    from cirrus_s_1a_b200.logprobs import token_logprobs

    with pytest.raises(ValueError):
        Kv8Cache(1, 1, 64, 64, "fp4")
    if not torch.cuda.is_available():
        with pytest.raises(_lib.CbError):
            Kv8Cache(1, 1, 64, 64)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_oracle_scale_is_the_smallest_power_of_two(fmt):
    q = ok.QMAX[fmt]
    for a in (q, math.nextafter(q, 0), math.nextafter(q, 1e9), 1.0, 2.0 ** -20, q / 2, 3.0, 1e30, 1e-20):
        e = ok.need_exponent(a, fmt)
        assert a <= math.ldexp(q, e) and a > math.ldexp(q, e - 1)
    assert ok.need_exponent(0.0, fmt) == ok.E_MIN == ok.need_exponent(1e-38, fmt)


def test_oracle_encode_is_the_e4m3_cast():
    x = torch.cat([torch.linspace(-448, 448, 40001), torch.randn(20000) * 2.0 ** -7,
                   torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()])
    x = x[torch.isfinite(x)]
    assert torch.equal(ok.encode(x.double(), "e4m3"), x.to(torch.float8_e4m3fn).double())
    y = torch.tensor([0.5, 1.5, -2.5, 200.0, -math.inf, math.nan], dtype=torch.float64)
    assert ok.encode(y, "int8").tolist() == [0.0, 2.0, -2.0, 127.0, -127.0, 0.0]


def test_oracle_attention_and_logprobs_against_torch():
    torch.manual_seed(0)
    H, L, D = 2, 128, 16
    c = {"k": torch.randn(1, H, L, D).double(), "v": torch.randn(1, H, L, D).double(),
         "ks": torch.full((1, H, 2), 0.5).double(), "vs": torch.full((1, H, 2), 2.0).double(),
         "mass": torch.zeros(1, H, L).double()}
    q = torch.randn(1, 5, 4, D).double()
    out, lse, _ = ok.attend(c, q, [90], [5], 0.25, True)
    mask = torch.arange(95) <= 90 + torch.arange(5)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(1, 2), 0.5 * c["k"][:, :, :95].repeat_interleave(2, 1),
        2.0 * c["v"][:, :, :95].repeat_interleave(2, 1), attn_mask=mask, scale=0.25)
    assert torch.allclose(out, want.transpose(1, 2), atol=1e-12)
    assert torch.allclose(c["mass"].sum(), torch.tensor(20.0).double())  # 5 rows of 4 heads
    x = torch.randn(3, 50).double()
    lp, ent, rank, tlp, tt = ok.token_logprobs(x, [4, -1, 9], 3)
    d = torch.distributions.Categorical(logits=x)
    assert torch.allclose(ent, d.entropy()) and float(lp[1]) == 0.0 and int(rank[1]) == -1
    assert torch.allclose(tlp, x.log_softmax(-1).topk(3).values)


def test_oracle_eviction_keeps_the_heaviest_and_the_latest():
    c = {"k": torch.arange(128.).view(1, 1, 128, 1).double() % 100, "v": torch.zeros(1, 1, 128, 1).double(),
         "ks": torch.ones(1, 1, 2).double(), "vs": torch.ones(1, 1, 2).double(), "mass": torch.zeros(1, 1, 128).double()}
    c["mass"][0, 0, [7, 3, 50]] = torch.tensor([2.0, 1.0, 1.0]).double()
    kept, pos = ok.evict(c, "int8", [100], 5, 2)
    assert kept[0, 0].tolist() == [3, 7, 50, 98, 99] and pos == [5]
    assert ok.values(c["k"], c["ks"])[0, 0, :5, 0].tolist() == [3, 7, 50, 98, 99]
