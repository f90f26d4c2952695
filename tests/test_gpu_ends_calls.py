"""Calls of the operators at the ends of a model that are refused, and what they leave as it was."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from cirrus_s_1a_b200 import _lib
from cirrus_s_1a_b200.loss import linear_cross_entropy
from test_gpu_ends import DEV, engine, ours
from test_gpu_linear_ce import PAIRS, TYPES, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv8", [None, "e4m3"])
@pytest.mark.parametrize("T", [5, 150])
def test_a_refused_loss_leaves_the_cache(kv8, T):
    cfg, eng = engine()
    ids = torch.randint(0, cfg.vocab_size, (2, T + 1), generator=torch.Generator().manual_seed(T))
    x, targets = ids[:, :T], ids[:, 1:]
    kw = dict(max_ctx=256, kv8=kv8) if kv8 else {}
    cache, clean = eng.new_cache(2, **kw), eng.new_cache(2, **kw)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    for kwargs in (dict(targets=targets, reduction="median"), dict(targets=targets.short()), dict(targets=targets.float()),
                   dict(targets=targets, status=torch.zeros(2, dtype=torch.int32, device=DEV)),
                   dict(targets=targets, status=word.long()), dict(targets=targets, status=word.cpu()),
                   dict(targets=targets[:1])):
        with pytest.raises(ValueError):
            eng.loss(x, cache=cache, **kwargs)
    with pytest.raises(ValueError):
        eng.loss(x.repeat(2, 1), targets.repeat(2, 1), cache)
    assert cache.pos == 0 and cache.pos_dev.tolist() == [0, 0]
    assert torch.equal(eng.loss(x, targets, cache).lse, eng.loss(x, targets, clean).lse)
    assert cache.pos == clean.pos == T


def test_a_captured_loss_wants_the_head_first():
    cfg, eng = engine()
    ids = torch.randint(0, cfg.vocab_size, (1, 6), device=DEV)
    cache = eng.new_cache(1)
    x, targets = ids[:, :5].contiguous(), ids[:, 1:].contiguous()
    eng(x, cache=cache.clone())  # the workspace
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(_lib.CbError):
            eng.loss(x, targets, cache)
    assert cache.pos == 0 and cache.pos_dev.tolist() == [0]
    eng.dense_head()
    want = eng.loss(x, targets, cache.clone(), "none")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = eng.loss(x, targets, cache, "none")
    graph.replay()
    assert torch.equal(got.loss, want.loss) and torch.equal(got.lse, want.lse)


@pytest.mark.parametrize("kv8", [None, "e4m3"])
@pytest.mark.parametrize("T", [5, 150])
def test_a_loss_notes_targets_outside_where_the_forward_notes_tokens(kv8, T):
    cfg, eng = engine()
    ids = torch.randint(0, cfg.vocab_size, (2, T + 1), generator=torch.Generator().manual_seed(T))
    x, targets = ids[:, :T], ids[:, 1:].clone()
    make = lambda: eng.new_cache(2, **(dict(max_ctx=256, kv8=kv8) if kv8 else {}))  # noqa: E731
    targets[1, 2] = -1
    cache = make()
    want = eng.loss(x, targets, cache, "none")
    assert eng.read_status(cache, T) == 0
    targets[1, 2] = cfg.vocab_size
    cache = make()
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert torch.equal(eng.loss(x, targets, cache.clone(), "none", word).loss, want.loss)
    assert int(word) == 6 and eng.read_status(cache, T) == 0  # the word that is given is the one that is used
    assert torch.equal(eng.loss(x, targets, cache, "none").loss, want.loss)
    assert eng.read_status(cache, T) == 6
    eng.clear_status(cache, T)
    assert eng.read_status(cache, T) == 0
    if not kv8:  # without a cache: that of any cache of this size
        eng.loss(x, targets)
        assert eng.read_status(eng.new_cache(2), T) == 6


def test_forward_mode_is_refused_on_the_device_and_of_gradients_from_above():
    embed, rms, ce = ours()
    table = torch.randn(20, 16, device=DEV)
    norm = torch.ones(16, device=DEV)
    ids = torch.arange(10, device=DEV)
    calls = (lambda x: embed(ids, x), lambda x: rms(x, norm), lambda x: ce(x, table, torch.arange(20, device=DEV)))
    for call in calls:
        with fw.dual_level():
            with pytest.raises(RuntimeError):
                call(fw.make_dual(table, torch.ones_like(table)))
            x = table.clone().requires_grad_()
            y = call(x)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(y, x, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("N,V,d", [(5, 300, 64), (200, 515, 72), (300, 90, 33)])
@pytest.mark.parametrize("step", [8, 16, 24, 1])
def test_hidden_rows_that_overlap(pair, N, V, d, step):
    """Rows closer together than they are long, as ``unfold`` gives."""
    _, w, t = inputs(N, V, d, pair, seed=N + step)
    line = torch.randn(N * step + d, generator=torch.Generator().manual_seed(step)).to(TYPES[pair[0]])
    h = line.unfold(0, d, step)[:N]
    hd = line.to(DEV).unfold(0, d, step)[:N]
    assert hd.stride() == (step, 1)
    check(h, w, t, dev=(hd, w.to(DEV)))


def test_saved_tensors_that_come_back_changed():
    """A hook that gives back another device's, type's or length's tensor: refused before a kernel
    reads it as what was saved."""
    embed, rms, _ = ours()
    table = torch.randn(20, 16, device=DEV)
    norm = torch.ones(16, device=DEV)
    ids = torch.arange(10, device=DEV)
    t = torch.arange(20, device=DEV)
    calls = {"embed": (1, lambda x: embed(ids + 0, x)), "norm": (2, lambda x: rms(x, norm + 0)),
             "mean": (5, lambda x: linear_cross_entropy(x, table + 0, t + 0).loss),
             "none": (5, lambda x: linear_cross_entropy(x, table + 0, t + 0, "none").loss)}
    for name, (saved, call) in calls.items():
        for which in range(saved):
            for change in (lambda x: x.cpu(), lambda x: x.to(torch.float16), lambda x: x[:-1]):
                seen = []

                def unpack(x):
                    seen.append(x)
                    return change(x) if len(seen) == which + 1 else x

                x = table.clone().requires_grad_()
                with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
                    y = call(x)
                with pytest.raises((ValueError, RuntimeError)):
                    torch.autograd.grad(y, x, torch.ones_like(y))
                assert len(seen) == saved, name
    torch.cuda.synchronize()
