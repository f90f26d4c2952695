"""The operators at the ends of a model together, as they are used: a tied table trained from
both ends, and the engine's loss from its hidden states."""

import math
from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def chain(ids, table, norm, targets, scale, ops):
    """embedding -> RMSNorm -> cross entropy over the same table."""
    embed, rms, ce = ops
    return ce(rms(embed(ids, table, scale), norm), table, targets)


def reference(ids, table, norm, targets, scale):
    table = table.double().requires_grad_()
    norm = norm.double().requires_grad_()
    x = torch.nn.functional.embedding(ids.clamp(min=0), table) * scale * (ids >= 0)[:, None]
    h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * norm
    loss = torch.nn.functional.cross_entropy(h @ table.T, targets, ignore_index=-1)
    return loss, *torch.autograd.grad(loss, (table, norm))


def ours():
    from cirrus_s_1a_b200.embedding import embedding
    from cirrus_s_1a_b200.loss import linear_cross_entropy
    from cirrus_s_1a_b200.norm import rms_norm

    return embedding, rms_norm, lambda h, w, t: linear_cross_entropy(h, w, t).loss


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,d", [(1, 40, 16), (37, 300, 72), (300, 2500, 128), (513, 900, 264)])
def test_tied_table_gets_both_gradients(dtype, n, V, d):
    """Against autograd in 64 bits on the same 16-bit values.  Between the operators values are
    rounded to the type (the embedding's row, the norm's, their gradients, and the table's two
    gradients and their sum): eight roundings of half a step, each of a quantity that its
    2-norm bounds, so that errors stay below 8 half steps of the gradient's 2-norm."""
    g = torch.Generator().manual_seed(n + d)
    table = (torch.randn(V, d, generator=g) / math.sqrt(d) * 2).to(TYPES[dtype])
    norm = 1 + 0.1 * torch.randn(d, generator=g)
    ids, targets = (torch.randint(0, V, (n,), generator=g) for _ in range(2))
    if n > 1:
        ids[::7], targets[::5] = -1, -1
    td, nd = table.to(DEV).requires_grad_(), norm.to(DEV).requires_grad_()
    loss = chain(ids.to(DEV), td, nd, targets.to(DEV), 3.0, ours())
    dt, dn = torch.autograd.grad(loss, (td, nd))
    want, wt, wn = reference(ids, table, norm, targets, 3.0)
    u = max(torch.finfo(TYPES[dtype]).eps / 2, 2.0 ** -20)
    assert abs(float(loss) - float(want)) <= 8 * u * (1 + abs(float(want)))
    for got, ref in ((dt, wt), (dn, wn)):
        assert (got.cpu().double() - ref).norm() <= 8 * u * ref.norm() + 1e-12


@pytest.mark.parametrize("dtype", TYPES)
def test_two_threads_on_streams_of_their_own(dtype):
    """Calls at the same time have their own scratch and give the bits of one alone."""
    from concurrent.futures import ThreadPoolExecutor

    g = torch.Generator().manual_seed(8)
    ids = [torch.randint(0, 2500, (n,), generator=g).to(DEV) for n in (900, 40)]
    targets = [torch.randint(-1, 2500, (len(i),), generator=g).to(DEV) for i in ids]
    table = (torch.randn(2500, 128, generator=g) / 8).to(TYPES[dtype]).to(DEV)
    norm = torch.ones(128, dtype=TYPES[dtype], device=DEV)

    def step(k):
        t, n = table.detach().requires_grad_(), norm.detach().requires_grad_()
        loss = chain(ids[k], t, n, targets[k], 2.0, ours())
        return loss.detach(), *torch.autograd.grad(loss, (t, n))

    def many(k):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            out = [step(k) for _ in range(20)]
        side.synchronize()
        return out

    alone = [step(k) for k in range(2)]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(2) as pool:
        for k, runs in enumerate(pool.map(many, range(2))):
            for out in runs:
                assert all(torch.equal(a, b) for a, b in zip(out, alone[k]))


def test_a_captured_training_step_and_an_eager_one():
    """A step of plain descent on the tied table, captured while an eager graph of the same
    table has lived: replays equal the eager steps bit for bit."""
    g = torch.Generator().manual_seed(1)
    table = (torch.randn(700, 64, generator=g) / 8).bfloat16().to(DEV)
    norm = torch.ones(64, device=DEV)
    batches = [(torch.randint(0, 700, (150,), generator=g).to(DEV), torch.randint(-1, 700, (150,), generator=g).to(DEV))
               for _ in range(3)]
    ops = ours()

    def step(tab, ids, targets):
        leaf, w = tab.detach().requires_grad_(), norm.detach().requires_grad_()
        loss = chain(ids, leaf, w, targets, 1.0, ops)
        dt, dn = torch.autograd.grad(loss, (leaf, w))
        return loss.detach(), dt, dn, tab - 0.5 * dt

    eager, t = [], table
    for b in batches:
        eager.append(step(t, *b))
        t = eager[-1][3]
    tab, ids, targets = table.clone(), batches[0][0].clone(), batches[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(tab, ids, targets)
        tab.copy_(outs[3])
    tab.copy_(table)
    for b, want in zip(batches, eager):
        ids.copy_(b[0])
        targets.copy_(b[1])
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(outs[:3], want[:3])) and torch.equal(tab, want[3])


@pytest.mark.parametrize("dtype", TYPES)
def test_saved_tensors_that_a_hook_moves(dtype):
    """Tensors kept on the host between forward and backward come back elsewhere, and rows of a
    wider matrix come back contiguous."""
    g = torch.Generator().manual_seed(2)
    big = (torch.randn(300, 100, generator=g) / 8).to(TYPES[dtype]).to(DEV)
    ids, targets = (torch.randint(0, 300, (200,), generator=g).to(DEV) for _ in range(2))
    norm = torch.ones(64, device=DEV)

    def step():
        table, w = big[:, 8:72].detach().requires_grad_(), norm.detach().requires_grad_()
        with torch.autograd.graph.save_on_cpu() if moved else torch.enable_grad():
            loss = chain(ids + 0, table, w, targets + 0, 1.0, ours())
        torch.full((1 << 22,), 7.0, device=DEV)  # over what has been freed
        return loss, *torch.autograd.grad(loss, (table, w))

    moved = False
    want = step()
    moved = True
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_a_gradient_of_a_gradient_is_refused():
    table = torch.randn(20, 16, device=DEV, requires_grad=True)
    norm = torch.ones(16, device=DEV, requires_grad=True)
    ids = torch.arange(10, device=DEV)
    embed, rms, ce = ours()
    for out in (embed(ids, table), rms(table, norm), ce(table, table, torch.arange(20, device=DEV))):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out.sum(), table, create_graph=True)


def engine(**kw):
    from cirrus_s_1a_b200 import synthetic
    from cirrus_s_1a_b200.config import get_config
    from cirrus_s_1a_b200.engine import CirrusB200

    cfg = replace(get_config("cirrus-s-1a-debug"), sparse_topk=None, **kw)
    return cfg, CirrusB200(cfg, synthetic.random_state_dict(cfg, seed=3, norm_jitter=0.1), device=DEV, max_ctx=640)


WIDE = dict(d_model=128, head_dim=64, n_q_heads=6, n_kv_heads=2, gdn_head_dim_k=64, gdn_head_dim_v=64, ffn_hidden=128)


@pytest.mark.parametrize("kw", [{}, WIDE], ids=["debug", "wide"])
@pytest.mark.parametrize("T", [1, 5, 150])
def test_engine_loss_equals_its_logits(kw, T):
    """The logits are sums of at most 128 products of exact weights and inputs carried in 22 to
    24 bits; the two ways differ by 2^-18 of the largest logit at most."""
    from cirrus_s_1a_b200.logprobs import token_logprobs

    cfg, eng = engine(**kw)
    ids = torch.randint(0, cfg.vocab_size, (2, T + 1), generator=torch.Generator().manual_seed(T))
    a, b = eng.new_cache(2), eng.new_cache(2)
    out = eng(ids[:, :T], cache=a)
    targets = ids[:, 1:].clone()
    if T > 1:
        targets[0, 1] = -1
    r = eng.loss(ids[:, :T], targets, b, reduction="none")
    lp = token_logprobs(out.logits.flatten(0, 1), targets.reshape(-1).int().to(DEV)).logprob.view(2, T)
    tol = 2.0 ** -18 * (1 + float(out.logits.abs().max()))
    assert ((r.loss + lp).abs() <= tol).all() and r.loss.shape == r.lse.shape == (2, T)
    assert ((r.lse - torch.logsumexp(out.logits.double(), -1)).abs() <= tol).all()
    assert a.pos_dev.tolist() == b.pos_dev.tolist() == [T, T] and b.pos == T
    mean = eng.loss(ids[:, :T], targets).loss
    n = int((targets >= 0).sum())
    assert abs(float(mean) - float(r.loss.double().sum() / n)) <= 2 * tol
    assert eng.read_status(b, T) == 0
    with pytest.raises(ValueError):
        eng.loss(ids[:, :T], targets[:, :0])


def test_dense_head_is_exact_and_made_once():
    cfg, eng = engine()
    head = eng.dense_head()
    assert head.dtype == torch.bfloat16 and head is eng.dense_head()
    x = torch.randn(3, cfg.d_model, device=DEV)
    from cirrus_s_1a_b200 import _lib

    rows = torch.arange(cfg.vocab_size, device=DEV)
    w = torch.empty(cfg.vocab_size, cfg.d_model, device=DEV)
    import ctypes as C

    assert _lib.lib().cb_embed(C.byref(eng.model.desc.lm_head), rows.data_ptr(), cfg.vocab_size, w.data_ptr(), None, 0) == 0
    torch.cuda.synchronize()
    assert torch.equal(head.float(), w) and x.shape[1] == head.shape[1]


def test_mean_loss_of_a_long_text():
    """Over a bf16 cache and a bounded 8-bit one, against the scores that go through logits."""
    from cirrus_s_1a_b200 import _lib
    from cirrus_s_1a_b200.longtext import mean_loss, score_text

    cfg, eng = engine(**WIDE)
    ids = torch.randint(0, cfg.vocab_size, (2, 300), generator=torch.Generator().manual_seed(9))
    for make, kw in ((lambda: eng.new_cache(2), {}),
                     (lambda: eng.new_cache(2, max_ctx=256, kv8="e4m3", add_mass=True), dict(keep=128, recent=32))):
        s = score_text(eng, ids, make(), **kw)
        m = mean_loss(eng, ids, make(), **kw)
        assert abs(float(m) + float(s.logprob.double().mean())) <= 2.0 ** -16 * (1 + abs(float(m)))
    with pytest.raises(ValueError):
        mean_loss(eng, ids[:, :1], eng.new_cache(2))
    with pytest.raises(ValueError):
        mean_loss(eng, ids, eng.new_cache(2), keep=64)
    for bad in (cfg.vocab_size, -3):
        ids[1, 299] = bad
        with pytest.raises(_lib.CbError):
            mean_loss(eng, ids, eng.new_cache(2))
