"""The 8-bit shared cache inside the model (cb_forward_kv8), with scoring and
eviction: the operators run together as they are used."""

from dataclasses import replace

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def model(**kw):
    from cirrus_s_1a_b200 import synthetic
    from cirrus_s_1a_b200.config import get_config
    from cirrus_s_1a_b200.engine import CirrusB200

    cfg = replace(get_config("cirrus-s-1a-debug"), sparse_topk=None, **kw)
    return cfg, CirrusB200(cfg, synthetic.random_state_dict(cfg, seed=3, norm_jitter=0.1), device=DEV, max_ctx=640)


def text(cfg, n, batch=1, seed=5):
    return torch.randint(0, cfg.vocab_size, (batch, n), generator=torch.Generator().manual_seed(seed))


WIDE = dict(d_model=128, head_dim=64, n_q_heads=6, n_kv_heads=2, gdn_head_dim_k=64, gdn_head_dim_v=64, ffn_hidden=128)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("kw", [{}, WIDE], ids=["debug", "wide"])
def test_steps_equal_the_bf16_path_on_the_same_keys_and_values(fmt, kw):
    """Prompts (several chunk lengths), verify and decode steps.  The 8-bit cache's
    values are exact in bf16, so the bf16 path can be given the same keys and values:
    what is left is one step's own tokens (bf16 there, 8 bits here) and the rounding
    of queries, probabilities and outputs to f16."""
    cfg, eng = model(**kw)
    B = 2
    a, b = eng.new_cache(B, kv8=fmt, add_mass=True), eng.new_cache(B)
    ids = text(cfg, 300, B)
    at = 0
    for T in (150, 1, 5, 40, 1, 1, 70):
        step = ids[:, at:at + T]
        x, y = eng(step, cache=a).logits, eng(step, cache=b).logits
        at += T
        # the first chunk differs by the quantisation of its own keys alone; later ones by their own tokens'
        tol = 6e-2 if T > 8 else 2e-2
        torch.testing.assert_close(x, y, rtol=tol, atol=tol)
        k, v = a.kv8.values()
        b.kv_k[:, :at] = k[:, :, :at].transpose(1, 2).bfloat16()
        b.kv_v[:, :at] = v[:, :, :at].transpose(1, 2).bfloat16()
        assert torch.equal(k, k.bfloat16().float())
        assert a.slots_dev.tolist() == a.pos_dev.tolist() == [at] * B == a.slots_host
    # every query row of every layer and head spreads a weight of 1
    G = cfg.n_q_heads // cfg.n_kv_heads
    want = float(at * G * cfg.n_cross_layers)
    assert (a.kv8.mass.sum(-1) - want).abs().max() < 1e-3 * want
    assert eng.read_status(a, 70) == 0


def test_scoring_with_and_without_a_bound():
    from cirrus_s_1a_b200.longtext import score_text

    cfg, eng = model(**WIDE)
    ids = text(cfg, 500)
    full = score_text(eng, ids, eng.new_cache(), top=3)
    assert full.logprob.shape == (1, 499) and full.top_token.shape == (1, 499, 3)
    logits = eng(ids[:, :-1], use_cache=True).logits.double().log_softmax(-1)
    want = logits.gather(2, ids[:, 1:, None].to(DEV))[..., 0]
    assert (full.logprob - want).abs().max() < 1e-2
    held = eng.new_cache(max_ctx=640, kv8="int8")
    near = score_text(eng, ids, held)
    assert (near.logprob - full.logprob).abs().max() < 0.1
    cache = eng.new_cache(max_ctx=192 + 128, kv8="int8", add_mass=True)
    bound = score_text(eng, ids, cache, keep=192, recent=64)
    assert cache.slots_host == [192] and cache.pos == 499 and cache.slots_dev.tolist() == [192]
    assert torch.equal(bound.logprob[:, :128], near.logprob[:, :128])  # nothing was evicted yet
    assert torch.isfinite(bound.logprob).all()
    assert (bound.logprob.mean() - near.logprob.mean()).abs() < 0.2
    assert float(cache.kv8.mass[:, :, :192].min()) >= 0.0


def test_clones_and_refusals():
    from cirrus_s_1a_b200 import _lib
    from cirrus_s_1a_b200.engine import CirrusB200, DecodeGraph
    from cirrus_s_1a_b200.longtext import score_text
    from cirrus_s_1a_b200.speculative import SpecDecoder
    from cirrus_s_1a_b200 import synthetic
    from cirrus_s_1a_b200.config import get_config

    cfg, eng = model()
    ids = text(cfg, 40)
    cache = eng.new_cache(max_ctx=64, kv8="e4m3", add_mass=True)
    eng(ids[:, :30], cache=cache)
    fork = cache.clone()
    x = eng(ids[:, 30:35], cache=cache).logits
    y = eng(ids[:, 30:35], cache=fork).logits
    assert torch.equal(x, y) and fork.slots_host == cache.slots_host == [35]
    with pytest.raises(_lib.CbError):
        eng(ids[:, :30], cache=cache)  # 35 + 30 > 64 slots
    with pytest.raises(ValueError):
        cache.to_reference()
    with pytest.raises(ValueError):
        DecodeGraph(eng, cache)
    with pytest.raises(ValueError):
        SpecDecoder(eng, cache)
    plain = eng.new_cache()
    with pytest.raises(ValueError):
        plain.evict(4, 2)
    with pytest.raises(ValueError):
        score_text(eng, ids, plain, keep=8)
    with pytest.raises(ValueError):
        score_text(eng, ids, eng.new_cache(kv8="int8"), keep=8)
    with pytest.raises(ValueError):
        score_text(eng, ids[:, :1], plain)
    sparse = get_config("cirrus-s-1a-debug")
    other = CirrusB200(sparse, synthetic.random_state_dict(sparse, seed=0), device=DEV, max_ctx=64)
    with pytest.raises(ValueError):
        other.new_cache(kv8="int8")


def test_a_capture_wants_its_workspace_first():
    """A workspace zeroed inside a capture would not be zero before the first replay."""
    from cirrus_s_1a_b200 import _lib

    cfg, eng = model()
    cache = eng.new_cache(kv8="int8")
    ids = text(cfg, 1).to(DEV)
    logits = torch.empty(1, 1, cfg.vocab_size, device=DEV)
    hidden = torch.empty(1, 1, cfg.d_model, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.CbError):
        with torch.cuda.graph(graph):
            torch.zeros(1, device=DEV)
            eng.launch(cache, ids, 1, 1, logits, hidden, None)
    eng(ids, cache=cache)
    slots, state = cache.slots_dev.clone(), (cache.pos_dev.clone(), cache.gdn_state.clone(), cache.gdn_conv.clone())
    eng.launch(cache, ids, 1, 1, logits, hidden, None)
    want = logits.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eng.launch(cache, ids, 1, 1, logits, hidden, None)
    cache.slots_dev.copy_(slots)
    for t, was in zip((cache.pos_dev, cache.gdn_state, cache.gdn_conv), state):
        t.copy_(was)
    graph.replay()
    torch.testing.assert_close(logits, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("kw", [{}, WIDE], ids=["debug", "wide"])
def test_values_past_the_range_of_f16(kw):
    """The 8-bit cache holds keys and values alone in fewer bits: values of 1e6 pass through
    the attention as they do on the bf16 path."""
    from cirrus_s_1a_b200 import synthetic
    from cirrus_s_1a_b200.config import get_config
    from cirrus_s_1a_b200.engine import CirrusB200

    cfg = replace(get_config("cirrus-s-1a-debug"), sparse_topk=None, **kw)
    sd = synthetic.random_state_dict(cfg, seed=3, norm_jitter=0.1)
    name = [n for n in sd if "shared" in n and "norm" in n and "k_norm" not in n]
    assert len(name) == 1, name
    sd[name[0]] = sd[name[0]] * 1e6
    eng = CirrusB200(cfg, sd, device=DEV, max_ctx=640)
    ids = text(cfg, 22)
    a, b = eng.new_cache(kv8="int8"), eng.new_cache()
    for lo, hi in ((0, 16), (16, 17), (17, 22)):  # (the many-token GEMM takes inputs up to 65504)
        x, y = eng(ids[:, lo:hi], cache=a).logits, eng(ids[:, lo:hi], cache=b).logits
        assert float(a.kv8.values()[1].abs().max()) > 65504
        # int8 values are within 2^-7 of their block's largest (1.6 % of a typical one); the
        # layers behind may double that
        assert float((x - y).norm() / y.norm()) < 0.1


@pytest.mark.parametrize("kw", [{}, WIDE], ids=["debug", "wide"])
def test_weights_come_from_every_token_whatever_logits_are_asked_for(kw):
    cfg, eng = model(**kw)
    ids = text(cfg, 300, 2)
    full, last = (eng.new_cache(2, kv8="int8", add_mass=True) for _ in range(2))
    for lo, hi in ((0, 290), (290, 295), (295, 300)):
        x = eng(ids[:, lo:hi], cache=full)
        y = eng(ids[:, lo:hi], cache=last, n_logits=2)
        assert y.logits.shape[1] == y.hidden.shape[1] == 2
        assert torch.equal(x.hidden[:, -2:], y.hidden)
        # the LM head of few rows runs on the GEMV, of many on the tensor cores (22-bit inputs)
        torch.testing.assert_close(x.logits[:, -2:], y.logits, rtol=1e-4, atol=1e-4)
        assert torch.equal(full.kv8.mass, last.kv8.mass)
    assert torch.equal(full.evict(100, 20), last.evict(100, 20))


def test_status_of_an_8_bit_cache_is_seen_and_cleared():
    cfg, eng = model()
    ids = text(cfg, 60)
    cache = eng.new_cache(max_ctx=64, kv8="e4m3")
    eng(ids[:, :40], cache=cache)
    eng(ids[:, 40:41], cache=cache)
    assert eng.read_status(cache) == 0
    cache.slots_host = [0]  # the host's count does not stop it: the device drops the tokens and says so
    eng(ids[:, :40], cache=cache)
    assert eng.read_status(cache) == 5 and eng.read_status(cache, 40) == 5
    eng.clear_status(cache)
    assert eng.read_status(cache) == 0 and eng.read_status(cache, 40) == 0
    held = len(eng._ws)
    for wrong in (lambda: eng.intermediates(cache), lambda: eng.phase_trace(cache), lambda: eng.set_wait_limit(cache, 0)):
        with pytest.raises(ValueError):
            wrong()
    assert len(eng._ws) == held


def test_scoring_reports_what_the_device_reports():
    from cirrus_s_1a_b200 import _lib
    from cirrus_s_1a_b200.longtext import score_text

    cfg, eng = model()
    ids = text(cfg, 60)
    cache = eng.new_cache(max_ctx=64, kv8="e4m3")
    cache.slots_dev.fill_(30)  # more than the host knows of
    with pytest.raises(_lib.CbError):
        score_text(eng, ids, cache)
    for at, bad in ((50, cfg.vocab_size), (50, -1), (59, cfg.vocab_size), (59, -1), (59, 2 ** 32 + 5)):
        wrong = ids.clone()
        wrong[0, at] = bad
        with pytest.raises(_lib.CbError):
            score_text(eng, wrong, eng.new_cache())
    assert bool(torch.isfinite(score_text(eng, ids, eng.new_cache()).logprob).all())


def test_weights_without_an_8_bit_cache_are_refused():
    cfg, eng = model()
    with pytest.raises(ValueError):
        eng.new_cache(add_mass=True)
