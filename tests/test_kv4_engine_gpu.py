"""Engines with a cache in 4 bits, against the plain model whose keys and values pass through the plain 4-bit form."""
import math

import pytest
import torch

from conftest import random_tokens
from grout_b200.engine import Engine
from grout_b200.kernels import ops
from helpers import run_batch, run_tail_decoded, run_whole
from plain import kv4, qwen3

pytestmark = pytest.mark.gpu

BASE = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", vocab_size=200, hidden_size=128, intermediate_size=192,
            num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=20000.0,
            rms_norm_eps=2e-6, max_position_embeddings=512, tie_word_embeddings=True, use_sliding_window=False,
            eos_token_id=199)
CONFIGS = {"64": BASE, "128": dict(BASE, head_dim=128, num_attention_heads=3, num_key_value_heads=1, hidden_size=96),
           "windowed": dict(BASE, use_sliding_window=True, sliding_window=24, max_window_layers=1)}
# Keys differ from the plain ones by the rounding of what is in front of them.  In 32 bits that turns a code (a step of
# a fifteenth of its group's range) once in about a million elements; in bfloat16, whose own step is about a fifteenth of
# a code's, for one element in fifteen, by one step: as much again as the 16-bit cache's tolerance for each, times four
# for the four bits that the step is larger than what bfloat16 rounds by.
TOL = {"float32": dict(atol=2e-4, rtol=2e-3), "bfloat16": dict(atol=0.1, rtol=0.15)}


def engine_of(name, dtype, **kw):
    torch.manual_seed(0)
    return Engine.random(CONFIGS[name], 5, dtype=dtype, max_tokens=4096, max_batch=8, cache_bits=4, **kw)


def weights_of(name):
    from grout_b200.parts.base import BuildContext
    from grout_b200.config import resolve_architecture
    from grout_b200.engine.model import Model
    from grout_b200.weights import random_tensor
    arch = resolve_architecture(CONFIGS[name])
    m = Model(arch.plan(arch.config_cls.from_dict(CONFIGS[name])), BuildContext(torch.bfloat16, torch.device("cpu")))
    return {n: random_tensor(n, s, 5, torch.bfloat16, torch.device("cuda:0")).cpu() for n, s in m.expected().items()}


def held(x):
    """[T, heads, D] as a cache in 4 bits holds it."""
    return kv4.value(*kv4.quantise(x.float())).double()


def plain_logits(name, tokens, monkeypatch, seen=None, rows=None):
    """The plain model's logits with keys and values through 4 bits; ``seen(T)`` -> [nkv, T, T] of what is visible."""
    usual = qwen3.causal_attention

    def attention(q, k, v, window=None):
        k, v = held(k), held(v)
        if seen is None:
            return usual(q, k, v, window)
        T, nq, D = q.shape
        see, out = seen(T), torch.empty_like(q)
        for h in range(nq):
            g = h // (nq // k.shape[1])
            s = (q[:, h] @ k[:, g].T / math.sqrt(D)).masked_fill(~see[g], -math.inf)
            out[:, h] = torch.softmax(s, -1) @ v[:, g]
        return out
    with monkeypatch.context() as m:
        m.setattr(qwen3, "causal_attention", attention)
        return qwen3.logits(weights_of(name), CONFIGS[name], tokens, rows)


def close(got, want, dtype, what):
    off, tol = (got.double().cpu() - want).abs(), TOL[dtype]
    bound = tol["atol"] + tol["rtol"] * want.abs()
    assert bool((off <= bound).all()), (what, float(off.max()), float((off / bound).max()))


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(CONFIGS))
def test_logits(name, dtype, graphs, monkeypatch):
    eng = engine_of(name, dtype, use_graphs=graphs)
    tokens = random_tokens(90, 200, 3)
    want = plain_logits(name, tokens, monkeypatch)
    close(run_whole(eng, tokens), want, dtype, "whole")
    close(run_tail_decoded(eng, tokens, 40), want, dtype, "one by one")
    requests = [random_tokens(n, 200, 10 + n) for n in (70, 5, 33)]
    for got, toks in zip(run_batch(eng, requests, [40, 3, 32]), requests):
        close(got, plain_logits(name, toks, monkeypatch), dtype, "batch")
    eng.cache.check()
    eng.check()


def test_the_kernels_in_four_bits_run_and_the_cache_is_smaller():
    eng = engine_of("64", "bfloat16", use_graphs=False)
    usual = Engine.random(BASE, 5, max_tokens=4096, max_batch=8)
    store = eng.cache.stores[0]
    assert store.pages.numel() * 32 == (usual.cache.stores[0].k.numel() + usual.cache.stores[0].v.numel()) * 2 * 9
    ops.LAUNCH_LOG = []
    try:
        s = eng.open_sequence()
        eng.step([(s, [1, 2, 3])], [[2]])
        eng.step([(s, [4])], [[0]])
        log = list(ops.LAUNCH_LOG)
    finally:
        ops.LAUNCH_LOG = None
    assert log.count("kv4_write") == 4 and log.count("attn_prefill_kv4") == 2 and log.count("attn_kv4_decode") == 2
    assert not [x for x in log if x in ("attn_prefill_tc", "attn_decode_bf16", "attn_decode_tma", "decode_stack")]


def test_generation_is_the_same_with_and_without_graphs():
    a, b = engine_of("128", "bfloat16"), engine_of("128", "bfloat16", use_graphs=False)
    prompts = [random_tokens(n, 200, n) for n in (17, 60, 3)]
    outs = [[o.token_ids for o in e.generate(prompts, 20, ignore_eos=True, look_ahead=False)] for e in (a, b)]
    assert outs[0] == outs[1]


@pytest.mark.parametrize("graphs", [True, False])
def test_a_sequence_that_is_cut(graphs, monkeypatch):
    """One layer, so that the weights of the tokens are the plain model's sums of probabilities: the prompt's last 32 rows
    and every single token's row.  What follows the cut sees what was kept, at its own positions."""
    config = dict(BASE, num_hidden_layers=1)
    monkeypatch.setitem(CONFIGS, "one", config)
    eng = engine_of("one", "bfloat16", cache_weights=True, use_graphs=graphs)
    n, keep, recent, first = 150, 70, 10, 2
    tokens = random_tokens(n + 12, 200, 8)
    s, other = eng.open_sequence(), eng.open_sequence()
    eng.step([(other, tokens[:100])])
    before = eng.step([(other, tokens[100:101])], [[0]]).clone()
    eng.step([(s, tokens[:n - 3])])
    for t in tokens[n - 3:n]:
        eng.step([(s, [t])])
    # the weights against the plain model's
    probs = {}

    def attention(q, k, v, window=None):
        k, v = held(k), held(v)
        out, _l, p = kv4.attend(q, k.transpose(0, 1), v.transpose(0, 1), 1 / math.sqrt(q.shape[2]))
        probs["p"] = p
        return out
    with monkeypatch.context() as m:
        m.setattr(qwen3, "causal_attention", attention)
        qwen3.logits(weights_of("one"), config, tokens[:n])
    p = probs["p"]                                          # [nq, n, n]
    want = p[:, n - 35:].sum(1).view(2, 2, n).sum(1)         # 32 rows of the prompt, three tokens
    view = eng.cache.view(0)
    table = view.block_table[s].tolist()
    got = torch.stack([view.weights[table[j // 64], :, j % 64] for j in range(n)], 1).double().cpu()
    # scores are off by the turned codes of the keys, as the logits are: a fifth of a probability at most
    assert float(((got - want).abs() / (want + 0.02)).max()) < 0.35
    assert abs(float(got.sum()) - 35 * 4) < 0.5               # every row's probabilities add up to one
    kept = {}
    usual = ops.kv4_evict

    def evict(*a, **kw):
        kept["k"], kept["n"] = usual(*a, **kw)
        return kept["k"], kept["n"]
    monkeypatch.setattr(ops, "kv4_evict", evict)
    held_before = eng.cache.stores[0].pool.n_held
    eng.evict([s], keep, recent, first)
    assert eng.length(s) == keep and eng.cache.dropped[s] == n - keep
    assert held_before - eng.cache.stores[0].pool.n_held == 1   # 3 pages of 64, then 2
    k = kept["k"][0].cpu()
    for h in range(2):
        assert k[h].tolist() == kv4.choose(got[h].tolist(), n, keep, recent, first)
    # what follows, one by one and several at once
    rows = [eng.step([(s, [t])], [[0]]).clone() for t in tokens[n:n + 4]]
    rows.append(eng.step([(s, tokens[n + 4:n + 12])], [list(range(8))]).clone())
    assert eng.length(s) == keep + 12

    def seen(T):
        see = torch.ones((2, T, T), dtype=torch.bool).tril()
        for h in range(2):
            gone = torch.ones(T, dtype=torch.bool)
            gone[k[h].long()] = False
            gone[n:] = False
            see[h, n:] &= ~gone
        return see
    want = plain_logits("one", tokens, monkeypatch, seen, list(range(n, n + 12)))
    close(torch.cat(rows), want, "bfloat16", "behind the cut")
    full = plain_logits("one", tokens, monkeypatch, None, list(range(n, n + 12)))
    got_rows = torch.cat(rows).double().cpu()
    assert float((got_rows - want).norm()) < 0.5 * float((full - want).norm())      # and not what was there before
    # the other sequence is as it was
    eng.close_sequence(s)
    again = eng.step([(other, tokens[101:102])], [[0]])
    assert bool(torch.isfinite(again).all()) and bool(torch.isfinite(before).all())
    eng.cache.check()


def test_evictions_that_are_refused():
    eng = engine_of("64", "bfloat16")
    s = eng.open_sequence()
    eng.step([(s, random_tokens(20, 200, 1))])
    with pytest.raises(ValueError):
        eng.evict([s], 10, 2)                               # no weights are kept
    usual = Engine.random(BASE, 5, max_tokens=1024, max_batch=2)
    t = usual.open_sequence()
    with pytest.raises(ValueError):
        usual.evict([t], 10, 2)
    with pytest.raises(ValueError):
        Engine.random(dict(BASE, head_dim=32), 5, max_tokens=1024, max_batch=2, cache_bits=4)
    with pytest.raises(ValueError):
        Engine.random(BASE, 5, dtype="float32", max_tokens=1024, max_batch=2, cache_bits=4, cache_weights=True)


def test_positions_end_where_the_architecture_does():
    eng = Engine.random(dict(BASE, max_position_embeddings=200), 5, max_tokens=1024, max_batch=2, cache_bits=4,
                        cache_weights=True)
    s = eng.open_sequence()
    eng.step([(s, random_tokens(190, 200, 1))])
    eng.evict([s], 50, 20)
    eng.step([(s, random_tokens(10, 200, 2))])
    with pytest.raises(ValueError):
        eng.step([(s, [1])])
    assert eng.length(s) == 60


# ---------------------------------------------------------------- the other designs
def _designs():
    from test_kakotar_engine_gpu import YARN, _att, _light, _rot
    from test_mananex_engine_gpu import MAN
    from test_sonalorn_engine_gpu import _attn, _delta
    from test_suvazen_engine_gpu import SUV
    # rotations, caps, sinks, windows, loops and values that are the unrotated keys; kept first keys and head gates beside
    # a state; a layer that reads another's keys; a query temperature and values narrower than the keys
    return {
        "suvazen": SUV["R"], "mananex": MAN["Q"],
        "kakotar": dict(architecture="Kakotar", vocab=300, width=128, norm={"eps": 3e-6}, layers=[
            dict(type="attention", mixer=_att(4, 2, 64, 64, 0.3, 70, _rot(1e5, 32, YARN)), mlp=None),
            dict(type="lightning", mixer=_light(2, 16, 16, 0.5, 0.9), mlp=None),
            dict(type="attention", mixer=_att(8, 2, 64, 64, 0.25, 40, _rot(1e5, 32, YARN), kv_from=0), mlp=None)]),
        "sonalorn": dict(architecture="Sonalorn", vocab=200, width=96, max_positions=512, norm={"eps": 1e-5}, layers=[
            dict(type="delta", mixer=_delta(heads=2, kv_heads=2, dim=32, vdim=32, conv=4), mlp=None),
            dict(type="attention", mixer=_attn(heads=4, kv_heads=1, dim=64, vdim=40, scale=0.15), mlp=None)])}


@pytest.mark.parametrize("name", ["suvazen", "mananex", "kakotar", "sonalorn"])
def test_the_other_designs(name, monkeypatch):
    """In 32 bits, against the same engine with a 32-bit cache whose keys and values pass through the plain 4-bit form
    in front of every attention: the same keys, so the logits differ by the attention kernels' 32-bit sums."""
    config = _designs()[name]
    tokens = random_tokens(170, 150, 4)
    eng = Engine.random(config, 3, dtype="float32", max_tokens=4096, max_batch=4, cache_bits=4, use_graphs=False)
    rows = [run_whole(eng, tokens), run_tail_decoded(eng, tokens, 50)]
    usual = ops.attention

    def through(q, k_pages, v_pages, *a, **kw):
        f = lambda x: kv4.value(*kv4.quantise(x.cpu())).to(x.device)
        return usual(q, f(k_pages), f(v_pages), *a, **kw)
    oracle = Engine.random(config, 3, dtype="float32", max_tokens=512, max_batch=4, use_graphs=False)
    with monkeypatch.context() as m:
        m.setattr(ops, "attention", through)
        want = run_whole(oracle, tokens)
    spread = float((want - want.mean(-1, keepdim=True)).pow(2).mean().sqrt())
    for got in rows:
        assert float((got - want).abs().max()) < 1e-3 * spread, float((got - want).abs().max()) / spread
    # (it does matter: without the 4-bit form the logits are elsewhere)
    plain = run_whole(oracle, tokens)
    assert float((plain - want).abs().max()) > 0.01 * spread


def test_designs_without_the_form():
    from test_keralix_engine_gpu import KER
    from test_zutazen_engine_gpu import ZUT
    for config in (next(iter(KER.values())), next(iter(ZUT.values()))):
        with pytest.raises(ValueError, match="4 bits"):
            Engine.random(config, 3, max_tokens=512, max_batch=4, cache_bits=4)
