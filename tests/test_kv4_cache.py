"""The host side of a cache in 4 bits: what layers ask for, pages given back by an eviction, positions ahead of places."""
import numpy as np
import pytest
import torch

from conftest import TINY
from grout_b200.cache import CacheLayout, KVSpec, Kv4Store, SequenceCache, SideBySideSpec, StateSpec
from grout_b200.config import resolve_architecture
from grout_b200.engine.batch import make_context, pack_step, pack_step_padded
from grout_b200.engine.model import Model
from grout_b200.engine.stack import stack_layers
from grout_b200.parts.base import BuildContext

WEIGHED = KVSpec(2, 64, bits=4, weighed=True)


def cache_of(*specs, max_tokens=64 * 12, **kw):
    return SequenceCache(CacheLayout.from_specs(specs), max_tokens=max_tokens, max_slots=4, max_seq_len=64 * 12,
                         dtype=torch.bfloat16, device="cpu", allocate=False, **kw)


def model_of(name, **ctx):
    arch = resolve_architecture(TINY[name])
    return Model(arch.plan(arch.config_cls.from_dict(TINY[name])), BuildContext(torch.bfloat16, torch.device("cpu"), **ctx))


def grow(c, slot, n):
    c.reserve(slot, n)
    c.advance(slot, n)


def test_an_eviction_gives_pages_back_and_remembers_positions():
    c = cache_of(WEIGHED, StateSpec((3,)), SideBySideSpec((WEIGHED, StateSpec((2,)))))
    a, b = c.open(), c.open()
    grow(c, a, 300)
    grow(c, b, 100)
    assert c.stores[0].pool.n_held == 5 + 2
    c.evict([a, b, a], keep=100, recent=10)
    assert (c.length[a], c.dropped[a], c.length[b], c.dropped[b]) == (100, 200, 100, 0)
    assert c.stores[0].pool.n_held == 2 + 2 and c.stores[2].stores[0].pool.n_held == 4
    c.check()
    grow(c, a, 40)
    assert c.stores[0].pool.n_held == 3 + 2
    c.evict([a], keep=64, recent=64)
    assert (c.length[a], c.dropped[a]) == (64, 276) and c.stores[0].pool.n_held == 1 + 2
    c.close(a)
    assert a not in c.dropped
    d = c.open()
    assert c.dropped[d] == 0
    c.check()


@pytest.mark.parametrize("args", [dict(keep=0, recent=0), dict(keep=10, recent=11), dict(keep=10, recent=5, first=6),
                                  dict(keep=10, recent=-1), dict(keep=10, recent=1, first=-1)])
def test_evictions_that_do_not_add_up(args):
    c = cache_of(WEIGHED)
    a = c.open()
    grow(c, a, 100)
    with pytest.raises(ValueError):
        c.evict([a], **args)
    assert c.length[a] == 100 and c.stores[0].pool.n_held == 2


@pytest.mark.parametrize("spec", [KVSpec(2, 64), KVSpec(2, 64, bits=4), KVSpec(2, 64, window=32, bits=4, weighed=True),
                                  KVSpec(2, 64, chunk=32, bits=4, weighed=True)], ids=str)
def test_stores_that_keep_all(spec):
    c = cache_of(WEIGHED, spec)
    a = c.open()
    grow(c, a, 100)
    with pytest.raises(ValueError):
        c.evict([a], keep=10, recent=1)
    assert c.length[a] == 100 and c.stores[0].pool.n_held == 2


def test_a_closed_slot_is_refused():
    c = cache_of(WEIGHED)
    with pytest.raises(ValueError):
        c.evict([1], keep=10, recent=1)


def test_stores_in_four_bits():
    s = KVSpec(2, 128, bits=4, weighed=True).make_store(3, cache_of(WEIGHED).sizes, torch.bfloat16, "cpu")
    assert isinstance(s, Kv4Store)
    v = s.layer(1)
    assert v.pages.shape == (12, 2, 4, 18 * 128) and v.weights.shape == (12, 2, 64) and v.page == 64
    assert KVSpec(2, 128, bits=4).make_store(1, cache_of(WEIGHED).sizes, torch.bfloat16, "cpu").layer(0).weights is None
    for bad in (KVSpec(2, 96, bits=4), KVSpec(2, 64, bits=8), KVSpec(2, 64, values_in_keys=True, bits=4)):
        with pytest.raises(ValueError):
            bad.make_store(1, cache_of(WEIGHED).sizes, torch.bfloat16, "cpu")


def test_which_models_have_the_form():
    m = model_of("D", cache_bits=4)
    m.check_cache()
    (spec, layers), = m.cache_layout().groups
    assert (spec.bits, spec.weighed, layers) == (4, False, [0, 1])
    m = model_of("D", cache_bits=4, cache_weights=True)
    m.check_cache()
    assert m.cache_layout().groups[0][0].weighed
    assert stack_layers(m) is None and all(b.mixer.weighed and b.mixer.kv_bits == 4 for b in m.blocks)
    model_of("A").check_cache()
    for name in ("A", "B", "C", "E"):                       # heads of 16, 32, 48, 80
        with pytest.raises(ValueError, match="4 bits"):
            model_of(name, cache_bits=4).check_cache()
    with pytest.raises(ValueError, match="8 bits"):
        model_of("D", cache_bits=8).check_cache()
    with pytest.raises(ValueError, match="weights"):
        model_of("D", cache_weights=True).check_cache()
    arch = resolve_architecture(TINY["D"])
    plan = arch.plan(arch.config_cls.from_dict(TINY["D"]))
    with pytest.raises(ValueError, match="weights"):
        Model(plan, BuildContext(torch.float32, torch.device("cpu"), cache_bits=4, cache_weights=True)).check_cache()


def test_a_cache_of_the_usual_kind_asks_for_what_it_did():
    (spec, _layers), = model_of("D").cache_layout().groups
    assert spec == KVSpec(2, 64) and spec.bits is None


def test_positions_ahead_of_places():
    ctx = make_context([(2, 10, [7, 8, 9]), (0, 5, [1], 100)], None, "cpu", pad_seqs=1)
    assert ctx.token_pos.tolist() == [10, 11, 12, 105, 0]
    assert ctx.kv_len.tolist() == [13, 6, 1] and ctx.cu_q.tolist() == [0, 3, 4, 5]
    plain, _m = pack_step([(2, 10, [7, 8, 9]), (0, 5, [1])], None)
    ahead, meta = pack_step([(2, 10, [7, 8, 9], 0), (0, 5, [1], 0)], None)
    assert np.array_equal(plain, ahead) and meta["starts"] == (10, 5)
    out, meta = pack_step_padded([(0, 5, [1, 2], 40)], [[1]], 4, 3, 1)
    o = meta["off"]["token_pos"][0]
    assert out[o:o + 4].tolist() == [45, 46, 0, 1]


def test_the_command_line_takes_it():
    from grout_b200.cli import build_parser
    ap = build_parser()
    assert ap.parse_args(["--model", "m", "--prompt-ids", "1", "--cache-bits", "4"]).cache_bits == 4
    assert ap.parse_args(["--model", "m", "--prompt-ids", "1"]).cache_bits is None
    with pytest.raises(SystemExit):
        ap.parse_args(["--model", "m", "--prompt-ids", "1", "--cache-bits", "8"])
