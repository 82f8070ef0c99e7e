"""Evictions that cannot be made leave everything as it was."""
import pytest
import torch

from grout_b200.cache import CacheLayout, KVSpec, SequenceCache, StateSpec
from grout_b200.kernels import ops

A, B = KVSpec(2, 64, bits=4, weighed=True), KVSpec(1, 128, bits=4, weighed=True)


def test_without_memory_for_one_store_no_store_is_cut(monkeypatch):
    """The second store's memory is not to be had: no kernel has run, lengths, positions and pages are the old ones."""
    c = SequenceCache(CacheLayout.from_specs((A, StateSpec((3,)), B)), max_tokens=64 * 12, max_slots=4, max_seq_len=64 * 12,
                      dtype=torch.bfloat16, device="cpu")
    a = c.open()
    c.reserve(a, 300)
    c.advance(a, 300)
    cut, sizes = [], []

    def memory(n_seqs, nkv, D, keep, device):
        sizes.append((n_seqs, nkv, D, keep))
        if D == 128:
            raise torch.OutOfMemoryError("no memory")
        return ()
    monkeypatch.setattr(ops, "kv4_evict_memory", memory)
    monkeypatch.setattr(ops, "kv4_evict", lambda *args, **kw: cut.append(kw))
    with pytest.raises(torch.OutOfMemoryError):
        c.evict([a], keep=100, recent=10)
    assert not cut and sizes == [(1, 2, 64, 100), (1, 1, 128, 100)]
    assert (c.length[a], c.dropped[a]) == (300, 0) and all(st.pool.n_held == 5 for st in (c.stores[0], c.stores[2]))
    c.check()
    monkeypatch.setattr(ops, "kv4_evict_memory", lambda *args: ())
    c.evict([a], keep=100, recent=10)
    assert len(cut) == 2 and all(kw["memory"] == () and kw["keep"] == 100 for kw in cut)
    assert (c.length[a], c.dropped[a]) == (100, 200) and all(st.pool.n_held == 2 for st in (c.stores[0], c.stores[2]))


@pytest.mark.gpu
@pytest.mark.parametrize("D,keep", [(64, 100), (128, 33)])
def test_eviction_with_memory_of_the_callers(D, keep):
    from test_kv4_gpu import DEV, Cache, ints
    c, d = (Cache([300, 20], 2, D, weights=True, seed=9) for _ in range(2))
    args = dict(slots=ints(*c.slots), kv_len=ints(300, 20), page=64, keep=keep, recent=10)
    memory = ops.kv4_evict_memory(2, 2, D, keep, DEV)
    a = ops.kv4_evict(c.pages, c.weights, c.table, **args)
    b = ops.kv4_evict(d.pages, d.weights, d.table, memory=memory, **args)
    assert b[0] is memory[0] and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for x, y in ((c.pages, d.pages), (c.weights.view(torch.int32), d.weights.view(torch.int32))):
        assert torch.equal(x, y)
    before = d.pages.clone()
    for bad in (ops.kv4_evict_memory(2, 2, D, keep + 1, DEV), ops.kv4_evict_memory(1, 2, D, keep, DEV),
                (memory[0], memory[1], memory[2][..., :-16], memory[3]), (memory[0].long(),) + memory[1:],
                ops.kv4_evict_memory(2, 2, D, keep, "cpu")):
        with pytest.raises(ops.KernelError):
            ops.kv4_evict(d.pages, d.weights, d.table, memory=bad, **args)
    assert torch.equal(d.pages, before)
