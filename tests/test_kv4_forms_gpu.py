"""Forms of attention over a 4-bit cache that only some sizes reach, each of them forced: prompts in blocks of both sizes with
packed heads and without, splits that have a workspace in captured graphs and on two streams at once, more sequences than
can share the keys out."""
import pytest
import torch

from grout_b200.kernels import ops
from test_kv4_gpu import DEV, NAN, SEEN, Cache, attend, ints, queries

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------- prompts
@pytest.mark.parametrize("seen", SEEN + [dict(window=130, softcap=15.0)], ids=str)
@pytest.mark.parametrize("pack", [1, 64])
@pytest.mark.parametrize("rows", [128, 256])
@pytest.mark.parametrize("nq,nkv,D", [(20, 4, 64), (8, 2, 64), (8, 2, 128), (6, 2, 128)])
def test_prompts_in_blocks_of_every_kind(nq, nkv, D, rows, pack, seen, monkeypatch):
    """128 and 256 query rows a block, heads of 64 and 128, packed (the four or two that a group has as a power of two) and one a block;
    two query blocks that share tiles and end at different keys, partial second halves, padding, sinks."""
    monkeypatch.setattr(ops, "PREFILL_TC_PACK", pack)
    taken = []

    def forced(blocks, nq, nkv, sms, one_head=False):
        taken.append((ops.prefill_tc_pack(nq, nkv), rows))
        return taken[-1]
    monkeypatch.setattr(ops, "prefill_tc_plan", forced)
    q_lens, before = [257, 1, 140, 30], [70, 64, 0, 500]
    c = Cache([a + b for a, b in zip(q_lens, before)], nkv, D, BF16, seed=rows)
    attend(c, q_lens, nq, BF16, sinks=True, pad=1, **seen)
    assert set(taken) == {(min(pack, nq // nkv & -(nq // nkv)), rows)}


@pytest.mark.parametrize("rows", [128, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_tokens_in_prompts_of_large_blocks(D, rows, monkeypatch):
    """A NaN key and a NaN value leave the rows that do not see them as they are, in both query blocks of a block."""
    monkeypatch.setattr(ops, "PREFILL_TC_ROWS", rows)

    def edit(kv):
        kv[150, 0] = NAN                 # a key of kv head 0
        kv[300, 3] = NAN                 # a value of kv head 1
    n = 600
    c, fine = Cache([n], 2, D, BF16, seed=2, edit=edit), Cache([n], 2, D, BF16, seed=2)
    step, q = c.step([n]), queries(n, 8, D, BF16, 1).to(DEV)
    for seen in (dict(window=60), dict(chunk=100), dict()):
        out, lse = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True, **seen)
        want, want_lse = ops.attention_kv4(q, fine.pages, fine.table, step=step, page=64, scale=0.1, want_lse=True, **seen)
        for first, heads in ((150, slice(0, 4)), (300, slice(4, 8))):
            end = {"window": first + 60, "chunk": (first // 100 + 1) * 100}.get(next(iter(seen), ""), n)
            hit = torch.zeros(n, dtype=torch.bool)
            hit[first:end] = True
            assert bool(out[hit, heads].isnan().all(-1).all())
            assert torch.equal(out[~hit, heads], want[~hit, heads]) and torch.equal(lse[~hit, heads], want_lse[~hit, heads])


# ---------------------------------------------------------------- workspaces
PLANS = [(BF16, 2, 0), (BF16, 2, 1), (BF16, 8, 1), (F32, 2, 0)]


class Job:
    """Two sequences of one cache with queries of their own, whose lengths, slots and queries change in place."""

    def __init__(self, c, k, nq, dtype):
        self.c, self.k, self.nq, self.dtype = c, k, nq, dtype
        self.step = c.step([1, 1])
        self.step.max_kv_len = 2000
        self.q = queries(2, nq, c.D, dtype, k).to(DEV)

    def turn(self, t):
        self.q.copy_(queries(2, self.nq, self.c.D, self.dtype, 50 * t + self.k))
        self.step.kv_len.copy_(ints(1900 - 130 * t - 70 * self.k, 1 + 61 * t))
        self.step.slots.copy_(ints(self.c.slots[0], self.c.slots[1] if (t + self.k) % 3 else -1))

    def run(self):
        return ops.attention_kv4(self.q, self.c.pages, self.c.table, step=self.step, page=64, scale=0.1, want_lse=True)


def jobs(dtype, stretches, way, monkeypatch, n=2):
    monkeypatch.setattr(ops, "KV4_SPLIT_OVERRIDE", stretches)
    monkeypatch.setattr(ops, "KV4_SHARE_OVERRIDE", way)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    plan = ops.kv4_split_plan(2, 4, 2000, 33, sms) if dtype == BF16 else ops.kv4_split_plan_f32(2 * 4, 2000, sms)
    assert plan[0] > 1 and plan[2] != 2                             # merged by a second kernel, from a workspace
    c = Cache([1900, 1000], 2, 64, dtype, seed=4)
    return [Job(c, k, 16, dtype) for k in range(n)]


@pytest.mark.parametrize("dtype,stretches,way", PLANS)
def test_captured_graphs_share_no_workspace(dtype, stretches, way, monkeypatch):
    """Two graphs replayed at once on two streams, again and again with other lengths, slots and queries, beside an eager
    call on a third: every one gives what it gives alone."""
    three = jobs(dtype, stretches, way, monkeypatch, 3)
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs = []
    for job in three[:2]:
        job.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = job.run()
        graphs.append((graph, got))
    for t in range(12):
        want = []
        for job in three:
            job.turn(t)
            want.append(job.run())
        torch.cuda.synchronize()
        for _ in range(3):
            for (graph, _g), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                eager = three[2].run()
        torch.cuda.synchronize()
        for got, w in zip([g for _x, g in graphs] + [eager], want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


@pytest.mark.parametrize("dtype,stretches,way", PLANS)
def test_calls_on_two_streams_at_once(dtype, stretches, way, monkeypatch):
    two = jobs(dtype, stretches, way, monkeypatch)
    want = [job.run() for job in two]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in two]
    got = [[], []]
    for _ in range(20):
        for k, (job, s) in enumerate(zip(two, streams)):
            with torch.cuda.stream(s):
                got[k].append(job.run())
    torch.cuda.synchronize()
    for k in range(2):
        for out, lse in got[k]:
            assert torch.equal(out, want[k][0]) and torch.equal(lse, want[k][1])


# ---------------------------------------------------------------- many sequences
@pytest.mark.parametrize("least,way", [(None, None), (2, 1), (2, 0)])
def test_more_sequences_than_share_the_keys_out(least, way, monkeypatch):
    """From 257 on the keys of a pair are split by themselves."""
    monkeypatch.setattr(ops, "KV4_SPLIT_OVERRIDE", least)
    monkeypatch.setattr(ops, "KV4_SHARE_OVERRIDE", way)
    lens = [1 + 29 * i % 90 for i in range(300)]
    lens[7], lens[290] = 2600, 1500
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert ops.kv4_split_plan(302, 302, 2600, 42, sms)[2] == 0
    c = Cache(lens, 1, 64, BF16, seed=6)
    attend(c, [1] * 300, 2, BF16, pad=2)
    assert ops.kv4_split_plan(256, 256, 2600, 42, sms)[2] == (1 if way != 0 else 0)


# ---------------------------------------------------------------- the profile
def test_what_the_profile_counts_for_the_weights():
    """Of a token and kv head the key's codes and pairs, 9 D / 16 bytes, and the weight in and out; one product."""
    c = Cache([200, 30], 2, 64, BF16, weights=True)
    prof = ops.OpProfile()
    for q_lens, last in (([1, 1], 0), ([50, 20], 8)):
        step = c.step(q_lens)
        q = queries(sum(q_lens), 8, 64, BF16, 0).to(DEV)
        out, lse = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True)
        ops.set_profile(prof)
        try:
            ops.kv4_weigh(q, lse, c.pages, c.weights, c.table, step=step, page=64, scale=0.1, last=last)
        finally:
            ops.set_profile(None)
    rows = 2 + 2 * 8
    pairs = 230 + sum(range(193, 201)) + sum(range(23, 31))
    calls, _ms, moved, flops = prof.totals()["kv4_weigh"]
    assert (calls, moved, flops) == (2, 2 * 230 * 2 * (36 + 8) + rows * 8 * (128 + 4), 2.0 * 8 * 64 * pairs)


# ---------------------------------------------------------------- a large pool
@pytest.mark.parametrize("D,nkv", [(128, 8), (64, 9)])
def test_pages_beyond_four_gigabytes(D, nkv):
    """Pages whose bytes lie more than 2^32 into the pool: every operator gives what it gives in a small pool, and the
    pages at the front, where an offset of 32 bits would end, are as they were."""
    small = Cache([300, 90, 65], nkv, D, BF16, seed=12, weights=True, spare_pages=4)
    n, page = small.pages.shape[0], nkv * 4 * ops.kv4_record(D)
    n_pages = (1 << 32) // page + 2 * n
    if torch.cuda.mem_get_info()[0] < n_pages * page + (4 << 30):
        pytest.skip("no room for the pool")
    pages = torch.zeros((n_pages, nkv, 4, ops.kv4_record(D)), dtype=torch.uint8, device=DEV)
    weights = torch.zeros((n_pages, nkv, 64), device=DEV)
    weights[-n:] = small.weights
    table = small.table + (n_pages - n)
    assert int(table.min()) * page > 1 << 32
    lens, nq = small.lens, 4 * nkv
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(lens)).int().to(DEV)
    pos = torch.cat([torch.arange(x) for x in lens]).int().to(DEV)
    far = dict(small.at, block_table=table)
    pages[-n:] = 0xFF                                               # (as Cache leaves what nobody has)
    ops.kv4_write(small.kv.to(DEV), nkv, D, token_seq=seq, token_pos=pos, pages=pages, **far)
    assert torch.equal(pages[-n:], small.pages)
    for dtype in (BF16, F32):
        a = ops.kv4_read(pages, token_seq=seq, token_pos=pos, dtype=dtype, **far)
        assert torch.equal(a, ops.kv4_read(small.pages, token_seq=seq, token_pos=pos, dtype=dtype, **small.at))
        for q_lens in ([1, 1, 1], [70, 3, 65]):
            step, q = small.step(q_lens), queries(sum(q_lens), nq, D, dtype, 1).to(DEV)
            got = ops.attention_kv4(q, pages, table, step=step, page=64, scale=0.1, want_lse=True)
            want = ops.attention_kv4(q, small.pages, small.table, step=step, page=64, scale=0.1, want_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            if dtype == BF16:
                ops.kv4_weigh(q, got[1], pages, weights, table, step=step, page=64, scale=0.1)
                ops.kv4_weigh(q, got[1], small.pages, small.weights, small.table, step=step, page=64, scale=0.1)
                assert torch.equal(weights[-n:], small.weights)
    cut = dict(slots=ints(*small.slots), kv_len=ints(*lens), page=64, keep=80, recent=10)
    got, want = ops.kv4_evict(pages, weights, table, **cut), ops.kv4_evict(small.pages, small.weights, small.table, **cut)
    assert torch.equal(got[0], want[0]) and torch.equal(pages[-n:], small.pages) and torch.equal(weights[-n:], small.weights)
    assert not bool(pages[:-n].view(-1, 1152).any()) and not bool(weights[:-n].any())
