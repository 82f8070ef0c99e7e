"""The operators on a 4-bit cache against their plain form in 64 bits (plain.kv4)."""
import math
import types

import pytest
import torch

from grout_b200.kernels import ops
from plain import kv4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # the most that one rounding takes off
NAN = float("nan")


def ints(*v, shape=None):
    t = torch.tensor(v, dtype=torch.int32, device=DEV)
    return t.view(shape) if shape else t


class Cache:
    """A pool with every sequence's pages in some order, each sequence's tokens written by kv4_write; what lies
    behind a sequence's last token, and in pages that nobody has, is NaN."""

    def __init__(self, lens, nkv, D, dtype=torch.bfloat16, seed=0, slots=None, spare_pages=2, scale=1.0, weights=False,
                 edit=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.nkv, self.D, n = list(lens), nkv, D, len(lens)
        need = [(x + 63) // 64 for x in lens]
        self.n_slots, self.max_pages = n + 2, max(need + [1]) + 1
        order = torch.randperm(sum(need) + spare_pages, generator=g).int()
        self.slots = list(slots) if slots else torch.randperm(self.n_slots, generator=g)[:n].tolist()
        self.table = torch.full((self.n_slots, self.max_pages), 0, dtype=torch.int32)
        at = 0
        for s, k in zip(self.slots, need):
            self.table[s, :k] = order[at:at + k]
            at += k
        self.free = order[at:].tolist()
        self.table = self.table.to(DEV)
        self.pages = torch.full((sum(need) + spare_pages, nkv, 4, ops.kv4_record(D)), 0xFF, dtype=torch.uint8, device=DEV)
        self.weights = torch.rand((self.pages.shape[0], nkv, 64), generator=g).to(DEV) if weights else None
        kv = torch.randn((sum(lens), 2 * nkv, D), generator=g) * scale
        kv[:, :nkv, 3] += 4.0                                      # a channel that stands out
        if edit:
            edit(kv)
        self.kv = kv.to(dtype)
        seq = torch.repeat_interleave(torch.arange(n), torch.tensor(lens)).int()
        pos = torch.cat([torch.arange(x) for x in lens]).int() if sum(lens) else torch.zeros(0).int()
        self.at = dict(block_table=self.table, page=64, slots=ints(*self.slots))
        ops.kv4_write(self.kv.to(DEV), nkv, D, token_seq=seq.to(DEV), token_pos=pos.to(DEV), pages=self.pages, **self.at)
        self.c, self.s, self.m = kv4.quantise(self.kv)             # what the pool should hold
        self.held = kv4.value(self.c, self.s, self.m)

    def sequence(self, i, what=None):
        """Keys and values [nkv, n, D] that sequence i holds."""
        a = sum(self.lens[:i])
        x = (self.held if what is None else what)[a:a + self.lens[i]].transpose(0, 1)
        return x[:self.nkv], x[self.nkv:]

    def step(self, q_lens, pad=0):
        slots = [s for s in self.slots] + [-1] * pad
        q_all, kv = list(q_lens) + [1] * pad, self.lens + [1] * pad
        cu = [0]
        for x in q_all:
            cu.append(cu[-1] + x)
        return types.SimpleNamespace(
            n_tokens=cu[-1], n_seqs=len(slots), slots=ints(*slots), kv_len=ints(*kv), cu_q=ints(*cu),
            token_seq=torch.repeat_interleave(torch.arange(len(slots)), torch.tensor(q_all)).int().to(DEV),
            decode=all(x == 1 for x in q_all), max_kv_len=max(kv), q_lens=tuple(q_all))


def queries(T, nq, D, dtype, seed):
    return torch.randn((T, nq, D), generator=torch.Generator().manual_seed(100 + seed)).to(dtype)


# ---------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,nkv,D", [([1], 1, 64), ([70, 3, 129], 3, 128), ([64], 2, 128), ([17, 16, 15], 5, 64),
                                        ([1, 1, 1, 1, 1], 8, 128)])
def test_what_is_written_is_what_is_read(dtype, lens, nkv, D):
    c = Cache(lens, nkv, D, dtype, seed=sum(lens))
    for i in range(len(lens)):
        n = lens[i]
        want = torch.cat(c.sequence(i)).transpose(0, 1)
        got = ops.kv4_read(c.pages, token_seq=ints(*[i] * n), token_pos=ints(*range(n)), **c.at)
        # the same 32-bit arithmetic: the same codes and pairs, and s c + m is rounded once on both sides
        assert torch.equal(got.cpu(), want)
        got = ops.kv4_read(c.pages, token_seq=ints(*[i] * n), token_pos=ints(*range(n)), dtype=torch.bfloat16, **c.at)
        assert torch.equal(got.cpu(), want.bfloat16())


@pytest.mark.parametrize("D", [64, 128])
def test_bytes_of_a_record(D):
    c = Cache([50], 2, D, torch.float32, seed=3)
    k, v = c.sequence(0, c.kv)
    page = int(c.table[c.slots[0], 0])
    got = c.pages[page].cpu()
    for h in range(2):
        for r in range(3):
            assert torch.equal(got[h, r], kv4.record(k[h, 16 * r:16 * r + 16], v[h, 16 * r:16 * r + 16])), (h, r)
        # of the last record two tokens are written; the others' bytes are as they were
        want = kv4.record(torch.cat([k[h, 48:], torch.zeros(14, D)]), torch.cat([v[h, 48:], torch.zeros(14, D)]))
        rows = got[h, 3, :16 * D].view(2, 16, D // 2)
        assert torch.equal(rows[:, :2], want[:16 * D].view(2, 16, D // 2)[:, :2])
        assert bool((rows[:, 2:] == 0xFF).all()) and bool((got[h, 3, 16 * D:].view(16, -1)[2:] == 0xFF).all())


def test_groups_that_are_not_held_and_ranges_at_the_ends():
    def edit(kv):
        kv[0, 0, 3], kv[1, 1, 70], kv[2, 2, 5] = NAN, float("inf"), float("-inf")
        kv[3, 3, 64:66] = torch.tensor([3.3e38, -3.3e38])
        kv[4, 0] = 0.0
        kv[5, 0] = 1.2345678
        kv[6, 0] = torch.randn(128) * 1e-40                        # below the smallest normal number
        kv[7, 0] = torch.linspace(-1, 1, 128) * 1e37
        kv[8, 0] = -5.0
        kv[9, 0, :64] = torch.linspace(100, 101, 64)               # a large offset and a small range
    c = Cache([12], 2, 128, torch.float32, edit=edit)
    got = ops.kv4_read(c.pages, token_seq=ints(*[0] * 12), token_pos=ints(*range(12)), **c.at).cpu()
    want = c.held
    assert torch.equal(got.isnan(), want.isnan()) and int(want.isnan().sum()) == 4 * 64
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    off = (got.double() - c.kv.double()).unflatten(-1, (-1, 64)).abs()
    fine = ~want.isnan().unflatten(-1, (-1, 64))
    # half a step, and what the 32-bit quotient and sum are rounded by
    most = (c.s.double() * (0.5 + 2.0 ** -20))[..., None] + c.kv.double().abs().unflatten(-1, (-1, 64)) * 2.0 ** -23 + 1e-45
    assert bool((off <= most)[fine].all())


def test_rows_that_are_nowhere():
    c = Cache([20], 1, 64)
    before = c.pages.clone()
    kv = torch.randn((5, 2, 64), device=DEV).bfloat16()
    seq, pos = ints(0, 1, 0, 0, 7), ints(-1, 3, c.max_pages * 64, 0x7FFFFFFF, 0)
    at = dict(c.at, slots=ints(c.slots[0], -1))
    ops.kv4_write(kv, 1, 64, token_seq=seq, token_pos=pos, pages=c.pages, **at)
    assert torch.equal(c.pages, before)
    assert bool((ops.kv4_read(c.pages, token_seq=seq, token_pos=pos, **at) == 0).all())
    bad = c.table.clone()
    bad[c.slots[0], 0] = 1 << 20                                   # a number that is no page's
    at = dict(c.at, block_table=bad)
    ops.kv4_write(kv[:1], 1, 64, token_seq=ints(0), token_pos=ints(3), pages=c.pages, **at)
    assert torch.equal(c.pages, before)
    assert bool((ops.kv4_read(c.pages, token_seq=ints(0), token_pos=ints(3), **at) == 0).all())
    assert ops.kv4_read(c.pages, token_seq=ints(), token_pos=ints(), **c.at).shape == (0, 2, 64)


# ---------------------------------------------------------------- attention
def term(x, p):
    """sum_j p_j |x_j| for x [rows.., n, D] of one kv head."""
    return p @ x.abs()


def check(got, lse, c, i, q, step_rows, scale, dtype, rounded, **seen):
    """The rows of sequence i against the plain form.  Off by at most:
      the output's rounding, HALF |o|;
      in bfloat16, P's: a probability times s is rounded (2^-8 of it) where it multiplies the value less an offset, the
        middle of the codes for single tokens (an element is at most 8 s from it), nothing for prompts;
      the scores' 32-bit sums and the exponentials: 2^-17 of the sum of the products' magnitudes (128 terms of up to 31
        times a code's weight), as a factor on every probability."""
    k, v = c.sequence(i)
    if rounded:
        k, v = k.bfloat16().float(), v.bfloat16().float()
    want, want_lse, p = kv4.attend(q, k, v, scale, **seen)
    G = q.shape[1] // c.nkv
    a = sum(c.lens[:i])
    s = c.s[a:a + c.lens[i]].transpose(0, 1)                      # [2 nkv, n, groups]
    m = c.m[a:a + c.lens[i]].transpose(0, 1)
    for h in range(q.shape[1]):
        kv = h // G
        size = (q[:, h].double().abs() @ (k[kv].double().abs() + 31 * s[kv].double().repeat_interleave(64, -1)).T).amax() * scale
        delta = 2.0 ** -17 * (1 + float(size))
        av = v[kv].double().abs()
        tol = HALF[dtype] * want[:, h].abs() + 2 * delta * (term(av, p[h]) + want[:, h].abs()) + 1e-30
        if dtype == torch.bfloat16:
            if rounded:
                spread = av
            else:
                spread = 8 * s[c.nkv + kv].double().repeat_interleave(64, -1)
            tol = tol + HALF[dtype] * term(spread, p[h]) * (1 + 2.0 ** -7)
        off = (got[:, h].double() - want[:, h]).abs()
        assert bool((off <= tol).all()), (i, h, float((off / tol).max()), float(off.max()))
        if lse is not None:
            assert bool(((lse[:, h].double() - want_lse[:, h]).abs() <= delta + 2.0 ** -20 * want_lse[:, h].abs()).all()), (i, h)


SEEN = [dict(), dict(window=20), dict(window=100, keep_first=5), dict(chunk=48), dict(softcap=15.0),
        dict(window=64, keep_first=70, softcap=30.0)]


def attend(c, q_lens, nq, dtype, seed=0, sinks=False, pad=0, **seen):
    step = c.step(q_lens, pad)
    q = queries(step.n_tokens, nq, c.D, dtype, seed)
    sk = torch.randn(nq, generator=torch.Generator().manual_seed(7)) if sinks else None
    scale = 0.6 / math.sqrt(c.D)
    kw = {k: v for k, v in seen.items()}
    out, lse = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=scale, want_lse=True,
                                 sinks=None if sk is None else sk.to(DEV), **kw)
    again = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=scale,
                              sinks=None if sk is None else sk.to(DEV), **kw)
    assert torch.equal(out, again)
    out, lse = out.cpu(), lse.cpu()
    rounded = dtype == torch.bfloat16 and not step.decode
    at = 0
    for i, n in enumerate(q_lens):
        check(out[at:at + n], lse[at:at + n], c, i, q[at:at + n], n, scale, dtype, rounded, sinks=sk, **seen)
        at += n
    assert bool((out[at:] == 0).all()) and bool((lse[at:] == -math.inf).all())
    return q, out, lse, step, scale


@pytest.mark.parametrize("seen", SEEN, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,nq,nkv,D", [([1], 1, 1, 64), ([1, 2, 16, 17, 63, 64, 65], 8, 2, 128),
                                           ([300, 5, 129, 128], 20, 4, 64), ([700, 33], 17, 1, 128), ([515], 12, 4, 128)])
def test_single_tokens(lens, nq, nkv, D, dtype, seen):
    c = Cache(lens, nkv, D, dtype, seed=len(lens))
    attend(c, [1] * len(lens), nq, dtype, sinks=len(lens) % 2 == 1, pad=len(lens) % 3, **seen)


@pytest.mark.parametrize("way", [0, 2])
@pytest.mark.parametrize("stretches", [1, 3, 4, 8, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_splits_of_the_keys(stretches, dtype, way, monkeypatch):
    monkeypatch.setattr(ops, "KV4_SPLIT_OVERRIDE", stretches)
    monkeypatch.setattr(ops, "KV4_SHARE_OVERRIDE", way)
    c = Cache([1000, 1, 130], 2, 128, dtype)
    attend(c, [1, 1, 1], 8, dtype, sinks=True, pad=1)
    attend(c, [1, 1, 1], 8, dtype, window=200, keep_first=3)


@pytest.mark.parametrize("seen", SEEN, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_lens,before,nq,nkv,D", [
    ([2], [0], 1, 1, 64), ([130, 1, 64], [0, 40, 3], 8, 2, 128), ([33, 7], [100, 0], 20, 4, 64), ([300], [5], 6, 2, 128),
    ([1, 70, 2, 129], [63, 64, 190, 0], 12, 1, 64)])
def test_prompts(q_lens, before, nq, nkv, D, dtype, seen):
    c = Cache([a + b for a, b in zip(q_lens, before)], nkv, D, dtype, seed=sum(q_lens))
    attend(c, q_lens, nq, dtype, sinks=len(q_lens) % 2 == 0, pad=len(q_lens) % 2, **seen)


@pytest.mark.parametrize("n", [500, 1200])
def test_prompts_in_large_blocks(n):
    """Enough rows and heads that a block takes 256 query rows."""
    c = Cache([n, n // 3], 8, 128, seed=n)
    attend(c, [n, n // 3], 32, torch.bfloat16)


@pytest.mark.parametrize("lens", [[3000, 1, 200, 64, 2500], [33] * 40 + [2000], [700], [2100, 2100, 2100]], ids=lambda x: str(len(x)))
@pytest.mark.parametrize("least,way", [(None, None), (2, 1), (3, 1), (9, 1), (1, 1), (5, 0), (15, 2), (40, 2)])
def test_ways_to_split_the_keys(lens, least, way, monkeypatch):
    """A block a split; clusters of them; runs of stretches that end inside a pair, hold several pairs, or one pair's
    middle; padding rows between."""
    monkeypatch.setattr(ops, "KV4_SPLIT_OVERRIDE", least)
    monkeypatch.setattr(ops, "KV4_SHARE_OVERRIDE", way)
    c = Cache(lens, 2, 64, seed=len(lens))
    attend(c, [1] * len(lens), 12, torch.bfloat16, sinks=True, pad=2)
    attend(c, [1] * len(lens), 4, torch.bfloat16, window=300, keep_first=40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bound", [1, 700, 1500])
def test_a_bound_of_the_lengths_that_is_too_low(dtype, bound):
    """Rows with more keys than the caller's bound are right or NaN, and the others right."""
    c = Cache([3000, 90], 2, 64, dtype, seed=3)
    step, q = c.step([1, 1]), queries(2, 8, 64, dtype, 0).to(DEV)
    want = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
    step.max_kv_len = bound
    got = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
    assert bool(got[0].isnan().all()) or float((got[0] - want[0]).abs().max()) < 0.01
    assert float((got[1] - want[1]).abs().max()) < 0.01


def test_a_capped_score_far_beyond_the_cap():
    c = Cache([90], 1, 64, scale=30.0)
    attend(c, [1], 4, torch.bfloat16, softcap=2.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_seen_may_be_anything(dtype):
    """The pool is NaN wherever nothing was written (Cache), and NaN tokens in front of the window, behind the row and
    in another sequence leave a row as it is."""
    def edit(kv):
        kv[10, 0] = NAN            # sequence 0: a key in front of the window
        kv[11, 1] = NAN            # ... and a value
        kv[200:230] = NAN          # sequence 1
    c = Cache([200, 30, 100], 1, 64, dtype, edit=edit)
    step = c.step([1, 1, 1])
    q = queries(3, 4, 64, dtype, 0)
    out = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.125, window=100).cpu()
    assert bool(out[1].isnan().all())
    for i in (0, 2):
        want, _l, _p = kv4.attend(q[i:i + 1], *[x.nan_to_num(0.0) for x in c.sequence(i)], 0.125, window=100)
        assert float((out[i:i + 1].double() - want).abs().max()) < 0.03
    # as prompts: only the rows that see the NaN tokens
    step = c.step([200, 30, 100])
    q = queries(330, 4, 64, dtype, 1)
    out = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.125, window=50).cpu()
    seen = torch.zeros(330, dtype=torch.bool)
    seen[10:61] = True             # key 10 is seen by rows 10 .. 59, value 11 by 11 .. 60
    seen[200:230] = True
    assert torch.equal(out.isnan().any(-1).any(-1), seen)


def test_a_page_that_there_is_not():
    c = Cache([100, 70, 40], 2, 128, seed=1)
    table = c.table.clone()
    table[c.slots[1], 0] = -5
    table[c.slots[2], 0] = 1 << 30
    for q_lens in ([1, 1, 1], [20, 30, 40]):
        for dtype in (torch.bfloat16, torch.float32):
            step = c.step(q_lens)
            q = queries(step.n_tokens, 4, 128, dtype, 0).to(DEV)
            out = ops.attention_kv4(q, c.pages, table, step=step, page=64, scale=0.1)
            fine = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
            a = q_lens[0]
            assert torch.equal(out[:a], fine[:a]) and bool(out[a:].isnan().all())
    # a length beyond what the table holds
    step = c.step([1, 1, 1])
    step.kv_len = ints(100, 70, c.max_pages * 64 + 1)
    q = queries(3, 4, 128, torch.bfloat16, 0).to(DEV)
    out = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
    assert bool(out[2].isnan().all()) and not bool(out[:2].isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sinks", [None, 0.5, -math.inf])
def test_a_sequence_without_keys(dtype, sinks):
    c = Cache([5], 1, 64)
    step = c.step([1])
    step.kv_len = ints(0)
    sk = None if sinks is None else torch.full((2,), sinks, device=DEV)
    out, lse = ops.attention_kv4(queries(1, 2, 64, dtype, 0).to(DEV), c.pages, c.table, step=step, page=64, scale=1.0,
                                 sinks=sk, want_lse=True)
    assert bool((out == 0).all())
    assert bool((lse == (-math.inf if sinks is None else sinks)).all())


# ---------------------------------------------------------------- weights
@pytest.mark.parametrize("seen", SEEN, ids=str)
@pytest.mark.parametrize("lens,nq,nkv,D", [([1], 1, 1, 64), ([70, 3, 129, 16], 20, 4, 128), ([300, 64], 17, 1, 64)])
def test_weights_of_single_tokens(lens, nq, nkv, D, seen):
    c = Cache(lens, nkv, D, weights=True, seed=2)
    before = c.weights.clone()
    q, _o, lse, step, scale = attend(c, [1] * len(lens), nq, torch.bfloat16, pad=1, sinks=True, **seen)
    ops.kv4_weigh(q.to(DEV), lse.to(DEV), c.pages, c.weights, c.table, step=step, page=64, scale=scale, **seen)
    check_weights(c, before, q, [1] * len(lens), [1] * len(lens), scale, **seen)


def check_weights(c, before, q, q_lens, last, scale, rel=None, **seen):
    want = before.double().cpu()
    tol = want.abs() * 2.0 ** -23
    sk = torch.randn(q.shape[1], generator=torch.Generator().manual_seed(7))
    at = 0
    for i, n in enumerate(q_lens):
        k, v = c.sequence(i)
        _o, _l, p = kv4.attend(q[at:at + n], k, v, scale, sinks=sk, **seen)
        p = p[:, n - last[i]:].sum(1).view(c.nkv, -1, c.lens[i]).sum(1)
        a = sum(c.lens[:i])
        size = float(q[at:at + n].double().abs().sum(-1).amax() * (k.abs().amax() + 31 * c.s[a:a + c.lens[i]].amax()) * scale)
        at += n
        for j in range(c.lens[i]):
            page = int(c.table[c.slots[i], j // 64])
            want[page, :, j % 64] += p[:, j]
            # both the score and the logarithm: 2^-17 of the products' magnitudes each (check)
            tol[page, :, j % 64] += p[:, j] * (rel if rel else 2 * 2.0 ** -17 * (1 + size)) + 1e-30
    off = (c.weights.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off / tol.clamp(min=1e-30)).max())


@pytest.mark.parametrize("last", [0, 1, 5, 1000])
@pytest.mark.parametrize("seen", [dict(), dict(window=20, keep_first=3), dict(softcap=15.0)], ids=str)
def test_weights_of_prompts(last, seen):
    q_lens, before_lens = [40, 1, 90], [30, 64, 0]
    c = Cache([a + b for a, b in zip(q_lens, before_lens)], 2, 64, weights=True, seed=5)
    before = c.weights.clone()
    q, _o, lse, step, scale = attend(c, q_lens, 6, torch.bfloat16, pad=1, sinks=True, **seen)
    ops.kv4_weigh(q.to(DEV), lse.to(DEV), c.pages, c.weights, c.table, step=step, page=64, scale=scale, last=last, **seen)
    rows = [min(n, last) if last else n for n in q_lens]
    # the prompt's lse comes from keys rounded to bfloat16: 2^-8 of the products' magnitudes (at most 6 here: |s| < 4
    # and the products' signs), as a factor
    check_weights(c, before, q, q_lens, rows, scale, rel=0.05, **seen)


def test_written_tokens_have_no_weight_yet():
    c = Cache([70], 2, 64, weights=True)
    ops.kv4_write(c.kv[:3].to(DEV), 2, 64, token_seq=ints(0, 0, 0), token_pos=ints(5, 64, 20), pages=c.pages,
                  weights=c.weights, **c.at)
    got = torch.stack([c.weights[int(c.table[c.slots[0], p // 64]), :, p % 64] for p in range(70)])
    zero = (got == 0).all(1)
    assert zero.nonzero().flatten().tolist() == [5, 20, 64]


# ---------------------------------------------------------------- eviction
def kept_of(c, i, kept, n):
    return kept[i, :, :n].cpu()


@pytest.mark.parametrize("place", ["in place", "elsewhere"])
@pytest.mark.parametrize("lens,nkv,D,keep,recent,first", [
    ([1], 1, 64, 4, 1, 0), ([200, 33, 64, 65], 2, 128, 64, 10, 4), ([500, 130], 3, 64, 100, 0, 0), ([70], 1, 128, 17, 17, 0),
    ([2100], 2, 64, 1500, 100, 3), ([90, 91], 1, 64, 1, 0, 1), ([40], 4, 128, 39, 0, 39)])
def test_eviction(lens, nkv, D, keep, recent, first, place):
    few = (keep + 63) // 64
    c = Cache(lens, nkv, D, torch.bfloat16, seed=keep, weights=True, spare_pages=len(lens) * few + 1)
    # equal weights, zeros and a NaN among them
    c.weights = (c.weights * 8).floor() / 8
    c.weights.view(-1)[::37] = NAN
    held = lambda i: torch.cat(c.sequence(i)).transpose(0, 1)
    weights = [torch.stack([c.weights[int(c.table[c.slots[i], p // 64]), :, p % 64] for p in range(n)], 1).cpu()
               for i, n in enumerate(lens)]
    into = None
    if place == "elsewhere":
        into = torch.full((c.n_slots, few), -1, dtype=torch.int32)
        for k, s in enumerate(c.slots):
            into[s] = torch.tensor(c.free[k * few:(k + 1) * few])
        into = into.to(DEV)
    before, w_before = c.pages.clone(), c.weights.clone()
    kept, new = ops.kv4_evict(c.pages, c.weights, c.table, slots=ints(*c.slots, -1), kv_len=ints(*lens, 9), page=64, keep=keep,
                              recent=recent, first=first, into=into)
    assert new.tolist() == [min(n, keep) for n in lens] + [0]
    assert bool((kept[-1] == -1).all())
    table = c.table if into is None else into
    for i, n in enumerate(lens):
        left = min(n, keep)
        got = ops.kv4_read(c.pages, token_seq=ints(*[i] * left), token_pos=ints(*range(left)), block_table=table, page=64,
                           slots=ints(*c.slots)).cpu()
        for h in range(nkv):
            want = kv4.choose(weights[i][h].tolist(), n, keep, recent, first)
            assert kept[i, h].tolist() == want + [-1] * (keep - left)
            assert torch.equal(got[:, h], held(i)[want, h]) and torch.equal(got[:, nkv + h], held(i)[want, nkv + h])
            w = torch.stack([c.weights[int(table[c.slots[i], p // 64]), h, p % 64] for p in range(left)]).cpu()
            assert torch.equal(w.nan_to_num(-1.0), weights[i][h][want].nan_to_num(-1.0))
    # every page that no kept token goes to is as it was
    touched = {int(p) for s, n in zip(c.slots, lens) for p in table[s, :(min(n, keep) + 63) // 64]}
    others = [p for p in range(before.shape[0]) if p not in touched]
    assert torch.equal(c.pages[others], before[others])
    assert torch.equal(c.weights[others].nan_to_num(-1.0), w_before[others].nan_to_num(-1.0))


def test_eviction_into_the_same_table():
    c = Cache([300], 2, 64, weights=True, seed=9)
    d = Cache([300], 2, 64, weights=True, seed=9)
    args = dict(slots=ints(*c.slots), kv_len=ints(300), page=64, keep=100, recent=10)
    a = ops.kv4_evict(c.pages, c.weights, c.table, **args)
    b = ops.kv4_evict(d.pages, d.weights, d.table, into=d.table, **args)
    assert torch.equal(a[0], b[0])
    n = dict(token_seq=ints(*[0] * 100), token_pos=ints(*range(100)))
    assert torch.equal(ops.kv4_read(c.pages, **n, **c.at), ops.kv4_read(d.pages, **n, **d.at))


# ---------------------------------------------------------------- together
def test_a_sequence_that_is_cut_and_goes_on():
    """Prompt, single tokens with account of the weights, a cut, and more single tokens behind it."""
    nq, nkv, D, keep, recent = 8, 2, 64, 48, 8
    g = torch.Generator().manual_seed(11)
    n, total = 90, 100
    kv = torch.randn((total, 2 * nkv, D), generator=g).bfloat16()
    held = kv4.value(*kv4.quantise(kv))
    table = ints(3, 1, 0, 2, shape=(1, 4))
    pages, weights = ops.kv4_pages(4, nkv, D, DEV), torch.full((4, nkv, 64), 9.0, device=DEV)
    at = dict(slots=ints(0), block_table=table, page=64)
    seen = dict(page=64, scale=0.125)
    ref_k = [[held[j, h] for j in range(n)] for h in range(nkv)]
    ref_v = [[held[j, nkv + h] for j in range(n)] for h in range(nkv)]
    ref_w = torch.zeros((nkv, n), dtype=torch.float64)

    def step(q_len, length):
        return types.SimpleNamespace(slots=ints(0), kv_len=ints(length), cu_q=ints(0, q_len), decode=q_len == 1, q_lens=(q_len,),
                                     token_seq=ints(*[0] * q_len), max_kv_len=length)

    ops.kv4_write(kv[:n].to(DEV), nkv, D, token_seq=ints(*[0] * n), token_pos=ints(*range(n)), pages=pages, weights=weights, **at)
    length = n
    for j in range(n, total):
        if j == 94:
            kept, new = ops.kv4_evict(pages, weights, table, slots=ints(0), kv_len=ints(length), page=64, keep=keep, recent=recent)
            assert int(new) == keep
            for h in range(nkv):
                want = kv4.choose(ref_w[h].tolist(), length, keep, recent, 0)
                assert kept[0, h].tolist() == want
                ref_k[h], ref_v[h] = [ref_k[h][x] for x in want], [ref_v[h][x] for x in want]
            ref_w = torch.stack([ref_w[h][kept[0, h].long().cpu()] for h in range(nkv)])
            length = keep
        ops.kv4_write(kv[j:j + 1].to(DEV), nkv, D, token_seq=ints(0), token_pos=ints(length), pages=pages, weights=weights, **at)
        length += 1
        for h in range(nkv):
            ref_k[h].append(held[j, h])
            ref_v[h].append(held[j, nkv + h])
        ref_w = torch.cat([ref_w, torch.zeros((nkv, 1), dtype=torch.float64)], 1)
        q = queries(1, nq, D, torch.bfloat16, j)
        s = step(1, length)
        out, lse = ops.attention_kv4(q.to(DEV), pages, table, step=s, want_lse=True, **seen)
        ops.kv4_weigh(q.to(DEV), lse, pages, weights, table, step=s, **seen)
        k = torch.stack([torch.stack(x) for x in ref_k])
        v = torch.stack([torch.stack(x) for x in ref_v])
        want, _l, p = kv4.attend(q, k, v, 0.125)
        ref_w += p.sum(1).view(nkv, -1, length).sum(1)
        # 2^-8 of the output and of the spread of the values around the middle of their codes (at most 8 s < 8 * 0.5)
        assert float((out.double().cpu() - want).abs().max()) <= 2.0 ** -8 * (4.0 + float(want.abs().max()))
    got = torch.stack([weights[int(table[0, p // 64]), :, p % 64] for p in range(length)], 1).double().cpu()
    assert float((got - ref_w).abs().max()) < 1e-3


def test_captured_and_replayed():
    """One graph of all operators, replayed with other lengths, tokens and queries; two graphs share nothing."""
    nq, nkv, D = 8, 2, 128
    c = Cache([700, 90], nkv, D, weights=True, seed=4)
    graphs = []
    for k in range(2):
        st = c.step([1, 1])
        st.max_kv_len = 1000
        q = queries(2, nq, D, torch.bfloat16, k).to(DEV)
        kv = c.kv[:2].to(DEV).clone()
        pos = ints(699, 89)

        def run(st=st, q=q, kv=kv, pos=pos):
            ops.kv4_write(kv, nkv, D, token_seq=st.token_seq, token_pos=pos, pages=c.pages, **dict(c.at, slots=st.slots))
            out, lse = ops.attention_kv4(q, c.pages, c.table, step=st, page=64, scale=0.1, want_lse=True)
            w = torch.zeros_like(c.weights)
            ops.kv4_weigh(q, lse, c.pages, w, c.table, step=st, page=64, scale=0.1)
            return out, w
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        graphs.append((graph, got, st, q, kv, run))
    for turn in range(3):
        for k, (graph, got, st, q, kv, run) in enumerate(graphs):
            q.copy_(queries(2, nq, D, torch.bfloat16, 10 * turn + k))
            st.kv_len.copy_(ints(700 - 100 * turn, 90 - turn))
            st.slots.copy_(ints(c.slots[0], c.slots[1] if turn else -1))
        for graph, *_ in graphs:
            graph.replay()
        for graph, got, st, q, kv, run in graphs:
            want = run()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_on_another_stream():
    c = Cache([300, 40], 2, 128, weights=True, seed=6)
    step, q = c.step([1, 1]), queries(2, 8, 128, torch.bfloat16, 0).to(DEV)
    want = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
    side.synchronize()
    assert torch.equal(got, want)


def test_on_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    c = Cache([300, 40], 2, 128, seed=6)
    step, q = c.step([1, 1]), queries(2, 8, 128, torch.bfloat16, 0).to(DEV)
    want = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1)
    with torch.cuda.device(1):
        assert torch.equal(ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1), want)


# ---------------------------------------------------------------- refusals
def test_refusals():
    c = Cache([40], 2, 64, weights=True)
    kv = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=DEV)
    one = dict(token_seq=ints(0), token_pos=ints(0), pages=c.pages, **c.at)
    q, step = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=DEV), c.step([1])
    seen = dict(step=step, page=64, scale=1.0)
    lse = torch.zeros((1, 4), device=DEV)
    cut = dict(slots=ints(*c.slots), kv_len=ints(40), page=64, keep=8, recent=2)
    other = types.SimpleNamespace(**{**vars(step), "kv_len": ints(1, 2)})
    odd = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(1, 4, 64)
    calls = [
        lambda: ops.kv4_write(kv.half(), 2, 64, **one),
        lambda: ops.kv4_write(kv, 4, 64, **one),
        lambda: ops.kv4_write(kv, 2, 128, **one),
        lambda: ops.kv4_write(kv[:, :3].contiguous(), 2, 64, **one),
        lambda: ops.kv4_write(odd, 2, 64, **one),
        lambda: ops.kv4_write(kv, 2, 64, **dict(one, page=32)),
        lambda: ops.kv4_write(kv, 2, 64, **dict(one, token_pos=ints(0, 1))),
        lambda: ops.kv4_write(kv, 2, 64, **dict(one, token_pos=ints(0).long())),
        lambda: ops.kv4_write(kv, 2, 64, **dict(one, pages=c.pages[:, :, :, :-1].contiguous())),
        lambda: ops.kv4_write(kv, 2, 64, **dict(one, pages=c.pages.view(torch.int8))),
        lambda: ops.kv4_write(kv, 2, 64, weights=c.weights[:1], **one),
        lambda: ops.kv4_read(c.pages, dtype=torch.float16, **{k: v for k, v in one.items() if k != "pages"}),
        lambda: ops.attention_kv4(q[:, :3].contiguous(), c.pages, c.table, **seen),
        lambda: ops.attention_kv4(q.half(), c.pages, c.table, **seen),
        lambda: ops.attention_kv4(q.repeat(1, 1, 2), c.pages, c.table, **seen),
        lambda: ops.attention_kv4(q.repeat(2, 1, 1), c.pages, c.table, **seen),
        lambda: ops.attention_kv4(q.transpose(1, 2), c.pages, c.table, **seen),
        lambda: ops.attention_kv4(odd, c.pages, c.table, **seen),
        lambda: ops.attention_kv4(q, c.pages, c.table.cpu(), **seen),
        lambda: ops.attention_kv4(q, c.pages, c.table, **dict(seen, page=16)),
        lambda: ops.attention_kv4(q, c.pages, c.table, **dict(seen, step=other)),
        lambda: ops.attention_kv4(q, c.pages, c.table, window=-1, **seen),
        lambda: ops.attention_kv4(q, c.pages, c.table, softcap=-2.0, **seen),
        lambda: ops.attention_kv4(q, c.pages, c.table, chunk=-1, **seen),
        lambda: ops.attention_kv4(q, c.pages, c.table, window=4, keep_first=2, chunk=8, **seen),
        lambda: ops.attention_kv4(q, c.pages, c.table, sinks=torch.zeros(3, device=DEV), **seen),
        lambda: ops.kv4_weigh(q.float(), lse, c.pages, c.weights, c.table, **seen),
        lambda: ops.kv4_weigh(q, lse[:, :2].contiguous(), c.pages, c.weights, c.table, **seen),
        lambda: ops.kv4_weigh(q, lse, c.pages, c.weights.double(), c.table, **seen),
        lambda: ops.kv4_weigh(q, lse, c.pages, c.weights, c.table, last=-1, **seen),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, **dict(cut, keep=0, recent=0)),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, **dict(cut, recent=9)),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, first=7, **cut),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, first=-1, **cut),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, **dict(cut, kv_len=ints(40, 1))),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, into=c.table[:1].contiguous(), **cut),
        lambda: ops.kv4_evict(c.pages, c.weights, c.table, into=c.table[:, :1].contiguous(), **dict(cut, keep=65)),
    ]
    before = c.pages.clone()
    for i, call in enumerate(calls):
        try:
            call()
        except ops.KernelError:
            continue
        raise AssertionError(f"call {i} was not refused")
    assert torch.equal(c.pages, before)
    torch.cuda.synchronize()


def test_the_profile_knows_the_operators():
    c = Cache([200, 30], 2, 64, weights=True)
    step, q = c.step([1, 1]), queries(2, 8, 64, torch.bfloat16, 0).to(DEV)
    prof = ops.OpProfile()
    ops.set_profile(prof)
    try:
        out, lse = ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True)
        ops.kv4_weigh(q, lse, c.pages, c.weights, c.table, step=step, page=64, scale=0.1)
        ops.kv4_read(c.pages, token_seq=ints(0), token_pos=ints(3), **c.at)
        ops.kv4_write(c.kv[:1].to(DEV), 2, 64, token_seq=ints(0), token_pos=ints(3), pages=c.pages, **c.at)
        ops.kv4_evict(c.pages, c.weights, c.table, slots=ints(*c.slots), kv_len=ints(200, 30), page=64, keep=50, recent=5)
    finally:
        ops.set_profile(None)
    totals = prof.totals()
    assert {"attn_kv4_decode", "kv4_weigh", "kv4_read", "kv4_write", "kv4_evict"} == set(totals)
    # 230 tokens of two heads of 72 bytes for keys and as many for values; eight heads in and out; 4 D flops a pair
    assert totals["attn_kv4_decode"][2:] == [230 * 2 * 144 // 2 * 1.0 + 2 * 2 * 8 * 64 * 2, 4.0 * 8 * 64 * 230]
    assert all(v[0] == 1 and v[1] > 0 and v[2] > 0 for v in totals.values())
