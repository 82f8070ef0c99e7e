"""Where the operators on a 4-bit cache could go wrong: at the edges of what they are given."""
import math
import types

import pytest
import torch

from grout_b200.kernels import ops
from plain import kv4
from test_kv4_gpu import DEV, NAN, Cache, check, ints, queries

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def split(monkeypatch, stretches, way):
    monkeypatch.setattr(ops, "KV4_SPLIT_OVERRIDE", stretches)
    monkeypatch.setattr(ops, "KV4_SHARE_OVERRIDE", way)


# ---------------------------------------------------------------- NaN and splits
SPLITS = [(BF16, 8, 0), (BF16, 1, 0), (BF16, 8, 1), (BF16, 2, 1), (BF16, 8, 2), (F32, 8, 0), (F32, 1, 0), (F32, 8, 2)]


@pytest.mark.parametrize("dtype,stretches,way", SPLITS)
@pytest.mark.parametrize("n", [257, 700])
def test_queries_that_are_nan(n, dtype, stretches, way, monkeypatch):
    """A row whose queries are NaN is NaN and so is its sum, however the keys are split; its neighbour is not."""
    split(monkeypatch, stretches, way)
    c = Cache([n, 90], 2, 64, dtype, seed=1)
    step, q = c.step([1, 1]), queries(2, 8, 64, dtype, 0)
    fine, fine_lse = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True)
    q[0] = NAN
    out, lse = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True)
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    assert torch.equal(out[1], fine[1]) and torch.equal(lse[1], fine_lse[1])


@pytest.mark.parametrize("dtype,stretches,way", SPLITS)
@pytest.mark.parametrize("n,first,last", [(257, 256, 257), (700, 256, 512), (700, 640, 700), (700, 699, 700), (257, 0, 257)])
def test_keys_that_are_nan(n, first, last, dtype, stretches, way, monkeypatch):
    """Tokens whose keys are NaN make the row NaN, also where they are all that a split has."""
    split(monkeypatch, stretches, way)

    def edit(kv):
        kv[first:last, :1] = NAN                                  # the keys of kv head 0
    c = Cache([n, 90], 2, 64, dtype, seed=1, edit=edit)
    step, q = c.step([1, 1]), queries(2, 8, 64, dtype, 0)
    out, lse = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True)
    assert bool(out[0, :4].isnan().all()) and bool(lse[0, :4].isnan().all())
    assert not bool(out[0, 4:].isnan().any()) and not bool(out[1].isnan().any()) and not bool(lse[0, 4:].isnan().any())


@pytest.mark.parametrize("dtype,stretches,way", SPLITS)
@pytest.mark.parametrize("n,first,last", [(700, 0, 256), (700, 699, 700), (257, 3, 4)])
def test_values_that_are_nan_and_of_no_weight(n, first, last, dtype, stretches, way, monkeypatch):
    """A token that a row sees makes its 64 elements NaN when they are stored as NaN, though 2^(its score) is 0."""
    split(monkeypatch, stretches, way)

    def edit(kv):
        kv[first:last, :2, 3] = -900.0
        kv[first:last, 3, :64] = NAN                              # the values of kv head 1
    c = Cache([n, 90], 2, 128, dtype, seed=1, edit=edit)
    step, q = c.step([1, 1]), queries(2, 8, 128, dtype, 0)
    q[..., 3] = 4.0
    out = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.1)
    assert bool(out[0, 4:, :64].isnan().all())
    assert not bool(out[0, :4].isnan().any()) and not bool(out[0, 4:, 64:].isnan().any()) and not bool(out[1].isnan().any())


# ---------------------------------------------------------------- scores far apart
def far_apart(nq, D, rows):
    """Keys whose scores lie 400 and more below those of the later ones (natural units), and queries of the last rows."""
    def edit(kv):
        nkv = kv.shape[1] // 2
        kv[:, :nkv, 3] = 0.0
        kv[:130, :nkv, 3] = -50.0
        kv[130:, :nkv, 3] = 50.0
        kv[:130, nkv:] += 6.0                                      # values that would be seen in the result
    c = Cache([260], 2, D, BF16, seed=3, edit=edit)
    q = queries(rows, nq, D, BF16, 5)
    q[..., 3] = 32.0
    return c, q


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [0, 128, 256])
def test_a_maximum_that_rises_beyond_the_numbers_range(rows, D, monkeypatch):
    """2^(old maximum - new) is 0 in 32 bits: nothing of the earlier keys is left, in a prompt's rows and a single token's."""
    monkeypatch.setattr(ops, "PREFILL_TC_ROWS", rows)
    c, q = far_apart(8, D, 260)
    scale = 1.0 / math.sqrt(D)
    for n in (260, 1):
        step = c.step([n])
        out, lse = ops.attention_kv4(q[260 - n:].to(DEV), c.pages, c.table, step=step, page=64, scale=scale, want_lse=True)
        check(out.cpu(), lse.cpu(), c, 0, q[260 - n:], n, scale, BF16, n > 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [128, 256])
def test_a_maximum_that_rises_beyond_the_range_over_pages_in_16_bits(rows, D):
    c, q = far_apart(8, D, 260)
    step, scale = c.step([260]), 1.0 / math.sqrt(D)
    rows_of = torch.arange(260)
    k, v = c.kv[:, :2].bfloat16(), c.kv[:, 2:].bfloat16()
    k_pages, v_pages = (torch.zeros((c.pages.shape[0], 2, 64, D), dtype=BF16, device=DEV) for _ in range(2))
    table = c.table.cpu()
    for p in range(5):
        at = rows_of[64 * p:64 * p + 64]
        k_pages[int(table[c.slots[0], p]), :, :len(at)] = k[at].transpose(0, 1).to(DEV)
        v_pages[int(table[c.slots[0], p]), :, :len(at)] = v[at].transpose(0, 1).to(DEV)
    out = ops.attn_prefill_tc(q.to(DEV), k_pages, v_pages, c.table, cu_q=step.cu_q, slots=step.slots, kv_len=step.kv_len,
                              q_lens=step.q_lens, page=64, scale=scale, rows_per_block=rows).cpu()
    want, _l, p = kv4.attend(q, k.transpose(0, 1), v.transpose(0, 1), scale)
    for h in range(8):
        av = v[:, h // 4].double().abs()
        # the output's rounding, the probabilities' (2^-8 each), and 2^-17 of scores up to 400 + 128 * 16
        delta = 2.0 ** -17 * 400
        tol = (2.0 ** -8 + 2 * delta) * want[:, h].abs() + (2.0 ** -8 * (1 + 2.0 ** -7) + 2 * delta) * (p[h] @ av)
        off = (out[:, h].double() - want[:, h]).abs()
        assert bool((off <= tol).all()), (h, float((off / tol).max()))


# ---------------------------------------------------------------- values of very different sizes
def sizes_apart(kind, nkv):
    def edit(kv):
        if kind == "a huge value that is paid nothing":
            kv[5, :nkv, 3] = -600.0
            kv[5, nkv:] *= 1e9
        elif kind == "huge values that a later key outweighs":
            kv[:200, :nkv, 3] = -600.0
            kv[:200, nkv:] *= 1e9
        elif kind == "huge values, then small ones that outweigh them":
            kv[:200, :nkv, 3] = -600.0
            kv[:200, nkv:] *= 1e20
            kv[200:, nkv:] *= 1e-15
        elif kind == "groups of different sizes":
            kv[:, nkv:, :64] *= 1e7
        elif kind == "small":
            kv[:, nkv:] *= 1e-25
        elif kind == "large":
            kv[:, nkv:] *= 1e35
        elif kind == "without a range":
            kv[:, nkv:] = 0.75
        elif kind == "growing":
            kv[:, nkv:] *= torch.logspace(-12, 12, kv.shape[0])[:, None, None]
        elif kind == "heads that pay to other tokens":
            kv[::2, :nkv, 3], kv[1::2, :nkv, 3] = 600.0, -600.0
            kv[::2, nkv:] *= 1e8
    return edit


KINDS = ["a huge value that is paid nothing", "huge values that a later key outweighs",
         "huge values, then small ones that outweigh them", "groups of different sizes", "small", "large", "without a range",
         "growing", "heads that pay to other tokens"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,stretches,way", [(BF16, None, None), (BF16, 2, 0), (BF16, 2, 1), (BF16, 2, 2), (F32, None, None)])
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_different_sizes(D, dtype, stretches, way, kind, monkeypatch):
    """A value's steps may be any size: a probability times a step keeps its bits whatever the values beside it."""
    split(monkeypatch, stretches, way)
    c = Cache([330, 40], 2, D, dtype, seed=8, edit=sizes_apart(kind, 2))
    q = queries(2, 16, D, dtype, 1)
    q[..., 3] = 4.0
    if kind == "heads that pay to other tokens":
        q[:, ::2, 3] = -4.0
    scale = 0.6 / math.sqrt(D)
    out, lse = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=c.step([1, 1]), page=64, scale=scale, want_lse=True)
    for i in range(2):
        check(out[i:i + 1].cpu(), lse[i:i + 1].cpu(), c, i, q[i:i + 1], 1, scale, dtype, False)


# ---------------------------------------------------------------- the end of the numbers' range
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_range_that_ends_beyond_the_numbers(dtype):
    """Fifteen steps above the least element no finite number is left (the step is rounded up): such a group is NaN like
    every other whose range is not held, and no row that does not see it has a part of it."""
    def edit(kv):
        kv[20, 1, :64] = 2e36
        kv[20, 1, 7] = 3.3895e38                                   # (bfloat16's largest; a 15th of the range rounds up)
        kv[21, 1, :64] = torch.linspace(0, 3.2e38, 64)             # held
    c = Cache([100], 1, 64, dtype, edit=edit)
    got = ops.kv4_read(c.pages, token_seq=ints(0, 0), token_pos=ints(20, 21), **c.at).cpu()
    assert bool(got[0, 1].isnan().all()) and bool(got[1, 1].isfinite().all())
    step, q = c.step([100]), queries(100, 4, 64, dtype, 1)
    out = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=0.125, window=10).cpu()
    seen = out.isnan().any(-1).any(-1)
    assert seen.nonzero().flatten().tolist() == list(range(20, 30))


# ---------------------------------------------------------------- eviction
@pytest.mark.parametrize("place", ["in place", "elsewhere"])
def test_eviction_of_tokens_that_no_page_holds(place):
    """They are kept as NaN without a weight, whatever lay in the memory that they go to."""
    n, keep, recent = 200, 100, 20
    c = Cache([n], 2, 64, BF16, seed=4, weights=True, spare_pages=3)
    good = torch.cat(c.sequence(0)).transpose(0, 1)
    table = c.table.clone()
    table[c.slots[0], 2], table[c.slots[0], 3] = -3, 1 << 30       # tokens 128 .. 191 and 192 .. 199
    into = None
    if place == "elsewhere":
        into = torch.full((c.n_slots, 2), -1, dtype=torch.int32)
        into[c.slots[0]] = torch.tensor(c.free[:2])
        into = into.to(DEV)
    kept, new = ops.kv4_evict(c.pages, c.weights, table, slots=ints(*c.slots), kv_len=ints(n), page=64, keep=keep, recent=recent,
                              first=70, into=into)
    assert new.tolist() == [keep]
    to = table if into is None else into
    got = ops.kv4_read(c.pages, token_seq=ints(*[0] * keep), token_pos=ints(*range(keep)), block_table=to, page=64,
                       slots=ints(*c.slots)).cpu()
    for h in range(2):
        places = kept[0, h].tolist()
        assert places[:70] == list(range(70)) and places[80:] == list(range(180, 200))
        for j, p in enumerate(places):
            w = float(c.weights[int(to[c.slots[0], j // 64]), h, j % 64])
            if p >= 128:
                assert bool(got[j, [h, 2 + h]].isnan().all()) and w == 0.0
            else:
                assert torch.equal(got[j, [h, 2 + h]], good[p, [h, 2 + h]])


# ---------------------------------------------------------------- workspaces
def peak(call):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("n_seqs,nq,nkv,bound", [(64, 64, 8, 32768), (200, 32, 8, 8192), (256, 16, 2, 32768), (3, 12, 1, 9000)])
def test_the_workspace_goes_by_the_parts(n_seqs, nq, nkv, bound):
    """Blocks that share the keys out make as many parts as there are blocks and pairs, whatever the bound of the lengths."""
    D = 64
    pages = ops.kv4_pages(4, nkv, D, DEV)
    table = torch.zeros((n_seqs, bound // 64 + 1), dtype=torch.int32, device=DEV)
    lens = [1 + 37 * i % 500 for i in range(n_seqs)]
    step = types.SimpleNamespace(slots=ints(*range(n_seqs)), kv_len=ints(*lens), cu_q=ints(*range(n_seqs + 1)), decode=True,
                                 max_kv_len=bound, q_lens=(1,) * n_seqs)
    q = torch.randn((n_seqs, nq, D), device=DEV).bfloat16()
    blocks, groups = ops.KV4_PER_SM * torch.cuda.get_device_properties(0).multi_processor_count, nkv * -(-nq // nkv // 8)
    call = lambda: ops.attention_kv4(q, pages, table, step=step, page=64, scale=0.1)
    call()
    most = (blocks + n_seqs * groups) * min(8, nq // nkv) * (D + 2) * 4 + q.nbytes + (1 << 20)
    assert peak(call) <= most


# ---------------------------------------------------------------- numbers without a bound
@pytest.mark.parametrize("n_rows", [1, 30])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_windows_and_bounds_beyond_32_bits(dtype, n_rows):
    """They are windows and bounds that reach everything."""
    c = Cache([300, 90], 2, 64, dtype, seed=7, weights=True)
    step, q = c.step([n_rows, n_rows]), queries(2 * n_rows, 8, 64, dtype, 0).to(DEV)
    call = lambda **seen: ops.attention_kv4(q, c.pages, c.table, step=step, page=64, scale=0.1, want_lse=True, **seen)
    want, want_lse = call()
    for seen in (dict(window=1 << 40), dict(window=(1 << 31) - 1), dict(window=20, keep_first=1 << 40), dict(chunk=1 << 40)):
        out, lse = call(**seen)
        # (another way through the kernel may add in another order: two results of which each is within half a unit)
        assert float((out.double() - want.double()).abs().max()) <= torch.finfo(dtype).eps * 4
        assert float((lse - want_lse).abs().max()) <= 2.0 ** -16
    step.max_kv_len = 1 << 40
    out, lse = call()
    assert float((out.double() - want.double()).abs().max()) <= torch.finfo(dtype).eps * 4
    if dtype == BF16:
        a, b = torch.zeros_like(c.weights), torch.zeros_like(c.weights)
        ops.kv4_weigh(q, lse, c.pages, a, c.table, step=step, page=64, scale=0.1, last=1 << 40)
        step.max_kv_len = 300
        ops.kv4_weigh(q, lse, c.pages, b, c.table, step=step, page=64, scale=0.1)
        assert torch.equal(a, b)
