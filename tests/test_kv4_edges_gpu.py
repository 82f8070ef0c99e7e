"""Where the operators on a 4-bit cache could go wrong: at the edges of what they are given."""
import pytest
import torch

from grout_b200.kernels import ops
from test_kv4_gpu import DEV, NAN, Cache, queries

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
