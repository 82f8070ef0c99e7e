"""The plain form of the 4-bit cache, and what its operators refuse, without a GPU."""
import types

import pytest
import torch

from grout_b200.kernels import ops
from plain import kv4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_code_is_cut_off_and_the_error_is_half_a_step(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn((40, 128), generator=g) * torch.logspace(-6, 6, 40)[:, None] + 3.0).to(dtype)
    c, s, m = kv4.quantise(x)
    raw = (x.double().unflatten(-1, (-1, 64)) - m.double()[..., None]) / s.double()[..., None]
    raw = torch.where(s[..., None] > 0, raw, torch.zeros_like(raw))      # (a group without a range: all of it is m)
    assert int(c.min()) >= 0 and int(c.max()) <= 15
    # the largest is at most 15 steps above the least: half a step and the quotient's rounding (2^-24 of 15)
    assert float((c.double().unflatten(-1, (-1, 64)) - raw).abs().max()) <= 0.5 + 15 * 2.0 ** -23
    off = (kv4.value(c, s, m).double() - x.double()).unflatten(-1, (-1, 64)).abs()
    assert bool((off <= s.double()[..., None] * (0.5 + 15 * 2.0 ** -23) + 2.0 ** -23 * x.double().abs().amax()).all())


def test_groups_that_are_not_held():
    x = torch.zeros((5, 64))
    x[0, 3], x[1, 4], x[2, 5] = float("nan"), float("inf"), float("-inf")
    x[3, 0], x[3, 1] = 3.3e38, -3.3e38
    x[4] = 0.1                                           # no range: every element is m, up to what bfloat16 holds
    c, s, m = kv4.quantise(x)
    y = kv4.value(c, s, m)
    assert bool(y[:4].isnan().all())
    assert float((y[4] - 0.1).abs().max()) <= 0.1 * 2.0 ** -7 / 15


def test_choice_by_weight():
    w = [5.0, 1.0, 1.0, 7.0, 1.0, float("nan"), 0.0, 3.0, 0.0, 0.0]
    assert kv4.choose(w, 10, 12, 2, 1) == list(range(10))
    assert kv4.choose(w, 10, 6, 2, 1) == [0, 3, 5, 7, 8, 9]
    assert kv4.choose(w, 10, 8, 2, 1) == [0, 1, 2, 3, 5, 7, 8, 9]
    assert kv4.choose(w, 10, 3, 2, 1) == [0, 8, 9]


def test_records():
    assert ops.kv4_record(64) == 1152 and ops.kv4_record(128) == 2304
    assert kv4.record(torch.randn((16, 64)), torch.randn((16, 64))).numel() == 1152
    assert ops.kv4_pages(3, 2, 128, "cpu").shape == (3, 2, 4, 2304)
    for D in (0, 16, 96, 192, 256):
        with pytest.raises(ops.KernelError):
            ops.kv4_record(D)


def test_there_is_no_cpu_path():
    pages = ops.kv4_pages(4, 2, 64, "cpu")
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    table = i(0, 1, 2, 3).view(2, 2)
    at = dict(token_seq=i(0), token_pos=i(0), slots=i(0), block_table=table, page=64)
    step = types.SimpleNamespace(slots=i(0), kv_len=i(1), cu_q=i(0, 1), token_seq=i(0), decode=True, max_kv_len=1, q_lens=(1,))
    weights = torch.zeros((4, 2, 64))
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16)
    for call in (lambda: ops.kv4_write(torch.zeros((1, 4, 64)), 2, 64, pages=pages, **at),
                 lambda: ops.kv4_read(pages, **at),
                 lambda: ops.attention_kv4(q, pages, table, step=step, page=64, scale=1.0),
                 lambda: ops.kv4_weigh(q, torch.zeros((1, 4)), pages, weights, table, step=step, page=64, scale=1.0),
                 lambda: ops.kv4_evict(pages, weights, table, slots=i(0), kv_len=i(1), page=64, keep=4, recent=1)):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()
