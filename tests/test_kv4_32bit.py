"""Attention in 32 bits over a 4-bit cache, held to what 32-bit arithmetic gives: the bound that the GPU's results have to
meet is one that a rounding of the queries, the probabilities, the keys and values or the result to 16 bits breaks."""
import math

import pytest
import torch

from grout_b200.kernels import ops
from plain import kv4

U = 2.0 ** -24                     # the most that one rounding takes off
SEEN = [dict(), dict(window=40, keep_first=5), dict(chunk=48), dict(softcap=15.0)]
# sequences' lengths and the rows of each that a step brings (0: one, as a step of single tokens)
SHAPES = [([2, 16, 17, 33, 64, 129], 0, 8, 2, 128), ([300, 5, 128], 0, 20, 4, 64), ([700, 33], 0, 17, 1, 128),
          ([1500, 40], 0, 4, 2, 64), ([130, 64], 40, 8, 2, 128), ([70, 190], 33, 12, 1, 64)]
SCALE = 0.6


def tokens(lens, nkv, D, seed):
    g = torch.Generator().manual_seed(seed)
    kv = torch.randn((sum(lens), 2 * nkv, D), generator=g)
    kv[:, :nkv, 3] += 4.0                                          # a channel that stands out
    return kv


def bound(q, k, v, s, m, scale, *, softcap=None, **seen):
    """(want, lse, tolerance, tolerance of lse) for q [rows, nq, D] over k, v [nkv, n, D] with the pairs s, m [nkv, n, groups]
    of the keys.

    A score is the sum over the groups of s (q . code) + (m + 8 s) (q's sum), codes around 0: every partial sum is at most
    A = scale sum_g (8 s + |m + 8 s|) |q|_1 in size.  Some 64 roundings of at most U A, independent of one another, add up to
    at most 8 U A at two times their spread or more; 8 U more for the power; the cap's tanh 2^-21 of the cap.  So a
    probability is off by a factor 1 + d_j, d_j independent: six times their spread in the result, sqrt(sum (p d (v - o))^2).
    What the keys have in common (the roundings of the query's sum, at most 3 U A) goes in with its size.  The sums over n
    keys round n times, independently, and the result once."""
    want, lse, p = kv4.attend(q, k, v, scale, softcap=softcap, **seen)
    nq, G = q.shape[1], q.shape[1] // k.shape[0]
    tol, tol_lse = torch.zeros_like(want), torch.zeros_like(lse)
    n = k.shape[1]
    for h in range(nq):
        sd, md, vd = s[h // G].double(), m[h // G].double(), v[h // G].double()
        size = q[:, h].double().abs().unflatten(-1, (-1, 64)).sum(-1)                     # [rows, groups]
        A = scale * size @ (8 * sd + (md + 8 * sd).abs()).T                               # [rows, n]
        d = 8 * U * A + 8 * U + (2.0 ** -21 * softcap if softcap else 0.0)
        far = (vd[None] - want[:, h, None]).abs()                                         # [rows, n, D]
        o, P = want[:, h].abs(), p[h][..., None]
        many = 2 * U * math.sqrt(n + 16)
        tol[:, h] = (6 * ((P * d[..., None] * far) ** 2).sum(1).sqrt() + (P * 3 * U * A[..., None] * far).sum(1)
                     + many * ((P * vd.abs()).sum(1) + o) + U * o + 1e-30)
        tol_lse[:, h] = (6 * ((p[h] * d) ** 2).sum(1).sqrt() + (p[h] * 3 * U * A).sum(1) + many + 4 * U * (1 + lse[:, h].abs()))
    return want, lse, tol, tol_lse


def case(lens, rows, nq, nkv, D, seed=0):
    kv = tokens(lens, nkv, D, seed)
    c, s, m = kv4.quantise(kv)
    held = kv4.value(c, s, m)
    q = torch.randn((sum(min(rows or 1, n) for n in lens), nq, D), generator=torch.Generator().manual_seed(100 + seed))
    at = a = 0
    parts = []
    for n in lens:
        r = min(rows or 1, n)
        x, xs, xm = (t[a:a + n].transpose(0, 1) for t in (held, s, m))
        parts.append((slice(at, at + r), q[at:at + r], x[:nkv], x[nkv:], xs[:nkv], xm[:nkv]))
        at, a = at + r, a + n
    return kv, q, parts


def plain32(q, k, v, scale, *, p_to=None, out_to=None, softcap=None, **seen):
    """The same in 32-bit tensor code, with roundings to a 16-bit type where asked for."""
    G = q.shape[1] // k.shape[0]
    see = kv4.mask(q.shape[0], k.shape[1], **seen)
    out = torch.zeros_like(q)
    for h in range(q.shape[1]):
        x = q[:, h] @ k[h // G].T * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        x = torch.where(see, x, torch.full_like(x, -math.inf))
        p = torch.exp(x - x.amax(1, keepdim=True))
        total = p.sum(1, keepdim=True)
        if p_to:
            p = p.to(p_to).float()
        out[:, h] = p @ v[h // G] / total
    return out.to(out_to).float() if out_to else out


@pytest.mark.parametrize("seen", SEEN, ids=str)
@pytest.mark.parametrize("lens,rows,nq,nkv,D", SHAPES)
def test_the_bound_tells_16_bits_from_32(lens, rows, nq, nkv, D, seen):
    scale, half = SCALE / math.sqrt(D), torch.bfloat16
    worst = {}
    for _at, q, k, v, s, m in case(lens, rows, nq, nkv, D)[2]:
        want, _lse, tol, _t = bound(q, k, v, s, m, scale, **seen)
        forms = dict(plain=plain32(q, k, v, scale, **seen), queries=plain32(q.to(half).float(), k, v, scale, **seen),
                     probabilities=plain32(q, k, v, scale, p_to=half, **seen),
                     keys=plain32(q, k.to(half).float(), v, scale, **seen), values=plain32(q, k, v.to(half).float(), scale, **seen),
                     result=plain32(q, k, v, scale, out_to=half, **seen))
        for name, got in forms.items():
            worst[name] = max(worst.get(name, 0.0), float(((got.double() - want).abs() / tol).max()))
    assert worst.pop("plain") <= 1.0
    assert all(x > 2.0 for x in worst.values()), worst


@pytest.mark.gpu
@pytest.mark.parametrize("stretches,way", [(None, None), (1, 0), (3, 0), (2, 2)])
@pytest.mark.parametrize("seen", SEEN, ids=str)
@pytest.mark.parametrize("lens,rows,nq,nkv,D", SHAPES)
def test_attention_in_32_bits(lens, rows, nq, nkv, D, seen, stretches, way, monkeypatch):
    from test_kv4_gpu import DEV, Cache
    monkeypatch.setattr(ops, "KV4_SPLIT_OVERRIDE", stretches)
    monkeypatch.setattr(ops, "KV4_SHARE_OVERRIDE", way)
    scale = SCALE / math.sqrt(D)
    kv, q, parts = case(lens, rows, nq, nkv, D)

    def edit(x):
        x.copy_(kv)
    c = Cache(lens, nkv, D, torch.float32, edit=edit)
    step = c.step([min(rows or 1, n) for n in lens])
    out, lse = ops.attention_kv4(q.to(DEV), c.pages, c.table, step=step, page=64, scale=scale, want_lse=True, **seen)
    for at, qi, k, v, s, m in parts:
        want, want_lse, tol, tol_lse = bound(qi, k, v, s, m, scale, **seen)
        off = (out[at].double().cpu() - want).abs()
        assert bool((off <= tol).all()), float((off / tol).max())
        off = (lse[at].double().cpu() - want_lse).abs()
        assert bool((off <= tol_lse).all()), float((off / tol_lse).max())
