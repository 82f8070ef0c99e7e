"""The 4-bit cache in plain tensor code, from its definition: what keys and values become, the bytes of a record,
attention over them in 64 bits, the weights that tokens gather and the eviction that goes by them."""
import math

import torch

PAGE, TOKENS, GROUP = 64, 16, 64


def _down(x):
    """x rounded down to bfloat16 (float32 in and out)."""
    y = x.to(torch.bfloat16)
    over = y.float() > x
    bits = y.view(torch.int16).int()
    # one step towards minus infinity in the order of the numbers
    lower = torch.where(bits < 0, bits + 1, torch.where(bits == 0, torch.full_like(bits, -0x7FFF), bits - 1))
    return torch.where(over, lower, bits).to(torch.int16).view(torch.bfloat16).float()


def quantise(x):
    """x [..., D] -> (codes int64 [..., D], s, m float32 [..., D / 64]); NaN pairs where a group is not held."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    m = _down(lo)
    s = -_down(-((hi - m) / torch.full_like(m, 15.0)))
    d = g - m[..., None]                          # rounded to 32 bits; then the nearest code, of two the even one
    c = torch.where(s[..., None] > 0, torch.round(d.double() / s.double()[..., None]), torch.zeros_like(g, dtype=torch.float64))
    bad = ~(g.isfinite().all(-1) & s.isfinite() & m.isfinite())
    nan = torch.full_like(s, float("nan"))
    c = torch.where(bad[..., None], torch.zeros_like(c), c)
    return c.long().flatten(-2), torch.where(bad, nan, s), torch.where(bad, nan, m)


def value(c, s, m):
    """What codes stand for, 32-bit (s c is exact there)."""
    g = c.float().unflatten(-1, (-1, GROUP))
    return (g.double() * s.double()[..., None] + m.double()[..., None]).float().flatten(-2)


def record(k, v):
    """Keys and values [16, D] -> the bytes of their record, uint8 [18 D]."""
    D = k.shape[-1]
    out = torch.zeros(18 * D, dtype=torch.uint8)
    pairs = torch.zeros((TOKENS, 2, D // GROUP, 2), dtype=torch.bfloat16)
    for which, x in enumerate((k, v)):
        c, s, m = quantise(x)
        pairs[:, which, :, 0], pairs[:, which, :, 1] = s.bfloat16(), m.bfloat16()
        for tok in range(TOKENS):
            for n in range(D // 8):
                if which == 0:
                    place = n % 4 * (D // 32) + n // 4
                else:
                    place = ((n % 8) ^ (4 if tok % 4 >= 2 else 0)) * (D // 64) + n // 8
                word = 0
                for e in range(8):
                    word |= int(c[tok, 8 * n + e]) << (4 * (e // 2) + 16 * (e % 2))
                at = which * 8 * D + tok * (D // 2) + 4 * place
                out[at:at + 4] = torch.tensor(list(word.to_bytes(4, "little")), dtype=torch.uint8)
    out[16 * D:] = pairs.view(torch.uint8).flatten()
    return out


def visible(pos, key, window=None, keep_first=0, chunk=0):
    """Whether a query at `pos` sees the key at `key`."""
    if key > pos:
        return False
    if window and key <= pos - window and key >= keep_first:
        return False
    return not (chunk and key // chunk != pos // chunk)


def mask(n_rows, n, window=None, keep_first=0, chunk=0):
    """[n_rows, n] for the last n_rows positions of n."""
    pos, key = torch.arange(n - n_rows, n)[:, None], torch.arange(n)[None]
    see = key <= pos
    if window:
        see &= (key > pos - window) | (key < keep_first)
    if chunk:
        see &= key // chunk == pos // chunk
    return see


def attend(q, k, v, scale, *, softcap=None, sinks=None, **seen):
    """q [rows, nq, D] of one sequence's last rows over k, v [nkv, n, D], in 64 bits: (out, lse, p [nq, rows, n])."""
    q, k, v = q.double(), k.double(), v.double()
    rows, nq, _D = q.shape
    G = nq // k.shape[0]
    see = mask(rows, k.shape[1], **seen)
    out, lse, ps = torch.zeros_like(q), torch.full((rows, nq), -math.inf, dtype=torch.float64), []
    for h in range(nq):
        s = q[:, h] @ k[h // G].T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        if sinks is not None:
            s = torch.cat([s, sinks[h].double().expand(rows, 1)], 1)
        lse[:, h] = torch.logsumexp(s, 1)
        p = torch.softmax(s, 1)[:, :k.shape[1]]
        p = torch.where(see, p, torch.zeros_like(p))
        # a key that is not seen has no part, whatever its value is
        out[:, h] = torch.where(see[..., None], p[..., None] * v[h // G][None], torch.zeros((), dtype=torch.float64)).sum(1)
        ps.append(p)
    return out, lse, torch.stack(ps)


def choose(weights, n, keep, recent, first):
    """The places that are kept of n tokens with the given weights (float, one head)."""
    if n <= keep:
        return list(range(n))
    sure = set(range(first)) | set(range(n - recent, n))
    rank = lambda i: (0 if weights[i] != weights[i] else 1, -weights[i] if weights[i] == weights[i] else 0, i)
    others = sorted((i for i in range(n) if i not in sure), key=rank)
    return sorted(sure | set(others[:keep - len(sure)]))
