"""What the speed of the operators on a 4-bit cache is measured on: writing and reading it, attention over it,
the weights that its tokens gather and the eviction that goes by them.

The cache is paged: a page has 64 tokens of every kv head, as four records of 16 tokens.  A record of heads of D
holds, one behind the other, the codes of 16 keys (D / 2 bytes each), the codes of 16 values, and for every token
the pairs (s, m) of its key's groups of 64 elements and of its value's, two bfloat16 each.  An element is s c + m,
c its code of 4 bits; m is the group's smallest value rounded down, s its range over 15 rounded up, so every
code is the nearest one and none is cut off.  Eight elements share a 32-bit word, the even ones in its low half;
the words of a row are in the order in which a kernel's threads take them (``_key_words``, ``_value_words``).

A pass is one call of an operator (with the read-back that shows its result where that is the cache itself)."""
import math
import random
import types

import torch

own = False

PAGE, GROUP = 64, 64
BF16, F32 = "bfloat16", "float32"


def listed():
    def case(name, kind, seqs, rows, longest, nq, nkv, D=128, dtype=BF16, mix=0, **more):
        return dict(dict(name=name, kind=kind, seqs=seqs, rows=rows, longest=longest, nq=nq, nkv=nkv, D=D, dtype=dtype,
                         mix=mix, window=0, cap=0.0, sinks=False, pad=0, keep=0, recent=0, first=0), **more)

    return [
        # a document of 2,048 tokens goes into the cache, one layer
        case("write-prompt", "write", 1, 2048, 2048, 32, 8),
        # a full server's decode step: 64 sequences bring a token each
        case("write-step", "write", 64, 1, 700, 32, 8, mix=1),
        # one user's short chat: the call whose latency counts
        case("decode-one", "decode", 1, 1, 300, 16, 8),
        # a full server with unequal contexts up to the default limit, some of the batch's rows padding
        case("decode-server", "decode", 60, 1, 4096, 32, 8, mix=2, pad=4),
        # two users with a book each, many query heads on a kv head
        case("decode-long", "decode", 2, 1, 32768, 64, 8),
        # the true 32-bit path, small heads
        case("decode-32bit", "decode", 4, 1, 1500, 16, 8, D=64, dtype=F32, mix=3),
        # reading one document of 2,048 tokens
        case("prompt", "prompt", 1, 2048, 2048, 32, 8),
        # prompts in chunks of up to 384 tokens behind what is there: windowed, capped scores with sinks, odd groups
        case("prompt-chunks", "prompt", 6, 384, 2500, 20, 4, D=64, mix=4, window=1024, cap=30.0, sinks=True),
        # a decode step that keeps account of what is attended to: one user, and a server
        case("weigh-one", "weigh", 1, 1, 1100, 32, 8),
        case("weigh-server", "weigh", 24, 1, 4096, 32, 8, mix=5),
        # one long sequence cut to half, and a batch cut to a quarter
        case("evict-one", "evict", 1, 1, 8192, 32, 8, keep=4096, recent=256, first=4),
        case("evict-batch", "evict", 16, 1, 4096, 16, 8, mix=6, keep=1024, recent=128, first=4),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))

    kind = rng.choice(["write", "decode", "decode", "prompt", "weigh", "evict"])
    D = rng.choice([64, 128, 128])
    nq, nkv = rng.choice([(16, 8), (32, 8), (64, 8), (20, 4), (8, 2), (5, 5), (12, 1), (28, 4)])
    case = dict(kind=kind, seqs=log(1, 64), rows=1, longest=log(1, 32768), nq=nq, nkv=nkv, D=D, dtype=BF16,
                mix=rng.randrange(1, 1 << 20), window=0, cap=0.0, sinks=False, pad=0, keep=0, recent=0, first=0)
    if kind == "write":
        case.update(rows=log(1, 2048), dtype=rng.choice([BF16, BF16, F32]))
        case["seqs"] = min(case["seqs"], max(1, 4096 // case["rows"]))
        case["longest"] = min(case["rows"] + log(1, 4096), 131072 // case["seqs"])
        case["rows"] = min(case["rows"], case["longest"])
        return case
    if kind in ("decode", "weigh"):
        case["longest"] = min(case["longest"], 131072 // case["seqs"])
        case.update(pad=rng.choice([0, 0, 3]))
        if kind == "decode" and rng.random() < 0.25:
            case.update(dtype=F32, longest=min(case["longest"], 4096), seqs=min(case["seqs"], 16))
    if kind == "prompt":
        case.update(seqs=log(1, 8), rows=log(2, 1500))
        case["longest"] = case["rows"] + log(1, 4000)
        most = (1 << 27) // (nq * case["rows"] * case["longest"])
        case["seqs"] = max(1, min(case["seqs"], most))
    if kind == "evict":
        case["longest"] = min(max(case["longest"], 8), 65536 // case["seqs"])
        keep = max(4, int(case["longest"] * rng.uniform(0.05, 0.9)))
        return dict(case, keep=keep, recent=rng.randrange(0, keep // 2 + 1), first=rng.randrange(0, min(5, keep // 2 + 1)))
    if rng.random() < 0.4:
        case.update(window=log(8, 4096))
    if rng.random() < 0.3:
        case.update(cap=rng.choice([15.0, 30.0, 50.0]))
    if rng.random() < 0.3:
        case.update(sinks=True)
    return case


# ---------------------------------------------------------------- sizes of a case
def _lens(case):
    """(rows that every sequence brings, tokens that it holds with them)."""
    n, rows, longest = case["seqs"], case["rows"], case["longest"]
    r = random.Random(case["mix"])
    if not case["mix"]:
        return [rows] * n, [longest] * n
    q = [rows] + [r.randint(max(1, rows // 3), rows) for _ in range(n - 1)]
    kv = [longest] + [r.randint(max(a, longest // 6), longest) for a in q[1:]]
    return q, kv


def _pairs(q, kv, window):
    """(query, visible key) pairs of one sequence, and the keys that some query sees."""
    if not window:
        return q * (kv - q) + q * (q + 1) // 2, kv
    pairs = sum(min(p + 1, window) for p in range(kv - q, kv))
    return pairs, min(kv, q + window - 1)


def work(case):
    q, kv = _lens(case)
    nq, nkv, D = case["nq"], case["nkv"], case["D"]
    el = 4 if case["dtype"] == F32 else 2
    token = nkv * (D + D // 8)                     # bytes of a token's keys and values in the cache
    if case["kind"] == "write":                    # rows in, records out, records in, values out
        return {"bytes": sum(q) * (2 * 2 * nkv * D * el + 2 * token), "flops": 0}
    if case["kind"] == "evict":                    # weights in and out, kept records in and out, read back in 16 bits
        kept = sum(min(n, case["keep"]) for n in kv)
        return {"bytes": sum(kv) * nkv * 4 + kept * (nkv * 8 + 2 * token) + kept * (token + 2 * nkv * D * 2), "flops": 0}
    pairs, seen = map(sum, zip(*(_pairs(a, b, case["window"]) for a, b in zip(q, kv))))
    nbytes = seen * token + 2 * sum(q) * nq * D * el
    if case["kind"] == "weigh":
        nbytes += sum(q) * nq * 4 + seen * nkv * 8
    return {"bytes": nbytes, "flops": 4 * nq * D * pairs}


# ---------------------------------------------------------------- the cache's format
_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)            # of the elements of a word


def _key_words(D, device):
    """Where word n of a key (elements 8 n .. 8 n + 7) stands among the words of its row."""
    n = torch.arange(D // 8, device=device)
    return (n % 4) * (D // 32) + n // 4


def _value_words(D, device):
    """The same for a value, by the token's place in its record: [16, D / 8]."""
    n = torch.arange(D // 8, device=device)[None]
    turn = (torch.arange(16, device=device)[:, None] // 2 % 2) * 4
    return ((n % 8) ^ turn) * (D // 64) + n // 8


def _quantise(x):
    """x [..., D] in 32 bits -> codes int32 [..., D], s and m float32 [..., D / 64] (values of bfloat16)."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    bits = lo.view(torch.int32)
    m = torch.where(bits < 0, bits + 0xFFFF, bits).bitwise_and(-0x10000).view(torch.float32)
    # (a quotient, not the product with 1 / 15 that a division by a number becomes: where it is exact it stays so)
    s = ((hi - m) / torch.full_like(m, 15)).view(torch.int32)
    s = (s + 0xFFFF).bitwise_and(-0x10000).view(torch.float32)
    c = torch.where(s[..., None] > 0, torch.round((g - m[..., None]) / s[..., None]), torch.zeros_like(g))
    return c.to(torch.int32).flatten(-2), s, m


def _pack(k, v):
    """Keys and values [..., 16, D] -> records uint8 [..., record]."""
    D = k.shape[-1]
    parts, pairs = [], []
    for x, words in ((k, _key_words(D, k.device).expand(16, -1)), (v, _value_words(D, k.device))):
        c, s, m = _quantise(x)
        shifts = torch.tensor(_SHIFTS, dtype=torch.int32, device=x.device)
        w = (c.unflatten(-1, (-1, 8)) << shifts).sum(-1, dtype=torch.int32)
        placed = torch.empty_like(w).scatter_(-1, words.expand_as(w), w)
        parts.append(placed.contiguous().view(torch.uint8).flatten(-2))
        pairs.append(torch.stack([s, m], -1).bfloat16())
    parts.append(torch.cat(pairs, -2).contiguous().view(torch.uint8).flatten(-3))
    return torch.cat(parts, -1)


def _unpack(records, D):
    """Records uint8 [..., record] -> keys and values float32 [..., 16, D]."""
    out = []
    pairs = records[..., 16 * D:].contiguous().view(torch.bfloat16).float()
    pairs = pairs.unflatten(-1, (16, 2, D // GROUP, 2))
    for i, words in enumerate((_key_words(D, records.device).expand(16, -1), _value_words(D, records.device))):
        w = records[..., i * 8 * D:(i + 1) * 8 * D].contiguous().view(torch.int32).unflatten(-1, (16, D // 8))
        w = torch.gather(w, -1, words.expand_as(w))
        shifts = torch.tensor(_SHIFTS, dtype=torch.int32, device=w.device)
        c = ((w[..., None] >> shifts) & 15).flatten(-2).float().unflatten(-1, (-1, GROUP))
        s, m = pairs[..., i, :, 0], pairs[..., i, :, 1]
        out.append((c * s[..., None] + m[..., None]).flatten(-2))
    return out


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    q_lens, kv_lens = _lens(case)
    n, nq, nkv, D = case["seqs"], case["nq"], case["nkv"], case["D"]
    dtype = getattr(torch, case["dtype"])
    # the order of the slots and of the pages is what a server's cache comes to after a while
    most = max((x + PAGE - 1) // PAGE for x in kv_lens)
    slots = torch.randperm(n + 3, generator=g, device=dev)[:n].to(torch.int32)
    n_pages = n * most + 1
    order = torch.randperm(n_pages - 1, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((n + 3, most), dtype=torch.int32, device=dev)
    table[slots.long()] = order.view(n, most)
    into = None
    if case["kind"] == "evict":                     # free pages that the kept tokens go to
        few = (case["keep"] + PAGE - 1) // PAGE
        into = torch.zeros((n + 3, few), dtype=torch.int32, device=dev)
        into[slots.long()] = (n_pages + torch.randperm(n * few, generator=g, device=dev).to(torch.int32)).view(n, few)
        n_pages += n * few
    # keys with a few strong channels and values around zero, as attention layers have them
    strong = 1.0 + 3.0 * (torch.rand((nkv, 1, 1, D), generator=g, device=dev) < 0.05)
    made = lambda: torch.randn((n_pages, nkv, 4, 16, D), generator=g, device=dev)
    if case["kind"] == "write":
        pages = torch.zeros((n_pages, nkv, 4, 16 * D + D // 2 * 4), dtype=torch.uint8, device=dev)
    else:
        pages = _pack(made() * strong, made())
    T = sum(q_lens)
    pad = case["pad"]
    state = types.SimpleNamespace(case=case, pages=pages, table=table, into=into)
    state.q = torch.randn((T + pad, nq, D), generator=g, device=dev).to(dtype)
    if case["kind"] == "write":
        kv = torch.randn((T, 2 * nkv, D), generator=g, device=dev)
        kv[:, :nkv] *= strong[:, 0, 0]
        state.kv = kv.to(dtype)
    if case["kind"] in ("weigh", "evict"):           # gathered so far; the newest tokens have none yet
        w = torch.empty((n_pages, nkv, PAGE), device=dev).exponential_(1.0, generator=g) ** 2
        state.weights = torch.where(torch.rand(w.shape, generator=g, device=dev) < 0.05, torch.zeros_like(w), w)
    state.sinks = torch.randn((nq,), generator=g, device=dev) if case["sinks"] else None
    state.scale = 1.0 / math.sqrt(D)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    starts = [b - a for a, b in zip(q_lens, kv_lens)]
    q_all = q_lens + [1] * pad
    cu = [0]
    for a in q_all:
        cu.append(cu[-1] + a)
    state.step = types.SimpleNamespace(
        n_tokens=T + pad, n_seqs=n + pad, slots=torch.cat([slots, ints([-1] * pad)]), kv_len=ints(kv_lens + [1] * pad),
        token_seq=torch.repeat_interleave(torch.arange(n + pad, device=dev), ints(q_all).long()).to(torch.int32),
        token_pos=torch.cat([torch.arange(s, s + a, device=dev) for s, a in zip(starts + [0] * pad, q_all)]).to(torch.int32),
        cu_q=ints(cu), decode=case["rows"] == 1, max_q_len=max(q_all), max_kv_len=max(kv_lens), q_lens=tuple(q_all))
    if case["kind"] == "evict":                      # where the kept tokens are read back
        kept = [min(x, case["keep"]) for x in kv_lens]
        state.kept_seq = torch.repeat_interleave(torch.arange(n, device=dev), ints(kept).long()).to(torch.int32)
        state.kept_pos = torch.cat([torch.arange(x, device=dev) for x in kept]).to(torch.int32)
    return state


# ---------------------------------------------------------------- the operators in their plain form
def _sequences(state):
    """Keys and values [seqs, tokens, nkv, D] of the step's sequences (what padding rows get is masked)."""
    step = state.step
    pages = state.pages[state.table[step.slots.clamp(min=0).long()].long()]   # [seqs, pages, nkv, 4, record]
    k, v = _unpack(pages, state.case["D"])                                   # [seqs, pages, nkv, 4, 16, D]
    join = lambda x: x.permute(0, 1, 3, 4, 2, 5).flatten(1, 3)
    return join(k), join(v)


def _scores(state, k):
    """Scores [seqs, nkv, heads of a kv head, rows, keys] with -inf where a query does not see a key; and where its
    rows stand among the step's: [seqs, rows], with the truth of each."""
    case, step = state.case, state.step
    nkv, G = case["nkv"], case["nq"] // case["nkv"]
    n = step.cu_q[1:] - step.cu_q[:-1]
    at = torch.arange(step.max_q_len, device=n.device)[None]
    real = at < n[:, None]
    rows = torch.where(real, step.cu_q[:-1, None] + at, torch.zeros_like(at)).long()
    pos = (step.kv_len - n)[:, None] + at
    q = state.q.float()[rows].unflatten(2, (nkv, G))                          # [seqs, rows, nkv, G, D]
    s = torch.einsum("brngd,bknd->bngrk", q, k) * state.scale
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    key = torch.arange(k.shape[1], device=n.device)
    seen = (key <= pos[..., None]) & real[..., None] & (step.slots >= 0)[:, None, None]
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    return s.masked_fill(~seen[:, None, None], -math.inf), rows, real


def _attend(state):
    """The heads' outputs [tokens, nq, D], the logarithm of every softmax's sum, and its terms over the sum."""
    case = state.case
    k, v = _sequences(state)
    s, rows, real = _scores(state, k)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    if state.sinks is not None:
        sink = state.sinks.view(case["nkv"], -1)[None, :, :, None, None]
        top = torch.maximum(top, sink)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    if state.sinks is not None:
        total = total + torch.exp(sink - top)
    p = e / total.clamp(min=1e-30)
    o = torch.einsum("bngrk,bknd->brngd", p, v).flatten(2, 3)
    lse = (torch.log(total) + top)[..., 0].permute(0, 3, 1, 2).flatten(2)     # [seqs, rows, nq]
    lse = lse.masked_fill((state.step.slots < 0)[:, None, None], -math.inf)
    out = torch.empty(state.q.shape, dtype=torch.float32, device=k.device)
    out[rows[real]] = o[real]
    sums = torch.empty(state.q.shape[:2], dtype=torch.float32, device=k.device)
    sums[rows[real]] = lse[real]
    return out.to(state.q.dtype), sums, p


def _token_weights(state, weights):
    """The weights of the step's sequences by token: [seqs, nkv, tokens], and where they stand."""
    at = state.table[state.step.slots.clamp(min=0).long()].long()
    return weights[at].permute(0, 2, 1, 3).flatten(2), at


def _plain(state):
    case, step = state.case, state.step
    kind = case["kind"]
    if kind == "write":
        c, s, m = _quantise(state.kv)
        x = c.float().unflatten(-1, (-1, GROUP)) * s[..., None] + m[..., None]
        return x.flatten(-2).to(state.kv.dtype)
    if kind in ("decode", "prompt"):
        return _attend(state)[0]
    if kind == "weigh":
        out, lse, p = _attend(state)
        add = p.sum((2, 3)).unflatten(2, (-1, PAGE)).permute(0, 2, 1, 3)     # [seqs, pages, nkv, 64]
        live = step.slots >= 0
        at = state.table[step.slots.clamp(min=0).long()].long()
        state.weights.index_add_(0, at[live].flatten(), add[live].flatten(0, 1))
        return {"out": out, "lse": lse, "weights": state.weights}
    # eviction: the first, the newest and the heaviest, in the order that they stand in
    w, at = _token_weights(state, state.weights)
    place = torch.arange(w.shape[-1], device=w.device)
    n = step.kv_len[:, None, None]
    rank = torch.where((place < case["first"]) | (place >= n - case["recent"]), torch.full_like(w, math.inf), w)
    rank = torch.where(place < n, rank, torch.full_like(w, -math.inf))
    few = min(case["keep"], w.shape[-1])
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :few]
    best = torch.where(best < n, best, torch.full_like(best, w.shape[-1])).sort(-1).values
    valid = best < w.shape[-1]
    kept = torch.full((*w.shape[:2], case["keep"]), -1, dtype=torch.int32, device=w.device)
    kept[..., :few] = torch.where(valid, best, torch.full_like(best, -1))
    best = best.clamp(max=w.shape[-1] - 1)
    k, v = _sequences(state)                                                  # [seqs, tokens, nkv, D]
    pick = best.transpose(1, 2)[..., None].expand(-1, -1, -1, case["D"])
    kv = torch.cat([torch.gather(k, 1, pick), torch.gather(v, 1, pick)], 2)[valid[:, 0]]
    to = state.into[step.slots.long()].long()                                 # [seqs, pages]
    page, spot = to[:, torch.arange(few, device=w.device) // PAGE], torch.arange(few, device=w.device) % PAGE
    heads = torch.arange(case["nkv"], device=w.device)[None, :, None]
    where = (page[:, None].expand_as(valid)[valid], heads.expand_as(valid)[valid], spot.expand_as(valid)[valid])
    state.weights.index_put_(where, torch.gather(w, 2, best)[valid])
    return {"kept": kept, "kv": kv.to(torch.bfloat16), "weights": state.weights}


def run(state):
    if not own:
        return _plain(state)
    from grout_b200.kernels import ops
    case, step = state.case, state.step
    kind = case["kind"]
    at = dict(token_seq=step.token_seq, token_pos=step.token_pos, slots=step.slots, block_table=state.table, page=PAGE)
    if kind == "write":
        ops.kv4_write(state.kv, case["nkv"], case["D"], pages=state.pages, **at)
        return ops.kv4_read(state.pages, dtype=state.kv.dtype, **at)
    if kind == "evict":
        kept, _len = ops.kv4_evict(state.pages, state.weights, state.table, slots=step.slots, kv_len=step.kv_len,
                                   page=PAGE, keep=case["keep"], recent=case["recent"], first=case["first"],
                                   into=state.into)
        kv = ops.kv4_read(state.pages, dtype=torch.bfloat16, token_seq=state.kept_seq, token_pos=state.kept_pos,
                          slots=step.slots, block_table=state.into, page=PAGE)
        return {"kept": kept, "kv": kv, "weights": state.weights}
    seen = dict(step=step, page=PAGE, scale=state.scale, window=case["window"] or None, softcap=case["cap"] or None)
    if kind in ("decode", "prompt"):
        return ops.attention_kv4(state.q, state.pages, state.table, sinks=state.sinks, **seen)
    out, lse = ops.attention_kv4(state.q, state.pages, state.table, sinks=state.sinks, want_lse=True, **seen)
    ops.kv4_weigh(state.q, lse, state.pages, state.weights, state.table, **seen)
    return {"out": out, "lse": lse, "weights": state.weights}


# ---------------------------------------------------------------- in 64 bits, sequence by sequence
def _read64(pages, D):
    """Pages [pages, nkv, 4, record] of one sequence -> keys and values float64 [nkv, tokens, D], byte by byte."""
    P, nkv = pages.shape[:2]
    dev = pages.device
    out = []
    d = torch.arange(D, device=dev)
    byte, high = d % 8 // 4 + 2 * (d % 2), d % 4 // 2
    tok = torch.arange(16, device=dev)[:, None]
    for i in range(2):
        rows = pages[..., i * 8 * D:(i + 1) * 8 * D].reshape(P, nkv, 4, 16, D // 2)
        word = d // 8
        if i == 0:
            place = (word % 4 * (D // 32) + word // 4).expand(16, -1)
        else:
            place = (word % 8 ^ (tok // 2 % 2 * 4)) * (D // 64) + word // 8
        b = torch.gather(rows, -1, (place * 4 + byte).expand(P, nkv, 4, 16, D)).long()
        c = torch.where(high.bool(), b // 16, b % 16).double()
        sm = pages[..., 16 * D:].contiguous().view(torch.bfloat16).double().reshape(P, nkv, 4, 16, 2, D // 64, 2)
        s, m = sm[..., i, :, 0][..., d // 64], sm[..., i, :, 1][..., d // 64]
        out.append((s * c + m).permute(1, 0, 2, 3, 4).reshape(nkv, P * 64, D))
    return out


def _quantised64(x):
    """The values that the cache holds for x, with the definition's real numbers rounded to bfloat16 up and down."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values

    def step(v):       # the spacing of bfloat16 around v, exactly
        e = v.abs().float().view(torch.int32) >> 23
        return ((e - 7).clamp(min=1) << 23).view(torch.float32).double()

    m = torch.floor(lo / step(lo)) * step(lo)
    s = (hi - m) / 15
    s = torch.ceil(s / step(s)) * step(s)
    c = torch.where(s > 0, torch.round((g - m) / s.clamp(min=1e-300)), torch.zeros_like(g))
    return (s * c + m).reshape(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    step, nkv, G, D = state.step, case["nkv"], case["nq"] // case["nkv"], case["D"]
    kind = case["kind"]
    if kind == "write":
        return _quantised64(state.kv)
    cu, lens, slots = step.cu_q.tolist(), step.kv_len.tolist(), step.slots.tolist()
    if kind == "evict":
        weights, kvs = state.weights.double(), []
        for n, slot in zip(lens, slots):
            pages = (n + PAGE - 1) // PAGE
            at, keep = state.table[slot, :pages].long(), min(n, case["keep"])
            k, v = _read64(state.pages[at], D)
            k, v = k[:, :n], v[:, :n]
            w = weights[at].transpose(0, 1).reshape(nkv, -1)[:, :n].clone()
            w[:, :case["first"]] = math.inf
            w[:, max(0, n - case["recent"]):] = math.inf
            order = torch.argsort(-w, dim=-1, stable=True)[:, :keep].sort(-1).values
            plain = weights[at].transpose(0, 1).reshape(nkv, -1)
            rows = []
            for h in range(nkv):
                to = torch.arange(keep, device=w.device)
                weights[state.into[slot].long()[to // PAGE], h, to % PAGE] = plain[h, order[h]]
                rows.append((k[h, order[h]], v[h, order[h]]))
            kvs.append(torch.stack([r[0] for r in rows] + [r[1] for r in rows], 1))
        return {"kept": None, "kv": torch.cat(kvs), "weights": weights}
    out = torch.zeros(state.q.shape, dtype=torch.float64, device=state.q.device)
    lse = torch.full(state.q.shape[:2], -math.inf, dtype=torch.float64, device=state.q.device)
    weights = state.weights.double() if kind == "weigh" else None
    for i, slot in enumerate(slots):
        if slot < 0:
            continue
        n, a, b = lens[i], cu[i], cu[i + 1]
        at = state.table[slot, :(n + PAGE - 1) // PAGE].long()
        k, v = _read64(state.pages[at], D)
        pos = torch.arange(n - (b - a), n, device=k.device)[:, None]
        key = torch.arange(n, device=k.device)[None]
        hidden = key > pos
        if case["window"]:
            hidden |= key <= pos - case["window"]
        for h in range(case["nq"]):
            s = state.q[a:b, h].double() @ k[h // G, :n].T * state.scale
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            s = s.masked_fill(hidden, -math.inf)
            if state.sinks is not None:
                s = torch.cat([s, state.sinks[h].double().expand(b - a, 1)], 1)
            lse[a:b, h] = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)[:, :n]
            out[a:b, h] = p @ v[h // G, :n]
            if weights is not None:
                spot = torch.arange(n, device=k.device)
                weights[at[spot // PAGE], h // G, spot % PAGE] += p.sum(0)
    if kind == "weigh":
        return {"out": out, "lse": lse, "weights": weights}
    return out
