"""Cases of the text-transformer operators: packed prompt attention, the paged key-value cache
(written, quantised on the way, and read back) and the attention of one new token over it.

`run` computes a case either with elementary torch operations (`own` false) or with the calls a
user makes of mold_b200 (`own` true), on the same inputs. Lengths of a batch are drawn from the
case's own numbers, so `work` knows them; values come from the seed.
"""
import math
import random

import torch

own = False

LARGEST = {"bytes": 8e8, "flops": 5.5e11}  # no drawn case costs more than the largest listed ones

CODES = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # A handful of image prompts on their way through a text encoder: latency counts.
        dict(name="prompt_few", op="prompt", n=4, low=19, high=77, past=0, heads=28, kv_heads=4, dim=128, causal=True,
             mix=1),
        # A serving batch of prompts of very different lengths, packed without padding.
        dict(name="prompt_ragged", op="prompt", n=24, low=32, high=2048, past=0, heads=32, kv_heads=8, dim=128,
             causal=True, mix=2),
        # One long prompt of odd length.
        dict(name="prompt_long", op="prompt", n=1, low=8201, high=8201, past=0, heads=32, kv_heads=8, dim=128,
             causal=True, mix=3),
        # The next piece of prompts whose beginnings are already cached.
        dict(name="prompt_chunk", op="prompt", n=3, low=300, high=1024, past=5000, heads=28, kv_heads=4, dim=128,
             causal=True, mix=4),
        # An encoder without a causal mask, one key head for each query head, heads of 64.
        dict(name="prompt_both_ways", op="prompt", n=16, low=40, high=512, past=0, heads=32, kv_heads=32, dim=64,
             causal=False, mix=5),
        # One generation step's new keys and values, short sequences.
        dict(name="cache_step", op="cache", codes="bf16", n=32, low=1, high=1, past=64, kv_heads=4, dim=128, page=16,
             mix=6),
        # Pieces of prompts written as int8 and read back for the next piece's attention.
        dict(name="cache_chunk_int8", op="cache", codes="int8", n=8, low=1000, high=2048, past=4096, kv_heads=8,
             dim=128, page=64, mix=7),
        # Many middling prompts, fp8, heads of 64.
        dict(name="cache_chunk_e4m3", op="cache", codes="e4m3", n=40, low=17, high=1500, past=700, kv_heads=8, dim=64,
             page=32, mix=8),
        # One user, a short conversation: latency counts.
        dict(name="token_one", op="token", codes="bf16", n=1, low=700, high=700, heads=28, kv_heads=4, dim=128,
             page=16, mix=9),
        # A serving batch with lengths far apart.
        dict(name="token_batch", op="token", codes="bf16", n=64, low=64, high=4096, heads=32, kv_heads=8, dim=128,
             page=64, mix=10),
        # Two very long contexts: the work has to be split along the length.
        dict(name="token_long", op="token", codes="int8", n=2, low=100001, high=131072, heads=32, kv_heads=8, dim=128,
             page=128, mix=11),
        # A full server.
        dict(name="token_many", op="token", codes="e4m3", n=160, low=256, high=8192, heads=64, kv_heads=8, dim=128,
             page=32, mix=12),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(["prompt", "cache", "token"])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 16])
        group = rng.choice([1, 2, 3, 4, 6, 7, 8, 12])
        dim = rng.choice([64, 128, 128])
        mix = rng.randrange(1, 1 << 20)
        if op == "prompt":
            n, high = _log(rng, 1, 64), _log(rng, 4, 8000)
            case = dict(op=op, n=n, low=_log(rng, 1, high), high=high, past=rng.choice([0, 0, _log(rng, 1, 6000)]),
                        heads=kv_heads * group, kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.75, mix=mix)
        elif op == "cache":
            n, high = _log(rng, 1, 128), rng.choice([1, _log(rng, 2, 4000)])
            case = dict(op=op, codes=rng.choice(list(CODES)), n=n, low=_log(rng, 1, high), high=high,
                        past=_log(rng, 1, 6000), kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]),
                        mix=mix)
        else:
            n, high = _log(rng, 1, 256), _log(rng, 8, 130000)
            case = dict(op=op, codes=rng.choice(list(CODES)), n=n, low=_log(rng, 1, high), high=high,
                        heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]),
                        mix=mix)
        w = work(case)
        # the plain forms pad a batch to its longest sequence, in 32 bits
        padded = case["n"] * case["high"] * kv_heads * dim * 4 if op == "token" else 0
        if case["heads" if op == "prompt" else "kv_heads"] <= 64 and padded <= 6e9 and all(
                w[k] <= LARGEST[k] for k in w) and (op != "prompt" or _pairs_padded(case) <= 3e9):
            return case


def _pairs_padded(case):
    return (case["high"] + case["past"]) * case["high"] * case["heads"]


def _lengths(case):
    """(new tokens, all tokens) of each sequence; the last one has the largest new length."""
    r = random.Random(case["mix"])
    new = [_log(r, case["low"], case["high"]) for _ in range(case["n"] - 1)] + [case["high"]]
    past = case.get("past", 0)
    return new, [m + (r.randint(0, past) if past else 0) for m in new]


def work(case):
    new, full = _lengths(case)
    kv, d = case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        # each query row against the keys its mask leaves: two products of d multiply-adds a pair
        pairs = sum(m * n - (m * (m - 1) // 2 if case["causal"] else 0) for m, n in zip(new, full))
        return {"bytes": 2.0 * d * (2 * case["heads"] * sum(new) + 2 * kv * sum(full)),
                "flops": 4.0 * d * case["heads"] * pairs}
    row = 2.0 * d if case["codes"] == "bf16" else d + 4.0
    if case["op"] == "cache":
        # new rows in and their codes out; every row's codes in and its values out
        return {"bytes": 2.0 * kv * (sum(new) * (2 * d + row) + sum(full) * (row + 2 * d)), "flops": 0.0}
    return {"bytes": 2.0 * kv * row * sum(new) + 4.0 * case["heads"] * d * case["n"],
            "flops": 4.0 * d * case["heads"] * sum(new)}


# ---------------------------------------------------------------- inputs

def _sum_up(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _values(shape, g, spread=None):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    return x if spread is None else x * spread


def _channels(kv, d, g):
    """Keys of trained models have a few channels far larger than the others."""
    s = torch.ones((kv, d), device="cuda", dtype=torch.bfloat16)
    s[:, torch.randperm(d, generator=g, device="cuda")[:3]] = 5.0
    return s


def _encode(x, codes):
    """Codes and scales of rows x [..., d]. A row's scale is its largest magnitude over the type's, in 32 bits; a
    value's code is the one nearest to its 32-bit product with the inverse; a row below 2^-100 is all zeros."""
    if codes == "bf16":
        return x, None
    x = x.float()
    top = x.abs().amax(-1)
    most = torch.full_like(top, TOP[codes])
    some = top >= 2.0 ** -100
    y = x * torch.where(some, most / top, 0.0)[..., None]
    y = y.round().clamp(-127, 127) if codes == "int8" else y.clamp(-448, 448)
    return y.to(CODES[codes]), torch.where(some, top / most, 0.0)


def _pool(case, n_pages, spread, g):
    """Page pools of keys and values [pages, kv heads, page, d], every row of them in use at some time."""
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    got = {}
    for name in ("k", "v"):
        codes = torch.empty(shape, device="cuda", dtype=CODES[case["codes"]])
        scale = None if case["codes"] == "bf16" else torch.empty(shape[:3], device="cuda")
        step = max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))
        for i in range(0, n_pages, step):
            m = min(step, n_pages - i)
            x = _values((m,) + shape[1:], g, spread[:, None] if name == "k" else None)
            c, s = _encode(x, case["codes"])
            codes[i:i + m] = c
            if scale is not None:
                scale[i:i + m] = s
        got[name], got[name + "_scale"] = codes, scale
    return got


def _tables(case, full, g):
    """Pages of each sequence, in no order, and a few pages of the pool that nobody has."""
    need = [-(-n // case["page"]) for n in full]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["n"], max(need)), device="cuda", dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    return table, sum(need) + 3


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["mix"])
    new, full = _lengths(case)
    kv, d = case["kv_heads"], case["dim"]
    ints = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
    state = {"case": case, "new": new, "full": full}
    spread = _channels(kv, d, g)
    if case["op"] == "prompt":
        state["q"] = _values((sum(new), case["heads"], d), g, 1.5)
        state["k"] = _values((sum(full), kv, d), g, spread)
        state["v"] = _values((sum(full), kv, d), g)
        state["cu_q"], state["cu_k"] = ints(_sum_up(new)), ints(_sum_up(full))
        return state
    state["table"], n_pages = _tables(case, full, g)
    state["pool"] = _pool(case, n_pages, spread, g)
    state["lens"] = ints(full)
    if case["op"] == "token":
        state["q"] = _values((case["n"], case["heads"], d), g, 1.5)
        return state
    # new rows as a fused projection leaves them: key heads, then value heads, in one row
    rows = _values((sum(new), 2 * kv, d), g)
    rows[:, :kv] *= spread
    state["k"], state["v"] = rows[:, :kv], rows[:, kv:]
    state["cu_new"], state["cu"] = ints(_sum_up(new)), ints(_sum_up(full))
    return state


# ---------------------------------------------------------------- plain forms

def _prompt(s):
    """softmax(q k^T / sqrt(d)) v of each sequence, query i at the end of its keys."""
    case, outs, a, c = s["case"], [], 0, 0
    group = case["heads"] // case["kv_heads"]
    for m, n in zip(s["new"], s["full"]):
        q = s["q"][a:a + m].float().transpose(0, 1).reshape(case["kv_heads"], group * m, -1)
        k, v = (s[x][c:c + n].float().transpose(0, 1) for x in "kv")
        p = torch.matmul(q, k.transpose(1, 2)).mul_(case["dim"] ** -0.5).view(-1, m, n)
        if case["causal"]:
            p.masked_fill_(torch.ones(m, n, device=p.device, dtype=torch.bool).triu_(n - m + 1), -math.inf)
        p = p.sub_(p.amax(-1, keepdim=True)).exp_()
        total = p.sum(-1)
        o = torch.matmul(p.view(case["kv_heads"], group * m, n), v).view(case["heads"], m, -1)
        outs.append((o / total[..., None]).transpose(0, 1))
        a, c = a + m, c + n
    return torch.cat(outs).to(torch.bfloat16)


def _rows(s, cu, first):
    """Pool places (page, offset) of the tokens that cu packs; first: each sequence's first position."""
    t = torch.arange(sum(s["new"]) if cu is s["cu_new"] else sum(s["full"]), device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu[1:], t, right=True)
    pos = (t - cu[b] + first[b]).long()
    page = s["case"]["page"]
    return s["table"][b, pos // page].long(), pos % page


def _bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _cache(s):
    codes, pool = s["case"]["codes"], s["pool"]
    page, at = _rows(s, s["cu_new"], s["lens"] - (s["cu_new"][1:] - s["cu_new"][:-1]))
    for x in "kv":
        c, scale = _encode(s[x], codes)
        _bits(pool[x])[page, :, at] = _bits(c)
        if scale is not None:
            pool[x + "_scale"][page, :, at] = scale
    page, at = _rows(s, s["cu"], torch.zeros_like(s["lens"]))
    out = []
    for x in "kv":
        y = _bits(pool[x])[page, :, at].view(pool[x].dtype).float()
        if codes != "bf16":
            y = y * pool[x + "_scale"][page, :, at][..., None]
        out.append(y.to(torch.bfloat16))
    return out


def _token(s):
    case, pool = s["case"], s["pool"]
    b, kv, d = case["n"], case["kv_heads"], case["dim"]
    got = []
    for x in "kv":
        y = _bits(pool[x])[s["table"].long()].view(pool[x].dtype).float()  # [b, pages, kv, page, d]
        if case["codes"] != "bf16":
            y = y * pool[x + "_scale"][s["table"].long()][..., None]
        got.append(y.transpose(1, 2).reshape(b, kv, -1, d))
    k, v = got
    q = s["q"].float().view(b, kv, -1, d)
    p = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    out = torch.arange(k.shape[2], device="cuda")[None] >= s["lens"][:, None]
    p = p.masked_fill_(out[:, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    o = torch.matmul(p, v.masked_fill_(out[:, None, :, None], 0.0)) / p.sum(-1, keepdim=True)
    return o.view(b, -1, d).to(torch.bfloat16)


# ---------------------------------------------------------------- the framework's calls

def _handle(s):
    """The cache handle, which a program makes once over its page pools and keeps."""
    import mold_b200 as mb
    if "cache" not in s:
        p = s["pool"]
        s["cache"] = mb.KVCache.from_tensors(p["k"], p["v"], p["k_scale"], p["v_scale"])
    return s["cache"]


def _own(s):
    import mold_b200 as mb
    op = s["case"]["op"]
    if op == "prompt":
        return mb.attention_varlen(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"])
    cache = _handle(s)
    if op == "token":
        return mb.attention_paged(s["q"], cache, s["table"], s["lens"])
    cache.write(s["k"], s["v"], s["table"], s["lens"], cu=s["cu_new"])
    return cache.read(s["table"], s["cu"], sum(s["full"]))


def run(state):
    if own:
        return _own(state)
    return {"prompt": _prompt, "cache": _cache, "token": _token}[state["case"]["op"]](state)


# ---------------------------------------------------------------- 64 bits

def _softmax64(scores, keep):
    e = torch.where(keep, scores, torch.tensor(-math.inf, dtype=torch.float64, device=scores.device))
    e = torch.exp(e - e.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


def _nearest64(y, codes):
    """The type's value nearest to y, ties to the even code."""
    if codes == "int8":
        return torch.round(y).clamp(-127, 127)
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _decoded64(s, name, b):
    """Sequence b's cached rows [kv heads, length, d] as numbers."""
    n, page = s["full"][b], s["case"]["page"]
    pages = s["table"][b, :-(-n // page)].long()
    y = _bits(s["pool"][name])[pages].view(s["pool"][name].dtype).to(torch.float64)
    if s["pool"][name + "_scale"] is not None:
        y = y * s["pool"][name + "_scale"][pages].double().unsqueeze(-1)
    return y.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    d, kv = case["dim"], case["kv_heads"]
    rows = []
    if case["op"] == "prompt":
        qs, ks, vs = (x.double() for x in (s["q"], s["k"], s["v"]))
        at_q, at_k = _sum_up(s["new"]), _sum_up(s["full"])
        for b in range(case["n"]):
            m, n = s["new"][b], s["full"][b]
            o = torch.empty((m, case["heads"], d), dtype=torch.float64, device="cuda")
            keep = torch.arange(n, device="cuda")[None] <= torch.arange(m, device="cuda")[:, None] + (n - m)
            keep = keep if case["causal"] else torch.ones_like(keep)
            for h in range(case["heads"]):
                j = h // (case["heads"] // kv)
                w = _softmax64(qs[at_q[b]:at_q[b + 1], h] @ ks[at_k[b]:at_k[b + 1], j].T / math.sqrt(d), keep)
                o[:, h] = w @ vs[at_k[b]:at_k[b + 1], j]
            rows.append(o)
        return torch.cat(rows)
    if case["op"] == "token":
        for b in range(case["n"]):
            k, v = _decoded64(s, "k", b), _decoded64(s, "v", b)
            q = s["q"][b].double().view(kv, -1, d)
            w = _softmax64(q @ k.mT / math.sqrt(d), torch.ones((), dtype=torch.bool, device="cuda"))
            rows.append((w @ v).reshape(-1, d))
        return torch.stack(rows)
    out = []
    for name in ("k", "v"):
        x = s[name].double()
        if case["codes"] != "bf16":
            # scale, inverse and product are held in 32 bits by definition: they decide at ties, which are frequent
            top = x.abs().amax(-1, keepdim=True)
            y = (x * (TOP[case["codes"]] / top).float().double()).float().double()
            x = _nearest64(y, case["codes"]) * (top / TOP[case["codes"]]).float().double()
        parts, at = [], 0
        for b in range(case["n"]):
            m, n = s["new"][b], s["full"][b]
            parts += [_decoded64(s, name, b)[:, :n - m].transpose(0, 1), x[at:at + m]]
            at += m
        out.append(torch.cat(parts))
    return out
