"""The attention half of a decoder layer over a paged cache held in 4 bits, as cases that can be timed: what a serving
engine has done for every step (``plan``: positions, slots and block tables from request lengths), for every layer
before attention (``rope``: norms of queries and keys for each head with the rotation; ``store``: keys and values into
the cache, and read back) and the attention itself (``attend``), from one sequence that waits for its next token to
whole prompts of 8192 tokens.

Cache format. A page of one KV head is cut into blocks of 16 tokens. A block has 17*D bytes for head size D: 8*D bytes
of key codes, 8*D of value codes, then for each token the scales of its key and of its value, one bfloat16 for 64 dims.
A code is 8 + c, c from -7 to 7, and stands for s*c. Codes lie in the order in which the 32 lanes of a warp take
them as matrix operands, 16 bytes for a lane at a time; `_nibbles` gives the place of each.
"""
import math

import numpy as np
import torch

own = False

GROUP = 64                                   # dims that share a scale
TABLE = 131072                               # rows of the rotation table: the longest context
PAGES_SPARE = 8


def listed():
    return [
        # a quiet server: one sequence gets one token
        plan("plan, one request", batch=1, new=1, cached=777, page=16),
        # the decode step of a loaded server
        plan("plan, decode 256", batch=256, new=1, cached=4096, page=16),
        # a step of chunked prefill that fills the token budget with ragged chunks
        plan("plan, ragged chunks 16384", batch=37, new=886, cached=2000, page=64),
        # decode batch, wide heads of which a quarter is rotated
        rope("norm+rotation, 16 tokens", tokens=16, heads=16, kv=2, dim=256, rotary=64),
        # prefill batch
        rope("norm+rotation, 8192 tokens", tokens=8192, heads=32, kv=4, dim=128, rotary=128),
        # a short prompt's keys and values
        store("store and read, 61 tokens", tokens=61, kv=4, dim=128, page=16),
        # a prefill batch's
        store("store and read, 16384 tokens", tokens=16384, kv=4, dim=128, page=64),
        # one sequence waiting for its next token: launches and latency
        attend("one token, context 777", batch=1, new=1, context=777, heads=16, kv=2, dim=256, page=16),
        # the decode step of a loaded server, ragged contexts
        attend("decode 64, contexts to 8192", batch=64, new=1, context=8192, heads=32, kv=4, dim=128, page=16),
        # two long documents: few rows, the context has to be split
        attend("decode 2, context 131072", batch=2, new=1, context=131072, heads=32, kv=4, dim=128, page=64, spread=0.0),
        # ragged chunks of chunked prefill behind earlier chunks
        attend("chunks of 700, contexts to 4096", batch=7, new=700, context=4096, heads=32, kv=4, dim=128, page=16),
        # a whole prompt
        attend("prompt of 8192", batch=1, new=8192, context=8192, heads=16, kv=2, dim=256, page=64),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def plan(name, batch, new, cached, page):
    """`batch` requests of 0.5*new to new tokens (one where new is 1) behind 0 to `cached` tokens."""
    return _named(name, {"op": "plan", "batch": batch, "new": new, "cached": cached, "page": page})


def rope(name, tokens, heads, kv, dim, rotary, interleaved=False, unit=False):
    return _named(name, {"op": "rope", "tokens": tokens, "heads": heads, "kv": kv, "dim": dim, "rotary": rotary,
                         "interleaved": interleaved, "unit": unit})


def store(name, tokens, kv, dim, page):
    return _named(name, {"op": "store", "tokens": tokens, "kv": kv, "dim": dim, "page": page})


def attend(name, batch, new, context, heads, kv, dim, page, spread=0.5, window=0, lse=False):
    """Contexts from (1 - spread)*context to `context` tokens, the last 0.5*new to new of them (one where new is 1) the queries'."""
    return _named(name, {"op": "attend", "batch": batch, "new": new, "context": context, "heads": heads, "kv": kv, "dim": dim,
                         "page": page, "spread": spread, "window": window, "lse": lse})


def _spread(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    """Any operator, head layout and page size; sizes over their logarithm, never above the listed ones' cost."""
    op = rng.choice(["plan", "rope", "store", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "plan":
        batch = _spread(rng, 1, 1024)
        return plan(None, batch, _spread(rng, 1, max(1, 16384 // batch)), _spread(rng, 1, 8192), page)
    if op == "rope":
        tokens = _spread(rng, 1, max(1, 8192 * 36 * 128 // ((group + 1) * kv * dim)))
        return rope(None, min(tokens, 16384), group * kv, kv, dim, rng.choice([dim, dim, dim // 2, dim // 4]),
                    rng.random() < 0.3, rng.random() < 0.3)
    if op == "store":
        return store(None, _spread(rng, 1, min(32768, 16384 * 4 * 128 // (kv * dim))), kv, dim, page)
    if rng.random() < 0.5:                   # decode, some with a few tokens guessed ahead
        batch, new = _spread(rng, 1, 128), rng.choice([1, 1, 1, 1, 2, 4, 7])
    else:
        batch, new = _spread(rng, 1, 8), _spread(rng, 2, 4096)
    context = new + _spread(rng, 1, 65536)
    window = rng.choice([0, 0, 0, 0, 127, 1024])
    while context > new and (batch * context * kv * dim > 2 * 131072 * 4 * 128 or batch * new * group * kv * context > 16 * 8192 * 4096):
        context = max(new, context // 2)
    while new > 1 and batch * new * group * kv * context > 16 * 8192 * 4096:
        new, context = new // 2, max(context // 2, new // 2)
    return attend(None, batch, new, context, group * kv, kv, dim, page, rng.choice([0.0, 0.5, 0.9]), window, rng.random() < 0.25)


def _even(n, least, most):
    """n whole numbers spread evenly over [least, most]."""
    return [most] if n == 1 else [int(round(least + (most - least) * i / (n - 1))) for i in range(n)]


def _lengths(case):
    """(tokens before the step, tokens of the step) of every request, in an order that the seed shuffles."""
    n, new = case["batch"], case["new"]
    news = _even(n, new - new // 2, new) if new > 1 else [1] * n
    if case["op"] == "plan":
        return _even(n, 0, case["cached"]), news
    total = _even(n, max(1, int(case["context"] * (1.0 - case["spread"]))), case["context"])
    return [max(0, t - m) for t, m in zip(total, news)], news


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _nibbles(dim, values):
    """Place (in half bytes) of each code of a block among its key or value codes, [16 tokens, dim]."""
    groups = dim // 64
    r, d = np.meshgrid(np.arange(16), np.arange(dim), indexing="ij")
    if values:
        part, lane = (r >> 3) * 2 + (r & 1), (d % 64 // 8) * 4 + (r >> 1) % 4
        o = part * 4 * groups + d // 64 * 4 + d % 8 // 2
    else:
        part, lane = r >> 3, (r & 7) * 4 + d % 64 // 16
        o = part * 8 * groups + d // 64 * 8 + d % 16 // 8 * 4 + d % 8 // 2
    return (o // 16 * 512 + lane * 16 + o % 16) * 2 + d % 2


_places = {}


def _place(dim, device, values):
    """(place of each code, the code at each place) as flat index tensors."""
    key = (dim, device, values)
    if key not in _places:
        at = torch.from_numpy(_nibbles(dim, values).reshape(-1)).to(device)
        _places[key] = (at, torch.argsort(at))
    return _places[key]


def _round5(s):
    """To five significant bits, ties to even."""
    m, e = torch.frexp(s)
    return torch.ldexp(torch.round(m * 32.0), e - 5)


def _quantise(x):
    """Codes (-7 to 7) and scales of x [..., D] in x's own precision."""
    g = x.unflatten(-1, (-1, GROUP))
    s = _round5(g.abs().amax(-1) / 7.0).clamp(2.0 ** -60, 2.0 ** 60)
    c = torch.round(g / s[..., None]).clamp(-7, 7)
    return c, s


def _pack(k, v):
    """Blocks [..., 17*D] from keys and values [..., 16, D]."""
    dim = k.shape[-1]
    parts, scales = [], []
    for values, x in ((False, k), (True, v)):
        c, s = _quantise(x.float())
        code = (c + 8).to(torch.uint8).flatten(-3)[..., _place(dim, k.device, values)[1]]
        parts.append(code[..., 0::2] | code[..., 1::2] << 4)
        scales.append(s.to(torch.bfloat16))
    parts.append(torch.cat(scales, -1).view(torch.uint8).flatten(-2))
    return torch.cat(parts, -1)


def _unpack(blocks, dtype):
    """Keys and values [..., 16, D] from blocks [..., 17*D]."""
    dim = blocks.shape[-1] // 17
    s = blocks[..., 16 * dim:].unflatten(-1, (16, -1)).contiguous().view(torch.bfloat16).to(dtype)
    got = []
    for values, x, sc in ((False, blocks[..., :8 * dim], s[..., :dim // 64]), (True, blocks[..., 8 * dim:16 * dim], s[..., dim // 64:])):
        code = torch.stack([x & 15, x >> 4], -1).flatten(-2)[..., _place(dim, x.device, values)[0]]
        c = code.to(dtype).sub_(8).unflatten(-1, (16, dim // GROUP, GROUP))
        got.append((c * sc[..., None]).flatten(-2))
    return got


def _cache(pages, kv, page, dim, gen, device):
    """A cache full of normal keys and values, [pages, kv, page/16, 17*dim]."""
    data = torch.empty(pages, kv, page // 16, 17 * dim, dtype=torch.uint8, device=device)
    at = max(1, (1 << 26) // (kv * page * dim))
    for p in range(0, pages, at):
        n = min(at, pages - p)
        kv_ = torch.randn(2, n, kv, page // 16, 16, dim, generator=gen, device=device)
        data[p:p + n] = _pack(kv_[0], kv_[1])
    return data


def _table(lens, page, width, pages, gen, device):
    """Block table [batch, width] of scattered pages for `lens` tokens, -1 behind them, and the pages left over."""
    need = torch.tensor([-(-n // page) for n in lens], device=device)
    order = torch.randperm(pages, generator=gen, device=device).to(torch.int32)
    first = torch.cumsum(need, 0) - need
    col = torch.arange(width, device=device)
    table = order[(first[:, None] + col).clamp(max=pages - 1)]
    return torch.where(col < need[:, None], table, -1).to(torch.int32).contiguous(), order[int(need.sum()):].contiguous()


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    s = {"case": case}

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=dev)

    if case["op"] == "rope":
        T, H, K, D, R = (case[n] for n in ("tokens", "heads", "kv", "dim", "rotary"))
        # q, k and v as the fused projection leaves them, one row of all heads for a token
        qkv = torch.randn(T, (H + 2 * K) * D, generator=gen, device=dev).to(torch.bfloat16).unflatten(1, (-1, D))
        s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + K]
        w = 0.2 * torch.randn(2, D, generator=gen, device=dev) + (0.0 if case["unit"] else 1.0)
        s["wq"], s["wk"] = w[0].to(torch.bfloat16), w[1].to(torch.bfloat16)
        angle = torch.arange(TABLE, device=dev, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["positions"] = torch.randint(0, TABLE, (T,), generator=gen, device=dev).to(torch.int32)
        return s
    if case["op"] == "store":
        T, K, D, P = (case[n] for n in ("tokens", "kv", "dim", "page"))
        pages = -(-T // P) + PAGES_SPARE
        s["data"] = _cache(pages, K, P, D, gen, dev)
        qkv = torch.randn(T, 2 * K * D, generator=gen, device=dev).to(torch.bfloat16).unflatten(1, (-1, D))
        s["k"], s["v"] = qkv[:, :K], qkv[:, K:]
        order = torch.randperm(pages, generator=gen, device=dev)
        t = torch.arange(T, device=dev) + int(rng.randint(P))     # prompts start inside a page
        s["slots"] = order[t // P] * P + t % P
        return s
    cached, news = _lengths(case)
    order = rng.permutation(case["batch"])
    cached, news = [cached[i] for i in order], [news[i] for i in order]
    P, total = case["page"], [a + b for a, b in zip(cached, news)]
    need = sum(-(-n // P) for n in total)
    width = -(-max(total) // P)
    if case["op"] == "plan":
        pages = need + PAGES_SPARE
        table, free = _table(cached, P, width, pages, gen, dev)
        s.update(cached=ints(cached), new=ints(news), table=table, free=free, taken=ints([0]), tokens=sum(news))
        return s
    pages = need + PAGES_SPARE
    s["data"] = _cache(pages, case["kv"], P, case["dim"], gen, dev)
    s["table"] = _table(total, P, width, pages, gen, dev)[0]
    start = np.concatenate([[0], np.cumsum(news)])
    s.update(lens=ints(total), start=ints(start), longest=max(news), tokens=int(start[-1]))
    s["q"] = torch.randn(s["tokens"], case["heads"], case["dim"], generator=gen, device=dev).to(torch.bfloat16)
    return s


def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    import unimonomoe_b200.attention as A
    c = s["case"]
    if c["op"] == "plan":
        p = A.plan_batch(s["cached"], s["new"], s["table"], s["free"], s["taken"], c["page"], s["tokens"])
        return {"start": p.query_start, "lens": p.seq_lens, "positions": p.positions, "slots": p.slots,
                "requests": p.requests, "taken": p.taken, "table": s["table"]}
    if c["op"] == "rope":
        q, k = A.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["table"], s["positions"], interleaved=c["interleaved"],
                              unit_offset=c["unit"])
        return {"q": q, "k": k}
    if "cache" not in s:                     # the handle that a program keeps
        s["cache"] = A.KV4Cache(s["data"])
    cache = s["cache"]
    if c["op"] == "store":
        A.kv4_append(s["k"], s["v"], cache, s["slots"])
        k, v = A.kv4_read(cache, s["slots"])
        return {"k": k, "v": v}
    got = A.kv4_attention(s["q"], cache, s["table"], s["lens"], s["start"], s["longest"], window=c["window"], return_lse=c["lse"])
    return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}


def _plain(s):
    c = s["case"]
    if c["op"] == "plan":
        return _plain_plan(s["cached"], s["new"], s["table"], s["free"], s["taken"], c["page"], s["tokens"])
    if c["op"] == "rope":
        return {"q": _plain_rope(s["q"].float(), s["wq"], s, c).to(torch.bfloat16),
                "k": _plain_rope(s["k"].float(), s["wk"], s, c).to(torch.bfloat16)}
    if c["op"] == "store":
        return _plain_store(s, c)
    return _plain_attend(s, c)


def _plain_plan(cached, new, table, free, taken, page, tokens):
    dev = cached.device
    total = cached + new
    start = torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), torch.cumsum(new, 0).to(torch.int32)])
    held, need = (cached + page - 1) // page, (total + page - 1) // page
    fresh = need - held
    first = taken + torch.cumsum(fresh, 0) - fresh
    col = torch.arange(table.shape[1], device=dev)
    source = (first[:, None] + col - held[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where((col >= held[:, None]) & (col < need[:, None]), free[source], table))
    at = torch.arange(tokens, device=dev)
    request = torch.searchsorted(start[1:], at, right=True)
    position = cached[request] + at - start[request]
    slots = table[request, position // page].long() * page + position % page
    return {"start": start, "lens": total, "positions": position.to(torch.int32), "slots": slots,
            "requests": request.to(torch.int32), "taken": (taken + fresh.sum()).to(torch.int32), "table": table}


def _plain_rope(x, w, s, c):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    y = y * (w.float() + 1.0 if c["unit"] else w.float())
    R = c["rotary"]
    cs = s["table"][s["positions"].long()][:, None]
    co, si = cs[..., :R // 2], cs[..., R // 2:]
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if c["interleaved"] else (y[..., :R // 2], y[..., R // 2:R])
    a, b = a * co - b * si, b * co + a * si
    rotated = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([rotated, y[..., R:]], -1)


def _plain_store(s, c):
    """Writes the codes and scales to their places in the cache; what they stand for comes back."""
    data, slots, P, D = s["data"], s["slots"], c["page"], c["dim"]
    flat = data.flatten()
    row = (slots // P * c["kv"])[:, None] + torch.arange(c["kv"], device=slots.device)
    base = (row * (P // 16) + (slots % P // 16)[:, None]) * (17 * D)                    # [T, kv]
    token = slots % 16
    back = {}
    for name, values in (("k", False), ("v", True)):
        code, scale = _quantise(s[name].float())
        nib = (code + 8).to(torch.uint8).flatten(-2)
        place = _place(D, slots.device, values)[0].view(16, D)[token][:, None, 0::2] // 2 + (8 * D if values else 0)
        flat[base[..., None] + place] = nib[..., 0::2] | nib[..., 1::2] << 4
        at = 16 * D + token[:, None, None] * (D // 16) + (D // 32 if values else 0) + torch.arange(D // 32, device=slots.device)
        flat[base[..., None] + at] = scale.to(torch.bfloat16).view(torch.uint8)
        got = flat[base[..., None] + place]
        sc = flat[base[..., None] + at].view(torch.bfloat16).float()
        c8 = torch.stack([got & 15, got >> 4], -1).flatten(-2).float() - 8
        back[name] = (c8.unflatten(-1, (-1, GROUP)) * sc[..., None]).flatten(-2).to(torch.bfloat16)
    return back


def _plain_attend(s, c):
    H, K, D = c["heads"], c["kv"], c["dim"]
    lens, start, dev = s["lens"].long(), s["start"].long(), s["q"].device
    blocks = s["data"][s["table"].clamp(min=0).long()]                                  # [B, pages, K, P/16, 17D]
    k, v = (x.permute(0, 2, 1, 3, 4, 5).flatten(2, 4) for x in _unpack(blocks, torch.float32))  # [B, K, L, D]
    del blocks
    n = start[1:] - start[:-1]
    i, j = torch.arange(s["longest"], device=dev), torch.arange(k.shape[2], device=dev)
    q = s["q"][(start[:-1, None] + i).clamp(max=s["tokens"] - 1)].float()                # [B, Q, H, D]
    q = q.unflatten(2, (K, H // K)).permute(0, 2, 3, 1, 4).flatten(2, 3)                # [B, K, G*Q, D]
    at = (lens - n)[:, None] + i                                                        # place of each query
    seen = (j <= at[..., None]) & (j < lens[:, None, None])
    if c["window"]:
        seen = seen & (j > at[..., None] - c["window"])
    x = (q @ k.transpose(-1, -2)).mul_(D ** -0.5).unflatten(2, (H // K, -1))            # [B, K, G, Q, L]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x.flatten(2, 3) @ v.masked_fill_(j[:, None] >= lens[:, None, None, None], 0.0)).unflatten(2, (H // K, -1))
    out = torch.where(total > 0, out / total, 0.0)
    token = torch.arange(s["tokens"], device=dev)
    b = torch.searchsorted(start[1:], token, right=True)
    row = token - start[b]
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[b, row].to(torch.bfloat16)
    if not c["lse"]:
        return {"out": out}
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).flatten(2, 3)[b, row]
    return {"out": out, "lse": lse.contiguous()}


def work(case):
    op = case["op"]
    if op == "plan":
        cached, news = _lengths(case)
        P, tokens = case["page"], sum(news)
        fresh = sum(-(-(a + b) // P) + -a // P for a, b in zip(cached, news))
        # lengths in; pages taken, and their table entries; starts and lengths; position, slot and request of a token; the table
        # entry of each page that a token lies in
        pages = sum(-(-(a + b) // P) - a // P for a, b in zip(cached, news))
        return {"bytes": 16.0 * case["batch"] + 8.0 * fresh + 4.0 * pages + 16.0 * tokens + 12, "flops": 8.0 * tokens}
    if op == "rope":
        T, D, R = case["tokens"], case["dim"], case["rotary"]
        n = T * (case["heads"] + case["kv"]) * D
        return {"bytes": 4.0 * n + 4.0 * T + 4.0 * min(T, TABLE) * R + 4.0 * D, "flops": 4.0 * n + 3.0 * n * R / D}
    if op == "store":
        n = 2.0 * case["tokens"] * case["kv"] * case["dim"]
        # in and back out in 16 bits, written and read once at 4 bits and a scale for 64
        return {"bytes": 4.0 * n + 2 * n * (0.5 + 2.0 / GROUP) + 16.0 * case["tokens"], "flops": 6.0 * n}
    cached, news = _lengths(case)
    w, read, pairs = case["window"], 0, 0
    for a, b in zip(cached, news):
        first = max(0, a + 1 - w) if w else 0
        read += a + b - first
        p = a + 1 + np.arange(b, dtype=np.int64)
        pairs += int((np.minimum(p, w) if w else p).sum())
    D, tokens = case["dim"], sum(news)
    entries = sum(-(-(a + b) // case["page"]) for a, b in zip(cached, news))
    return {"bytes": read * case["kv"] * D * 17.0 / 16.0 + 4.0 * tokens * case["heads"] * D + 4.0 * entries
            + (4.0 * tokens * case["heads"] if case["lse"] else 0.0),
            "flops": 4.0 * pairs * case["heads"] * D}


def exact(case, seed):
    if case["op"] == "plan":                 # whole numbers
        return None
    s = prepare(case, seed)
    if case["op"] == "rope":
        return {n: _exact_rope(s[n].double(), s["w" + n].double(), s, case) for n in "qk"}
    if case["op"] == "store":
        return {n: _exact_store(s[n].double()) for n in "kv"}
    return _exact_attend(s, case)


def _exact_rope(x, w, s, c):
    """The rotation as a product of complex numbers."""
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w + 1.0 if c["unit"] else w)
    R = c["rotary"]
    turn = torch.complex(*s["table"].double()[s["positions"].long()].chunk(2, -1))[:, None]
    if c["interleaved"]:
        z = torch.view_as_complex(y[..., :R].unflatten(-1, (-1, 2)).contiguous()) * turn
        y[..., :R] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :R // 2].contiguous(), y[..., R // 2:R].contiguous()) * turn
        y[..., :R] = torch.cat([z.real, z.imag], -1)
    return y


def _exact_store(x):
    """Nearest multiple within 7 steps of the group's scale: a seventh of its largest magnitude, to five bits."""
    g = x.unflatten(-1, (-1, GROUP))
    s = g.abs().amax(-1, keepdim=True) / 7.0
    unit = torch.exp2(torch.floor(torch.log2(s.clamp(min=2.0 ** -60))) - 4)
    s = (torch.round(s / unit) * unit).clamp(2.0 ** -60, 2.0 ** 60)
    return (s * torch.round(g / s).clamp(-7, 7)).flatten(-2)


def _exact_attend(s, c):
    K, G, P = c["kv"], c["heads"] // c["kv"], c["page"]
    lens, start = s["lens"].tolist(), s["start"].tolist()
    out = torch.zeros(s["tokens"], c["heads"], c["dim"], dtype=torch.float64, device=s["q"].device)
    lse = torch.full((s["tokens"], c["heads"]), -math.inf, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(lens):
        pages = s["table"][b, :-(-n // P)].long()
        for h in range(K):
            k, v = (x.reshape(-1, c["dim"])[:n] for x in _unpack(s["data"][pages, h], torch.float64))
            rows = 1 + (1 << 27) // (n * G)                       # of queries at a time
            for a in range(start[b], start[b + 1], rows):
                e = min(a + rows, start[b + 1])
                at = n - start[b + 1] + torch.arange(a, e, device=k.device)[:, None]
                j = torch.arange(n, device=k.device)
                hide = (j > at) | ((j <= at - c["window"]) if c["window"] else (j < 0))
                x = torch.einsum("tgd,nd->tgn", s["q"][a:e, h * G:(h + 1) * G].double(), k) / math.sqrt(c["dim"])
                x = x.masked_fill(hide[:, None], -math.inf)
                lse[a:e, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
                out[a:e, h * G:(h + 1) * G] = torch.softmax(x, -1).nan_to_num(0.0) @ v
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
