"""The block-FP8 products of a decoder layer outside of the one-launch MoE kernel, as cases that can be timed: rows to 8 bits
(``quantize``, with or without the gated activation in front), the dense projections (``linear``), and for experts of any
geometry the division of a batch among them (``plan``), their products over ragged runs of rows (``experts``) and the weighted
sum of each token's results (``combine``). From the one token of a quiet server to prefill batches of 16384 tokens.

Numbers. A row is cut into groups of 128 that share a scale: with m the largest magnitude (1 where that is below 2^-100, so that
448 / m stays finite), codes are e4m3 of x * (448 / m), to nearest, and the scale is m / 448. Weights [N, K] in e4m3 have one fp32
scale for each block of 128 x 128. A product sums codes * codes over a group of K, times both scales, over the groups.
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # hidden states of one token in front of a projection: a launch
        quantize("quantize, 1 token", rows=1, cols=2048),
        # gate and up halves of a prefill batch's routed rows, 8 for each of 16384 tokens
        quantize("silu quantize, 131072 rows", rows=131072, cols=512, silu=True),
        # query, key and value projection of one token that waits for its next
        linear("qkv, 1 token", rows=1, cols=5120, inner=2048),
        # output projection of a decode step with the residual stream added
        linear("output projection, 61 tokens", rows=61, cols=2048, inner=4096, residual=True),
        # a wide projection of a prefill batch
        linear("projection, 16384 tokens", rows=16384, cols=4096, inner=7168),
        # one token's eight experts
        plan("plan, 1 token", tokens=1, top=8, experts=256),
        # a prefill batch on one rank of two, which owns half of the experts
        plan("plan, 16384 tokens", tokens=16384, top=8, experts=128, owned=0.5),
        # up projection of a decode step, gated activation in the same call
        experts("experts up, 24 tokens", tokens=24, top=8, experts=256, cols=1024, inner=2048, silu=True),
        # the same of a prefill batch
        experts("experts up, 16384 tokens", tokens=16384, top=8, experts=256, cols=1024, inner=2048, silu=True),
        # down projection of a chunk of 3000 tokens, unevenly routed
        experts("experts down, 3000 uneven", tokens=3000, top=8, experts=256, cols=2048, inner=512, gather=False, skew=0.7),
        # results of a decode step
        combine("combine, 24 tokens", tokens=24, top=8, cols=2048, residual=True),
        # results of a prefill batch
        combine("combine, 16384 tokens", tokens=16384, top=8, cols=2048),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def quantize(name, rows, cols, silu=False):
    """`cols` columns of the result."""
    return _named(name, {"op": "quantize", "rows": rows, "cols": cols, "silu": silu})


def linear(name, rows, cols, inner, residual=False, silu=False, wide=False):
    """`cols` rows of the weight; `wide`: the result in fp32; `silu`: its halves gated, the result in 8 bits."""
    return _named(name, {"op": "linear", "rows": rows, "cols": cols, "inner": inner, "residual": residual, "silu": silu, "wide": wide})


def plan(name, tokens, top, experts, owned=1.0, skew=0.0):
    """`owned`: share of the slots whose expert lies on this rank."""
    return _named(name, {"op": "plan", "tokens": tokens, "top": top, "experts": experts, "owned": owned, "skew": skew})


def experts(name, tokens, top, experts, cols, inner, silu=False, gather=True, skew=0.0):
    """`gather`: rows are the tokens' (up projection), else those of the plan (down projection)."""
    return _named(name, {"op": "experts", "tokens": tokens, "top": top, "experts": experts, "cols": cols, "inner": inner, "silu": silu,
                         "gather": gather, "skew": skew})


def combine(name, tokens, top, cols, residual=False, owned=1.0):
    return _named(name, {"op": "combine", "tokens": tokens, "top": top, "cols": cols, "residual": residual, "owned": owned})


def _spread(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(max(least, most))))))


def draw(rng):
    """Any operator and geometry; sizes over their logarithm, never above the listed ones' cost."""
    op = rng.choice(["quantize", "linear", "linear", "linear", "plan", "experts", "experts", "combine"])
    inner = rng.choice([256, 512, 512, 768, 1024, 1536, 2048, 2048, 4096, 7168, 1040, 1808])
    if op == "quantize":
        silu = rng.random() < 0.5
        inner = max(128, inner // 128 * 128) if silu else inner
        return quantize(None, _spread(rng, 1, min(131072, 131072 * 512 // inner)), inner, silu)
    if op == "linear":
        silu = rng.random() < 0.2
        cols = 256 * rng.randint(1, 16) if silu else rng.choice([64, 129, 256, 576, 1000, 1536, 2048, 2112, 4096, 5120, 9216])
        rows = _spread(rng, 1, min(16384, 16384 * 4096 * 7168 // (cols * inner)))
        plain = not silu and rng.random() < 0.7
        return linear(None, rows, cols, inner, residual=plain and rng.random() < 0.4, silu=silu, wide=not silu and not plain)
    top = rng.choice([1, 2, 4, 6, 8, 8])
    count = rng.choice([8, 16, 60, 64, 128, 256])
    skew = rng.choice([0.0, 0.0, 0.5, 1.0])
    if op == "plan":
        return plan(None, _spread(rng, 1, 16384), top, count, rng.choice([1.0, 1.0, 0.5, 0.1]), skew)
    if op == "combine":
        return combine(None, _spread(rng, 1, min(16384, 16384 * 2048 * 8 // (inner * top))), top, inner, rng.random() < 0.4, rng.choice([1.0, 1.0, 0.5]))
    silu = rng.random() < 0.5
    cols = 256 * rng.randint(1, 8) if silu else rng.choice([192, 512, 1000, 2048, 2048, 4096])
    while count > 8 and count * cols * inner > 256 * 1024 * 2048:
        count //= 2
    while cols > 512 and count * cols * inner > 256 * 1024 * 2048:
        cols = cols // 512 * 256
    tokens = _spread(rng, 1, min(16384, 131072 * 1024 * 2048 // (top * cols * inner)))
    return experts(None, tokens, top, count, cols, inner, silu, rng.random() < 0.5, skew)


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _over(a, b):
    """a / b as a division of tensors (by or of a number it would be a product with a reciprocal)."""
    a, b = torch.broadcast_tensors(torch.as_tensor(a, dtype=torch.float32), torch.as_tensor(b, dtype=torch.float32))
    dev = a.device if a.is_cuda else b.device
    return a.to(dev).contiguous() / b.to(dev).contiguous()


def _codes(x):
    """Codes and scales of fp32 rows [..., K]."""
    k = x.shape[-1]
    g = torch.nn.functional.pad(x, (0, -k % 128)).unflatten(-1, (-1, 128))
    m = g.abs().amax(-1)
    m = torch.where(m < 2.0 ** -100, 1.0, m)
    q = (g * _over(448.0, m)[..., None]).clamp(-448, 448).to(E4M3).flatten(-2)[..., :k]
    return q.contiguous(), _over(m, 448.0)


def _values(q, s, blocks=False):
    """What codes [..., K] and their scales stand for, in fp32; `blocks`: a scale for 128 rows too."""
    s = s.repeat_interleave(128, -1)[..., :q.shape[-1]]
    if blocks:
        s = s.repeat_interleave(128, -2)[..., :q.shape[-2], :]
    return q.float() * s


def _weight(shape, gen, dev):
    """N(0, 0.02) in block FP8, [..., N, K], a few matrices at a time."""
    *lead, n, k = shape
    lead = lead[0] if lead else 1
    q = torch.empty(lead, n, k, dtype=E4M3, device=dev)
    s = torch.empty(lead, -(-n // 128), -(-k // 128), device=dev)
    step = max(1, (1 << 28) // (n * k))
    for a in range(0, lead, step):
        w = 0.02 * torch.randn(min(step, lead - a), n, k, generator=gen, device=dev)
        g = torch.nn.functional.pad(w, (0, -k % 128, 0, -n % 128)).unflatten(-1, (-1, 128)).unflatten(1, (-1, 128))
        sc = (g.abs().amax((2, 4)) / 448.0).clamp(min=1e-12)
        q[a:a + step] = (g / sc[:, :, None, :, None]).clamp(-448, 448).flatten(3, 4).flatten(1, 2)[:, :n, :k].to(E4M3)
        s[a:a + step] = sc
    return (q, s) if len(shape) == 3 else (q[0], s[0])


def _states(rows, cols, gen, dev):
    """Hidden states: some channels are larger than others."""
    return (torch.randn(rows, cols, generator=gen, device=dev) * torch.exp(0.5 * torch.randn(cols, generator=gen, device=dev))).to(torch.bfloat16)


def _routing(c, gen, dev):
    """int32 [tokens, top]: distinct experts, -1 where this rank does not own them."""
    n = c["experts"]
    score = torch.randn(c["tokens"], n, generator=gen, device=dev) + c.get("skew", 0.0) * torch.randn(n, generator=gen, device=dev)
    ids = score.topk(c["top"], dim=1).indices
    gone = torch.rand(ids.shape, generator=gen, device=dev) >= c.get("owned", 1.0)
    return torch.where(gone, -1, ids).to(torch.int32)


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    s, c = {"case": case}, case
    if c["op"] == "quantize":
        s["x"] = _states(c["rows"], c["cols"] * (2 if c["silu"] else 1), gen, dev)
    elif c["op"] == "linear":
        s["x"] = _states(c["rows"], c["inner"], gen, dev)
        s["w"], s["ws"] = _weight((c["cols"], c["inner"]), gen, dev)
        s["residual"] = _states(c["rows"], c["cols"], gen, dev) if c["residual"] else None
    elif c["op"] == "plan":
        s["ids"] = _routing(c, gen, dev)
    elif c["op"] == "experts":
        s["offsets"], s["tokens"], s["positions"] = _plain_plan(_routing(c, gen, dev), c["experts"])
        s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
        s["q"], s["qs"] = _codes(_states(c["tokens"] * (1 if c["gather"] else c["top"]), c["inner"], gen, dev).float())
        s["w"], s["ws"] = _weight((c["experts"], c["cols"], c["inner"]), gen, dev)
    else:
        rows = c["tokens"] * c["top"]
        s["partial"] = _states(rows, c["cols"], gen, dev)
        at = torch.randperm(rows, generator=gen, device=dev)
        gone = torch.rand(rows, generator=gen, device=dev) >= c["owned"]
        s["positions"] = torch.where(gone, -1, at).to(torch.int32).view(c["tokens"], c["top"])
        s["weights"] = torch.softmax(torch.randn(c["tokens"], c["top"], generator=gen, device=dev), 1)
        s["residual"] = _states(c["tokens"], c["cols"], gen, dev) if c["residual"] else None
    return s


def run(s):
    return (_own if own else _plain)(s)


def _own(s):
    import unimonomoe_b200 as U
    c = s["case"]
    if c["op"] == "quantize":
        return U.fp8_quantize(s["x"], silu_mul=c["silu"])
    if c["op"] == "linear":
        return U.fp8_linear(s["x"], s["w"], s["ws"], residual=s["residual"], silu_mul=c["silu"], out_dtype=torch.float32 if c["wide"] else None)
    if c["op"] == "plan":
        return tuple(U.plan_experts(s["ids"], c["experts"]))
    if c["op"] == "experts":
        p = U.ExpertPlan(s["offsets"], s["tokens"], s["positions"])
        return U.fp8_expert_linear(s["q"], s["w"], s["ws"], p, x_scale=s["qs"], gather=c["gather"], silu_mul=c["silu"])
    return U.combine_experts(s["partial"], s["positions"], s["weights"], residual=s["residual"])


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        return _codes(_gated(s["x"].float()) if c["silu"] else s["x"].float())
    if c["op"] == "linear":
        y = _values(*_codes(s["x"].float())) @ _values(s["w"], s["ws"], True).T
        if c["silu"]:
            return _codes(_gated(y))
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y if c["wide"] else y.to(torch.bfloat16)
    if c["op"] == "plan":
        return _plain_plan(s["ids"], c["experts"])
    if c["op"] == "experts":
        return _plain_experts(s, c)
    p = s["positions"].long()
    w = torch.where(p >= 0, s["weights"], 0.0)
    y = (s["partial"][p.clamp(min=0)].float() * w[..., None]).sum(1)
    return (y if s["residual"] is None else y + s["residual"].float()).to(torch.bfloat16)


def _gated(x):
    a, b = x.chunk(2, -1)
    return a / (1.0 + torch.exp(-a)) * b


def _plain_plan(ids, n):
    """Offsets of each expert's run of rows, the token of each row (-1 behind the last run), the row of each slot (-1: none)."""
    top, key = ids.shape[1], torch.where(ids < 0, n, ids).flatten().long()
    order = torch.argsort(key, stable=True)
    first = torch.searchsorted(key[order], torch.arange(n + 1, device=ids.device))
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=ids.device)
    return (first.to(torch.int32), torch.where(key[order] < n, order // top, -1).to(torch.int32),
            torch.where(key < n, row, -1).to(torch.int32).view(ids.shape))


def _plain_experts(s, c):
    """All experts' rows side by side, as many for each as the fullest has."""
    off, dev = s["offsets"].long(), s["q"].device
    rows = c["tokens"] * c["top"]
    at = (off[:-1, None] + torch.arange(s["most"], device=dev)).clamp(max=rows - 1)
    x = _values(s["q"], s["qs"])[s["tokens"].long()[at] if c["gather"] else at]             # [experts, most, K]
    y = torch.bmm(x, _values(s["w"], s["ws"], True).transpose(1, 2))
    row = torch.arange(rows, device=dev)
    e = torch.searchsorted(off[1:], row, right=True)
    y = y[e, row - off[e]]
    return _codes(_gated(y)) if c["silu"] else y.to(torch.bfloat16)


def work(case):
    c, op = case, case["op"]
    if op == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": (5.0 if c["silu"] else 3.0) * n + 4.0 * c["rows"] * -(-c["cols"] // 128), "flops": (8.0 if c["silu"] else 3.0) * n}
    if op == "linear":
        m, n, k = c["rows"], c["cols"], c["inner"]
        out = m * n * (0.5 + 2.0 / 128 if c["silu"] else 4.0 if c["wide"] else 2.0) + (2.0 * m * n if c["residual"] else 0.0)
        return {"bytes": 2.0 * m * k + n * k * (1.0 + 4.0 / 16384) + out, "flops": 2.0 * m * n * k}
    slots = c["tokens"] * c["top"]
    if op == "plan":
        return {"bytes": 12.0 * slots + 4.0 * (c["experts"] + 1), "flops": 1.0 * slots}
    if op == "combine":
        rows = slots * c["owned"]
        return {"bytes": 2.0 * c["cols"] * (rows + c["tokens"] * (2 if c["residual"] else 1)) + 8.0 * slots, "flops": 2.0 * rows * c["cols"]}
    n, k = c["cols"], c["inner"]
    reached = c["experts"] * (1.0 - (1.0 - c["top"] / c["experts"]) ** c["tokens"])          # of even routing
    rows = c["tokens"] if c["gather"] else slots
    out = slots * n * (0.5 + 2.0 / 128 if c["silu"] else 2.0)
    return {"bytes": reached * n * k * (1.0 + 4.0 / 16384) + rows * k * (1.0 + 4.0 / 128) + (4.0 * slots if c["gather"] else 0.0) + out,
            "flops": 2.0 * slots * n * k}


# ---- the same from the definition, in 64 bits
def _exact_e4m3(v):
    """Nearest e4m3 number: steps of an eighth of the power of two below, of 2^-9 under 2^-6, up to 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_codes(x):
    """Codes' values and scales of each piece of up to 128 columns."""
    codes, scales = [], []
    for g in x.split(128, -1):
        m = g.abs().amax(-1, keepdim=True)
        m = torch.where(m < 2.0 ** -100, torch.ones_like(m), m)
        codes.append(_exact_e4m3(g * 448.0 / m))
        scales.append(m / 448.0)
    return torch.cat(codes, -1), torch.cat(scales, -1)


def _exact_times(q, s, w, ws):
    """Sum over the groups of 128 of (codes x codes) times both scales."""
    y = torch.zeros(q.shape[0], w.shape[0], dtype=torch.float64, device=q.device)
    by_row = ws.double().repeat_interleave(128, 0)[:w.shape[0]]
    for i, k in enumerate(range(0, q.shape[1], 128)):
        y += (q[:, k:k + 128].double() @ w[:, k:k + 128].double().T) * s[:, i:i + 1].double() * by_row[:, i]
    return y


def _exact_gate(y):
    n = y.shape[-1] // 2
    return y[..., :n] * torch.sigmoid(y[..., :n]) * y[..., n:]


def exact(case, seed):
    c = case
    if c["op"] == "plan":                    # whole numbers
        return None
    s = prepare(case, seed)
    if c["op"] == "quantize":
        return _exact_codes(_exact_gate(s["x"].double()) if c["silu"] else s["x"].double())
    if c["op"] == "linear":
        y = _exact_times(*_exact_codes(s["x"].double()), s["w"], s["ws"])
        if c["silu"]:
            return _exact_codes(_exact_gate(y))
        return y if s["residual"] is None else y + s["residual"].double()
    if c["op"] == "experts":
        off = s["offsets"].tolist()
        y = torch.empty(c["tokens"] * c["top"], c["cols"], dtype=torch.float64, device=s["q"].device)
        for e, (a, b) in enumerate(zip(off, off[1:])):
            if a < b:
                rows = s["tokens"][a:b].long() if c["gather"] else slice(a, b)
                y[a:b] = _exact_times(s["q"][rows], s["qs"][rows], s["w"][e], s["ws"][e])
        return _exact_codes(_exact_gate(y)) if c["silu"] else y
    y = torch.zeros(c["tokens"], c["cols"], dtype=torch.float64, device=s["partial"].device)
    for j in range(c["top"]):
        p = s["positions"][:, j].long()
        y += torch.where(p[:, None] >= 0, s["partial"][p.clamp(min=0)].double() * s["weights"][:, j:j + 1].double(), 0.0)
    return y if s["residual"] is None else y + s["residual"].double()
