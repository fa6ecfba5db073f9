"""The attention operators against their definitions in 64 bits: sizes, layouts and masks where they can go wrong."""
import ctypes
import math
import random

import pytest
import torch

from tests import attention_ref as ref
from unimonomoe_b200 import attention as A

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _status():
    yield
    A.check_status(DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(shape, seed, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * scale).to(torch.bfloat16)


# ---------------------------------------------------------------------- plan
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("lens", [
    [(0, 1)], [(15, 1), (16, 1), (17, 1)], [(0, 0), (0, 33), (5, 0), (1023, 2)], [(0, 5000)], "ragged", "many"])
def test_plan(page, lens):
    rng = random.Random(7)
    if lens == "ragged":
        lens = [(rng.randrange(300), rng.randrange(200)) for _ in range(61)]
    elif lens == "many":
        lens = [(rng.randrange(70), rng.randrange(3)) for _ in range(7001)]
    cached, new = [list(x) for x in zip(*lens)]
    width = max(max(-(-(c + n) // page) for c, n in lens), 1) + 1
    held = [-(-c // page) for c in cached]
    need = sum(-(-(c + n) // page) for c, n in lens)
    order = list(range(need + 9))
    rng.shuffle(order)
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (width - h))
        at += h
    tokens, taken = sum(new) + 3, 2
    free = [10 ** 6, 10 ** 6] + order[at:]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    dev_table = i32(table)
    got = A.plan_batch(i32(cached), i32(new), dev_table, i32(free), i32([taken]), page, tokens)
    start, total, pos, slot, req, taken = ref.plan(cached, new, table, free, taken, page, tokens)
    assert got.query_start.tolist() == start and got.seq_lens.tolist() == total
    assert got.positions.tolist() == pos and got.slots.tolist() == slot and got.requests.tolist() == req
    assert got.taken.tolist() == [taken] and dev_table.tolist() == table


@pytest.mark.parametrize("what,code", [("pages", "more pages"), ("table", "longer than"), ("tokens", "more tokens"), ("negative", "negative"),
                                       ("entry", "block-table entry")])
def test_plan_faults_are_reported_and_kept_in_bounds(what, code):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cached, new, free, tokens, width = [10, 40], [20, 30], [5, 6, 7, 8], 50, 5
    table = [[1, -1, -1, -1, -1], [2, 3, 4, -1, -1]]
    if what == "pages":
        free = [5, 6]
    elif what == "table":
        width, table = 4, [r[:4] for r in table]
    elif what == "tokens":
        tokens = 49
    elif what == "negative":
        new = [20, -30]
    elif what == "entry":
        table[0][0] = -1
    guard = torch.full((tokens + 64,), 77, dtype=torch.int64, device=DEV)
    p = A.plan_batch(i32(cached), i32(new), i32(table), i32(free), i32([0]), 16, tokens)
    with pytest.raises(RuntimeError, match=code):
        A.check_status(DEV)
    assert (guard == 77).all()
    fine = p.slots[:6] if what != "entry" else p.slots[6:20]
    want = [26, 27, 28, 29, 30, 31] if what != "entry" else [5 * 16 + i for i in range(14)]
    assert fine.tolist() == want
    assert ((p.slots >= -1) & (p.slots < 9 * 16)).all()


# ---------------------------------------------------------------------- store and read
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("K,page,T", [(1, 16, 1), (3, 16, 37), (4, 64, 200), (8, 1024, 61)])
def test_append_and_read(D, K, page, T):
    pages = -(-T // page) + 2
    cache = A.KV4Cache.empty(pages, K, D, page, DEV)
    cache.data.fill_(0xA5)
    before = cache.data.clone()
    qkv = randn((T, 2 * K + 3, D), D + K + T, 3.0)
    qkv[0, 3] = 0                                            # a row of zeros, one of equal values, tiny and large groups
    qkv[T // 2, 4] = 7.0
    qkv[T - 1, 3, :64] *= 2.0 ** -70
    qkv[T - 1, 3 + K, :64] *= 2.0 ** 40
    k, v = qkv[:, 3:3 + K], qkv[:, 3 + K:]
    slots = torch.randperm(pages * page, generator=gen(1), device=DEV)[:T]
    if T > 5:
        slots[5] = -1
    A.kv4_append(k, v, cache, slots)
    kept = [i for i in range(T) if i != 5]
    gk, gv = A.kv4_read(cache, slots)
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got[kept].double(), ref.quantised(x)[kept])
        assert T <= 5 or not got[5].any()
    dk, dv = cache.dequantize()
    flat = slots[kept]
    assert torch.equal(dk[flat // page, flat % page].double(), ref.quantised(k)[kept])
    assert torch.equal(dv[flat // page, flat % page].double(), ref.quantised(v)[kept])
    # every other token's codes and scales are untouched
    other = A.KV4Cache(before)
    ok, ov = other.dequantize()
    rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    rest[flat] = False
    for a, b in ((dk, ok), (dv, ov)):
        assert torch.equal(a.flatten(0, 1)[rest].nan_to_num(9.0), b.flatten(0, 1)[rest].nan_to_num(9.0))


def test_every_bf16_value_against_the_definition():
    """Each finite bf16 of 40 octaves beside a group maximum that makes ties: the same codes as in 64 bits."""
    bits = torch.arange(87 << 7, 167 << 7, device=DEV, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    x = x[: x.numel() // 64 * 64].view(-1, 1, 64).clone()
    x[:, :, ::2] *= -1
    top = torch.tensor([231.0, 245.0, 7.0, 1.0, 3.5], device=DEV).to(torch.bfloat16)
    for t in top:
        y = x.clone()
        y[:, 0, 5] = x[:, 0].abs().amax(-1) * (t / 64)
        cache = A.KV4Cache.empty(-(-len(y) // 16), 1, 64, 16, DEV)
        slots = torch.arange(len(y), device=DEV)
        A.kv4_append(y, -y, cache, slots)
        k, v = A.kv4_read(cache, slots)
        assert torch.equal(k.double(), ref.quantised(y)) and torch.equal(v.double(), ref.quantised(-y))


def test_groups_that_are_not_finite_read_back_as_nan():
    x = randn((4, 2, 128), 3)
    x[0, 0, 3], x[1, 1, 70], x[2, 0, 127] = math.inf, math.nan, -math.inf
    cache = A.KV4Cache.empty(1, 2, 128, 16, DEV)
    cache.data.zero_()
    slots = torch.tensor([3, 2, 1, 0], device=DEV)
    A.kv4_append(x, -x, cache, slots)
    k, v = A.kv4_read(cache, slots)
    for got, want in ((k, ref.quantised(x)), (v, ref.quantised(-x))):
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(want).sum() == 3 * 64
        assert torch.equal(got.double().nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("slot", [-2, 32, 1 << 40])
def test_slots_outside_the_cache(slot):
    cache = A.KV4Cache.empty(2, 1, 64, 16, DEV)
    cache.data.fill_(0x88)
    slots = torch.tensor([slot], device=DEV)
    x = randn((1, 1, 64), 1)
    A.kv4_append(x, x, cache, slots)
    with pytest.raises(RuntimeError, match="slot outside"):
        A.check_status(DEV)
    assert (cache.data == 0x88).all()
    k, v = A.kv4_read(cache, slots)
    with pytest.raises(RuntimeError, match="slot outside"):
        A.check_status(DEV)
    assert not k.any() and not v.any()


# ---------------------------------------------------------------------- norms and rotation
ROPE = [(64, 4, 1, 64, 1), (64, 5, 5, 16, 33), (128, 32, 4, 128, 19), (128, 7, 1, 48, 3), (128, 1, 1, 0, 5), (256, 16, 2, 64, 9), (256, 6, 3, 256, 70)]


def _rope_inputs(D, H, K, R, T, fp32):
    qkv = randn((T, H + 2 * K, D), D + T, 2.0)
    qkv[0, 0] = 0
    w = torch.randn(2, D, generator=gen(3), device=DEV).to(torch.float32 if fp32 else torch.bfloat16)
    angle = torch.rand(50, R // 2, generator=gen(4), device=DEV) * 100
    table = torch.cat([angle.cos(), angle.sin()], 1).contiguous()
    pos = torch.randint(0, 50, (T,), generator=gen(5), device=DEV).to(torch.int32)
    return qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], w[0].contiguous(), w[1].contiguous(), table, pos


@pytest.mark.parametrize("D,H,K,R,T", ROPE)
@pytest.mark.parametrize("interleaved,unit,fp32", [(False, False, False), (True, True, True), (False, True, False)])
def test_norm_rope(D, H, K, R, T, interleaved, unit, fp32):
    q, k, _, wq, wk, table, pos = _rope_inputs(D, H, K, R, T, fp32)
    got = A.qk_norm_rope(q, k, wq, wk, table, pos, 1e-6, interleaved, unit)
    for y, x, w in zip(got, (q, k), (wq, wk)):
        want = ref.norm_rope(x, w, table, pos, 1e-6, interleaved, unit)
        assert y.is_contiguous() and y.shape == x.shape
        # fp32 arithmetic: the mean of D squares, a reciprocal root, four products and a sum, each within a few 2^-24 of its
        # terms, which are at most sqrt 2 of the pair's length; then one rounding to bf16
        pair = want.abs().amax(-1, keepdim=True)
        assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + pair * 2.0 ** -19 + 1e-30).all()


@pytest.mark.parametrize("D,H,K,R,T", ROPE)
def test_norm_rope_into_the_cache_is_append_of_its_results(D, H, K, R, T):
    q, k, v, wq, wk, table, pos = _rope_inputs(D, H, K, R, T, False)
    caches = [A.KV4Cache.empty(T // 32 + 2, K, D, 32, DEV) for _ in range(2)]
    slots = torch.randperm((T // 32 + 2) * 32, generator=gen(1), device=DEV)[:T]
    if T > 2:
        slots[2] = -1
    for c in caches:
        c.data.zero_()
    q1, k1 = A.qk_norm_rope(q, k, wq, wk, table, pos)
    A.kv4_append(k1, v, caches[0], slots)
    q2 = A.qk_norm_rope(q, k, wq, wk, table, pos, v=v, cache=caches[1], slots=slots)
    assert torch.equal(q1, q2) and torch.equal(caches[0].data, caches[1].data)


def test_norm_rope_takes_any_strides_and_positions_outside_are_reported():
    q, k, _, wq, wk, table, pos = _rope_inputs(128, 4, 2, 128, 6, False)
    want = A.qk_norm_rope(q, k, wq, wk, table, pos)
    odd = torch.empty(6, 4, 129, dtype=torch.bfloat16, device=DEV)[..., 1:]
    odd.copy_(q)
    turned = k.transpose(0, 1).contiguous().transpose(0, 1)
    got = A.qk_norm_rope(odd, turned, wq, wk, table, pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for bad in (-1, 50):
        p = pos.clone()
        p[3] = bad
        got = A.qk_norm_rope(q, k, wq, wk, table, p)
        with pytest.raises(RuntimeError, match="position outside"):
            A.check_status(DEV)
        rest = [0, 1, 2, 4, 5]
        assert torch.equal(got[0][rest], want[0][rest]) and torch.equal(got[1][rest], want[1][rest])


# ---------------------------------------------------------------------- attention
def make(lens, news, H, K, D, page, seed=0, extra=3):
    """Cache, table, lengths and queries; the pages' unused places and the spare pages hold garbage: scales of all kinds."""
    width = max(max(-(-n // page) for n in lens), 1) + 1
    pages = sum(-(-n // page) for n in lens) + extra
    cache = A.KV4Cache.empty(pages, K, D, page, DEV)
    cache.data.copy_(torch.randint(0, 256, cache.data.shape, generator=gen(seed + 9), device=DEV))
    order = torch.randperm(pages, generator=gen(seed + 1), device=DEV).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    keys, values, at = [], [], 0
    for b, n in enumerate(lens):
        mine = order[at:at + -(-n // page)]
        at += len(mine)
        table[b, :len(mine)] = torch.tensor(mine, dtype=torch.int32, device=DEV)
        k, v = randn((n, K, D), seed + 100 + b), randn((n, K, D), seed + 500 + b)
        if n:
            i = torch.arange(n, device=DEV)
            A.kv4_append(k, v, cache, table[b].long()[i // page] * page + i % page)
        keys.append(ref.quantised(k))
        values.append(ref.quantised(v))
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    q = randn((starts[-1], H, D), seed + 77)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return cache, table, i32(lens), i32(starts), q, keys, values, starts


def close(out, lse, want):
    """Scores: products of exact operands summed in fp32, weights rounded to fp16 or bf16 (2^-9 of each), sums in fp32, one rounding
    of the output to bf16 (2^-9): within 2^-8 of the output and of the sum of p |v|. Log-sum-exp: fp32 scores of a few tens,
    each within 2^-20 of it, and the exponentials' 2^-22."""
    o, l, size = want
    assert torch.equal(torch.isnan(out), torch.isnan(o))
    assert ((out.double() - o).abs() <= (o.abs() + size) * 2.0 ** -8 + 1e-30).nan_to_num(1).logical_or(torch.isnan(o)).all()
    if lse is not None:
        seen = l > -math.inf
        assert (lse[~seen] == -math.inf).all()
        assert ((lse.double() - l)[seen].abs() <= 2.0 ** -16 * (1 + l[seen].abs())).all()


SHAPES = [(1, 1, 64, 16), (8, 8, 64, 32), (6, 2, 128, 16), (8, 1, 128, 64), (16, 1, 128, 16), (10, 2, 256, 16), (16, 2, 256, 64),
          (14, 2, 128, 1024), (5, 1, 64, 16), (16, 1, 64, 128)]
BATCHES = [([1], [1]), ([16], [1]), ([17], [1]), ([777], [1]), ([33, 1, 128, 129, 500], [1] * 5), ([0, 5, 0], [1, 1, 1]),
           ([40, 3], [4, 3]), ([9, 300, 2], [7, 1, 5]), ([64, 70], [0, 2]), ([200, 31, 90], [100, 31, 17])]


@pytest.mark.parametrize("H,K,D,page", SHAPES)
@pytest.mark.parametrize("lens,news", BATCHES)
def test_attention(H, K, D, page, lens, news):
    cache, table, ln, st, q, keys, values, starts = make(lens, news, H, K, D, page, seed=H + D)
    out, lse = A.kv4_attention(q, cache, table, ln, st, max(news), return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, 0, D ** -0.5))


@pytest.mark.parametrize("window", [1, 5, 16, 33, 1000])
@pytest.mark.parametrize("H,K,D", [(8, 2, 64), (4, 1, 128), (16, 2, 256)])
def test_window(window, H, K, D):
    lens, news = [1, 50, 333, 200], [1, 1, 7, 60]
    cache, table, ln, st, q, keys, values, starts = make(lens, news, H, K, D, 16, seed=window)
    out, lse = A.kv4_attention(q, cache, table, ln, st, 60, window=window, scale=0.3, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, window, 0.3))


@pytest.mark.parametrize("H,K,D,n", [(8, 1, 128, 40000), (16, 2, 256, 9000), (4, 4, 64, 20011)])
def test_long_contexts_are_split_and_joined_the_same_way_every_time(H, K, D, n):
    cache, table, ln, st, q, keys, values, starts = make([n, 100], [1, 1], H, K, D, 64, seed=5)
    q = q * 3
    out, lse = A.kv4_attention(q, cache, table, ln, st, 1, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, 0, D ** -0.5))
    for _ in range(5):
        again = A.kv4_attention(q, cache, table, ln, st, 1)
        assert torch.equal(out, again)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news", [1, 3, 90])
def test_values_and_queries_of_very_different_sizes(D, news):
    """Value scales over 2^40, tokens with values of zero that take most of the weight, queries of 2^-20 to 2^6."""
    H, K, n = 4, 2, 400
    cache, table, ln, st, q, _, _, starts = make([n], [news], H, K, D, 16, seed=2)
    k, v = randn((n, K, D), 11), randn((n, K, D), 12)
    v *= torch.exp2(torch.randint(-20, 20, (n, 1, 1), generator=gen(13), device=DEV).float()).to(torch.bfloat16)
    v[7] = 0
    k[7] = q[0, 0] * 0.5
    i = torch.arange(n, device=DEV)
    A.kv4_append(k, v, cache, table[0].long()[i // 16] * 16 + i % 16)
    for size in (2.0 ** -20, 1.0, 64.0):
        x = q * size
        out, lse = A.kv4_attention(x, cache, table, ln, st, news, return_lse=True)
        o, l, s = ref.attention(x, [ref.quantised(k)], [ref.quantised(v)], starts, 0, D ** -0.5)
        assert ((out.double() - o).abs() <= (o.abs() + s) * 2.0 ** -8 + 1e-30).all()
        # scores of up to a thousand: fp32 sums within 2^-18 of the largest term
        top = (x.double().norm(dim=-1).max() * ref.quantised(k).norm(dim=-1).max()) * D ** -0.5
        assert ((lse.double() - l).abs() <= 2.0 ** -16 * (1 + l.abs()) + 2.0 ** -18 * top).all()


@pytest.mark.parametrize("news", [1, 2, 40])
def test_not_finite_keys_and_values_stay_where_they_are_seen(news):
    H, K, D, n = 4, 2, 128, 100
    cache, table, ln, st, q, _, _, starts = make([n], [news], H, K, D, 16, seed=4)
    k, v = randn((n, K, D), 21), randn((n, K, D), 22)
    v[n - 1, 0, 70] = math.nan                               # only the last query sees these
    k[n - 1, 1, 3] = math.inf
    i = torch.arange(n, device=DEV)
    A.kv4_append(k, v, cache, table[0].long()[i // 16] * 16 + i % 16)
    out = A.kv4_attention(q, cache, table, ln, st, news)
    want = ref.attention(q, [ref.quantised(k)], [ref.quantised(v)], starts, 0, D ** -0.5)
    close(out, None, want)
    assert torch.isnan(out[-1, :2, 64:]).all() and torch.isnan(out[-1, 2:]).all() and not torch.isnan(out[-1, :2, :64]).any()
    assert torch.isfinite(out[:-1]).all()


PROMPTS = [([1000], [1000]), ([2500], [70]), ([129, 1, 640, 0, 257], [129, 1, 500, 0, 128]), ([40], [100]), ([3, 900], [70, 300]),
           ([130, 130, 130, 130], [127, 128, 129, 130]), ([5000], [33])]


@pytest.mark.parametrize("H,K,D,page", [(8, 1, 64, 16), (16, 2, 128, 16), (4, 4, 128, 64), (10, 2, 256, 32), (7, 1, 256, 16), (128, 1, 128, 16),
                                        (130, 1, 64, 16)])
@pytest.mark.parametrize("lens,news", PROMPTS)
@pytest.mark.parametrize("window", [0, 100])
def test_prompts(H, K, D, page, lens, news, window):
    cache, table, ln, st, q, keys, values, starts = make(lens, news, H, K, D, page, seed=H + D)
    out, lse = A.kv4_attention(q, cache, table, ln, st, max(news), window=window, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, window, D ** -0.5))


@pytest.mark.parametrize("most", [1, 1000])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-3])
def test_other_scales_and_a_bound_that_is_too_low_or_too_high(most, scale):
    """The bound chooses kernels only; a negative scale prefers what is least alike, a zero scale weighs all the same."""
    H, K, D = 8, 2, 128
    cache, table, ln, st, q, keys, values, starts = make([300, 90], [120, 3], H, K, D, 16, seed=9)
    out, lse = A.kv4_attention(q, cache, table, ln, st, most, scale=scale, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, 0, scale))


@pytest.mark.parametrize("count", [1, 40, 200])
def test_many_values_that_are_not_numbers_in_a_prompt(count):
    """Groups that are not numbers at several places of a prompt: the rows before each do not see it, with a window neither do
    those far behind it."""
    H, K, D, n = 2, 1, 128, 400
    cache, table, ln, st, q, _, _, starts = make([n, n], [n, 300], H, K, D, 16, seed=4)
    k, v = randn((n, K, D), 31), randn((n, K, D), 32)
    v[torch.arange(count, device=DEV) + 150, 0, 70] = math.inf
    i = torch.arange(n, device=DEV)
    for b in range(2):
        A.kv4_append(k, v if b == 0 else k, cache, table[b].long()[i // 16] * 16 + i % 16)
    keys, values = [ref.quantised(k)] * 2, [ref.quantised(v), ref.quantised(k)]
    close(A.kv4_attention(q, cache, table, ln, st, n), None, ref.attention(q, keys, values, starts, 0, D ** -0.5))
    if count <= 40:
        got = A.kv4_attention(q, cache, table, ln, st, n, window=90)
        close(got, None, ref.attention(q, keys, values, starts, 90, D ** -0.5))


def test_attention_out_strides_streams_and_graphs():
    H, K, D = 8, 2, 128
    cache, table, ln, st, q, keys, values, starts = make([300, 65, 900], [1, 1, 1], H, K, D, 16, seed=6)
    want = ref.attention(q, keys, values, starts, 0, D ** -0.5)
    wide = torch.randn(3, H + 4, D, device=DEV).to(torch.bfloat16)
    wide[:, 2:2 + H] = q
    out = torch.full_like(q, math.nan)
    assert A.kv4_attention(wide[:, 2:2 + H], cache, table, ln, st, 1, out=out) is out
    close(out, None, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = A.kv4_attention(q, cache, table, ln, st, 5)
    torch.cuda.current_stream().wait_stream(side)
    close(other, None, want)
    graph, got = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        A.kv4_attention(q, cache, table, ln, st, 1, out=got)
    for _ in range(3):
        got.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


def test_rows_of_no_request_are_left_alone_and_faults_are_reported():
    H, K, D = 4, 1, 64
    cache, table, ln, st, q, keys, values, starts = make([30, 50], [1, 1], H, K, D, 16, seed=8)
    q5 = torch.cat([q, q, q[:1]])
    out = torch.full((5, H, D), 3.0, dtype=torch.bfloat16, device=DEV)
    A.kv4_attention(q5, cache, table, ln, st, 1, out=out)
    assert (out[2:] == 3.0).all()
    want = ref.attention(q, keys, values, starts, 0, D ** -0.5)
    close(out[:2], None, want)
    for name, fault in (("entry", "block-table entry"), ("long", "longer than"), ("offsets", "out of order"), ("length", "negative")):
        t2, l2, s2 = table.clone(), ln.clone(), st.clone()
        if name == "entry":
            t2[1, 0] = cache.num_pages
        elif name == "long":
            l2[1] = 10 ** 6
        elif name == "offsets":
            s2[2] = 9
        else:
            l2[1] = -3
        out = A.kv4_attention(q, cache, t2, l2, s2, 1)
        with pytest.raises(RuntimeError, match=fault):
            A.check_status(DEV)
        close(out[:1], None, [x[:1] for x in want])


def test_the_whole_step_against_its_parts_in_64_bits():
    """Plan, norm with rotation into the cache, attention: two steps of three requests, the second with single tokens."""
    H, K, D, page = 8, 2, 128, 16
    free = torch.randperm(64, generator=gen(1), device=DEV).to(torch.int32)
    table, taken = torch.full((3, 12), -1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    cache = A.KV4Cache.empty(64, K, D, page, DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    w = randn((2, D), 5)
    angle = torch.arange(200, device=DEV)[:, None] * 0.37 ** torch.arange(0, 64, 2, device=DEV)
    cs = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
    cached, keys, values = [0, 0, 0], [[], [], []], [[], [], []]
    for step, news in enumerate(([70, 16, 5], [1, 1, 1])):
        T = sum(news)
        p = A.plan_batch(i32(cached), i32(news), table, free, taken, page, T)
        taken = p.taken
        qkv = randn((T, H + 2 * K, D), 40 + step)
        q = A.qk_norm_rope(qkv[:, :H], qkv[:, H:H + K], w[0], w[1], cs, p.positions, v=qkv[:, H + K:], cache=cache, slots=p.slots)
        out = A.kv4_attention(q, cache, table, p.seq_lens, p.query_start, max(news))
        _, k = A.qk_norm_rope(qkv[:, :H], qkv[:, H:H + K], w[0], w[1], cs, p.positions)
        starts = p.query_start.tolist()
        for b in range(3):
            keys[b].append(ref.quantised(k[starts[b]:starts[b + 1]]))
            values[b].append(ref.quantised(qkv[starts[b]:starts[b + 1], H + K:]))
            cached[b] += news[b]
        close(out, None, ref.attention(q, [torch.cat(x) for x in keys], [torch.cat(x) for x in values], starts, 0, D ** -0.5))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 64])
def test_not_finite_keys_and_values_in_prompts_of_all_head_sizes(D, window):
    H, K, n = 4, 2, 300
    cache, table, ln, st, q, _, _, starts = make([n], [200], H, K, D, 16, seed=14)
    k, v = randn((n, K, D), 41), randn((n, K, D), 42)
    v[n - 1, 0, D - 1] = math.nan                            # only the last query sees these
    v[130, 1, 0] = -math.inf                                 # queries from 130 on, or to 193 with the window
    k[n - 1, 1, 3] = math.inf
    i = torch.arange(n, device=DEV)
    A.kv4_append(k, v, cache, table[0].long()[i // 16] * 16 + i % 16)
    out = A.kv4_attention(q, cache, table, ln, st, 200, window=window)
    close(out, None, ref.attention(q, [ref.quantised(k)], [ref.quantised(v)], starts, window, D ** -0.5))
    bad = torch.isnan(out).flatten(2).any(-1)[:, 2:].any(-1)
    assert not bad[:30].any() and bad[30:94].all() and bad[-1] and (window == 0 or not bad[94:-1].any())


@pytest.mark.parametrize("H,K,D,page", [(8, 2, 64, 16), (16, 2, 128, 32), (16, 2, 256, 16)])
@pytest.mark.parametrize("bound", [0, 7])
def test_batches_of_many_items_of_few_and_many_rows(H, K, D, page, bound):
    """40 (request, KV head) items and more: requests of one token, of a few, and of chunks side by side, some of them empty."""
    news = [1, 5, 6, 40, 0, 11, 1, 3, 64, 17, 10, 2, 1, 33, 5, 1, 0, 12, 9, 30]
    lens = [n + 37 * i * (i % 3) for i, n in enumerate(news)]
    cache, table, ln, st, q, keys, values, starts = make(lens, news, H, K, D, page, seed=D)
    out, lse = A.kv4_attention(q, cache, table, ln, st, max(news) + bound, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, 0, D ** -0.5))


@pytest.mark.parametrize("H,K,D", [(2, 1, 64), (4, 2, 128), (2, 1, 256)])
def test_chunks_over_long_contexts_are_joined_the_same_way_every_time(H, K, D):
    cache, table, ln, st, q, keys, values, starts = make([9000, 300], [150, 270], H, K, D, 64, seed=15)
    q = q * 3
    out, lse = A.kv4_attention(q, cache, table, ln, st, 270, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, 0, D ** -0.5))
    for _ in range(5):
        assert torch.equal(out, A.kv4_attention(q, cache, table, ln, st, 270))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_reading_into_outputs_on_16_byte_boundaries(D):
    """The C ABI takes outputs on any 16-byte boundary; those on 32 are written in wider pieces."""
    lib = ctypes.CDLL(A.attention_lib_path())
    K, n = 3, 37
    cache = A.KV4Cache.empty(4, K, D, 16, DEV)
    k, v, slots = randn((n, K, D), 1), randn((n, K, D), 2), torch.randperm(64, generator=gen(3), device=DEV)[:n].contiguous()
    A.kv4_append(k, v, cache, slots)
    want = A.kv4_read(cache, slots)
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    room = torch.full((2, n * K * D + 16), 7.0, dtype=torch.bfloat16, device=DEV)
    got = [x[8:8 + n * K * D] for x in room]
    assert got[0].data_ptr() % 32 == 16
    rc = lib.mono_attn_kv4_read(p(cache.data), ctypes.c_int64(4), 16, p(slots), n, K, D, p(got[0]), p(got[1]), p(status),
                                ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0 and torch.equal(got[0].view(n, K, D), want[0]) and torch.equal(got[1].view(n, K, D), want[1])
    assert (room[:, :8] == 7).all() and (room[:, 8 + n * K * D:] == 7).all() and not status.any()
