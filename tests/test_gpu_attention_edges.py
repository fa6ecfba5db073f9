"""The attention operators where something is missing, not finite or out of range, in shapes that the tests by size do not have."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

from tests import attention_ref as ref
from tests.test_gpu_attention import DEV, _rope_inputs, close, gen, make, randn
from unimonomoe_b200 import attention as A

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status():
    yield
    A.check_status(DEV)


def store(cache, table, b, k, v, page):
    """Keys and values of request b, from its first token on."""
    i = torch.arange(len(k), device=DEV)
    A.kv4_append(k, v, cache, table[b].long()[i // page] * page + i % page)


# ---------------------------------------------------------------------- values that are not numbers
@pytest.mark.parametrize("H,K,D", [(4, 4, 64), (8, 2, 64), (8, 4, 128), (16, 2, 128), (8, 4, 256)])
@pytest.mark.parametrize("window", [0, 40])
def test_values_that_are_not_numbers_in_many_short_prompts(H, K, D, window):
    """CTAs have many items of a single tile of keys one after another: a group that is not a number reaches the rows of its own
    request that see it, all of them, and no other request's."""
    count = 500
    lens = [60 + (37 * i) % 69 for i in range(count)]
    cache, table, ln, st, q, keys, values, starts = make(lens, lens, H, K, D, 16, seed=D + K)
    for b in range(0, count, 3):
        v = randn((lens[b], K, D), 500 + D + K + b)          # what make() has stored, with one value in it that is not finite
        at, head, dim = (11 * b) % lens[b], b % K, (29 * b) % D
        v[at, head, dim] = (math.nan, math.inf, -math.inf)[b % 3]
        store(cache, table, b, randn((lens[b], K, D), 100 + D + K + b), v, 16)
        values[b] = ref.quantised(v)
    want = ref.attention(q, keys, values, starts, window, D ** -0.5)
    assert torch.isnan(want[0]).any()
    for _ in range(3):
        out, lse = A.kv4_attention(q, cache, table, ln, st, 128, window=window, return_lse=True)
        close(out, lse, want)


@pytest.mark.parametrize("H,K,D", [(2, 1, 64), (8, 1, 128), (8, 2, 256)])
@pytest.mark.parametrize("window", [0, 60, 97])
def test_values_that_are_not_numbers_far_apart_in_a_window(H, K, D, window):
    """Two hundred of them in two places: with a window the rows between see none."""
    n = 500
    cache, table, ln, st, q, keys, values, starts = make([n, n], [n, 300], H, K, D, 16, seed=D)
    for b in range(2):
        v = randn((n, K, D), 500 + D + b)
        v[60:160, 0, 3] = math.inf
        v[390:490, K - 1, D - 1] = math.nan
        store(cache, table, b, randn((n, K, D), 100 + D + b), v, 16)
        values[b] = ref.quantised(v)
    want = ref.attention(q, keys, values, starts, window, D ** -0.5)
    close(A.kv4_attention(q, cache, table, ln, st, n, window=window), None, want)
    assert window == 0 or not torch.isnan(want[0][260:390]).any()


# ---------------------------------------------------------------------- pages that are not there
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("H,K,D", [(2, 2, 64), (16, 2, 128), (8, 2, 256)])
@pytest.mark.parametrize("news", [[1, 2], [5, 1], [150, 70], [300, 40]])
@pytest.mark.parametrize("window", [1, 30, 200])
def test_pages_before_the_window_may_be_gone(page, H, K, D, news, window):
    """A server that gives back what no later token sees: its entries are -1, and nothing is reported."""
    lens = [n + 600 + 77 * i for i, n in enumerate(news)]
    cache, table, ln, st, q, keys, values, starts = make(lens, news, H, K, D, page, seed=D)
    for b, (n, m) in enumerate(zip(lens, news)):
        table[b, :max(n - m + 1 - window, 0) // page] = -1
    out, lse = A.kv4_attention(q, cache, table, ln, st, max(news), window=window, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, window, D ** -0.5))
    A.check_status(DEV)


@pytest.mark.parametrize("H,K,D", [(8, 2, 64), (16, 2, 128), (10, 2, 256)])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
@pytest.mark.parametrize("news", [1, 3, 250])
def test_a_missing_page_is_zeros_and_no_other_requests_page(H, K, D, entry, news):
    lens = [400, 400]
    cache, table, ln, st, q, keys, values, starts = make(lens, [news] * 2, H, K, D, 32, seed=D)
    for b, col in ((0, 2), (0, 3), (1, 12)):
        table[b, col] = entry
        keys[b][32 * col:32 * (col + 1)] = 0
        values[b][32 * col:32 * (col + 1)] = 0
    out, lse = A.kv4_attention(q, cache, table, ln, st, news, return_lse=True)
    with pytest.raises(RuntimeError, match="block-table entry"):
        A.check_status(DEV)
    close(out, lse, ref.attention(q, keys, values, starts, 0, D ** -0.5))


def test_plan_without_pages_enters_none():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table = i32([[1, 90, 91, 92], [2, 93, 94, 95]])            # both rows hold what earlier requests had
    p = A.plan_batch(i32([16, 16]), i32([20, 17]), table, i32([5, 6, 7]), i32([0]), 16, 37)
    with pytest.raises(RuntimeError, match="more pages"):
        A.check_status(DEV)
    assert table.tolist() == [[1, 5, 6, 92], [2, 7, -1, 95]] and p.taken.tolist() == [4]
    assert p.slots.tolist() == [*range(80, 100), *range(112, 128), -1]


# ---------------------------------------------------------------------- scales
@pytest.mark.parametrize("H,K,D", [(4, 2, 64), (12, 2, 128), (10, 2, 256)])
@pytest.mark.parametrize("lens,news", [([700, 3], [1, 1]), ([300, 9], [5, 7]), ([260, 200], [250, 200])])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-38, -1e-30, 0.1])
def test_no_scale_and_queries_of_next_to_nothing_weigh_all_alike(H, K, D, lens, news, scale):
    cache, table, ln, st, q, keys, values, starts = make(lens, news, H, K, D, 16, seed=D)
    q[:, ::3] = 0
    q[:, 1::3] *= 2.0 ** -115
    for window in (0, 6):
        out, lse = A.kv4_attention(q, cache, table, ln, st, max(news), scale=scale, window=window, return_lse=True)
        close(out, lse, ref.attention(q, keys, values, starts, window, scale))


# ---------------------------------------------------------------------- the status word, graphs
FIRST_CALL_IN_A_CAPTURE = """
import torch
from unimonomoe_b200 import attention as A
dev = torch.device("cuda:0")
junk = [torch.full((1 << k,), -1, dtype=torch.int32, device=dev) for k in range(1, 24)]     # what a word made from freed memory would hold
del junk
x = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=dev)
cache = A.KV4Cache(torch.zeros(2, 1, 1, 17 * 64, dtype=torch.uint8, device=dev))
good, bad = torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), 99, dtype=torch.int64, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    k, v = A.kv4_read(cache, good)                           # the first call of the process
A.check_status(dev)                                          # nothing has run yet
def faulty():
    A.kv4_append(x, x, cache, bad)
def told():
    try:
        A.check_status(dev)
    except RuntimeError as e:
        assert "slot outside" in str(e), e
        return True
    return False
graph.replay()
assert not told()
faulty()
graph.replay()
assert told() and not told()
graph.replay()
faulty()
assert told() and not told()
print("fine")
"""


def test_the_first_call_of_a_process_may_be_captured():
    got = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert got.returncode == 0 and got.stdout.strip() == "fine", got.stdout + got.stderr


def test_graphs_captured_on_a_stream_without_a_workspace_run_one_after_another():
    H, K, D = 8, 2, 128
    cache, table, ln, st, q, keys, values, starts = make([3000, 900], [1, 60], H, K, D, 16, seed=6)
    want = [A.kv4_attention(x, cache, table, ln, st, 60) for x in (q, -q)]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    for x in (q, -q):
        graphs.append(torch.cuda.CUDAGraph())
        outs.append(torch.full_like(q, math.nan))
        with torch.cuda.graph(graphs[-1], stream=stream):
            A.kv4_attention(x, cache, table, ln, st, 60, out=outs[-1])
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            out.fill_(math.nan)
            graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---------------------------------------------------------------------- refusals
def _views():
    data = torch.zeros(4, 2, 2, 17 * 64, dtype=torch.uint8, device=DEV)
    yield "every other page", data[::2]
    yield "one page many times", data[:1].expand(9, -1, -1, -1)
    yield "half of the heads", data[:, :1]
    yield "flat", data.flatten(2)
    yield "another type", data.view(torch.int8)
    yield "no pages", data[:0]
    yield "a page size of 48", torch.zeros(4, 2, 3, 17 * 64, dtype=torch.uint8, device=DEV)
    yield "a page size of 2048", torch.zeros(1, 2, 128, 17 * 64, dtype=torch.uint8, device=DEV)
    yield "a head size of 96", torch.zeros(4, 2, 1, 17 * 96, dtype=torch.uint8, device=DEV)
    yield "not 17 bytes a dim", torch.zeros(4, 2, 1, 17 * 64 + 8, dtype=torch.uint8, device=DEV)
    yield "off its boundary", torch.zeros(4 * 2 * 17 * 64 + 8, dtype=torch.uint8, device=DEV)[8:].view(4, 2, 1, 17 * 64)


@pytest.mark.parametrize("what", ["every other page", "one page many times", "half of the heads", "flat", "another type", "no pages", "a page size of 48",
                                  "a page size of 2048", "a head size of 96", "not 17 bytes a dim", "off its boundary"])
def test_what_is_not_a_cache_is_refused_by_every_operator(what):
    class Looks:                                             # anything with `data`, as a tensor has too
        pass
    cache = Looks()
    cache.data = dict(_views())[what]
    x, slots = randn((1, 2, 64), 1), torch.zeros(1, dtype=torch.int64, device=DEV)
    one, w, cs = torch.ones(1, dtype=torch.int32, device=DEV), randn((64,), 2), torch.ones(4, 64, device=DEV)
    start = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for c in (cache, cache.data):
        for call in (lambda: A.kv4_append(x, x, c, slots), lambda: A.kv4_read(c, slots),
                     lambda: A.qk_norm_rope(x, x, w, w, cs, one, v=x, cache=c, slots=slots),
                     lambda: A.kv4_attention(x, c, one[None], one, start, 1)):
            with pytest.raises(ValueError):
                call()


# ---------------------------------------------------------------------- plans of what cannot be
def raw_plan(cached, new, table, free, taken, page, tokens):
    """The C entry with every output, and the table, inside one buffer of 0x5A bytes, 256 to each side: (outputs, table, what was reported); nothing else has
    been written."""
    lib = ctypes.CDLL(A.attention_lib_path())
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    batch, width = len(cached), len(table[0])
    sizes = {"table": 4 * batch * width, "start": 4 * (batch + 1), "lens": 4 * batch, "positions": 4 * tokens, "slots": 8 * tokens, "requests": 4 * tokens,
             "taken": 4}
    room = torch.full((sum(256 + (n + 255) // 256 * 256 for n in sizes.values()) + 256,), 0x5A, dtype=torch.uint8, device=DEV)
    view, at, mine = {}, 256, torch.zeros(room.numel(), dtype=torch.bool, device=DEV)
    for name, n in sizes.items():
        view[name] = room[at:at + n].view(torch.int64 if name == "slots" else torch.int32)
        mine[at:at + n] = True
        at += (n + 255) // 256 * 256 + 256
    view["table"].copy_(i32(table).flatten())
    given = i32(cached), i32(new), i32(free), i32([taken])
    status = torch.zeros(2, dtype=torch.int32, device=DEV)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rc = lib.mono_attn_plan(p(given[0]), p(given[1]), batch, p(view["table"]), width, p(given[2]), len(free), p(given[3]), page, tokens, p(view["start"]),
                            p(view["lens"]), p(view["positions"]), p(view["slots"]), p(view["requests"]), p(view["taken"]), p(status),
                            ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    got = {name: x.tolist() for name, x in view.items()}
    assert (room[~mine] == 0x5A).all()
    return got, [got["table"][i * width:(i + 1) * width] for i in range(batch)], A.STATUS_CODES[status.tolist()[0]]


TOP = 2 ** 31 - 1


@pytest.mark.parametrize("cached,new,taken,said", [
    ([TOP], [1], 0, "longer"), ([TOP - 20], [40], 0, "longer"), ([TOP - 16], [TOP], 0, "longer"), ([0, TOP - 5], [TOP, TOP], 0, ""),
    ([40] * 1100, [TOP - 70000] * 1100, 0, ""), ([40] * 600, [2 ** 22] * 600, 0, ""), ([3, 70], [20, 5], TOP, "more pages"),
    ([3, 70], [20, 5], -TOP, "more pages"), ([3, 70], [20, 5], -1, "more pages"), ([TOP - 70000, 3], [60000, 20], TOP, "")])
@pytest.mark.parametrize("page", [16, 1024])
def test_lengths_at_the_end_of_32_bits_stay_in_bounds(cached, new, taken, said, page):
    width, tokens = 6, 200
    table = [[1, 2, 3, 4, 5, 6]] * len(cached)
    got, after, told = raw_plan(cached, new, table, [7, 8, 9], taken, page, tokens)
    assert said in told and told != "ok"
    assert all(-1 <= s < 10 * page for s in got["slots"])
    assert all(0 <= p < 2 ** 31 for p in got["positions"]) and all(-1 <= r < len(cached) for r in got["requests"])
    assert got["start"][0] == 0 and got["start"] == sorted(got["start"]) and all(0 <= n < 2 ** 31 for n in got["lens"])
    assert all(e in range(-1, 10) for row in after for e in row)


@pytest.mark.parametrize("what,code", [("pages", "more pages"), ("table", "longer than"), ("tokens", "more tokens"), ("negative", "negative"),
                                       ("entry", "block-table entry")])
def test_plan_faults_touch_nothing_but_the_outputs(what, code):
    cached, new, free, tokens, width = [10, 40], [20, 30], [5, 6, 7, 8], 50, 5
    table = [[1, -1, -1, -1, -1], [2, 3, 4, -1, -1]]
    want = [[1, 5, -1, -1, -1], [2, 3, 4, 6, 7]]
    if what == "pages":
        free, want[1][4] = [5, 6], -1
    elif what == "table":
        width, table, want = 4, [r[:4] for r in table], [r[:4] for r in want]
    elif what == "tokens":
        tokens = 49
    elif what == "negative":
        new, want[1][3:] = [20, -30], [-1, -1]
    elif what == "entry":
        table[0][0] = want[0][0] = -1
    got, after, told = raw_plan(cached, new, table, free, 0, 16, tokens)
    assert code in told and after == want
    ref_table = [r[:] for r in table]
    if what == "tokens":                                     # all but the token that has no row
        start, lens, pos, slot, req, taken = ref.plan(cached, new, ref_table, free, 0, 16, 50)
        assert (got["start"], got["lens"], got["positions"], got["slots"], got["requests"], got["taken"]) == (start, lens, pos[:49], slot[:49], req[:49], [taken])


# ---------------------------------------------------------------------- sizes past 32 bits
def test_more_rows_than_32_bits_of_threads():
    """2^28 + 5 tokens of one head of 256, the same row for all of them (strides of 0), of which a few are stored."""
    T = 2 ** 28 + 5
    cache = A.KV4Cache.empty(1, 1, 256, 16, DEV)
    cache.data.fill_(0x88)
    k, v = randn((1, 1, 256), 1), randn((1, 1, 256), 2)
    slots = torch.full((T,), -1, dtype=torch.int64, device=DEV)
    for i, at in enumerate((0, T // 2 - 1, T // 2, T // 2 + 1, T - 2, T - 1)):
        slots[at] = 2 * i
    A.kv4_append(k.expand(T, 1, 256), v.expand(T, 1, 256), cache, slots)
    got = A.kv4_read(cache, torch.arange(12, device=DEV))
    for x, y in zip(got, (k, v)):
        assert torch.equal(x[::2].double(), ref.quantised(y).expand(6, 1, 256))


@pytest.mark.parametrize("news", [1, 200])
def test_a_cache_of_more_than_4_gib(news):
    """Pages on both sides of byte 2^32 and of element 2^32 / 2, read and written by every operator."""
    H, K, D, page, n = 8, 2, 128, 1024, 5000
    pages = 2 ** 32 // (K * page * 17 * D // 16) + 40            # of 278 528 bytes
    cache = A.KV4Cache.empty(pages, K, D, page, DEV)
    assert cache.data.numel() > 2 ** 32
    edge = [i * 2 ** 31 // (K * page * 17 * D // 16) for i in (1, 2)]
    table = torch.tensor([[edge[0], pages - 1, edge[1], edge[1] + 1, edge[0] + 1, 0]], dtype=torch.int32, device=DEV)
    i = torch.arange(n, device=DEV)
    slots = table[0].long()[i // page] * page + i % page
    k, v, q = randn((n, K, D), 1), randn((n, K, D), 2), randn((news, H, D), 3)
    cs, w = torch.cat([torch.ones(1, 32, device=DEV), torch.zeros(1, 32, device=DEV)], 1), randn((D,), 4)
    A.kv4_append(k[1000:], v[1000:], cache, slots[1000:])
    raw = randn((1000, K, D), 5)                                # the first page's keys come by way of their norm
    zeros = torch.zeros(1000, dtype=torch.int32, device=DEV)
    _, k0 = A.qk_norm_rope(raw, raw, w, w, cs, zeros)
    A.qk_norm_rope(raw, raw, w, w, cs, zeros, v=v[:1000], cache=cache, slots=slots[:1000])
    keys, values = ref.quantised(torch.cat([k0, k[1000:]])), ref.quantised(v)
    got = A.kv4_read(cache, slots)
    assert torch.equal(got[0].double(), keys) and torch.equal(got[1].double(), values)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out, lse = A.kv4_attention(q, cache, table, i32([n]), i32([0, news]), news, return_lse=True)
    close(out, lse, ref.attention(q, [keys], [values], [0, news], 0, D ** -0.5))


# ---------------------------------------------------------------------- norms and rotation
@pytest.mark.parametrize("D,R", [(64, 0), (64, 32), (128, 48), (256, 64), (256, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_an_infinity_reaches_what_turns_with_it_and_nothing_else(D, R, interleaved):
    q, k = randn((D, 3, D), D), randn((D, 1, D), D + 1)
    i = torch.arange(D, device=DEV)
    q[i, 1, i], k[i, 0, i] = math.inf, -math.inf                # token t: dim t
    q[5, 0, 7] = math.nan
    w = randn((2, D), 3)
    angle = torch.rand(9, R // 2, generator=gen(4), device=DEV) + 0.1
    table, pos = torch.cat([angle.cos(), angle.sin()], 1).contiguous(), torch.randint(0, 9, (D,), generator=gen(5), device=DEV).to(torch.int32)
    for got, x, y in zip(A.qk_norm_rope(q, k, w[0], w[1], table, pos, 1e-6, interleaved), (q, k), w):
        want = ref.norm_rope(x, y, table, pos, 1e-6, interleaved, False)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        bad = torch.isinf(x).any(-1)
        assert not got[bad].nan_to_num(0.0).any()


@pytest.mark.parametrize("D,H,K,R,T", [(64, 4, 1, 64, 7), (64, 5, 5, 16, 33), (128, 7, 3, 48, 19), (128, 32, 4, 128, 3), (256, 16, 2, 64, 9)])
@pytest.mark.parametrize("fp32", [False, True])
def test_neighbours_into_the_cache_are_append_of_their_results(D, H, K, R, T, fp32):
    q, k, v, wq, wk, table, pos = _rope_inputs(D, H, K, R, T, fp32)
    caches = [A.KV4Cache.empty(T // 32 + 2, K, D, 32, DEV) for _ in range(2)]
    slots = torch.randperm((T // 32 + 2) * 32, generator=gen(1), device=DEV)[:T]
    slots[1] = -1
    for c in caches:
        c.data.zero_()
    q1, k1 = A.qk_norm_rope(q, k, wq, wk, table, pos, 1e-5, True, True)
    A.kv4_append(k1, v, caches[0], slots)
    q2 = A.qk_norm_rope(q, k, wq, wk, table, pos, 1e-5, True, True, v=v, cache=caches[1], slots=slots)
    assert torch.equal(q1, q2) and torch.equal(caches[0].data, caches[1].data)


def test_more_steps_than_32_bits_are_reported_and_not_begun():
    B, K, D, page, width = 16384, 8, 64, 1024, 5000              # 2.6e9 steps of 256 tokens, all in one page
    cache = A.KV4Cache(torch.zeros(1, K, page // 16, 17 * D, dtype=torch.uint8, device=DEV))
    table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    lens = torch.full((B,), width * page, dtype=torch.int32, device=DEV)
    out = torch.full((B, K, D), 3.0, dtype=torch.bfloat16, device=DEV)
    A.kv4_attention(torch.zeros_like(out), cache, table, lens, torch.arange(B + 1, dtype=torch.int32, device=DEV), 1, out=out)
    with pytest.raises(RuntimeError, match="longer than"):
        A.check_status(DEV)
    assert (out == 3.0).all()


@pytest.mark.parametrize("news", [1, 100])
@pytest.mark.parametrize("window", [400, 4096, 2 ** 31, 2 ** 62])
def test_windows_as_wide_as_the_sequence_and_wider(news, window):
    H, K, D = 8, 2, 128
    cache, table, ln, st, q, keys, values, starts = make([400], [news], H, K, D, 16, seed=3)
    out, lse = A.kv4_attention(q, cache, table, ln, st, news, window=window, return_lse=True)
    close(out, lse, ref.attention(q, keys, values, starts, 0, D ** -0.5))


FIRST_CALL_IN_INFERENCE_MODE = """
import torch
from unimonomoe_b200 import attention as A
dev = torch.device("cuda:0")
x = torch.ones(1, 1, 64, dtype=torch.bfloat16, device=dev)
cache, bad = A.KV4Cache.empty(2, 1, 64, 16, dev), torch.full((1,), 99, dtype=torch.int64, device=dev)
def told():
    try:
        A.check_status(dev)
    except RuntimeError as e:
        assert "slot outside" in str(e), e
        return True
    return False
with torch.inference_mode():
    A.kv4_append(x, x, cache, bad)                           # the first call of the process
assert told() and not told()
A.kv4_append(x, x, cache, bad)
with torch.inference_mode():
    assert told() and not told()
print("fine")
"""


def test_the_first_call_of_a_process_may_be_in_inference_mode():
    got = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_INFERENCE_MODE], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert got.returncode == 0 and got.stdout.strip() == "fine", got.stdout + got.stderr
