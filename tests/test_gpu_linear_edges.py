"""The block-FP8 operators where values are not finite, numbers from the device are wrong, calls overlap, are captured or are very large."""
import math

import pytest
import torch

from tests import linear_ref as ref
from tests.test_gpu_linear import gen, routed
from unimonomoe_b200 import (ExpertPlan, combine_experts, fp8_expert_linear, fp8_linear, fp8_quantize, moe_experts,
                             plan_experts)
from unimonomoe_b200.linear import check_status

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_fault(linear_lib):
    yield
    check_status()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), 7e30), torch.nan_to_num(b.float(), 7e30)) and torch.equal(a.isnan(), b.isnan())


# ---------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_group_that_is_not_finite_is_nan_and_no_other(value):
    x = ref.states(6, 400, gen(1)).cuda()
    clean = fp8_quantize(x)
    x[2, 130], x[4, 399] = value, value
    q, s = fp8_quantize(x)
    bad = torch.zeros(6, 4, dtype=torch.bool)
    bad[2, 1] = bad[4, 3] = True
    assert torch.equal(s.isnan().cpu(), bad)
    keep = ~ref.spread(bad, 400).cuda()
    assert torch.equal(q.view(torch.uint8)[keep], clean[0].view(torch.uint8)[keep]) and torch.equal(s[~bad.cuda()], clean[1][~bad.cuda()])
    y = ref.states(6, 800, gen(2)).cuda()
    y[3, 5], y[1, 405] = value, value        # half a of group 0, half b of group 0
    s = fp8_quantize(y, silu_mul=True)[1]
    # a / (1 + exp(-a)) is the quotient of two infinities where a is -inf
    assert s[1, 0].isnan() and s[3, 0].isnan() and int(s.isnan().sum()) == 2


@pytest.mark.parametrize("m", [7, 40, 1500])
@pytest.mark.parametrize("silu", [False, True])
def test_a_row_that_is_not_finite_reaches_its_own_results(m, silu):
    g = gen(m, 3)
    w, ws = (t.cuda() for t in ref.weight(512, 640, g))
    x = ref.states(m, 640, g).cuda()
    clean = fp8_linear(x, w, ws, silu_mul=silu)
    x[m - 3, 200], x[1, 639] = math.nan, math.inf
    got = fp8_linear(x, w, ws, silu_mul=silu)
    rows = torch.ones(m, dtype=torch.bool)
    rows[m - 3] = rows[1] = False
    for a, b in zip(got, clean) if silu else [(got, clean)]:
        assert torch.equal(a[rows].view(torch.uint8), b[rows].view(torch.uint8))
    assert bool((got[1] if silu else got)[~rows].isnan().all())
    w.view(torch.uint8)[300, 17] = 0x7F       # NaN in a row of the weight
    got = fp8_linear(x[rows], w, ws)
    assert bool(got[:, 300].isnan().all()) and int(got.isnan().sum()) == int(rows.sum())


def test_rows_that_are_not_finite_stay_with_their_expert():
    g = gen(9)
    for tokens, experts in ((12, 16), (900, 4)):
        ids = routed(tokens, 2, experts, g).cuda()
        w, ws = (t.cuda() for t in ref.weight(256, 256, g, (experts,)))
        x = ref.states(tokens, 256, g).cuda()
        plan = plan_experts(ids, experts)
        clean = fp8_expert_linear(x, w, ws, plan)
        x[5] = math.nan
        got = fp8_expert_linear(x, w, ws, plan)
        hit = plan.tokens == 5
        assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("m", [1, 9, 30, 60])
@pytest.mark.parametrize("k", [128, 384, 1040])
def test_infinite_scales_are_infinite_results(m, k):
    """Of an odd number of groups the last one has an infinite scale: sums of one sign, so that nothing of it is NaN."""
    g = k // 128 + (k % 128 > 0)
    x = torch.ones(m, k, device="cuda").to(ref.E4M3)
    w = torch.ones(200, k, device="cuda").to(ref.E4M3)
    xs, ws = torch.ones(m, g, device="cuda"), torch.ones(2, g, device="cuda")
    ws[1, -1] = math.inf
    got = fp8_linear(x, w, ws, x_scale=xs)
    assert bool((got[:, 128:] == math.inf).all()) and bool((got[:, :128] == k).all())
    assert torch.equal(fp8_linear(torch.ones(m, k, dtype=torch.bfloat16, device="cuda"), w, ws).isinf(), got.isinf())
    xs[0, -1], ws[1, -1] = math.inf, 1.0
    got = fp8_linear(x, w, ws, x_scale=xs)
    assert bool((got[0] == math.inf).all()) and bool((got[1:] == k).all())


def test_one_row_whose_values_lie_apart():
    x = ref.states(1, 1024, gen(5)).cuda()[0]
    for a, b in zip(fp8_quantize(x[::2]), fp8_quantize(x[::2].contiguous())):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    w, ws = (t.cuda() for t in ref.weight(256, 512, gen(6)))
    assert torch.equal(fp8_linear(x[::2], w, ws), fp8_linear(x[::2].contiguous(), w, ws))
    assert torch.equal(fp8_linear(x[:512].expand(3, 512), w, ws), fp8_linear(x[:512].repeat(3, 1), w, ws))


def test_gates_of_every_size():
    """Every finite value as the gate of 1 and of 2^60, one to a group, so that its scale shows the product: off by the roundings of the exponential
    (2 + 1.2 |a| units of 2^-24 at most), the sum, quotient, product and scale (8 units); below -88.72 it is nothing, however large a and b are."""
    a = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    a = a[torch.isfinite(a)]
    for b in (1.0, 2.0 ** 60):
        x = torch.zeros(len(a), 256, dtype=torch.bfloat16)
        x[:, 0], x[:, 128] = a, b
        m = fp8_quantize(x.cuda(), silu_mul=True)[1][:, 0].double().cpu() * 448
        v = (a.double() * torch.sigmoid(a.double()) * b).abs()
        plain = (a > -88.5) & (v > 2.0 ** -99) & (v < 2.0 ** 127)
        assert bool(((m - v).abs()[plain] <= (v * (10 + 1.2 * a.double().abs().clamp(max=90)) * 2.0 ** -24)[plain]).all())
        assert bool(((m - 1).abs()[(a < -88.72) | (v < 2.0 ** -101)] <= ref.HALF32).all())          # 1 / 448, rounded, times 448
    x[:, 128] = 3e38
    a = a[a < -88.72]
    x = x[:len(a)]
    x[:, 0] = a
    m = fp8_quantize(x.cuda(), silu_mul=True)[1][:, 0].double() * 448
    assert bool(((m - 1).abs() <= ref.HALF32).all())


def test_groups_of_next_to_nothing_and_of_very_much():
    x = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    x[0, :128], x[0, 128:256], x[0, 256:384] = 1e-39, 2.0 ** -100, 2.0 ** -101
    x[1, :128], x[1, 200] = 3e38, -3.3e38
    q, s = fp8_quantize(x)
    wq, wsc = ref.codes32(x.float().cpu())
    assert torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s.cpu(), wsc)
    assert bool(torch.isfinite(s).all()) and bool((q[0, 256:].float() == 0).all()) and bool((q[0, 128:256].float() == 448).all())
    w = torch.eye(512, device="cuda").to(ref.E4M3)
    y = fp8_linear(x, w, torch.ones(4, 4, device="cuda"), out_dtype=torch.float32)
    assert torch.equal(y, ref.values(q, s).float()) and bool((y[2:] == 0).all())


def test_zero_times_a_row_of_the_plan():
    """A weight of zero still multiplies; a slot that is elsewhere does not."""
    partial = torch.full((2, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    pos = torch.tensor([[0, -1], [-1, -1]], dtype=torch.int32, device="cuda")
    got = combine_experts(partial, pos, torch.zeros(2, 2, device="cuda"))
    assert bool(got[0].isnan().all()) and bool((got[1] == 0).all())


# ---------------------------------------------------------------------- wrong numbers on the device
def reported(text):
    with pytest.raises(RuntimeError, match=text):
        check_status()


@pytest.mark.parametrize("dtype,value", [(torch.int32, 8), (torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 40)])
@pytest.mark.parametrize("tokens", [40, 3000])
def test_ids_past_the_last_expert_are_nowhere_and_reported(dtype, value, tokens):
    ids = torch.randint(0, 8, (tokens, 3), generator=gen(tokens)).to(dtype)
    want = ids.clone()
    ids[17, 1], want[17, 1] = value, -1
    for a, b in zip(plan_experts(ids.cuda(), 8), ref.plan(want, 8)):
        assert torch.equal(a.cpu().long(), b)
    reported("past the last expert")
    ids[17, 1] = -(2 ** 31) if dtype == torch.int32 else -(2 ** 62)
    assert int(plan_experts(ids.cuda(), 8).positions[17, 1]) == -1


@pytest.mark.parametrize("tokens", [30, 2000])
@pytest.mark.parametrize("change", [(2, 1000000), (2, -5), (4, 1000000), (0, -1), (1, 2 ** 31 - 1)])
@pytest.mark.parametrize("silu", [False, True])
def test_offsets_out_of_order_compute_nothing_and_are_reported(tokens, change, silu):
    g = gen(tokens, 4)
    w, ws = (t.cuda() for t in ref.weight(256, 128, g, (4,)))
    plan = plan_experts(routed(tokens, 2, 4, g).cuda(), 4)
    good = fp8_expert_linear(ref.states(tokens, 128, gen(1)).cuda(), w, ws, plan, silu_mul=silu)
    offsets = plan.offsets.clone()
    offsets[change[0]] = change[1]
    fp8_expert_linear(ref.states(tokens, 128, gen(1)).cuda(), w, ws, ExpertPlan(offsets, plan.tokens, plan.positions), silu_mul=silu)
    reported("offsets")
    again = fp8_expert_linear(ref.states(tokens, 128, gen(1)).cuda(), w, ws, plan, silu_mul=silu)
    for a, b in zip(again, good) if silu else [(again, good)]:
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("tokens", [30, 2000])
@pytest.mark.parametrize("value", [-1, 1000000, -(2 ** 31)])
def test_rows_that_x_does_not_have_are_reported(tokens, value):
    g = gen(tokens, 6)
    w, ws = (t.cuda() for t in ref.weight(384, 256, g, (4,)))
    x, plan = ref.states(tokens, 256, g).cuda(), plan_experts(routed(tokens, 2, 4, g).cuda(), 4)
    good = fp8_expert_linear(x, w, ws, plan)
    rows = plan.tokens.clone()
    rows[7] = value
    got = fp8_expert_linear(x, w, ws, ExpertPlan(plan.offsets, rows, plan.positions))
    reported("row outside")
    keep = torch.arange(tokens * 2, device="cuda") != 7
    assert torch.equal(got[keep], good[keep])


def test_positions_past_the_partial_rows_add_nothing_and_are_reported():
    g = gen(8)
    partial, pos = ref.states(20, 64, g), torch.randint(0, 20, (10, 2), generator=g).to(torch.int32)
    wt = torch.rand(10, 2, generator=g)
    bad = pos.clone()
    bad[3, 1], pos[3, 1] = 20, -1
    got = combine_experts(partial.cuda(), bad.cuda(), wt.cuda())
    reported("position")
    assert torch.equal(got, combine_experts(partial.cuda(), pos.cuda(), wt.cuda()))


# ---------------------------------------------------------------------- streams, graphs, what comes before and after
def layer(tokens, seed):
    g = gen(tokens, seed, 77)
    experts, inter, hidden, top = 8, 256, 512, 2
    (w13, s13), (w2, s2) = ref.weight(2 * inter, hidden, g, (experts,)), ref.weight(hidden, inter, g, (experts,))
    return [t.cuda() for t in (ref.states(tokens, hidden, g), routed(tokens, top, experts, g), torch.rand(tokens, top, generator=g), w13, s13, w2, s2)]


@pytest.mark.parametrize("m,n,k", [(1, 640, 512), (30, 640, 512), (70, 2048, 1024), (2000, 640, 512)])
def test_what_is_written_just_before_is_read(m, n, k):
    """Weights, scales, rows and residual change on the stream right before the call, and its result is used right behind it: the product
    begins while the rows are still being quantised."""
    g = gen(m, n)
    w, ws = (t.cuda() for t in ref.weight(n, k, g))
    x, res = ref.states(m, k, g).cuda(), ref.states(m, n, g).cuda()
    sets, wants = [], []
    for i in range(6):
        sets.append((w.view(torch.uint8).roll(i, 0), ws * (1 + i), x.roll(i, 1), res.roll(3 * i, 1)))
        wants.append(fp8_linear(sets[i][2], sets[i][0], sets[i][1], residual=sets[i][3]))
        torch.cuda.synchronize()
    a, b, c, d = (torch.empty_like(t) for t in sets[0])
    big = torch.empty(1 << 26, device="cuda")
    got = []
    for i in range(48):
        if i % 12 == 0:
            big.zero_()                      # the launches queue up behind it
        for to, t in zip((a, b, c, d), sets[i % 6]):
            to.copy_(t)
        got.append(fp8_linear(c, a, b, residual=d).clone())
    for i, t in enumerate(got):
        assert torch.equal(t, wants[i % 6]), i


def test_two_streams_at_once():
    inputs = [layer(t, i) for i, t in enumerate((3, 40, 700, 1))]
    want = [moe_experts(*a) for a in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[] for _ in inputs]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(moe_experts(*inputs[i]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(t, w) for t in got[i])


def captured(f, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = f()
    return graph, out


@pytest.mark.parametrize("tokens", [1, 24, 900])
def test_captured_and_replayed_also_two_graphs_at_once(tokens):
    one, two = layer(tokens, 1), layer(tokens, 2)
    dense = ref.weight(384, 512, gen(5))
    w, ws = dense[0].cuda(), dense[1].cuda()

    def run(a):
        y = moe_experts(*a, residual=a[0])
        return fp8_linear(y, w, ws), y

    fresh = [(layer(tokens, 3), layer(tokens, 4)), (layer(tokens, 1), layer(tokens, 2))]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = [captured(lambda a=a: run(a), s) for a, s in zip((one, two), streams)]
    for inputs in fresh:
        for a, b in zip((one, two), inputs):
            for to, t in zip(a, b):
                to.copy_(t)
        torch.cuda.synchronize()
        for _ in range(10):
            for (graph, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, got), b in zip(graphs, inputs):
            assert all(torch.equal(x, y) for x, y in zip(got, run(b)))


def test_the_first_call_of_a_process_may_be_captured(linear_lib):
    import os
    import subprocess
    import sys
    code = """
import torch
import unimonomoe_b200 as U
from unimonomoe_b200.linear import check_status
x = torch.randn(5, 256, device="cuda").to(torch.bfloat16)
w, s = torch.ones(128, 256, device="cuda").to(torch.float8_e4m3fn), torch.ones(1, 2, device="cuda")
ids = torch.tensor([[9]], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = U.fp8_linear(x, w, s)
    U.plan_experts(ids, 4)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, U.fp8_linear(x, w, s))
try:
    check_status()
except RuntimeError as e:
    assert "past the last expert" in str(e)
    check_status()
    print("fine")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert got.returncode == 0 and got.stdout.strip() == "fine", f"{got.returncode}: {got.stdout}{got.stderr}"


def test_inference_mode_and_repeated_calls():
    a = layer(33, 9)
    want = moe_experts(*a)
    with torch.inference_mode():
        assert torch.equal(moe_experts(*a), want)
    assert all(torch.equal(moe_experts(*a), want) for _ in range(20))


# ---------------------------------------------------------------------- past 32 bits
def test_results_past_32_bits():
    g = gen(12)
    rows, n, k = 300001, 8192, 128           # 2.46e9 values
    w, ws = (t.cuda() for t in ref.weight(n, k, g))
    x = torch.randn(rows, k, device="cuda").to(torch.bfloat16)
    y = fp8_linear(x, w, ws)
    for part in (slice(0, 40), slice(262140, 262150), slice(rows - 33, rows)):
        assert torch.equal(y[part], fp8_linear(x[part], w, ws))
    del y
    ids = torch.randint(0, 5, (rows, 1), device="cuda", dtype=torch.int32)
    ew, es = w[None].expand(5, -1, -1).contiguous(), ws[None].expand(5, -1, -1).contiguous()
    plan = plan_experts(ids, 5)
    y = fp8_expert_linear(x, ew, es, plan)
    last = torch.arange(rows - 40, rows, device="cuda")
    assert torch.equal(y[last], fp8_linear(x[plan.tokens[last].long()], w, ws))
    out = combine_experts(y, plan.positions, torch.ones(rows, 1, device="cuda"))
    assert torch.equal(out[-40:], y[plan.positions[-40:, 0].long()])


def test_rows_past_32_bits():
    rows, k = 1100001, 2048                  # 2.25e9 values
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-3000:] = ref.states(3000, k, gen(13)).cuda()
    x[:-3000] = 1.0
    q, s = fp8_quantize(x)
    a, b = fp8_quantize(x[-3000:])
    assert torch.equal(q[-3000:].view(torch.uint8), a.view(torch.uint8)) and torch.equal(s[-3000:], b)
    w, ws = (t.cuda() for t in ref.weight(64, k, gen(14)))
    del x
    y = fp8_linear(q, w, ws, x_scale=s)
    assert ref.near(y[-70:].cpu(), *ref.product(a[-70:].cpu(), b[-70:].cpu(), w.cpu(), ws.cpu()), ref.HALF16)
    tokens = torch.arange(rows - 3000, rows, device="cuda", dtype=torch.int32)
    plan = ExpertPlan(torch.tensor([0, 1000, 3000], dtype=torch.int32, device="cuda"), tokens, tokens[:, None])
    y = fp8_expert_linear(q, w[None].expand(2, -1, -1).contiguous(), ws[None].expand(2, -1, -1).contiguous(), plan, x_scale=s)
    assert ref.near(y[-70:].cpu(), *ref.product(a[-70:].cpu(), b[-70:].cpu(), w.cpu(), ws.cpu()), ref.HALF16)


def test_weights_past_32_bits():
    experts, n, k = 140, 4096, 4096          # 2.35e9 bytes
    w = torch.zeros(experts, n, k, dtype=torch.uint8, device="cuda")
    one, ws = ref.weight(n, k, gen(15))
    w[-1] = one.view(torch.uint8).cuda()
    es = ws.cuda()[None].expand(experts, -1, -1).contiguous()
    for tokens in (9, 700):
        x = ref.states(tokens, k, gen(16)).cuda()
        y = fp8_expert_linear(x, w, es, plan_experts(torch.full((tokens, 1), experts - 1, dtype=torch.int32, device="cuda"), experts))
        q, s = ref.codes32(x.float().cpu())
        assert ref.near(y.cpu(), *ref.product(q, s, one, ws), ref.HALF16)


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="one device")
def test_on_another_device_than_the_current_one():
    a = layer(20, 1)
    want = moe_experts(*a)
    b = [t.to("cuda:1") for t in a]
    assert torch.cuda.current_device() == 0 and torch.equal(moe_experts(*b).cpu(), want.cpu())
    check_status("cuda:1")
