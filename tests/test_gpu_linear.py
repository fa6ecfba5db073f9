"""The block-FP8 operators against 64-bit forms (linear_ref.py) at the sizes where they can go wrong."""
import pytest
import torch

from tests import linear_ref as ref
from unimonomoe_b200 import (ExpertPlan, combine_experts, fp8_expert_linear, fp8_linear, fp8_quantize, moe_experts,
                             plan_experts)
from unimonomoe_b200.linear import check_status

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_fault(linear_lib):
    yield
    check_status()


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 2048), (3, 128), (7, 144), (61, 1040), (130, 7168), (1000, 512), (5, 2032)])
def test_quantize_is_the_definition_bit_for_bit(rows, cols):
    x = ref.states(rows, cols, gen(rows, cols))
    x[0, :16] = 0
    q, s = fp8_quantize(x.cuda())
    wq, ws = ref.codes32(x.float())
    assert q.dtype == ref.E4M3 and torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s.cpu(), ws)


@pytest.mark.parametrize("rows,cols", [(1, 128), (3, 16), (61, 512), (130, 1040), (1000, 256)])
def test_gated_quantize(rows, cols):
    x = ref.states(rows, 2 * cols, gen(rows, cols, 1))
    q, s = fp8_quantize(x.cuda(), silu_mul=True)
    y = x.double()
    assert ref.gate_near(q.cpu().view(ref.E4M3), s.cpu(), y, torch.zeros_like(y))


def check_linear(m, n, k, seed, mode):
    g = gen(m, n, k, seed)
    x, (w, ws) = ref.states(m, k, g), ref.weight(n, k, g)
    residual = ref.states(m, n, g) if mode == "residual" else None
    q, s = ref.codes32(x.float())
    y, off = ref.product(q, s, w, ws)
    dev = dict(residual=residual.cuda()) if residual is not None else {}
    if mode == "fp32":
        got = fp8_linear(x.cuda(), w.cuda(), ws.cuda(), out_dtype=torch.float32)
        assert got.dtype == torch.float32 and ref.near(got.cpu(), y, off, ref.HALF32)
    elif mode == "silu":
        cq, cs = fp8_linear(x.cuda(), w.cuda(), ws.cuda(), silu_mul=True)
        assert cq.shape == (m, n // 2) and cs.shape == (m, n // 256) and ref.gate_near(cq.cpu(), cs.cpu(), y, off)
    else:
        got = fp8_linear(x.cuda(), w.cuda(), ws.cuda(), **dev)
        if residual is not None:
            off = off + (y.abs() + off + residual.double().abs()) * ref.HALF32
            y = y + residual.double()
        assert got.dtype == torch.bfloat16 and ref.near(got.cpu(), y, off, ref.HALF16)
        again = fp8_linear(q.cuda(), w.cuda(), ws.cuda(), x_scale=s.cuda(), **dev)
        assert torch.equal(got, again)


@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 5120, 2048), (3, 40000, 144), (20, 20000, 400), (32, 512, 4096), (2, 64, 16), (15, 1000, 1040), (16, 2048, 4096), (17, 129, 272), (33, 384, 7168),
                                   (61, 2048, 4096), (64, 576, 1808), (65, 640, 512), (100, 1, 256), (128, 200, 144), (129, 512, 1024)])
@pytest.mark.parametrize("mode", ["plain", "residual", "fp32"])
def test_linear_few_rows(m, n, k, mode):
    check_linear(m, n, k, 0, mode)


@pytest.mark.parametrize("m,n,k", [(1000, 2048, 512), (1500, 1000, 1040), (2049, 577, 272), (700, 4096, 2048), (4099, 264, 144)])
@pytest.mark.parametrize("mode", ["plain", "residual", "fp32"])
def test_linear_many_rows(m, n, k, mode):
    check_linear(m, n, k, 1, mode)


@pytest.mark.parametrize("m,n,k", [(256, 2048, 4096), (130, 300, 7168), (500, 1000, 4112), (129, 2057, 6160), (1000, 264, 7168), (256, 4096, 7168)])
@pytest.mark.parametrize("mode", ["plain", "residual", "fp32"])
def test_linear_with_k_divided_among_ctas(m, n, k, mode):
    check_linear(m, n, k, 9, mode)


@pytest.mark.parametrize("m,n,k", [(300, 2048, 7168), (130, 512, 8208), (600, 1024, 4112), (257, 4096, 6160)])
def test_gated_activation_with_k_divided_among_ctas(m, n, k):
    check_linear(m, n, k, 10, "silu")


@pytest.mark.parametrize("m,n,k", [(1, 256, 128), (1, 1024, 2048), (2, 40960, 400), (32, 512, 2048), (16, 512, 1040), (17, 4096, 512), (33, 768, 1808), (64, 256, 7168), (200, 512, 272), (1500, 1024, 1040),
                                   (2300, 512, 2048)])
def test_linear_with_gated_activation(m, n, k):
    check_linear(m, n, k, 2, "silu")


def test_linear_takes_leading_dimensions_and_strides():
    g = gen(7)
    w, ws = (t.cuda() for t in ref.weight(256, 512, g))
    x = ref.states(12, 1024, g).cuda()
    wide = x[:, 256:768]
    assert torch.equal(fp8_linear(wide, w, ws), fp8_linear(wide.contiguous(), w, ws))
    cube = x.view(3, 4, 1024)[..., :512]
    assert torch.equal(fp8_linear(cube, w, ws), fp8_linear(x[:, :512].contiguous(), w, ws).view(3, 4, 256))
    assert torch.equal(fp8_linear(x[0, :512], w, ws), fp8_linear(x[:1, :512], w, ws)[0])
    odd = torch.empty(12 * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(12, 512).copy_(wide)
    assert torch.equal(fp8_linear(odd, w, ws), fp8_linear(wide, w, ws))
    turned = wide.t().contiguous().t()
    assert torch.equal(fp8_linear(turned, w, ws), fp8_linear(wide, w, ws))
    q, s = fp8_quantize(cube)
    assert q.shape == (3, 4, 512) and s.shape == (3, 4, 4) and torch.equal(fp8_linear(q, w.view(torch.uint8), ws, x_scale=s), fp8_linear(cube, w, ws))
    none = x[:0, :512]
    assert fp8_linear(none, w, ws).shape == (0, 256) and fp8_linear(none, w, ws, silu_mul=True)[1].shape == (0, 1)


@pytest.mark.parametrize("tokens,top,experts,dtype", [(0, 2, 4, torch.int32), (1, 1, 1, torch.int32), (1, 8, 256, torch.int64), (33, 6, 60, torch.int32), (500, 8, 1024, torch.int64),
                                                      (700, 8, 128, torch.int32), (3001, 3, 17, torch.int32), (9000, 2, 300, torch.int64)])
@pytest.mark.parametrize("kind", ["all", "some", "none", "one"])
def test_plan(tokens, top, experts, dtype, kind):
    g = gen(tokens, top, experts)
    ids = torch.randint(0, experts, (tokens, top), generator=g)
    if kind == "some":
        ids = torch.where(torch.rand(tokens, top, generator=g) < 0.4, -1 - ids, ids)
    elif kind == "none":
        ids = torch.full_like(ids, -1)
    elif kind == "one":
        ids = torch.full_like(ids, experts - 1)
    got = plan_experts(ids.to(dtype).cuda(), experts)
    assert all(t.dtype == torch.int32 for t in got)
    for a, b in zip(got, ref.plan(ids, experts)):
        assert torch.equal(a.cpu().long(), b)


def routed(tokens, top, experts, g, skew=0.0, gone=0.0):
    score = torch.randn(tokens, experts, generator=g) + skew * torch.randn(experts, generator=g)
    ids = score.topk(top, dim=1).indices
    return torch.where(torch.rand(ids.shape, generator=g) < gone, -1, ids).to(torch.int32)


def check_experts(tokens, top, experts, n, k, gather, silu, skew=0.0, gone=0.0, ids=None):
    g = gen(tokens, top, experts, n, k, gather)
    ids = routed(tokens, top, experts, g, skew, gone) if ids is None else ids
    off, toks, _ = ref.plan(ids, experts)
    rows = int(off[-1])
    w, ws = ref.weight(n, k, g, (experts,))
    x = ref.states(tokens if gather else tokens * top, k, g)
    q, s = ref.codes32(x.float())
    plan = plan_experts(ids.cuda(), experts)
    got = fp8_expert_linear(x.cuda(), w.cuda(), ws.cuda(), plan, gather=gather, silu_mul=silu)
    again = fp8_expert_linear(q.cuda(), w.cuda(), ws.cuda(), plan, x_scale=s.cuda(), gather=gather, silu_mul=silu)
    for a, b in zip(got, again) if silu else [(got, again)]:
        assert torch.equal(a[:rows].view(torch.uint8), b[:rows].view(torch.uint8))
    for e in range(experts):
        a, b = int(off[e]), int(off[e + 1])
        if a == b:
            continue
        src = toks[a:b] if gather else torch.arange(a, b)
        y, slack = ref.product(q[src], s[src], w[e], ws[e])
        if silu:
            assert ref.gate_near(got[0][a:b].cpu(), got[1][a:b].cpu(), y, slack), e
        else:
            assert ref.near(got[a:b].cpu(), y, slack, ref.HALF16), e


@pytest.mark.parametrize("tokens,top,experts,n,k", [(1, 1, 1, 128, 128), (1, 8, 16, 256, 512), (3, 2, 5, 1000, 272), (24, 8, 64, 512, 256), (100, 6, 60, 192, 1040),
                                                    (40, 4, 8, 256, 1808), (300, 4, 8, 129, 256), (700, 2, 4, 512, 256), (1500, 2, 3, 577, 144), (2000, 4, 16, 256, 512)])
@pytest.mark.parametrize("gather", [True, False])
def test_experts(tokens, top, experts, n, k, gather):
    check_experts(tokens, top, experts, n, k, gather, False, skew=0.5)


@pytest.mark.parametrize("tokens,top,experts,n,k", [(1, 1, 1, 256, 128), (2, 8, 16, 512, 512), (30, 8, 32, 256, 272), (100, 6, 60, 768, 256), (600, 2, 8, 256, 1040), (2000, 4, 16, 512, 256)])
@pytest.mark.parametrize("gather", [True, False])
def test_experts_with_gated_activation(tokens, top, experts, n, k, gather):
    check_experts(tokens, top, experts, n, k, gather, True, skew=1.0)


@pytest.mark.parametrize("n,silu", [(384, False), (512, True)])
def test_experts_elsewhere_and_without_rows(n, silu):
    check_experts(90, 4, 32, n, 256, True, silu, skew=2.0, gone=0.6)
    check_experts(1200, 4, 12, n, 256, True, silu, skew=2.0, gone=0.6)
    check_experts(50, 2, 8, n, 256, False, silu, ids=torch.full((50, 2), 7, dtype=torch.int32))
    check_experts(900, 2, 4, n, 256, False, silu, ids=torch.full((900, 2), 3, dtype=torch.int32))


def test_rows_behind_the_last_run_are_left_as_they_were():
    g = gen(11)
    for tokens, experts in ((20, 8), (1500, 4)):
        ids = torch.where(torch.rand(tokens, 4, generator=g) < 0.5, -1, torch.randint(0, experts, (tokens, 4), generator=g)).cuda()
        plan = plan_experts(ids, experts)
        rows = int(plan.offsets[-1])
        w, ws = (t.cuda() for t in ref.weight(256, 256, g, (experts,)))
        x = ref.states(tokens, 256, g).cuda()
        torch.cuda.empty_cache()
        mark = torch.full((tokens * 4, 256), 7.0, dtype=torch.bfloat16, device="cuda")
        at = mark.data_ptr()
        del mark                             # its memory is what the result gets
        got = fp8_expert_linear(*fp8_quantize(x)[:1], w, ws, plan, x_scale=fp8_quantize(x)[1])
        if got.data_ptr() == at:
            assert bool((got[rows:] == 7.0).all())
        assert bool(torch.isfinite(got[:rows].float()).all())


@pytest.mark.parametrize("tokens,top,cols", [(1, 1, 8), (1, 8, 2048), (24, 8, 1040), (1000, 3, 512), (5, 64, 128), (300, 9, 264)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine(tokens, top, cols, residual):
    g = gen(tokens, top, cols)
    rows = tokens * top
    partial = ref.states(rows, cols, g)
    pos = torch.randperm(rows, generator=g).view(tokens, top).to(torch.int32)
    pos = torch.where(torch.rand(tokens, top, generator=g) < 0.2, -1, pos)
    wt = torch.rand(tokens, top, generator=g)
    res = ref.states(tokens, cols, g) if residual else None
    got = combine_experts(partial.cuda(), pos.cuda(), wt.cuda(), None if res is None else res.cuda())
    want, size = ref.combine(partial, pos, wt, res)
    assert ref.near(got.cpu(), want, size * (top + 1) * ref.HALF32, ref.HALF16)


def test_nothing_to_combine():
    pos = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    wt = torch.full((3, 2), float("nan"), device="cuda")
    assert bool((combine_experts(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), pos, wt) == 0).all())
    assert combine_experts(torch.empty(4, 64, dtype=torch.bfloat16, device="cuda"), pos[:0], wt[:0]).shape == (0, 64)


@pytest.mark.parametrize("tokens", [1, 30, 1300])
def test_operators_together_are_a_layer(tokens):
    """Experts in 64 bits from bf16 states: what is lost is the two roundings to e4m3, 2^-4 of a value at most, and 2^-4 / sqrt(3) on average; a
    dot product of values that are off by independent errors of that size is off by that share of its root mean square."""
    g = gen(tokens, 5)
    experts, inter, hidden, top = 12, 256, 512, 4
    x, ids = ref.states(tokens, hidden, g), routed(tokens, top, experts, g, gone=0.2)
    (w13, s13), (w2, s2) = ref.weight(2 * inter, hidden, g, (experts,)), ref.weight(hidden, inter, g, (experts,))
    wt = torch.softmax(torch.randn(tokens, top, generator=g), 1)
    res = ref.states(tokens, hidden, g)
    got = moe_experts(x.cuda(), ids.cuda(), wt.cuda(), w13.cuda(), s13.cuda(), w2.cuda(), s2.cuda()).cpu().double()
    with_res = moe_experts(x.cuda(), ids.cuda(), wt.cuda(), w13.cuda(), s13.cuda(), w2.cuda(), s2.cuda(), residual=res.cuda()).cpu().double()
    want = torch.zeros(tokens, hidden, dtype=torch.float64)
    for t in range(tokens):
        for j in range(top):
            e = int(ids[t, j])
            if e >= 0:
                v = ref.gated(values_of(x[t:t + 1]) @ ref.values(w13[e], s13[e], True).T)
                want[t] += float(wt[t, j]) * (v @ ref.values(w2[e], s2[e], True).T)[0]
    assert float((got - want).norm()) <= 2.0 ** -4 * float(want.norm()) + 1e-12
    assert ref.near(with_res, got + res.double(), (got.abs() + res.double().abs()) * 2.0 ** -7, ref.HALF16)


def values_of(x):
    return ref.values(*ref.codes32(x.float()))
