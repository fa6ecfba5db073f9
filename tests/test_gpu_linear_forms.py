"""Forms of the block-FP8 products together, and memory that is not theirs to write."""
import ctypes

import pytest
import torch

from tests import linear_ref as ref
from tests.test_gpu_linear import gen, routed
from unimonomoe_b200 import fp8_linear, fp8_quantize, plan_experts
from unimonomoe_b200.linear import check_status

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_fault(linear_lib):
    yield
    check_status()


# one row tile in one launch, more of them, many rows (aligned or not), K divided among CTAs of either kernel
SIZES = [(1, 256, 2048), (9, 1000, 1040), (40, 512, 4096), (61, 577, 272), (129, 2056, 6160), (256, 2048, 4096), (1000, 2048, 512), (1537, 512, 1040), (2049, 577, 272), (4099, 264, 144)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("eight_bits", [False, True])
def test_residual_and_fp32_together(m, n, k, eight_bits):
    g = gen(m, n, k, 21)
    x, (w, ws), res = ref.states(m, k, g), ref.weight(n, k, g), ref.states(m, n, g)
    q, s = ref.codes32(x.float())
    y, off = ref.product(q, s, w, ws)
    off = off + (y.abs() + off + res.double().abs()) * ref.HALF32        # the sum's own rounding; that to fp32 is none more
    rows = dict(x=q.cuda(), x_scale=s.cuda()) if eight_bits else dict(x=x.cuda())
    got = fp8_linear(**rows, weight=w.cuda(), weight_scale=ws.cuda(), residual=res.cuda(), out_dtype=torch.float32)
    assert got.dtype == torch.float32 and ref.near(got.cpu(), y + res.double(), off, ref.HALF32)
    half = fp8_linear(**rows, weight=w.cuda(), weight_scale=ws.cuda(), residual=res.cuda())
    assert torch.equal(half, got.to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", SIZES)
def test_rows_in_8_bits_give_the_same_bits_in_fp32(m, n, k):
    g = gen(m, n, k, 22)
    x, (w, ws) = ref.states(m, k, g).cuda(), (t.cuda() for t in ref.weight(n, k, g))
    q, s = fp8_quantize(x)
    got = fp8_linear(q, w, ws, x_scale=s, out_dtype=torch.float32)
    assert torch.equal(got, fp8_linear(x, w, ws, out_dtype=torch.float32))
    assert torch.equal(got.to(torch.bfloat16), fp8_linear(x, w, ws))


@pytest.mark.parametrize("m,n,k", [(1, 256, 2048), (16, 512, 1040), (33, 768, 1808), (64, 512, 4096), (130, 512, 8208), (300, 2048, 7168), (1500, 1024, 1040)])
def test_rows_in_8_bits_with_the_gated_activation(m, n, k):
    g = gen(m, n, k, 23)
    x, (w, ws) = ref.states(m, k, g), ref.weight(n, k, g)
    q, s = ref.codes32(x.float())
    cq, cs = fp8_linear(q.cuda(), w.cuda(), ws.cuda(), x_scale=s.cuda(), silu_mul=True)
    assert ref.gate_near(cq.cpu(), cs.cpu(), *ref.product(q, s, w, ws))
    for a, b in zip((cq, cs), fp8_linear(x.cuda(), w.cuda(), ws.cuda(), silu_mul=True)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---------------------------------------------------------------------- rows outside of a plan's runs, through the C ABI
def pointer(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("tokens,experts", [(20, 8), (90, 32), (1500, 4)])
@pytest.mark.parametrize("n", [512, 264])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gather", [False, True])
def test_rows_outside_of_the_runs_keep_every_byte(linear_lib, tokens, experts, n, silu, gather):
    """Rows in front of the first run, whose expert has been taken out, and behind the last one."""
    if silu and n % 256:
        n = 256
    lib = ctypes.CDLL(linear_lib)
    vp, i, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    lib.mono_lin_experts.argtypes = [vp, vp, i64, vp, vp, i64, i, vp, vp, i, i, vp, vp, vp, vp, vp]
    k, top = 272, 4
    g = gen(tokens, experts, n, silu, gather)
    ids = routed(tokens, top, experts, g, skew=0.5, gone=0.4)
    ids[0, 0] = 0                            # the first expert has a row
    rows = tokens * top
    plan = plan_experts(ids.cuda(), experts)
    offsets = plan.offsets.clone()
    offsets[0] = offsets[1]
    lo, hi = int(offsets[0]), int(offsets[-1])
    assert 0 < lo < hi < rows
    w, ws = (t.cuda() for t in ref.weight(n, k, g, (experts,)))
    q, s = fp8_quantize(ref.states(tokens if gather else rows, k, g).cuda())
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    results = []
    for mark in (0xA5, 0x5A):
        out = torch.full((rows, n // 2 if silu else 2 * n), mark, dtype=torch.uint8, device="cuda")
        scales = torch.full((rows, n // 256, 4), mark, dtype=torch.uint8, device="cuda") if silu else None
        torch.cuda.synchronize()
        rc = lib.mono_lin_experts(pointer(q), pointer(s), len(q), pointer(plan.tokens) if gather else None, pointer(offsets), rows, experts, pointer(w), pointer(ws), n, k,
                                  None if silu else pointer(out), pointer(out) if silu else None, pointer(scales), pointer(status), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0 and status.tolist() == [0, 0]
        for t in (out, scales) if silu else (out,):
            assert bool((t[:lo] == mark).all()) and bool((t[hi:] == mark).all())
        results.append(out[lo:hi])
        last = scales[lo:hi] if silu else out[lo:hi]
        results.append(last)
    assert torch.equal(results[0], results[2]) and torch.equal(results[1], results[3])          # and inside of them all is written
