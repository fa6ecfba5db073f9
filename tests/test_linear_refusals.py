"""What the block-FP8 operators refuse, and how: an exception that Python can catch, in a process that lives on."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CALLS = """
import torch
import unimonomoe_b200 as U
from unimonomoe_b200 import linear as L
dev = torch.device("cuda:0")
def i32(*shape): return torch.zeros(shape, dtype=torch.int32, device=dev)
def bf(*shape): return torch.zeros(shape, dtype=torch.bfloat16, device=dev)
def f8(*shape): return torch.zeros(shape, dtype=torch.float8_e4m3fn, device=dev)
def f32(*shape): return torch.ones(shape, device=dev)
x, w, ws = bf(3, 256), f8(512, 256), f32(4, 2)
ew, es = f8(4, 512, 256), f32(4, 4, 2)
plan = U.plan_experts(i32(3, 2), 4)
other = U.plan_experts(i32(3, 2), 5)
wrong = {
    "quantize: type": lambda: U.fp8_quantize(x.float()),
    "quantize: columns": lambda: U.fp8_quantize(bf(3, 40)),
    "quantize: no dimension": lambda: U.fp8_quantize(bf()),
    "quantize: no columns": lambda: U.fp8_quantize(bf(3, 0)),
    "quantize: halves": lambda: U.fp8_quantize(bf(3, 33), silu_mul=True),
    "quantize: columns of a half": lambda: U.fp8_quantize(bf(3, 48), silu_mul=True),
    "quantize: sparse": lambda: U.fp8_quantize(x.to_sparse()),
    "quantize: negative in memory": lambda: U.fp8_quantize(torch._neg_view(x)),
    "combine: negative in memory": lambda: U.combine_experts(bf(6, 64), plan.positions, torch._neg_view(f32(3, 2))),
    "linear: type": lambda: U.fp8_linear(x.half(), w, ws),
    "linear: type of the weight": lambda: U.fp8_linear(x, w.to(torch.bfloat16), ws),
    "linear: other 8 bits": lambda: U.fp8_linear(x, w.view(torch.float8_e5m2), ws),
    "linear: columns": lambda: U.fp8_linear(x[:, :128], w, ws),
    "linear: weight's dimensions": lambda: U.fp8_linear(x, ew, es),
    "linear: weight's strides": lambda: U.fp8_linear(x, f8(256, 512).t(), ws),
    "linear: scales": lambda: U.fp8_linear(x, w, f32(4, 1)),
    "linear: type of scales": lambda: U.fp8_linear(x, w, ws.half()),
    "linear: device": lambda: U.fp8_linear(x, w.cpu(), ws),
    "linear: device of scales": lambda: U.fp8_linear(x, w, ws.cpu()),
    "linear: K": lambda: U.fp8_linear(bf(3, 40), f8(512, 40), f32(4, 1)),
    "linear: codes without scales": lambda: U.fp8_linear(f8(3, 256), w, ws),
    "linear: scales without codes": lambda: U.fp8_linear(x, w, ws, x_scale=f32(3, 2)),
    "linear: rows of x_scale": lambda: U.fp8_linear(f8(3, 256), w, ws, x_scale=f32(2, 2)),
    "linear: groups of x_scale": lambda: U.fp8_linear(f8(3, 256), w, ws, x_scale=f32(3, 3)),
    "linear: residual": lambda: U.fp8_linear(x, w, ws, residual=bf(3, 256)),
    "linear: type of the residual": lambda: U.fp8_linear(x, w, ws, residual=bf(3, 512).float()),
    "linear: residual and gate": lambda: U.fp8_linear(x, w, ws, residual=bf(3, 512), silu_mul=True),
    "linear: fp32 and gate": lambda: U.fp8_linear(x, w, ws, silu_mul=True, out_dtype=torch.float32),
    "linear: halves": lambda: U.fp8_linear(x, f8(384, 256), f32(3, 2), silu_mul=True),
    "linear: out_dtype": lambda: U.fp8_linear(x, w, ws, out_dtype=torch.float16),
    "linear: no rows of the weight": lambda: U.fp8_linear(x, f8(0, 256), f32(0, 2)),
    "plan: type": lambda: U.plan_experts(f32(3, 2), 4),
    "plan: dimensions": lambda: U.plan_experts(i32(3), 4),
    "plan: too many a token": lambda: U.plan_experts(i32(3, 65), 4),
    "plan: experts": lambda: U.plan_experts(i32(3, 2), 0),
    "plan: too many experts": lambda: U.plan_experts(i32(3, 2), 1025),
    "experts: another plan": lambda: U.fp8_expert_linear(x, ew, es, other),
    "experts: dimensions of x": lambda: U.fp8_expert_linear(x[None], ew, es, plan),
    "experts: rows of the plan": lambda: U.fp8_expert_linear(x, ew, es, plan, gather=False),
    "experts: no tokens": lambda: U.fp8_expert_linear(x[:0], ew, es, plan),
    "experts: dense weight": lambda: U.fp8_expert_linear(x, w, ws, plan),
    "experts: scales": lambda: U.fp8_expert_linear(x, ew, es[:3], plan),
    "experts: halves": lambda: U.fp8_expert_linear(x, f8(4, 128, 256), f32(4, 1, 2), plan, silu_mul=True),
    "experts: codes without scales": lambda: U.fp8_expert_linear(f8(3, 256), ew, es, plan),
    "experts: type of offsets": lambda: U.fp8_expert_linear(x, ew, es, U.ExpertPlan(plan.offsets.long(), plan.tokens, plan.positions)),
    "experts: tokens elsewhere": lambda: U.fp8_expert_linear(x, ew, es, U.ExpertPlan(plan.offsets, plan.tokens.cpu(), plan.positions)),
    "combine: type": lambda: U.combine_experts(f32(6, 64), plan.positions, f32(3, 2)),
    "combine: columns": lambda: U.combine_experts(bf(6, 60), plan.positions, f32(3, 2)),
    "combine: weights": lambda: U.combine_experts(bf(6, 64), plan.positions, f32(3, 3)),
    "combine: type of weights": lambda: U.combine_experts(bf(6, 64), plan.positions, bf(3, 2)),
    "combine: type of positions": lambda: U.combine_experts(bf(6, 64), plan.positions.long(), f32(3, 2)),
    "moe: other tokens": lambda: U.moe_experts(x, i32(2, 2), f32(2, 2), ew, es, f8(4, 256, 256), f32(4, 2, 2)),
    "moe: weights": lambda: U.moe_experts(x, i32(3, 2), f32(3, 1), ew, es, f8(4, 256, 256), f32(4, 2, 2)),
    "moe: width": lambda: U.moe_experts(x, i32(3, 2), f32(3, 2), ew, es, f8(4, 128, 256), f32(4, 1, 2)),
    "combine: residual": lambda: U.combine_experts(bf(6, 64), plan.positions, f32(3, 2), bf(2, 64)),
}
for name, call in wrong.items():
    try:
        call()
    except ValueError as e:
        assert str(e), name
    else:
        raise SystemExit(name + " was taken")
for call in (lambda: U.fp8_quantize([1.0]), lambda: U.fp8_linear(x, None, ws), lambda: U.plan_experts(i32(3, 2), 4.5), lambda: U.combine_experts(bf(6, 64), None, f32(3, 2))):
    try:
        call()
    except TypeError:
        continue
    raise SystemExit("a wrong type was taken")
L.check_status(dev)
assert U.fp8_linear(x, w, ws).shape == (3, 512)
print("fine")
"""


@pytest.mark.gpu
def test_every_wrong_argument_is_a_python_exception(linear_lib):
    got = subprocess.run([sys.executable, "-c", CALLS], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert got.returncode == 0 and got.stdout.strip() == "fine", f"{got.returncode}: {got.stdout}{got.stderr}"
