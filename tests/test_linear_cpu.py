"""The block-FP8 operators without a GPU: the library's symbols and return codes, refusals, the 64-bit forms that the GPU tests use."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import unimonomoe_b200 as U
from tests import linear_ref as ref
from unimonomoe_b200 import linear as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_declared_symbol_is_exported(linear_lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mono_linear.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(mono_lin_\w+)\s*\(", text))
    assert names == {"mono_lin_quantize", "mono_lin_product", "mono_lin_product_rows", "mono_lin_takes_rows", "mono_lin_plan", "mono_lin_experts", "mono_lin_combine"}
    lib = ctypes.CDLL(linear_lib)
    assert not [n for n in names if not hasattr(lib, n)]
    assert L.linear_lib_path() == linear_lib


def test_the_module_has_no_c_plus_plus_runtime_of_its_own(linear_lib):
    if shutil.which("readelf") is None:
        pytest.skip("no readelf")
    from unimonomoe_b200 import build
    symbols = subprocess.run(["readelf", "--dyn-syms", "-W", build.part_binding_path("linear")], capture_output=True, text=True, check=True).stdout
    throw = [line for line in symbols.splitlines() if "__cxa_throw" in line]
    assert throw and all(" UND " in line for line in throw)


def wrong(call, good, cases):
    for at, value, code in cases:
        a = list(good)
        for i, v in zip(at if isinstance(at, tuple) else (at,), value if isinstance(at, tuple) else (value,)):
            a[i] = v
        assert call(*a) == code, (at, value)


def test_return_codes_before_any_cuda_call(linear_lib):
    lib = ctypes.CDLL(linear_lib)
    vp, i, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    lib.mono_lin_quantize.argtypes = [vp, i64, i64, i, i, vp, vp, vp]
    lib.mono_lin_product.argtypes = [vp, vp, i64, vp, vp, i, i, vp, i, vp, vp, vp, i, vp, vp]
    lib.mono_lin_plan.argtypes = [vp, i, i64, i, i, vp, vp, vp, vp, vp]
    lib.mono_lin_experts.argtypes = [vp, vp, i64, vp, vp, i64, i, vp, vp, i, i, vp, vp, vp, vp, vp]
    lib.mono_lin_combine.argtypes = [vp, i64, vp, vp, i64, i, i, vp, vp, vp, vp]
    p = (ctypes.addressof(ctypes.create_string_buffer(64)) + 15) // 16 * 16
    wrong(lib.mono_lin_quantize, [p, 128, 2, 128, 0, p, p, 0],
          [(2, -1, -302), (3, 120, -302), (3, 0, -302), (0, 0, -301), (5, 0, -301), (6, 0, -301), (0, p + 2, -303), (5, p + 8, -303), (1, 130, -303), (2, 0, 0)])
    product = [p, p, 2, p, p, 256, 128, p, 0, 0, 0, 0, 0, p, 0]
    wrong(lib.mono_lin_product, product,
          [(5, 0, -302), (6, 136, -302), (6, 0, -302), (2, -1, -302), (2, 1 << 31, -302), ((2, 5), ((1 << 31) - 1, 1 << 20), -302), (0, 0, -301), (1, 0, -301), (3, 0, -301),
           (4, 0, -301), (7, 0, -301), (10, p, -301), (13, 0, -301), ((7, 10), (0, p), -301), (0, p + 4, -303), (3, p + 8, -303), (2, 0, 0)])
    wrong(lib.mono_lin_product, [*product[:7], 0, 0, 0, p, p, 0, p, 0], [(5, 384, -302), (5, 128, -302), (10, p + 8, -303), (11, 0, -301)])
    lib.mono_lin_product_rows.argtypes = [vp, i64, i, vp, vp, i, i, vp, i, vp, vp, vp, vp, vp]
    wrong(lib.mono_lin_product_rows, [p, 128, 2, p, p, 256, 128, p, 0, 0, 0, 0, p, 0],
          [(2, 17, -302), (2, -1, -302), (1, -8, -302), (5, 0, -302), (6, 24, -302), (0, 0, -301), (3, 0, -301), (7, 0, -301), (12, 0, -301), (0, p + 2, -303), (1, 129, -303), (2, 0, 0)])
    wrong(lib.mono_lin_plan, [p, 0, 4, 2, 8, p, p, p, p, 0],
          [(2, -1, -302), (3, 0, -302), (3, L.MAX_TOP + 1, -302), (4, 0, -302), (4, L.MAX_EXPERTS + 1, -302), (2, 1 << 31, -302), (0, 0, -301), (5, 0, -301), (7, 0, -301), (8, 0, -301)])
    wrong(lib.mono_lin_experts, [p, p, 4, p, p, 8, 3, p, p, 256, 128, p, 0, 0, p, 0],
          [(6, 0, -302), (6, L.MAX_EXPERTS + 1, -302), (9, 0, -302), (10, 24, -302), (5, -1, -302), ((3, 5), (0, 8), -302), (2, 0, -302), (4, 0, -301), (0, 0, -301), (11, 0, -301),
           (14, 0, -301), (7, p + 4, -303), (5, 0, 0)])
    wrong(lib.mono_lin_combine, [p, 4, p, p, 2, 2, 64, 0, p, p, 0],
          [(6, 60, -302), (6, 0, -302), (5, 0, -302), (5, L.MAX_TOP + 1, -302), (4, -1, -302), (0, 0, -301), (2, 0, -301), (3, 0, -301), (8, 0, -301), (9, 0, -301), (0, p + 8, -303),
           (7, p + 2, -303), (4, 0, 0)])


def test_operators_refuse_cpu_tensors(linear_lib):
    x, w, s = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(128, 128, dtype=ref.E4M3), torch.ones(1, 1)
    i = torch.zeros(2, 1, dtype=torch.int32)
    plan = U.ExpertPlan(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), i)
    for call in (lambda: U.fp8_quantize(x), lambda: U.fp8_linear(x, w, s), lambda: U.plan_experts(i, 4), lambda: U.fp8_expert_linear(x, w[None], s[None], plan),
                 lambda: U.combine_experts(x, i, torch.ones(2, 1)), lambda: U.moe_experts(x, i, torch.ones(2, 1), w[None], s[None], w[None], s[None])):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="float16"):
        U.fp8_linear(x, w, s, out_dtype=torch.float16)


def test_codes_of_the_reference_are_within_half_a_step():
    g = torch.Generator().manual_seed(1)
    x = ref.states(5, 300, g)
    q, s = ref.codes32(x.float())
    v = x.double()
    off = (ref.values(q, s) - v).abs()
    per = ref.spread(s.double(), 300)
    assert bool((off <= torch.maximum(ref.HALF8 * v.abs(), ref.LEAST8 * per) * (1 + 2.0 ** -20)).all())
    assert bool((q.float().abs().amax(-1) == 448).all())


def test_a_wrong_product_is_noticed():
    """The bounds of the GPU tests are of use: one scale left out, one group of K left out, one row of the weight for another."""
    g = torch.Generator().manual_seed(2)
    x, (w, ws) = ref.states(9, 512, g), ref.weight(256, 512, g)
    q, s = ref.codes32(x.float())
    y, off = ref.product(q, s, w, ws)
    assert ref.near(y.to(torch.bfloat16), y, off, ref.HALF16)
    one = ws.clone()
    one[0, 2] = ws[0, 1]
    for other in (ref.product(q, s, w, one)[0], ref.product(q[:, :384], s[:, :3], w[:, :384], ws[:, :3])[0], y.roll(1, 1)):
        assert not ref.near(other.to(torch.bfloat16), y, off, ref.HALF16)
    cq, cs = ref.codes32(ref.gated(y).float())
    assert ref.gate_near(cq, cs, y, off) and not ref.gate_near(cq, cs * 1.001, y, off) and not ref.gate_near(cq.roll(1, 1), cs, y, off)
