"""What the attention operators refuse, and how: an exception that Python can catch, in a process that lives on."""
import ctypes
import math
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_module_has_no_c_plus_plus_runtime_of_its_own(attention_lib):
    if shutil.which("readelf") is None:
        pytest.skip("no readelf")
    from unimonomoe_b200 import build
    dynamic = subprocess.run(["readelf", "-d", build.attention_binding_path()], capture_output=True, text=True, check=True).stdout
    assert "libstdc++.so.6" in dynamic
    symbols = subprocess.run(["readelf", "--dyn-syms", "-W", build.attention_binding_path()], capture_output=True, text=True, check=True).stdout
    throw = [line for line in symbols.splitlines() if "__cxa_throw" in line]
    assert throw and all(" UND " in line for line in throw)


CALLS = """
import torch
from unimonomoe_b200 import attention as A
dev = torch.device("cuda:0")
def i32(*shape): return torch.zeros(shape, dtype=torch.int32, device=dev)
def bf(*shape): return torch.zeros(shape, dtype=torch.bfloat16, device=dev)
cache = A.KV4Cache.empty(2, 2, 64, 16, dev)
i64, one, start, cs = torch.zeros(3, dtype=torch.int64, device=dev), i32(1), i32(2), torch.ones(4, 64, device=dev)
x, w = bf(3, 2, 64), bf(64)
wrong = {
    "plan: lengths": lambda: A.plan_batch(i32(2), i32(3), i32(2, 4), i32(8), one, 16, 4),
    "plan: type": lambda: A.plan_batch(i32(2), i32(2).long(), i32(2, 4), i32(8), one, 16, 4),
    "plan: table": lambda: A.plan_batch(i32(2), i32(2), i32(4, 2).t(), i32(8), one, 16, 4),
    "plan: rows of the table": lambda: A.plan_batch(i32(2), i32(2), i32(3, 4), i32(8), one, 16, 4),
    "plan: page size": lambda: A.plan_batch(i32(2), i32(2), i32(2, 4), i32(8), one, 24, 4),
    "plan: tokens": lambda: A.plan_batch(i32(2), i32(2), i32(2, 4), i32(8), one, 16, -1),
    "plan: no requests": lambda: A.plan_batch(i32(0), i32(0), i32(0, 4), i32(8), one, 16, 4),
    "plan: taken": lambda: A.plan_batch(i32(2), i32(2), i32(2, 4), i32(8), i32(2), 16, 4),
    "rope: type": lambda: A.qk_norm_rope(x.float(), x, w, w, cs, i32(3)),
    "rope: tokens": lambda: A.qk_norm_rope(x, x[:2], w, w, cs, i32(3)),
    "rope: head size": lambda: A.qk_norm_rope(bf(3, 2, 96), bf(3, 2, 96), bf(96), bf(96), cs, i32(3)),
    "rope: weights": lambda: A.qk_norm_rope(x, x, bf(128), w, cs, i32(3)),
    "rope: kinds of weights": lambda: A.qk_norm_rope(x, x, w, w.float(), cs, i32(3)),
    "rope: rotary dims": lambda: A.qk_norm_rope(x, x, w, w, torch.ones(4, 24, device=dev), i32(3)),
    "rope: table": lambda: A.qk_norm_rope(x, x, w, w, cs.half(), i32(3)),
    "rope: positions": lambda: A.qk_norm_rope(x, x, w, w, cs, i32(4)),
    "rope: v alone": lambda: A.qk_norm_rope(x, x, w, w, cs, i32(3), v=x),
    "rope: cache alone": lambda: A.qk_norm_rope(x, x, w, w, cs, i32(3), cache=cache),
    "rope: heads of v": lambda: A.qk_norm_rope(x, x, w, w, cs, i32(3), v=bf(3, 1, 64), cache=cache, slots=i64),
    "append: slots": lambda: A.kv4_append(x, x, cache, i64[:2]),
    "append: type of slots": lambda: A.kv4_append(x, x, cache, i32(3)),
    "append: v": lambda: A.kv4_append(x, bf(3, 2, 128), cache, i64),
    "append: heads": lambda: A.kv4_append(bf(3, 4, 64), bf(3, 4, 64), cache, i64),
    "append: dims": lambda: A.kv4_append(x[0], x[0], cache, i64),
    "read: slots": lambda: A.kv4_read(cache, i64[:, None]),
    "read: device": lambda: A.kv4_read(cache, i64.cpu()),
    "attend: head size": lambda: A.kv4_attention(bf(1, 2, 128), cache, i32(1, 4), one, start, 1),
    "attend: heads": lambda: A.kv4_attention(bf(1, 3, 64), cache, i32(1, 4), one, start, 1),
    "attend: table": lambda: A.kv4_attention(x, cache, i32(2, 4), one, start, 1),
    "attend: offsets": lambda: A.kv4_attention(x, cache, i32(1, 4), one, i32(1), 1),
    "attend: window": lambda: A.kv4_attention(x, cache, i32(1, 4), one, start, 1, window=-1),
    "attend: out": lambda: A.kv4_attention(x, cache, i32(1, 4), one, start, 1, out=bf(3, 2, 128)),
    "attend: type of out": lambda: A.kv4_attention(x, cache, i32(1, 4), one, start, 1, out=x.half()),
}
for name, call in wrong.items():
    try:
        call()
    except ValueError as e:
        assert str(e), name
    else:
        raise SystemExit(name + " was taken")
for call in (lambda: A.kv4_append(x, x, cache, None), lambda: A.kv4_attention(x, cache, i32(1, 4), one, start, 1.5),
             lambda: A.plan_batch([1], one, i32(1, 4), i32(8), one, 16, 4)):
    try:
        call()
    except TypeError:
        continue
    raise SystemExit("a wrong type was taken")
A.check_status(dev)
print("fine")
"""


@pytest.mark.gpu
def test_every_wrong_argument_is_a_python_exception(attention_lib):
    got = subprocess.run([sys.executable, "-c", CALLS], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert got.returncode == 0 and got.stdout.strip() == "fine", f"{got.returncode}: {got.stdout}{got.stderr}"


def test_the_c_entry_refuses_scales_that_are_not_numbers(attention_lib):
    lib = ctypes.CDLL(attention_lib)
    vp, i, i64, f, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
    lib.mono_attn_kv4_attention.argtypes = [vp, i64, i64, vp, i64, i, vp, i, vp, vp, i, i, i, i, i, i, f, i, vp, vp, vp, z, vp, vp]
    p = ctypes.addressof(ctypes.create_string_buffer(64))
    for scale, code in ((math.nan, -202), (math.inf, -202), (-math.inf, -202), (0.1, -204)):
        assert lib.mono_attn_kv4_attention(p, 128, 128, p, 4, 16, p, 4, p, p, 1, 1, 1, 4, 2, 128, scale, 0, p, 0, p, 100, p, 0) == code


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_scales_that_are_not_numbers_are_refused(attention_lib, scale):
    import torch
    from unimonomoe_b200 import attention as A
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    cache, x = A.KV4Cache.empty(1, 1, 64), torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="scale"):
        A.kv4_attention(x, cache, one[None] * 0, one, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1, scale=scale)
