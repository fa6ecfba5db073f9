"""The attention operators without a GPU: the library's symbols and return codes, the cache's layout, refusals."""
import ctypes
import os
import re

import pytest
import torch

from tests import attention_ref as ref
from unimonomoe_b200 import attention as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_declared_symbol_is_exported(attention_lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mono_attention.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(mono_attn_\w+)\s*\(", text))
    assert len(names) >= 6
    lib = ctypes.CDLL(attention_lib)
    assert not [n for n in names if not hasattr(lib, n)]
    assert A.attention_lib_path() == attention_lib


def test_return_codes_before_any_cuda_call(attention_lib):
    lib = ctypes.CDLL(attention_lib)
    vp, i, i64, f, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
    lib.mono_attn_plan.argtypes = [vp, vp, i, vp, i, vp, i, vp, i, i, vp, vp, vp, vp, vp, vp, vp, vp]
    lib.mono_attn_qk_norm_rope.argtypes = [vp, i64, i64, vp, i64, i64, vp, vp, i, i, f, vp, i, i, i, vp, i, i, i, i, vp, vp, vp, i64, i64, vp, i64, i,
                                           vp, vp, vp]
    lib.mono_attn_kv4_append.argtypes = [vp, i64, i64, vp, i64, i64, i, i, i, vp, i64, i, vp, vp, vp]
    lib.mono_attn_kv4_attention.argtypes = [vp, i64, i64, vp, i64, i, vp, i, vp, vp, i, i, i, i, i, i, f, i, vp, vp, vp, z, vp, vp]
    p = ctypes.addressof(ctypes.create_string_buffer(64))
    good = [p, p, 2, p, 4, p, 8, p, 16, 5, p, p, p, p, p, p, p, 0]
    for at, value, code in ((2, 0, -202), (2, A.MAX_REQUESTS + 1, -202), (8, 24, -202), (8, 8, -202), (0, 0, -201), (12, 0, -201), (16, 0, -201)):
        a = list(good)
        a[at] = value
        assert lib.mono_attn_plan(*a) == code, at
    append = [p, 128, 128, p, 128, 128, 3, 1, 128, p, 4, 16, p, p, 0]
    for at, value, code in ((8, 96, -203), (7, 0, -202), (11, 20, -202), (9, 0, -201), (12, 0, -201)):
        a = list(append)
        a[at] = value
        assert lib.mono_attn_kv4_append(*a) == code, at
    append[6] = 0
    assert lib.mono_attn_kv4_append(*append) == 0
    attend = [p, 128, 128, p, 4, 16, p, 4, p, p, 1, 1, 1, 4, 2, 128, 0.1, 0, p, 0, p, 1 << 30, p, 0]
    for at, value, code in ((15, 80, -203), (13, 3, -202), (17, -1, -202), (7, 0, -202), (3, 0, -201), (20, 0, -201), (21, 100, -204)):
        a = list(attend)
        a[at] = value
        assert lib.mono_attn_kv4_attention(*a) == code, at
    rope = [p, 128, 128, p, 128, 128, p, p, 0, 0, 1e-6, p, 10, 64, 0, p, 1, 2, 1, 128, p, p, 0, 0, 0, 0, 0, 16, 0, p, 0]
    for at, value, code in ((13, 40, -202), (13, 144, -202), (19, 32, -203), (0, 0, -201), (11, 0, -201), (21, 0, -201), (25, p, -201)):
        a = list(rope)
        a[at] = value
        assert lib.mono_attn_qk_norm_rope(*a) == code, at


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_code_has_a_place_of_its_own_and_dequantize_reads_it(dim):
    for values in (False, True):
        at = A._code_places(dim, values)
        assert sorted(at.flatten().tolist()) == list(range(16 * dim))
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randn(3, 32, 2, dim, generator=g) for _ in range(2))    # [pages, page_size, heads, dim]
    cache = A.KV4Cache.empty(3, 2, dim, 32, "cpu")
    for i, x in enumerate((k, v)):
        q = ref.quantised(x.to(torch.bfloat16)).view(3, 2, 16, 2, dim).permute(0, 3, 1, 2, 4)    # [pages, heads, blocks, 16, dim]
        grouped = x.to(torch.bfloat16).double().view(3, 2, 16, 2, dim).permute(0, 3, 1, 2, 4).unflatten(-1, (-1, 64))
        s = ref.round_bits(grouped.abs().amax(-1) / 7, 5)
        codes = (torch.round(q.unflatten(-1, (-1, 64)) / s[..., None]) + 8).flatten(-2).to(torch.uint8)
        nib = torch.zeros(3, 2, 2, 16 * dim, dtype=torch.uint8)
        nib[..., A._code_places(dim, bool(i)).flatten()] = codes.flatten(-2)
        cache.data[..., 8 * dim * i:8 * dim * (i + 1)] = nib[..., 0::2] | nib[..., 1::2] << 4
        cache.data[..., 16 * dim:].view(3, 2, 2, 16, 2, dim // 32)[..., i, :] = s.to(torch.bfloat16).contiguous().view(torch.uint8).view(3, 2, 2, 16, dim // 32)
    got = cache.dequantize()
    assert torch.equal(got[0].double(), ref.quantised(k.to(torch.bfloat16))) and torch.equal(got[1].double(), ref.quantised(v.to(torch.bfloat16)))
    some = cache.dequantize(torch.tensor([2, 0]))
    assert torch.equal(some[0], got[0][[2, 0]])


@pytest.mark.parametrize("shape", [(1, 1, 1, 100), (1, 1, 3, 17 * 64), (0, 1, 1, 17 * 64), (1, 17 * 64), (1, 1, 1, 17 * 32)])
def test_cache_refuses_other_layouts(shape):
    with pytest.raises(ValueError):
        A.KV4Cache(torch.zeros(shape, dtype=torch.uint8))


def test_cache_refuses_other_types_sizes_and_strides():
    with pytest.raises(ValueError):
        A.KV4Cache(torch.zeros(1, 1, 1, 17 * 64))
    with pytest.raises(ValueError):
        A.KV4Cache(torch.zeros(2, 1, 2, 17 * 64, dtype=torch.uint8)[:, :, ::2])
    for page, dim in ((8, 64), (48, 64), (2048, 64), (16, 96)):
        with pytest.raises(ValueError):
            A.KV4Cache.empty(1, 1, dim, page, "cpu")


def test_operators_refuse_cpu_tensors(attention_lib):
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    cache = A.KV4Cache.empty(1, 1, 64, 16, "cpu")
    for call in (lambda: A.plan_batch(i, i, i[None], i, i, 16, 1), lambda: A.kv4_append(x, x, cache, i.long()), lambda: A.kv4_read(cache, i.long()),
                 lambda: A.qk_norm_rope(x, x, x[0, 0], x[0, 0], torch.zeros(1, 64), i),
                 lambda: A.kv4_attention(x, cache, i[None], i, torch.zeros(2, dtype=torch.int32), 1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
