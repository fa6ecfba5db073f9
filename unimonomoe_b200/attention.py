"""The attention half of a decoder layer, next to the MoE half of loader.py, over a paged key/value cache held in 4 bits:

* ``plan_batch``      positions, cache slots and block-table entries of a step, on the GPU, from the lengths of its requests
* ``qk_norm_rope``    norms of query and key heads with the position rotation, and the keys and values into the cache
* ``kv4_append``, ``kv4_read``   keys and values into the cache by slot, and back
* ``kv4_attention``   attention of single tokens, guessed tokens, chunks and whole prompts over the cache

Host side of ``libmono_attention.so`` (include/mono_attention.h): arguments are checked, outputs and workspaces made, the
launch goes to the current stream. Shapes, types and devices raise ValueError before anything is launched. What only the
device knows (slots, pages, lengths) is checked there: the access is left out and the first fault kept in a status word, which
``check_status`` reads. There is no CPU or library fallback.
"""
from __future__ import annotations

import ctypes
import os
from typing import NamedTuple, Optional

import torch

STATUS_CODES = {
    0: "ok", 1: "position outside the rotation table", 2: "slot outside the cache", 3: "block-table entry outside the cache",
    4: "sequence longer than its row of the block table", 5: "more pages needed than are free",
    6: "more tokens than num_tokens", 7: "negative length, or query offsets out of order", 8: "a wait inside a kernel ran out",
}
GROUP = 64                                   # dims that share a scale
BLOCK = 16                                   # tokens of a block
HEAD_DIMS = (64, 128, 256)
MAX_REQUESTS = 16384

_lib = None


def attention_lib_path() -> str:
    """Path of the in-tree library (see unimonomoe_b200/build.py)."""
    return os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libmono_attention.so")


def _load():
    global _lib
    if _lib is None:
        path = attention_lib_path()
        try:
            lib = ctypes.CDLL(path)
        except OSError as e:
            raise RuntimeError(f"{path} cannot be loaded; build it with `python -m unimonomoe_b200.build attention`") from e
        p, i, l, f, z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
        lib.mono_attn_plan.argtypes = [p, p, i, p, i, p, i, p, i, i, p, p, p, p, p, p, p, p]
        lib.mono_attn_qk_norm_rope.argtypes = [p, l, l, p, l, l, p, p, i, i, f, p, i, i, i, p, i, i, i, i, p, p, p, l, l, p, l, i,
                                               p, p, p]
        lib.mono_attn_kv4_append.argtypes = [p, l, l, p, l, l, i, i, i, p, l, i, p, p, p]
        lib.mono_attn_kv4_read.argtypes = [p, l, i, p, i, i, i, p, p, p, p]
        lib.mono_attn_kv4_attention.argtypes = [p, l, l, p, l, i, p, i, p, p, i, i, i, i, i, i, f, i, p, p, p, z, p, p]
        lib.mono_attn_workspace_bytes.restype = z
        _lib = lib
    return _lib


_ERRORS = {-201: "a required pointer is null", -202: "a size is out of its range", -203: "head size is not 64, 128 or 256",
           -204: "workspace too small"}


def _launched(name: str, rc: int) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed: rc={rc}" + (f" ({_ERRORS[rc]})" if rc in _ERRORS else ""))


# ---------------------------------------------------------------------- device state
_status = {}
_workspaces = {}


def _status_word(device: torch.device) -> torch.Tensor:
    s = _status.get(device.index)
    if s is None:
        s = _status[device.index] = torch.zeros(2, dtype=torch.int32, device=device)
    return s


def check_status(device=None) -> None:
    """Synchronise and raise if a launch on this device has reported a fault since the last call."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = _status.get(torch.cuda.current_device() if dev.index is None else dev.index)
    if word is None:
        return
    torch.cuda.synchronize(word.device)
    code, where = word.tolist()
    if code:
        word.zero_()
        raise RuntimeError(f"attention device status: {STATUS_CODES.get(code, code)} (code {code}, at {where})")


def _workspace(device: torch.device, stream: int) -> torch.Tensor:
    """Scratch of the attention launches, one per device and stream, its counters zero between launches. A capture that finds
    none gets buffers of its own, so that the capture's memory pool owns them."""
    key = (device.index, stream)
    ws = _workspaces.get(key)
    if ws is None:
        ws = torch.empty(_load().mono_attn_workspace_bytes(), dtype=torch.uint8, device=device)
        ws[:1 << 16].zero_()
        if not torch.cuda.is_current_stream_capturing():
            _workspaces[key] = ws
    return ws


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _cuda(name: str, t: torch.Tensor, dtype=None, device=None) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}; these operators need a CUDA device, there is no CPU path")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _ints(name: str, t: torch.Tensor, shape, device, dtype=torch.int32) -> torch.Tensor:
    _cuda(name, t, dtype, device)
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(name: str, t: torch.Tensor, device=None) -> torch.Tensor:
    """bf16 [tokens, heads, head_dim] with 16-byte rows; any other layout is copied into one."""
    _cuda(name, t, torch.bfloat16, device)
    if t.dim() != 3:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [tokens, heads, head_dim]")
    a, b, c = t.stride()
    if c != 1 or (a | b) & 7 or t.data_ptr() & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
    return t


def _head_dim(d: int) -> int:
    if d not in HEAD_DIMS:
        raise ValueError(f"head size {d}; the kernels have {HEAD_DIMS}")
    return d


def _page_size(p: int) -> int:
    if p < 16 or p > 1024 or p & (p - 1):
        raise ValueError(f"page size {p}; a power of two from 16 to 1024 is needed")
    return p


class _On:
    """The tensor's device as the current one, where it is not already."""

    def __init__(self, device):
        self.device, self.before = device, None

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self.device.index:
            self.before = now
            torch.cuda.set_device(self.device)

    def __exit__(self, *exc):
        if self.before is not None:
            torch.cuda.set_device(self.before)


# ---------------------------------------------------------------------- the cache
def _code_places(dim: int, values: bool) -> torch.Tensor:
    """Place, in half bytes, of the code of each token and dim among the key or value codes of a block: [16, dim]."""
    ng = dim // GROUP
    r, d = torch.meshgrid(torch.arange(BLOCK), torch.arange(dim), indexing="ij")
    if values:
        lane, o = (d % 64 // 8) * 4 + r // 2 % 4, (r // 8 * 2 + r % 2) * 4 * ng + d // 64 * 4 + d % 8 // 2
    else:
        lane, o = r % 8 * 4 + d % 64 // 16, r // 8 * 8 * ng + d // 64 * 8 + d % 16 // 8 * 4 + d % 8 // 2
    return (o // 16 * 512 + lane * 16 + o % 16) * 2 + d % 2


class KV4Cache:
    """Paged keys and values of one layer in 4 bits: ``data`` is uint8 [num_pages, kv_heads, page_size / 16, 17 * head_dim].

    64 dims of a token's key or value share a scale: a seventh of their largest magnitude, rounded to five significant bits
    and kept within 2^-60 and 2^60; codes are the nearest multiples from -7 to 7. A multiple of such a scale is exact in
    bfloat16. A group that is not finite is stored as NaN. 4.25 bits a value."""

    def __init__(self, data: torch.Tensor):
        if data.dim() != 4 or data.dtype != torch.uint8 or not data.is_contiguous():
            raise ValueError(f"cache data must be contiguous uint8 [num_pages, kv_heads, page_size / 16, 17 * head_dim], got "
                             f"{tuple(data.shape)} {data.dtype}")
        self.num_pages, self.kv_heads, blocks, width = data.shape
        if width % 17:
            raise ValueError(f"cache blocks of {width} bytes; expected 17 * head_dim")
        self.head_dim, self.page_size = _head_dim(width // 17), _page_size(blocks * BLOCK)
        if not self.num_pages or not self.kv_heads:
            raise ValueError("a cache needs at least one page and one KV head")
        if data.data_ptr() & 15:
            raise ValueError("cache data must begin on a 16-byte boundary")
        self.data = data

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 16, device="cuda") -> "KV4Cache":
        return cls(torch.empty(num_pages, kv_heads, _page_size(page_size) // BLOCK, 17 * _head_dim(head_dim), dtype=torch.uint8, device=device))

    @property
    def device(self) -> torch.device:
        return self.data.device

    def dequantize(self, pages: Optional[torch.Tensor] = None):
        """Keys and values of whole pages in fp32, [pages, page_size, kv_heads, head_dim] each, by torch operations on any
        device: for tests and for moving a cache into another format."""
        d, ng = self.head_dim, self.head_dim // GROUP
        blocks = self.data if pages is None else self.data[pages.long()]
        scales = blocks[..., 16 * d:].contiguous().view(torch.bfloat16).float().unflatten(-1, (BLOCK, 2, ng))
        got = []
        for i in range(2):
            x = blocks[..., 8 * d * i:8 * d * (i + 1)]
            codes = torch.stack([x & 15, x >> 4], -1).flatten(-2)[..., _code_places(d, bool(i)).to(x.device)]
            v = (codes.float() - 8).unflatten(-1, (ng, GROUP)) * scales[..., i, :, None]
            got.append(v.flatten(-2).flatten(2, 3).transpose(1, 2))
        return got[0], got[1]


# ---------------------------------------------------------------------- operators
class BatchPlan(NamedTuple):
    query_start: torch.Tensor                # int32 [batch + 1]
    seq_lens: torch.Tensor                   # int32 [batch]
    positions: torch.Tensor                  # int32 [num_tokens]
    slots: torch.Tensor                      # int64 [num_tokens], -1: no place
    requests: torch.Tensor                   # int32 [num_tokens], -1: no request
    taken: torch.Tensor                      # int32 [1], pages handed out so far


def plan_batch(cached_lens, new_lens, block_table, free_pages, taken, page_size: int, num_tokens: int) -> BatchPlan:
    """Where the tokens of a step go. ``cached_lens`` and ``new_lens`` (int32 [batch]) are each request's tokens in the cache and
    in this step, ``block_table`` (int32 [batch, width]) its pages, ``free_pages`` (int32) the free list, of which the first
    ``taken`` (int32 [1]) are in use. New pages are taken from the list in the order of the requests and entered into
    ``block_table`` in place. ``num_tokens`` is the number of rows of the result: rows behind the last token hold position
    0, slot -1, request -1, so a captured graph serves any smaller step. Nothing is read back to the host."""
    dev = _cuda("cached_lens", cached_lens, torch.int32).device
    B = cached_lens.numel()
    if not 1 <= B <= MAX_REQUESTS:
        raise ValueError(f"{B} requests; 1 to {MAX_REQUESTS} are planned at a time")
    cached_lens, new_lens = _ints("cached_lens", cached_lens, (B,), dev), _ints("new_lens", new_lens, (B,), dev)
    _cuda("block_table", block_table, torch.int32, dev)
    if block_table.dim() != 2 or block_table.size(0) != B or block_table.size(1) < 1 or not block_table.is_contiguous():
        raise ValueError(f"block_table must be contiguous int32 [{B}, pages], got {tuple(block_table.shape)}")
    free_pages, taken = _ints("free_pages", free_pages, (free_pages.numel(),), dev), _ints("taken", taken, (1,), dev)
    num_tokens = int(num_tokens)
    if num_tokens < 0:
        raise ValueError(f"num_tokens is {num_tokens}")
    _page_size(page_size)
    lib = _load()
    with _On(dev):
        new = lambda n, dt=torch.int32: torch.empty(n, dtype=dt, device=dev)  # noqa: E731
        p = BatchPlan(new(B + 1), new(B), new(num_tokens), new(num_tokens, torch.int64), new(num_tokens), new(1))
        _launched("mono_attn_plan", lib.mono_attn_plan(
            cached_lens.data_ptr(), new_lens.data_ptr(), B, block_table.data_ptr(), block_table.size(1), free_pages.data_ptr(),
            free_pages.numel(), taken.data_ptr(), page_size, num_tokens, p.query_start.data_ptr(), p.seq_lens.data_ptr(),
            p.positions.data_ptr(), p.slots.data_ptr(), p.requests.data_ptr(), p.taken.data_ptr(), _status_word(dev).data_ptr(),
            _stream(dev)))
    return p


def _check_cache(cache: KV4Cache, kv_heads: int, head_dim: int, device) -> None:
    if cache.kv_heads != kv_heads or cache.head_dim != head_dim or cache.device != device:
        raise ValueError(f"cache holds {cache.kv_heads} KV heads of {cache.head_dim} on {cache.device}, the call has {kv_heads} of "
                         f"{head_dim} on {device}")


def qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps: float = 1e-6, interleaved: bool = False,
                 unit_offset: bool = False, v=None, cache: Optional[KV4Cache] = None, slots=None):
    """Root-mean-square norm of every head of ``q`` [tokens, heads, head_dim] and ``k`` [tokens, kv_heads, head_dim] (bf16; views of
    a fused projection are taken as they are), weights ``q_weight`` and ``k_weight`` [head_dim] (bf16 or fp32; ``unit_offset``: 1 + w),
    then the rotation of the first ``cos_sin.size(1)`` dims by the row ``positions[t]`` of ``cos_sin`` (fp32 [positions, rotary_dim],
    cosines then sines): halves against each other, or neighbours where ``interleaved``. Returns contiguous (q, k).

    With ``cache``, ``v`` and ``slots`` the rotated keys and the values are stored in the cache in the same launch, the same
    codes as ``kv4_append`` of the results; only q is returned."""
    q = _rows("q", q)
    dev = q.device
    k = _rows("k", k, dev)
    T, H, D = q.shape
    K = k.size(1)
    _head_dim(D)
    if k.size(0) != T or k.size(2) != D or not H or not K:
        raise ValueError(f"q is {tuple(q.shape)}, k is {tuple(k.shape)}: tokens and head size must agree")
    if q_weight.dtype not in (torch.bfloat16, torch.float32) or k_weight.dtype != q_weight.dtype:
        raise ValueError(f"norm weights must both be bfloat16 or float32, got {q_weight.dtype} and {k_weight.dtype}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if _cuda(name, w, None, dev).shape != (D,) or not w.is_contiguous() or w.data_ptr() & 15:
            raise ValueError(f"{name} must be contiguous [{D}] on a 16-byte boundary, got {tuple(w.shape)}")
    _cuda("cos_sin", cos_sin, torch.float32, dev)
    if cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.data_ptr() & 15:
        raise ValueError(f"cos_sin must be contiguous fp32 [positions, rotary_dim], got {tuple(cos_sin.shape)}")
    R = cos_sin.size(1)
    if R % 16 or R > D:
        raise ValueError(f"rotary dim {R}; a multiple of 16 up to the head size {D} is needed")
    if R and not cos_sin.size(0):
        raise ValueError("cos_sin has no rows")
    positions = _ints("positions", positions, (T,), dev)
    stored = (0, 0, 0, 0, 0, 16, 0)
    if cache is not None:
        if v is None or slots is None:
            raise ValueError("storing into a cache needs v and slots")
        v = _rows("v", v, dev)
        if v.shape != k.shape:
            raise ValueError(f"v is {tuple(v.shape)}, k is {tuple(k.shape)}")
        _check_cache(cache, K, D, dev)
        slots = _ints("slots", slots, (T,), dev, torch.int64)
        stored = (v.data_ptr(), v.stride(0), v.stride(1), cache.data.data_ptr(), cache.num_pages, cache.page_size, slots.data_ptr())
    elif v is not None or slots is not None:
        raise ValueError("v and slots are stored in a cache, and none is given")
    lib = _load()
    with _On(dev):
        q_out = torch.empty((T, H, D), dtype=torch.bfloat16, device=dev)
        k_out = None if cache is not None else torch.empty((T, K, D), dtype=torch.bfloat16, device=dev)
        _launched("mono_attn_qk_norm_rope", lib.mono_attn_qk_norm_rope(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), q_weight.data_ptr(), k_weight.data_ptr(),
            q_weight.dtype == torch.float32, bool(unit_offset), float(eps), cos_sin.data_ptr(), cos_sin.size(0), R, bool(interleaved),
            positions.data_ptr(), T, H, K, D, q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(), *stored,
            _status_word(dev).data_ptr(), _stream(dev)) if T else 0)
    return q_out if k_out is None else (q_out, k_out)


def kv4_append(k, v, cache: KV4Cache, slots) -> None:
    """Stores ``k`` and ``v`` (bf16 [tokens, kv_heads, head_dim], any strides) in the cache at ``slots`` (int64 [tokens], -1: not
    stored). No slot may be given twice."""
    k = _rows("k", k)
    dev = k.device
    v = _rows("v", v, dev)
    T, K, D = k.shape
    if v.shape != k.shape:
        raise ValueError(f"v is {tuple(v.shape)}, k is {tuple(k.shape)}")
    _check_cache(cache, K, D, dev)
    slots = _ints("slots", slots, (T,), dev, torch.int64)
    if not T:
        return
    lib = _load()
    with _On(dev):
        _launched("mono_attn_kv4_append", lib.mono_attn_kv4_append(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), T, K, D, cache.data.data_ptr(),
            cache.num_pages, cache.page_size, slots.data_ptr(), _status_word(dev).data_ptr(), _stream(dev)))


def kv4_read(cache: KV4Cache, slots):
    """What the cache holds at ``slots`` (int64 [tokens]) as (k, v), bf16 [tokens, kv_heads, head_dim], exactly; zeros at -1."""
    dev = _cuda("cache", cache.data).device
    T = slots.numel()
    slots = _ints("slots", slots, (T,), dev, torch.int64)
    lib = _load()
    with _On(dev):
        k, v = (torch.empty((T, cache.kv_heads, cache.head_dim), dtype=torch.bfloat16, device=dev) for _ in range(2))
        if T:
            _launched("mono_attn_kv4_read", lib.mono_attn_kv4_read(
                cache.data.data_ptr(), cache.num_pages, cache.page_size, slots.data_ptr(), T, cache.kv_heads, cache.head_dim,
                k.data_ptr(), v.data_ptr(), _status_word(dev).data_ptr(), _stream(dev)))
    return k, v


def kv4_attention(q, cache: KV4Cache, block_table, seq_lens, query_start, max_query_len: int, scale: Optional[float] = None,
                  window: int = 0, out=None, return_lse: bool = False):
    """Attention of ``q`` (bf16 [tokens, heads, head_dim]) over the cache. Rows ``query_start[b]`` to ``query_start[b + 1]`` (int32
    [batch + 1]) are the last tokens of sequence b, which is ``seq_lens[b]`` (int32 [batch]) long with them and lies in the pages
    ``block_table[b]`` (int32 [batch, width]). Each query sees the keys up to its own place; with ``window`` > 0, the last
    ``window`` of those. heads / kv_heads query heads share a KV head. ``scale`` is 1 / sqrt(head_dim) unless given.

    Returns ``out`` (bf16 [tokens, heads, head_dim], made unless given) or (out, lse) with the fp32 natural log-sum-exp [tokens,
    heads]. A query that sees no key gets zeros and -inf. Rows that belong to no request are left as they are.

    ``max_query_len``: the largest number of queries of a request, or anything above; it chooses kernels, never results."""
    q = _rows("q", q)
    dev = q.device
    T, H, D = q.shape
    K = cache.kv_heads
    _check_cache(cache, K, D, dev)
    if not H or H % K:
        raise ValueError(f"{H} query heads over {K} KV heads")
    B = seq_lens.numel()
    _cuda("block_table", block_table, torch.int32, dev)
    if block_table.dim() != 2 or block_table.size(0) != B or not block_table.size(1) or not block_table.is_contiguous():
        raise ValueError(f"block_table must be contiguous int32 [{B}, pages], got {tuple(block_table.shape)}")
    if B > MAX_REQUESTS:
        raise ValueError(f"{B} requests; up to {MAX_REQUESTS} are taken at a time")
    seq_lens, query_start = _ints("seq_lens", seq_lens, (B,), dev), _ints("query_start", query_start, (B + 1,), dev)
    if window < 0 or max_query_len < 0:
        raise ValueError(f"window is {window}, max_query_len is {max_query_len}")
    if out is None:
        out = torch.empty((T, H, D), dtype=torch.bfloat16, device=dev)
    elif out.shape != (T, H, D) or _cuda("out", out, torch.bfloat16, dev).data_ptr() & 15 or not out.is_contiguous():
        raise ValueError(f"out must be contiguous bfloat16 [{T}, {H}, {D}] on a 16-byte boundary, got {tuple(out.shape)}")
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    if T and B:
        lib = _load()
        with _On(dev):
            stream = _stream(dev)
            ws = _workspace(dev, stream)
            _launched("mono_attn_kv4_attention", lib.mono_attn_kv4_attention(
                q.data_ptr(), q.stride(0), q.stride(1), cache.data.data_ptr(), cache.num_pages, cache.page_size,
                block_table.data_ptr(), block_table.size(1), seq_lens.data_ptr(), query_start.data_ptr(), B, T, int(max_query_len),
                H, K, D, D ** -0.5 if scale is None else float(scale), int(window), out.data_ptr(),
                0 if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(), _status_word(dev).data_ptr(), stream))
    return (out, lse) if return_lse else out
