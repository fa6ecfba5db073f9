"""The attention half of a decoder layer, next to the MoE half of loader.py, over a paged key/value cache held in 4 bits:

* ``plan_batch``      positions, cache slots and block-table entries of a step, on the GPU, from the lengths of its requests
* ``qk_norm_rope``    norms of query and key heads with the position rotation, and the keys and values into the cache
* ``kv4_append``, ``kv4_read``   keys and values into the cache by slot, and back
* ``kv4_attention``   attention of single tokens, guessed tokens, chunks and whole prompts over the cache

Host side of ``libmono_attention.so`` (include/mono_attention.h): arguments are checked, outputs and workspaces made (in C++,
csrc/attention/binding.cpp), the launch goes to the current stream. Shapes, types and devices raise ValueError before anything is
launched. The workspace of ``kv4_attention`` is kept for each stream: launches on one stream, or graphs captured on it, must
not overlap. What only the device knows (slots, pages, lengths) is checked there: the access is left out and the first fault kept in a status word, which
``check_status`` reads. Forward only: results carry no graph. There is no CPU or library fallback.
"""
from __future__ import annotations

import importlib.util
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

_C = None


def attention_lib_path() -> str:
    """Path of the in-tree library (see unimonomoe_b200/build.py)."""
    return os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libmono_attention.so")


def _load():
    """The Python module next to the library (csrc/attention/binding.cpp): checks, outputs, launches."""
    global _C
    if _C is None:
        path = os.path.join(os.path.dirname(attention_lib_path()), "_mono_attention.so")
        try:
            spec = importlib.util.spec_from_file_location("_mono_attention", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as e:
            raise RuntimeError(f"{path} cannot be loaded; build it with `python -m unimonomoe_b200.build attention`") from e
        _C = module
    return _C


def check_status(device=None) -> None:
    """Synchronise and raise if a launch on this device has reported a fault since the last call."""
    dev = torch.device("cuda" if device is None else device)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    word = _load().status_tensor(index)
    torch.cuda.synchronize(index)
    code, where = word.tolist()
    if code:
        word.zero_()
        torch.cuda.synchronize(index)                           # a launch on any stream behind this one may report again
        raise RuntimeError(f"attention device status: {STATUS_CODES.get(code, code)} (code {code}, at {where})")


def _head_dim(d: int) -> int:
    if d not in HEAD_DIMS:
        raise ValueError(f"head size {d}; the kernels have {HEAD_DIMS}")
    return d


def _page_size(p: int) -> int:
    if p < 16 or p > 1024 or p & (p - 1):
        raise ValueError(f"page size {p}; a power of two from 16 to 1024 is needed")
    return p


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
    ``block_table`` in place; where the list is too short, -1 is entered and ``taken`` of the result lies behind its end. ``num_tokens`` is the number of rows of the result: rows behind the last token hold position
    0, slot -1, request -1, so a captured graph serves any smaller step. Nothing is read back to the host."""
    return BatchPlan(*(_C or _load()).plan(cached_lens, new_lens, block_table, free_pages, taken, page_size, num_tokens))



def qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps: float = 1e-6, interleaved: bool = False,
                 unit_offset: bool = False, v=None, cache: Optional[KV4Cache] = None, slots=None):
    """Root-mean-square norm of every head of ``q`` [tokens, heads, head_dim] and ``k`` [tokens, kv_heads, head_dim] (bf16; views of
    a fused projection are taken as they are), weights ``q_weight`` and ``k_weight`` [head_dim] (bf16 or fp32; ``unit_offset``: 1 + w),
    then the rotation of the first ``cos_sin.size(1)`` dims by the row ``positions[t]`` of ``cos_sin`` (fp32 [positions, rotary_dim],
    cosines then sines): halves against each other, or neighbours where ``interleaved``. Returns contiguous (q, k).

    With ``cache``, ``v`` and ``slots`` the rotated keys and the values are stored in the cache in the same launch, the same
    codes as ``kv4_append`` of the results; only q is returned."""
    return (_C or _load()).qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved, unit_offset, v,
                                        None if cache is None else cache.data, slots)



def kv4_append(k, v, cache: KV4Cache, slots) -> None:
    """Stores ``k`` and ``v`` (bf16 [tokens, kv_heads, head_dim], any strides) in the cache at ``slots`` (int64 [tokens], -1: not
    stored). No slot may be given twice."""
    (_C or _load()).kv4_append(k, v, cache.data, slots)



def kv4_read(cache: KV4Cache, slots):
    """What the cache holds at ``slots`` (int64 [tokens]) as (k, v), bf16 [tokens, kv_heads, head_dim], exactly; zeros at -1."""
    return (_C or _load()).kv4_read(cache.data, slots)



def kv4_attention(q, cache: KV4Cache, block_table, seq_lens, query_start, max_query_len: int, scale: Optional[float] = None,
                  window: int = 0, out=None, return_lse: bool = False):
    """Attention of ``q`` (bf16 [tokens, heads, head_dim]) over the cache. Rows ``query_start[b]`` to ``query_start[b + 1]`` (int32
    [batch + 1]) are the last tokens of sequence b, which is ``seq_lens[b]`` (int32 [batch]) long with them and lies in the pages
    ``block_table[b]`` (int32 [batch, width]). Each query sees the keys up to its own place; with ``window`` > 0, the last
    ``window`` of those. A page that is missing from the table is reported, its keys and values are zeros. heads / kv_heads query heads share a KV head. ``scale`` is 1 / sqrt(head_dim) unless given.

    Returns ``out`` (bf16 [tokens, heads, head_dim], made unless given) or (out, lse) with the fp32 natural log-sum-exp [tokens,
    heads]. A query that sees no key gets zeros and -inf. Rows that belong to no request are left as they are (what
    is made here is unset there).

    ``max_query_len``: the largest number of queries of a request, or anything above; it chooses kernels, never results."""
    return (_C or _load()).kv4_attention(q, cache.data, block_table, seq_lens, query_start, max_query_len, scale, window, out, return_lse)
