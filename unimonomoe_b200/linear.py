"""The block-FP8 products of a decoder layer outside of the one-launch MoE kernel of loader.py: the projections around attention,
whose checkpoints hold them in the experts' format, and experts of geometries that no binary was compiled for:

* ``fp8_quantize``        rows to 8 bits, with the gated activation in front of it where asked for
* ``fp8_linear``          dense projections, with a residual added or the gated activation behind it
* ``plan_experts``        which rows belong to which expert, on the GPU
* ``fp8_expert_linear``   the products of ragged runs of rows with an expert's weight each
* ``combine_experts``     the weighted sum of each token's results
* ``moe_experts``         these together: a MoE layer's experts from router ids and weights

Numbers: a row has a scale for 128 columns, m / 448 with m their largest magnitude, and e4m3 codes of x * (448 / m), to nearest; a weight has one fp32 scale
for each block of 128 x 128, as checkpoints have it (last blocks may be partial). Where m is below 2^-100 it counts as 1; a group that holds an infinity or a
NaN is NaN, and so are the products of its row. Codes and scales are the MoE kernel's, bit for bit, but for these groups: there m counts as 1 only below
2^-126, a NaN is no group's largest magnitude, and the scale of a group with an infinity is infinite. A group's sum is multiplied by the row's scale times the weight's, which is one fp32 number.

Host side of ``libmono_linear.so`` (include/mono_linear.h): arguments are checked and outputs made (in C++, csrc/linear/binding.cpp), the launch
goes to the current stream. Shapes, types and devices raise ValueError before anything is launched. What only the device knows (expert ids,
offsets, positions) is checked there: the access is left out and the first fault kept in a status word, which ``check_status`` reads.
Nothing is kept between calls, so calls on several streams and captured graphs do not meet. Forward only: results carry no
graph. There is no CPU or library fallback.
"""
from __future__ import annotations

import importlib.util
import os
from typing import NamedTuple, Optional

import torch

STATUS_CODES = {
    0: "ok", 1: "expert id past the last expert", 2: "offsets of experts out of order or outside the rows", 3: "row outside the rows of x",
    4: "position outside the partial rows", 5: "a wait inside a kernel ran out",
}
GROUP = 128                                  # columns that share a scale; rows too in a weight
MAX_EXPERTS = 1024
MAX_TOP = 64                                 # experts of a token

_C = None


def linear_lib_path() -> str:
    """Path of the in-tree library (see unimonomoe_b200/build.py)."""
    return os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libmono_linear.so")


def _load():
    """The Python module next to the library (csrc/linear/binding.cpp): checks, outputs, launches."""
    global _C
    if _C is None:
        path = os.path.join(os.path.dirname(linear_lib_path()), "_mono_linear.so")
        try:
            spec = importlib.util.spec_from_file_location("_mono_linear", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as e:
            raise RuntimeError(f"{path} cannot be loaded; build it with `python -m unimonomoe_b200.build linear`") from e
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
        raise RuntimeError(f"linear device status: {STATUS_CODES.get(code, code)} (code {code}, at {where})")


def fp8_quantize(x, silu_mul: bool = False):
    """``x`` (bf16 [..., K], K a multiple of 16; views whose rows are evenly spaced are taken as they are) in 8 bits: (codes, scales), e4m3 [..., K]
    and fp32 [..., ceil(K / 128)]. With ``silu_mul`` x is [..., 2 K], and the silu of its first half times its second is what
    is quantised."""
    return (_C or _load()).quantize(x, silu_mul)


def fp8_linear(x, weight, weight_scale, x_scale=None, residual=None, silu_mul: bool = False, out_dtype: Optional[torch.dtype] = None):
    """``x`` [..., K] times the transpose of ``weight`` (e4m3 [N, K], K a multiple of 16, any N) with ``weight_scale`` (fp32 [ceil(N / 128),
    ceil(K / 128)]). x is bf16, and quantised as by ``fp8_quantize``, or e4m3 with its scales ``x_scale``. Returns [..., N] in
    bfloat16, or in float32 if that is ``out_dtype``; ``residual`` (bf16 [..., N]) is added before the one rounding.

    With ``silu_mul`` (N a multiple of 256) the silu of the first half of the result times its second half comes back in 8 bits, as
    (codes, scales) of [..., N / 2]: what the next projection takes."""
    if out_dtype not in (None, torch.bfloat16, torch.float32):
        raise ValueError(f"out_dtype {out_dtype}; results are bfloat16 or float32")
    return (_C or _load()).linear(x, weight, weight_scale, x_scale, residual, silu_mul, out_dtype is torch.float32)


class ExpertPlan(NamedTuple):
    offsets: torch.Tensor                    # int32 [experts + 1]: rows offsets[e] to offsets[e + 1] are expert e's
    tokens: torch.Tensor                     # int32 [tokens * top]: the token of each row, -1 behind the last run
    positions: torch.Tensor                  # int32 [tokens, top]: the row of each slot, -1 for a slot computed elsewhere


def plan_experts(ids, num_experts: int) -> ExpertPlan:
    """Division of a batch among experts. ``ids`` (int32 or int64 [tokens, top]) are the experts of each token, negative for those that are
    computed elsewhere (by another rank). Rows are sorted by expert, those of one expert in the order of their slots: the same ids
    give the same plan. Nothing is read back to the host."""
    return ExpertPlan(*(_C or _load()).plan(ids, num_experts))


def fp8_expert_linear(x, weight, weight_scale, plan: ExpertPlan, x_scale=None, gather: bool = True, silu_mul: bool = False):
    """Rows of a plan times their experts' weights (``weight`` e4m3 [experts, N, K], ``weight_scale`` fp32 [experts, ceil(N / 128), ceil(K / 128)]).
    With ``gather``, ``x`` [tokens, K] has the tokens' rows (an up projection), else [tokens * top, K] the plan's (a down projection). x, ``x_scale``,
    ``silu_mul`` and the result, [tokens * top, N] bf16 or (codes, scales) of half the width, are as in ``fp8_linear``. Rows behind the
    last run are not written."""
    return (_C or _load()).experts(x, weight, weight_scale, plan.offsets, plan.tokens, x_scale, gather, silu_mul)


def combine_experts(partial, positions, weights, residual=None):
    """bf16 [tokens, H]: for each token the sum of ``weights[t, j]`` (fp32 [tokens, top]) times row ``positions[t, j]`` (int32, -1: nothing) of
    ``partial`` (bf16 [rows, H], H a multiple of 8), plus ``residual`` (bf16 [tokens, H]); in fp32, in the order of j, rounded once."""
    return (_C or _load()).combine(partial, positions, weights, residual)


def moe_experts(x, ids, weights, w13, w13_scale, w2, w2_scale, residual=None):
    """The experts of a MoE layer, for any geometry: bf16 [tokens, H] = sum over j of weights[t, j] * (silu(x w1^T) * (x w3^T)) w2^T (+ ``residual``)
    with the experts ``ids[t, j]`` (negative: computed elsewhere). ``w13`` [experts, 2 I, H] holds gate rows, then up rows, I a multiple of 128; ``w2``
    is [experts, H, I]. Activations are in 8 bits in front of both projections, as in the MoE launch."""
    (_C or _load()).check_layer(x, ids, weights, w13, w13_scale, w2, w2_scale, residual)
    plan = plan_experts(ids, w13.size(0))
    codes, scales = fp8_quantize(x)
    codes, scales = fp8_expert_linear(codes, w13, w13_scale, plan, x_scale=scales, silu_mul=True)
    partial = fp8_expert_linear(codes, w2, w2_scale, plan, x_scale=scales, gather=False)
    return combine_experts(partial, plan.positions, weights, residual)
