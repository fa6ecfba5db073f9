"""The block-FP8 operators where the package uses them: a whole MoE layer against the one launch, and the example decoder."""
import os
import sys

import pytest
import torch

from unimonomoe_b200 import MonoKernel, fp8_quantize, linear, moe_experts, plan_experts, synth, variant_path

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(scope="module")
def one_launch(built_libs, linear_lib):
    return MonoKernel(variant_path("qwen_w1")), synth.make_layer(synth.QWEN, seed=3, device="cuda", with_shared=False)


@pytest.mark.parametrize("tokens", [1, 24, 700, 5000])
def test_operators_and_the_one_launch_agree(one_launch, tokens):
    """Codes, scales and the order of rows are the same bits. Both have the same sums up to fp32's rounding, which moves one code in some 10^4 of the
    activation in the middle, and round each expert's row to bf16, one before its weight and one behind it: 2^-9 of a row at
    most, 2^-9 / sqrt(3) on average, twice. A hundredth is several times that in root mean square."""
    kernel, layer = one_launch
    batch = synth.make_batch(synth.QWEN, layer, tokens, seed=tokens, device="cuda", skew=0.3)
    w = [layer[n] for n in ("w13", "w13_scale", "w2", "w2_scale")]
    out = torch.empty(tokens, synth.QWEN.hidden, dtype=torch.bfloat16, device="cuda")
    seen = kernel.prefill_impl(batch["hs"], batch["logits"], *w, 8, True, None, out, check=True)
    codes, scales = fp8_quantize(batch["hs"])
    assert torch.equal(codes.view(torch.uint8), seen["act_fp8"]) and torch.equal(scales, seen["act_scales"])
    plan = plan_experts(seen["topk_ids"], 256)
    assert torch.equal(plan.tokens, torch.div(seen["sorted_ids"], 8, rounding_mode="floor"))
    got = moe_experts(batch["hs"], seen["topk_ids"], seen["topk_weights"], *w)
    linear.check_status()
    assert float((got.double() - out.double()).norm()) <= 1e-2 * float(out.double().norm())


def test_the_decoder_by_operators(linear_lib, attention_lib):
    """Prompts in chunks, then decoding from a captured graph. The states behind the prompts are near to those with the one launch: layers differ by
    roundings to bf16 and codes next to one another, a few hundredths of the states in root mean square after two layers."""
    import decoder_layers
    gen = torch.Generator(device="cuda").manual_seed(5)
    prompts = [torch.randint(0, 8192, (n,), generator=gen, device="cuda") for n in (30, 1, 200)]
    last = []
    for operators in (False, True):
        server = decoder_layers.Server(2, 3, 260, fp8=True, operators=operators)
        states, inner = [], server.step
        server.step = lambda *a, inner=inner, states=states: states.append(inner(*a)) or states[-1]
        first = server.prefill(prompts, 231)
        last.append(states[-1][0].double())
        server.step = inner
        more = server.decode(first, 8)
        decoder_layers.check_status()
        linear.check_status()
        assert more.shape == (3, 8) and ((more >= 0) & (more < 8192)).all()
    assert last[0].shape == last[1].shape and torch.isfinite(last[1]).all()
    assert float((last[0] - last[1]).norm()) <= 5e-2 * float(last[0].norm())
