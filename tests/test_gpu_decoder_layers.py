"""The example decoder (examples/decoder_layers.py): plan_batch, qk_norm_rope with the store, kv4_attention and the MoE launch in
one step, as a server runs them. What the layer's attention returns must not depend on how a prompt was cut into steps."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def decoder(attention_lib):
    import decoder_layers
    return decoder_layers


def first_attention(decoder, prompts, budget):
    """The first layer's attention for every token, in the prompts' order, with the prompts cut at `budget` tokens a step."""
    server = decoder.Server(1, len(prompts), 400)
    got = [[] for _ in prompts]
    layer, inner = server.layers[0], server.layers[0].attention

    def seen(x, plan, *rest):
        out = inner(x, plan, *rest)
        start = plan.query_start.tolist()
        for b in range(len(prompts)):
            got[b].append(out[start[b]:start[b + 1]])
        return out

    layer.attention = seen
    server.prefill(prompts, budget)
    decoder.check_status()
    return torch.cat([torch.cat(g) for g in got]).double()


def test_chunks_and_whole_prompts_agree(decoder):
    gen = torch.Generator(device="cuda").manual_seed(3)
    prompts = [torch.randint(0, 8192, (n,), generator=gen, device="cuda") for n in (1, 37, 300)]
    whole, cut, single = (first_attention(decoder, prompts, n) for n in (338, 129, 5))
    # The embeddings are the same, so only projections of another batch size differ: by a rounding to bf16 in a few values, 2^-9,
    # and by one code where that moves a value over the middle between two (one in a hundred at most, a seventh of the group's largest).
    # Weighted sums of such values stay within 2e-2 of the whole in root mean square.
    for other in (cut, single):
        assert other.shape == whole.shape and torch.isfinite(other).all()
        assert ((other - whole).square().mean() / whole.square().mean()).sqrt() < 2e-2


def test_decoding_goes_on_behind_the_prompts(decoder):
    gen = torch.Generator(device="cuda").manual_seed(4)
    lengths = (20, 1, 150)
    prompts = [torch.randint(0, 8192, (n,), generator=gen, device="cuda") for n in lengths]
    server = decoder.Server(2, 3, 200)
    more = server.decode(server.prefill(prompts, 64), 12)
    decoder.check_status()
    assert more.shape == (3, 12) and ((more >= 0) & (more < 8192)).all()
    assert server.cached.tolist() == [n + 12 for n in lengths]
    pages = [-(-(n + 12) // 16) for n in lengths]
    assert int(server.taken) == sum(pages)
    held = server.table[server.table >= 0]
    assert held.numel() == sum(pages) and held.unique().numel() == held.numel()
