"""A small decoder that serves: whole layers made of this package's two halves, the attention of attention.py over a paged
4-bit cache and the MoE launch of loader.py, on one GPU.

Requests of ragged lengths are prefilled in chunks under a token budget, then decoded together, one captured CUDA graph a step.
Weights are random (synth.py; width and experts of its first geometry), projections and the embedding are plain library products.

    python examples/decoder_layers.py --layers 2 --prompts 700 33 1500 --budget 1024 --new 32
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from unimonomoe_b200 import KV4Cache, MonoKernel, kv4_attention, plan_batch, qk_norm_rope, synth, variant_path  # noqa: E402
from unimonomoe_b200.attention import check_status  # noqa: E402
from unimonomoe_b200.loader import prepare_shared_expert  # noqa: E402

HEADS, KV_HEADS, HEAD_DIM, ROTARY = 16, 2, 256, 64


class Layer:
    """norm, q/k/v projection, norm and rotation of heads with the store into the cache, attention, output projection; norm,
    router, routed and shared experts in one launch."""

    def __init__(self, moe: MonoKernel, pages: int, page_size: int, seed: int, device):
        spec = synth.QWEN
        gen = torch.Generator(device=device).manual_seed(1000 + seed)

        def weight(*shape, std=0.02, mean=0.0):
            return (mean + std * torch.randn(*shape, generator=gen, device=device)).to(torch.bfloat16)

        self.moe, self.cache = moe, KV4Cache.empty(pages, KV_HEADS, HEAD_DIM, page_size, device)
        self.norms = weight(2, spec.hidden, mean=1.0)
        self.q_norm, self.k_norm = weight(HEAD_DIM, mean=1.0), weight(HEAD_DIM, mean=1.0)
        self.qkv = weight((HEADS + 2 * KV_HEADS) * HEAD_DIM, spec.hidden)
        self.o = weight(spec.hidden, HEADS * HEAD_DIM)
        self.experts = synth.make_layer(spec, seed=seed, device=device)
        self.router = self.experts["router_w"].to(torch.bfloat16)
        sh = self.experts["shared"]
        self.shared = prepare_shared_expert(sh["w13"], sh["w13_scale"], sh["w2"], sh["w2_scale"], sh["gate"])

    def attention(self, x, plan, table, cos_sin, longest):
        qkv = F.linear(F.rms_norm(x, x.shape[-1:], self.norms[0], 1e-6), self.qkv).unflatten(1, (-1, HEAD_DIM))
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
        q = qk_norm_rope(q, k, self.q_norm, self.k_norm, cos_sin, plan.positions, v=v, cache=self.cache, slots=plan.slots)
        return kv4_attention(q, self.cache, table, plan.seq_lens, plan.query_start, longest)

    def __call__(self, x, plan, table, cos_sin, longest):
        x = x + F.linear(self.attention(x, plan, table, cos_sin, longest).flatten(1), self.o)
        y, w = F.rms_norm(x, x.shape[-1:], self.norms[1], 1e-6), self.experts
        return x + self.moe.prefill(y, F.linear(y, self.router), w["w13"], w["w13_scale"], w["w2"], w["w2_scale"], shared=self.shared)


class Server:
    """Layers with one page pool. All lengths and tables stay on the GPU; a step reads nothing back but its tokens."""

    def __init__(self, layers: int, batch: int, context: int, page_size: int = 16, vocabulary: int = 8192, device="cuda"):
        self.device, self.batch, self.page_size = torch.device(device), batch, page_size
        width = -(-context // page_size)
        moe = MonoKernel(variant_path("qwen_w1"))
        self.layers = [Layer(moe, batch * width, page_size, i, device) for i in range(layers)]
        gen = torch.Generator(device=device).manual_seed(7)
        self.embedding, self.head = torch.randn(2, vocabulary, synth.QWEN.hidden, generator=gen, device=device).to(torch.bfloat16)
        angle = torch.arange(context, device=device, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, ROTARY, 2, device=device, dtype=torch.float64) / ROTARY)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
        self.free = torch.randperm(batch * width, generator=gen, device=device).to(torch.int32)
        self.taken = torch.zeros(1, dtype=torch.int32, device=device)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.cached = torch.zeros(batch, dtype=torch.int32, device=device)

    def step(self, tokens, new_lens, longest):
        """`tokens` (all requests' new ones in order) through all layers; the hidden states behind them."""
        plan = plan_batch(self.cached, new_lens, self.table, self.free, self.taken, self.page_size, tokens.numel())
        x = self.embedding[tokens]
        for layer in self.layers:
            x = layer(x, plan, self.table, self.cos_sin, longest)
        self.cached.copy_(plan.seq_lens)
        self.taken.copy_(plan.taken)
        return x, plan

    def next_tokens(self, x, plan):
        """The likeliest token behind each request's last one."""
        last = x[(plan.query_start[1:] - 1).clamp(min=0)]
        return F.linear(F.rms_norm(last, last.shape[-1:]), self.head).argmax(-1)

    def prefill(self, prompts, budget: int):
        """Prompts (lists of token tensors) in chunks of at most `budget` tokens a step; the first token that follows each."""
        done, first = [0] * self.batch, torch.zeros(self.batch, dtype=torch.long, device=self.device)
        while any(d < len(p) for d, p in zip(done, prompts)):
            left, take = budget, []
            for d, p in zip(done, prompts):
                take.append(min(left, len(p) - d))
                left -= take[-1]
            tokens = torch.cat([p[d:d + n] for d, n, p in zip(done, take, prompts)])
            x, plan = self.step(tokens, torch.tensor(take, dtype=torch.int32, device=self.device), max(take))
            nxt = self.next_tokens(x, plan)
            for b, n in enumerate(take):
                done[b] += n
                if n and done[b] == len(prompts[b]):
                    first[b] = nxt[b]
        return first

    def decode(self, tokens, steps: int):
        """`steps` tokens for every request, [batch, steps]: the first step as it is, the others as replays of one graph."""
        one = torch.ones(self.batch, dtype=torch.int32, device=self.device)
        got, now = [], tokens.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for i in range(steps):
                if i == 0:
                    now.copy_(self.next_tokens(*self.step(now, one, 1)))
                else:
                    if i == 1:
                        graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(graph, stream=side):
                            now.copy_(self.next_tokens(*self.step(now, one, 1)))
                    graph.replay()
                got.append(now.clone())
        torch.cuda.current_stream().wait_stream(side)
        return torch.stack(got, 1)


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--prompts", type=int, nargs="+", default=[700, 33, 1500], help="their lengths")
    p.add_argument("--budget", type=int, default=1024, help="tokens of a prefill step")
    p.add_argument("--new", type=int, default=32, help="tokens to decode for each request")
    args = p.parse_args()
    server = Server(args.layers, len(args.prompts), max(args.prompts) + args.new)
    gen = torch.Generator(device="cuda").manual_seed(11)
    prompts = [torch.randint(0, len(server.embedding), (n,), generator=gen, device="cuda") for n in args.prompts]

    def timed(f, *a):
        torch.cuda.synchronize()
        t = time.perf_counter()
        got = f(*a)
        torch.cuda.synchronize()
        return got, 1e3 * (time.perf_counter() - t)

    first, prefill_ms = timed(server.prefill, prompts, args.budget)
    more, decode_ms = timed(server.decode, first, args.new)
    check_status()
    print(f"prefilled {sum(args.prompts)} tokens in {prefill_ms:.1f} ms, decoded {args.new} x {len(prompts)} in {decode_ms:.1f} ms (both with first-call set-up)")
    for b, n in enumerate(args.prompts):
        print(f"  request {b}: {n} tokens, then {[int(first[b])] + more[b, :7].tolist()} ...")


if __name__ == "__main__":
    main()
