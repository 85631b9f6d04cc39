"""A flow-matching action expert on packed projections, block by block.

Several candidate action chunks are denoised at once for each observation.
All of an observation's chunks attend to the same prefix (its images and
prompt, whose keys and values the backbone left in a cache) and to their own
chunk; the time embedding modulates every norm and gates every block; each
chunk may carry a low-rank adapter of its own (a robot's fine-tune) beside the
shared resident bank. One denoising step is one graph:

    projections   packed linears (GroupedPaddedLinear), siblings in one launch
    attention     shared_prefix_attention
    adapters      AdaptedLinear beside the query and output projections
    between       block_norm: residual, gate, norm, scale and shift at once

Weights are random; widths are the action expert's (1024, 8 heads of 256 over
one key head, MLP 4096, chunks of 50 tokens).

    python examples/denoise_expert.py [--observations 2] [--samples 8] [--layers 4] [--prefix 816]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from actune_amd.graph import GraphReplay  # noqa: E402
from actune_amd.kernels.adapters import AdaptedLinear, adapter_scope  # noqa: E402
from actune_amd.kernels.attention import shared_prefix_attention  # noqa: E402
from actune_amd.kernels.grouped import GroupedPaddedLinear, gated_down_forward, grouped_sibling_forward  # noqa: E402
from actune_amd.kernels.norms import block_norm  # noqa: E402

HEADS, HEAD = 8, 256


def packed(inputs, outputs, mode="W4A8"):
    linear = torch.nn.Linear(inputs, outputs, bias=False, device="cuda", dtype=torch.bfloat16)
    torch.nn.init.normal_(linear.weight, std=inputs ** -0.5)
    return GroupedPaddedLinear(linear, {"q11": mode}, "q11", {mode: None})


def adapted(base, adapters, rank):
    a = torch.randn(adapters, rank, base.in_features, device="cuda", dtype=torch.bfloat16) * base.in_features ** -0.5
    b = torch.randn(adapters, base.out_features, rank, device="cuda", dtype=torch.bfloat16) * 0.1
    return AdaptedLinear(base, a, b, torch.full((adapters,), 0.5, device="cuda"))


class Block(torch.nn.Module):
    def __init__(self, width, mlp, adapters, rank):
        super().__init__()
        self.query = adapted(packed(width, HEADS * HEAD), adapters, rank)
        self.key, self.value = packed(width, HEAD), packed(width, HEAD)
        self.output = adapted(packed(HEADS * HEAD, width), adapters, rank)
        self.gate, self.up, self.down = packed(width, mlp), packed(width, mlp), packed(mlp, width)
        self.act = torch.nn.GELU(approximate="tanh")
        # gate, scale and shift of both norms from the time embedding
        self.modulation = torch.nn.Linear(width, 6 * width, device="cuda", dtype=torch.bfloat16)

    def attend(self, x, prefix_k, prefix_v, prefix_mask):
        b, t, _ = x.shape
        q, k, v = grouped_sibling_forward(x, [self.query, self.key, self.value])
        out = shared_prefix_attention(q.view(b, t, HEADS, HEAD), prefix_k, prefix_v, k.view(b, t, 1, HEAD),
                                      v.view(b, t, 1, HEAD), prefix_mask=prefix_mask)
        return self.output(out.view(b, t, HEADS * HEAD))

    def feed_forward(self, x):
        gate, up = grouped_sibling_forward(x, [self.gate, self.up])
        return gated_down_forward(self.down, gate, up, self.act)


class ActionExpert(torch.nn.Module):
    def __init__(self, layers=4, width=1024, mlp=4096, actions=32, adapters=4, rank=16):
        super().__init__()
        self.width = width
        self.enter = torch.nn.Linear(actions, width, device="cuda", dtype=torch.bfloat16)
        self.leave = torch.nn.Linear(width, actions, device="cuda", dtype=torch.bfloat16)
        self.blocks = torch.nn.ModuleList(Block(width, mlp, adapters, rank) for _ in range(layers))
        self.weight = torch.nn.Parameter(torch.zeros(width, device="cuda", dtype=torch.bfloat16), requires_grad=False)

    def packed_layers(self):
        return {n: m for n, m in self.named_modules() if isinstance(m, GroupedPaddedLinear)}

    def embed(self, time):
        """[B, width] sine embedding of the flow time [B]."""
        freq = torch.exp(torch.arange(self.width // 2, device=time.device) * (-9.0 / (self.width // 2)))
        angle = time[:, None] * freq * 100.0
        return torch.cat([angle.sin(), angle.cos()], -1).to(torch.bfloat16)

    def forward(self, actions, time, prefix_k, prefix_v, prefix_mask, ids):
        """The flow's velocity at actions [B, T, actions]; prefix_k, prefix_v: [layers, G, P, 1, 256]."""
        hidden, branch, gate = self.enter(actions), None, None
        embedding = self.embed(time)
        with adapter_scope(ids):
            for i, block in enumerate(self.blocks):
                gate1, scale1, shift1, gate2, scale2, shift2 = block.modulation(embedding).chunk(6, -1)
                hidden, normed = block_norm(hidden, branch, gate=gate, weight=self.weight, scale=scale1, shift=shift1,
                                            weight_offset=1.0)
                branch = block.attend(normed, prefix_k[i], prefix_v[i], prefix_mask)
                hidden, normed = block_norm(hidden, branch, gate=gate1, weight=self.weight, scale=scale2, shift=shift2,
                                            weight_offset=1.0)
                branch, gate = block.feed_forward(normed), gate2
            _, normed = block_norm(hidden, branch, gate=gate, weight=self.weight, weight_offset=1.0)
        return self.leave(normed)


def denoise(step, actions, prefix_k, prefix_v, prefix_mask, ids, steps=10):
    """Euler steps of the flow from noise (time 1) to actions (time 0)."""
    for i in range(steps):
        time = torch.full(actions.shape[:1], 1.0 - i / steps, device=actions.device)
        actions = actions - step(actions, time, prefix_k, prefix_v, prefix_mask, ids) / steps
    return actions


def inputs(observations, samples, layers, prefix, tokens=50, actions=32, adapters=4, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *shape: torch.randn(shape, device="cuda", generator=gen).to(torch.bfloat16)  # noqa: E731
    batch = observations * samples
    mask = torch.ones(observations, prefix, dtype=torch.bool, device="cuda")
    mask[0, prefix // 4:prefix // 2] = False  # the first observation misses a camera
    ids = torch.arange(batch, device="cuda", dtype=torch.int32) % (adapters + 1) - 1
    return (n(batch, tokens, actions), n(layers, observations, prefix, 1, HEAD), n(layers, observations, prefix, 1, HEAD),
            mask, ids)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--observations", type=int, default=2)
    parser.add_argument("--samples", type=int, default=8)
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--prefix", type=int, default=816)
    args = parser.parse_args()
    torch.manual_seed(0)
    with torch.inference_mode():
        expert = ActionExpert(args.layers)
        state = inputs(args.observations, args.samples, args.layers, args.prefix)
        eager = denoise(expert, *state)
        replay = GraphReplay(expert, expert.packed_layers(), shared_a8=True)
        replay.enabled = True
        chunks = denoise(replay, *state)
        torch.cuda.synchronize()
        begin = time.perf_counter()
        denoise(replay, *state)
        torch.cuda.synchronize()
        took = time.perf_counter() - begin
    print(f"{chunks.shape[0]} chunks of {chunks.shape[1]} actions in {took * 1e3:.2f} ms (10 steps of {args.layers} blocks, one "
          f"graph a step); equal to the eager run: {torch.equal(eager, chunks)}")


if __name__ == "__main__":
    main()
