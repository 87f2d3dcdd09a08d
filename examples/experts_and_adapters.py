"""A packed mixture-of-experts block: serve it, train LoRA adapters over it, merge them into it.

Everything stays in MXFP4 from beginning to end: products read the packed
weights, gradients pass through them, and a LoRA is merged in place.

    PYTHONPATH=piper-offload_amd python examples/experts_and_adapters.py
"""

from __future__ import annotations

import argparse

import torch

from piper_offload_amd import MxAdapter, MXWeight, expert_view, grouped_linear, mx_linear
from piper_offload_amd import kernels as K

FP4 = torch.float4_e2m1fn_x2


def pack(w: torch.Tensor) -> MXWeight:
    """A dense weight [rows, columns] in MXFP4 with swizzled scales."""
    q, s = K.requantize_mx(w, FP4, swizzled=True)
    return MXWeight(q, s, FP4, 32, w.dtype, True)


class Block:
    """``out(sum of the best experts of x)``: experts of one stack per projection, an MXFP4 projection after them."""

    def __init__(self, hidden: int, inner: int, experts: int, best: int, device: torch.device) -> None:
        def rand(rows: int, cols: int) -> torch.Tensor:
            return torch.randn(rows, cols, device=device, dtype=torch.bfloat16) * cols**-0.5

        self.experts, self.best = experts, best
        self.router = rand(experts, hidden)
        self.up = pack(rand(experts * 2 * inner, hidden))  # gate and up of every expert, one below the other
        self.down = pack(rand(experts * hidden, inner))
        self.out = pack(rand(hidden, hidden))

    def mixture(self, x: torch.Tensor, activation_dtype: torch.dtype | None = None) -> torch.Tensor:
        weight, expert = (x @ self.router.t()).float().softmax(-1).topk(self.best, -1)
        order = expert.reshape(-1).argsort(stable=True)  # rows of one expert side by side
        ends = torch.bincount(expert.reshape(-1), minlength=self.experts).cumsum(0).to(torch.int32)
        token = order // self.best
        h = grouped_linear(x[token], self.up, ends, activation_dtype=activation_dtype)
        gate, up = h.chunk(2, -1)
        h = grouped_linear(torch.nn.functional.silu(gate) * up, self.down, ends, activation_dtype=activation_dtype)
        h = h.float() * weight.reshape(-1)[order, None]
        return torch.zeros_like(x, dtype=torch.float32).index_add(0, token, h).to(x.dtype)

    def __call__(self, x: torch.Tensor, activation_dtype: torch.dtype | None = None) -> torch.Tensor:
        return mx_linear(self.mixture(x, activation_dtype), self.out, activation_dtype=activation_dtype)


def adapted(block: Block, h: torch.Tensor, down: torch.Tensor, up: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    """``out`` with one LoRA per group of rows: request ``e`` has rows ``ends[e-1] : ends[e]``."""
    return mx_linear(h, block.out) + grouped_linear(grouped_linear(h, down, ends), up, ends)


def main(argv: list[str] | None = None) -> dict[str, float]:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--inner", type=int, default=1408)
    p.add_argument("--experts", type=int, default=32)
    p.add_argument("--best", type=int, default=4)
    p.add_argument("--tokens", type=int, default=2000)
    p.add_argument("--rank", type=int, default=16)
    p.add_argument("--steps", type=int, default=30)
    a = p.parse_args(argv)
    torch.manual_seed(0)
    dev = torch.device("cuda")
    block = Block(a.hidden, a.inner, a.experts, a.best, dev)
    x = torch.randn(a.tokens, a.hidden, device=dev, dtype=torch.bfloat16)
    said = {}

    def say(name: str, value: float) -> None:
        said[name] = float(value)
        print(f"{name:48s} {value:.4g}", flush=True)

    def apart(u: torch.Tensor, v: torch.Tensor) -> float:
        return float((u.float() - v.float()).norm() / v.float().norm())

    with torch.no_grad():
        # a prompt with inputs in 16 and in 4 bits, then its last token alone
        h = block.mixture(x)
        y = block(x)
        say("prompt, 4-bit inputs: distance to 16-bit ones", apart(block(x, FP4), y))
        say("last token alone: distance to the prompt's", apart(block(x[-1:]), y[-1:]))

    # three requests train a LoRA each on the output projection, in one batch; the packed weight is frozen
    sizes = torch.tensor([a.tokens // 2, a.tokens // 3, a.tokens // 8])
    ends = sizes.cumsum(0).to(device=dev, dtype=torch.int32)
    down = torch.randn(3, a.rank, a.hidden, device=dev, dtype=torch.bfloat16) * a.hidden**-0.5
    up = torch.zeros(3, a.hidden, a.rank, device=dev, dtype=torch.bfloat16)
    goal_up = torch.randn_like(up) * 0.5
    with torch.no_grad():
        goal = adapted(block, h, down, goal_up, ends)
    down.requires_grad_()
    up.requires_grad_()
    optimizer = torch.optim.Adam([down, up], lr=0.03)
    for step in range(a.steps):
        loss = (adapted(block, h, down, up, ends).float() - goal.float()).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        if step in (0, a.steps - 1):
            say(f"LoRA loss, step {step + 1}", loss.item())

    with torch.no_grad():
        # the first request's adapter, merged: the projection alone now gives what both gave
        rows = slice(0, int(sizes[0]))
        both = adapted(block, h, down, up, ends)[rows]
        before = mx_linear(h[rows], block.out)
        MxAdapter.merge_lora_(block.out, up[0].detach(), down[0].detach(), 1.0)
        say("without the adapter: distance", apart(before, both))
        say("adapter merged: distance", apart(mx_linear(h[rows], block.out), both))

        # a LoRA merged into one expert of the stack
        counts = torch.full((a.experts,), a.tokens // a.experts, device=dev)
        ends = counts.cumsum(0).to(torch.int32)
        before = grouped_linear(x, block.up, ends)
        one = expert_view(block.up, 1, a.experts)
        MxAdapter.merge_lora_(one, torch.randn(2 * a.inner, a.rank, device=dev, dtype=torch.bfloat16) * 0.1,
                              torch.randn(a.rank, a.hidden, device=dev, dtype=torch.bfloat16) * 0.1, 1.0)
        changed = (grouped_linear(x, block.up, ends) != before).any(-1)
        n = a.tokens // a.experts
        say("rows of expert 1 that changed", changed[n:2 * n].sum().item())
        say("rows of other experts that changed", changed.sum().item() - changed[n:2 * n].sum().item())
    return said


if __name__ == "__main__":
    main()
