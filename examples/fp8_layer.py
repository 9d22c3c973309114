"""An MoE block in 8 bits: quantise its experts, run a prompt through it, decode a few tokens, train a head on its outputs.

    python examples/fp8_layer.py [--hidden 2880] [--experts 32] [--top-k 4] [--prompt 512] [--classes 1000]
"""
import argparse
import os
import sys
import types

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import yamoe_b200  # noqa: E402


def make_block(hidden, experts, top_k, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(0)

    def normal(*shape, std):
        return torch.empty(*shape, dtype=torch.bfloat16, device=device).normal_(0, std, generator=gen)
    block = yamoe_b200.Yamoe()
    block.router = types.SimpleNamespace(weight=normal(experts, hidden, std=hidden ** -0.5), bias=normal(experts, std=0.02))
    block.experts = types.SimpleNamespace(
        gate_up_proj=normal(experts, hidden, 2 * hidden, std=hidden ** -0.5), gate_up_proj_bias=normal(experts, 2 * hidden, std=0.02),
        down_proj=normal(experts, hidden, hidden, std=hidden ** -0.5), down_proj_bias=normal(experts, hidden, std=0.02))
    block.num_experts, block.top_k = experts, top_k
    return block


def milliseconds(fn, repeats=10):
    fn()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(repeats):
        fn()
    end.record()
    end.synchronize()
    return start.elapsed_time(end) / repeats


def difference(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("hidden", 2880), ("experts", 32), ("top-k", 4), ("prompt", 512), ("classes", 1000)):
        ap.add_argument("--" + name, type=int, default=default)
    a = ap.parse_args(argv)
    block = make_block(a.hidden, a.experts, a.top_k)
    layer = yamoe_b200.Fp8Yamoe.from_layer(block)
    results = {}
    for what, T in (("prompt", a.prompt), ("step", 1)):
        x = torch.randn(1, T, a.hidden, device="cuda").bfloat16()
        block.expert_capacity = layer.expert_capacity = T
        with torch.no_grad():
            wide, narrow = block(x)[0], layer(x)[0]
            results[what] = difference(narrow, wide)
            print(f"{what} of {T} tokens: bf16 {milliseconds(lambda: block(x)):.3f} ms, 8 bits {milliseconds(lambda: layer(x)):.3f} ms, "
                  f"difference {results[what]:.3f} of the output's norm")
    # a head on the block's outputs, trained with products in 8 bits
    layer.expert_capacity = a.prompt
    x = layer(torch.randn(1, a.prompt, a.hidden, device="cuda").bfloat16())[0][0].float()
    target = torch.randint(0, a.classes, (a.prompt,), device="cuda")
    head = torch.zeros(a.classes, a.hidden, device="cuda", requires_grad=True)
    losses = []
    for _ in range(20):
        loss = torch.nn.functional.cross_entropy(yamoe_b200.fp8_linear(x, head), target)
        losses.append(loss.item())
        (grad,) = torch.autograd.grad(loss, head)
        with torch.no_grad():
            head -= grad
    print(f"head: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    results["loss"] = losses
    return results


if __name__ == "__main__":
    main()
