"""An MoE block put together from the steps of the expert layer: served with weights in 8-bit integers, trained on products and checkpoints
in 8 bits.

    python examples/expert_steps.py [--hidden 2880] [--experts 32] [--top-k 4] [--tokens 512]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import yamoe_b200  # noqa: E402


def serve(x, indices, weights, gate_up, down):
    """gate_up, down: (codes, scales) of `quantize_int8(weights, transpose=True)`.  Rows of any number per expert, nothing is padded."""
    rows, row_of, offsets = yamoe_b200.sort_tokens(x, indices, gate_up[0].shape[0])
    pre = yamoe_b200.int8_mm(*yamoe_b200.quantize_int8(rows), *gate_up, torch.bfloat16, offsets)
    y = yamoe_b200.int8_mm(*yamoe_b200.quantize_int8(yamoe_b200.glu_fp8(pre)), *down, torch.bfloat16, offsets)
    return yamoe_b200.combine_tokens(y, row_of, weights)


def train(x, indices, weights, gate_up, down, capacity):
    """gate_up [E, 2H, H], down [E, H, H]: a place for `capacity` rows of each expert.  Between the passes live codes of the rows, of the
    pre-activations and of the activations, a byte per value."""
    rows, row_of, _ = yamoe_b200.sort_tokens(x, indices, gate_up.shape[0], capacity)
    act = yamoe_b200.glu_fp8(yamoe_b200.fp8_linear(rows, gate_up))
    return yamoe_b200.combine_tokens(yamoe_b200.fp8_linear(act, down), row_of, weights)


def difference(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("hidden", 2880), ("experts", 32), ("top-k", 4), ("tokens", 512)):
        ap.add_argument("--" + name, type=int, default=default)
    a = ap.parse_args(argv)
    H, E, K, T = a.hidden, a.experts, a.top_k, a.tokens
    gen = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape, std=1.0):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0, std, generator=gen)
    gate_up, down = normal(E, H, 2 * H, std=H ** -0.5), normal(E, H, H, std=H ** -0.5)
    x, up = normal(T, H), normal(T, H)
    best, indices = torch.topk(torch.randn(T, E, device="cuda", generator=gen), K, dim=-1)
    weights = torch.softmax(best, dim=-1).bfloat16()
    # (`experts` takes biases, the products here have none)
    biases = torch.zeros(E, 2 * H, device="cuda").bfloat16(), torch.zeros(E, H, device="cuda").bfloat16()

    # (`experts` takes [T, K] weights as dense where K is the number of experts)
    dense = torch.zeros(T, E, device="cuda", dtype=torch.bfloat16).scatter_(1, indices, weights)
    wide = yamoe_b200.experts(x, indices, dense, gate_up, biases[0], down, biases[1], T, E, K)
    quantised = yamoe_b200.quantize_int8(gate_up, True), yamoe_b200.quantize_int8(down, True)
    results = {"serve": difference(serve(x, indices, weights, *quantised), wide)}
    print(f"{T} tokens in 8-bit integers: difference {results['serve']:.4f} of the output's norm")

    leaves = [t.detach().requires_grad_(True) for t in (x, weights, gate_up.transpose(1, 2).contiguous(), down.transpose(1, 2).contiguous())]
    out = train(leaves[0], indices, leaves[1], leaves[2], leaves[3], T)
    grads = torch.autograd.grad(out, leaves, up)
    d_hidden, d_routing, d_gate_up, _, d_down, _ = yamoe_b200.experts_backward(up, x, indices, dense, gate_up, biases[0], down,
                                                                                    biases[1], T, E, K)
    results["train"] = difference(out.detach(), wide)
    for name, got, want in zip(("x", "weights", "gate_up", "down"), grads,
                               (d_hidden, d_routing.gather(1, indices), d_gate_up.transpose(1, 2), d_down.transpose(1, 2))):
        results["d_" + name] = difference(got, want)
    print("trained in 8 bits: differences " + ", ".join(f"{k} {v:.4f}" for k, v in results.items() if k != "serve"))
    return results


if __name__ == "__main__":
    main()
