"""Autograd glue for the expert op: saves the seven inputs in forward and calls
`experts_backward` in backward, returning gradients in the op's argument order.
reference: torch-ext/yamoe/layers.py:6-100 (`_ExpertsFn`)."""
from __future__ import annotations

import torch

from . import ops


class _ExpertsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden_flat, router_indices, routing_weights_dense, gate_up_proj, gate_up_proj_bias,
                down_proj, down_proj_bias, expert_capacity, num_experts, top_k, enable_router_grads):
        out = ops.experts(hidden_flat, router_indices, routing_weights_dense, gate_up_proj, gate_up_proj_bias,
                          down_proj, down_proj_bias, expert_capacity, num_experts, top_k)
        ctx.expert_capacity, ctx.num_experts, ctx.top_k = expert_capacity, num_experts, top_k
        ctx.enable_router_grads = bool(enable_router_grads)
        ctx.save_for_backward(hidden_flat, router_indices, routing_weights_dense, gate_up_proj,
                              gate_up_proj_bias, down_proj, down_proj_bias)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        saved = ctx.saved_tensors
        d_hidden, d_routing, d_wgu, d_bgu, d_wd, d_bd = ops.experts_backward(
            grad_output, *saved, ctx.expert_capacity, ctx.num_experts, ctx.top_k)
        return (d_hidden, None, d_routing if ctx.enable_router_grads else None, d_wgu, d_bgu, d_wd, d_bd,
                None, None, None, None)


class _ExpertsSavedFn(torch.autograd.Function):
    """Like `_ExpertsFn`, but the forward keeps the routing tables, gathered rows, pre-activations
    and weighted activations (about 12*S*H bytes in bf16), and the backward skips routing, the
    gather and the gate_up recompute: 12 instead of 16 S*H^2 of GEMM work."""

    @staticmethod
    def forward(ctx, hidden_flat, router_indices, routing_weights, gate_up_proj, gate_up_proj_bias,
                down_proj, down_proj_bias, expert_capacity, num_experts, top_k, enable_router_grads):
        out, saved = ops.experts_forward_saving(hidden_flat, router_indices, routing_weights, gate_up_proj,
                                                gate_up_proj_bias, down_proj, down_proj_bias, expert_capacity,
                                                num_experts, top_k)
        ctx.expert_capacity, ctx.num_experts, ctx.top_k = expert_capacity, num_experts, top_k
        ctx.enable_router_grads = bool(enable_router_grads)
        ctx.save_for_backward(saved, routing_weights, gate_up_proj, down_proj, down_proj_bias)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        saved, routing_weights, gate_up_proj, down_proj, down_proj_bias = ctx.saved_tensors
        d_hidden, d_routing, d_wgu, d_bgu, d_wd, d_bd = ops.experts_backward_saved(
            grad_output, saved, routing_weights, gate_up_proj, down_proj, down_proj_bias, ctx.expert_capacity,
            ctx.num_experts, ctx.top_k)
        return (d_hidden, None, d_routing if ctx.enable_router_grads else None, d_wgu, d_bgu, d_wd, d_bd,
                None, None, None, None)


def experts_autograd(hidden_flat, router_indices, routing_weights, gate_up_proj, gate_up_proj_bias, down_proj,
                     down_proj_bias, expert_capacity, num_experts, top_k, enable_router_grads=True,
                     save_activations=False):
    """Differentiable `experts`: forward through the CUDA op, backward through `experts_backward`
    (recomputing the forward, like the reference) or, with `save_activations`, through the pair
    that keeps the forward's intermediates.  A backward pass can run once per forward."""
    fn = _ExpertsSavedFn if save_activations else _ExpertsFn
    return fn.apply(hidden_flat, router_indices, routing_weights, gate_up_proj, gate_up_proj_bias,
                    down_proj, down_proj_bias, expert_capacity, num_experts, top_k, enable_router_grads)


def ceil_div(a, b):
    return (a + b - 1) // b


class Yamoe(torch.nn.Module):
    """Drop-in `forward` for a GPT-OSS MoE block (an object with `router.weight`, `router.bias`,
    `experts.gate_up_proj`, `experts.gate_up_proj_bias`, `experts.down_proj`,
    `experts.down_proj_bias`, and optionally `num_experts`, `top_k`), returning
    `(output [B,S,H], router_scores [T,E])` like the reference layer
    (torch-ext/yamoe/layers.py:103-218; oracle torch-ext/yamoe/vendored/gpt_oss_mlp.py:142-159).

    Differences from the reference layer, on purpose:
    * `expert_capacity` defaults to the reference's `ceil(T*K/E)` (layers.py:162), which drops
      assignments of over-subscribed experts; set the attribute `expert_capacity` (for example to
      the token count) for a run that never drops and therefore matches `GptOssMLP`.
    * gradients are not switched off: when autograd is recording, the router runs in PyTorch and
      the experts go through `_ExpertsFn`, so router and expert weights receive gradients.  Without
      autograd the whole router (projection, top-k, softmax, scatter) runs in the library: one
      tcgen05 kernel for bf16.
    """
    can_torch_compile: bool = False

    def forward(self, hidden_states: torch.Tensor):
        batch, seq, hidden = hidden_states.shape
        T = batch * seq
        E = getattr(self, "num_experts", self.router.weight.shape[0])
        K = getattr(self, "top_k", 4)
        x = hidden_states.reshape(T, hidden)
        needs_grad = torch.is_grad_enabled() and (
            x.requires_grad or self.router.weight.requires_grad or self.experts.gate_up_proj.requires_grad)
        if needs_grad:
            logits = torch.nn.functional.linear(x, self.router.weight, self.router.bias)
            top_v, router_indices = torch.topk(logits, K, dim=-1)
            top_w = torch.nn.functional.softmax(top_v, dim=-1, dtype=top_v.dtype)
            router_scores = torch.zeros_like(logits).scatter(1, router_indices, top_w)
        else:
            # router projection, top-k, softmax and scatter in the library (one kernel for bf16)
            router_indices, router_scores = ops.router_forward(x, self.router.weight, self.router.bias, K)
        cap = getattr(self, "expert_capacity", None)
        if cap is None:
            cap = ceil_div(T * K, E)
        gate_up = self.experts.gate_up_proj[:, :, : 2 * hidden]
        gate_up_bias = self.experts.gate_up_proj_bias[:, : 2 * hidden]
        down = self.experts.down_proj[:, :hidden, :]
        down_bias = self.experts.down_proj_bias
        if needs_grad:
            out = _ExpertsFn.apply(x, router_indices, router_scores, gate_up, gate_up_bias, down, down_bias,
                                   int(cap), E, K, True)
        else:
            out = ops.experts(x, router_indices, router_scores, gate_up, gate_up_bias, down, down_bias, int(cap), E, K)
        return out.view(batch, seq, hidden), router_scores


class Fp8Yamoe(torch.nn.Module):
    """The MoE block of `Yamoe` for serving, with expert weights in 8 bits.

        layer = Fp8Yamoe.from_layer(block)          # block: as for `Yamoe`; its bf16 expert weights are not kept
        out, router_scores = layer(hidden_states)   # [B, S, H] bf16

    Up to 32 tokens with up to 256 assignments (a decode step) run as `moe_layer`, two launches in
    all, activations at 11 bits and the router's logits unrounded.  Others run as `router_forward`, whose logits are bf16
    numbers, and `experts_fp8`, which quantises the token rows and the activations too; so where two logits of a token round to the
    same number its experts may depend on how many tokens come with it.  `expert_capacity` None: ceil(T K / E), as in `Yamoe`."""

    def __init__(self, router_weight, router_bias, gate_up, gate_up_scale, gate_up_bias, down, down_scale, down_bias,
                 top_k, expert_capacity=None):
        super().__init__()
        for name, t in (("router_weight", router_weight), ("router_bias", router_bias), ("gate_up", gate_up),
                        ("gate_up_scale", gate_up_scale), ("gate_up_bias", gate_up_bias), ("down", down),
                        ("down_scale", down_scale), ("down_bias", down_bias)):
            self.register_buffer(name, t)
        self.top_k, self.expert_capacity = int(top_k), expert_capacity

    @classmethod
    def from_layer(cls, block):
        hidden = block.router.weight.shape[1]
        e = block.experts
        gate_up, gate_up_scale, down, down_scale = ops.quantize_experts(e.gate_up_proj[:, :, : 2 * hidden].detach(),
                                                                        e.down_proj[:, :hidden, :].detach())
        bias = None if block.router.bias is None else block.router.bias.detach()
        return cls(block.router.weight.detach(), bias, gate_up, gate_up_scale,
                   e.gate_up_proj_bias[:, : 2 * hidden].detach(), down, down_scale, e.down_proj_bias.detach(),
                   getattr(block, "top_k", 4), getattr(block, "expert_capacity", None))

    @torch.no_grad()
    def forward(self, hidden_states):
        batch, seq, hidden = hidden_states.shape
        T, E, K = batch * seq, self.router_weight.shape[0], self.top_k
        x = hidden_states.reshape(T, hidden)
        cap = int(self.expert_capacity) if self.expert_capacity is not None else ceil_div(T * K, E)
        if T <= 32 and T * K <= 256 and x.dtype == torch.bfloat16:
            out, scores = ops.moe_layer(x, self.router_weight, self.router_bias, self.gate_up, self.gate_up_bias, self.down,
                                        self.down_bias, cap, E, K, self.gate_up_scale, self.down_scale)
        else:
            indices, scores = ops.router_forward(x, self.router_weight, self.router_bias, K)
            out = ops.experts_fp8(x, indices, scores, self.gate_up, self.gate_up_scale, self.gate_up_bias, self.down,
                                  self.down_scale, self.down_bias, cap, E, K)
        return out.view(batch, seq, hidden), scores
