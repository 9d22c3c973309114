"""The 8-bit operators as a layer uses them: `Fp8Yamoe` over decode and prefill, and the example that runs all of them."""
import importlib.util
import os
import types

import pytest
import torch

from test_gpu_fp8 import experts_ref, randn, rel
from test_gpu_moe_layer import BOUND, reference

pytestmark = pytest.mark.gpu


def make_layer(H, E, K, seed=0):
    import yamoe_b200
    d = dict(wr=randn(E, H, seed=seed, std=H ** -0.5), br=randn(E, seed=seed + 1, std=0.1),
             gu=randn(E, H, 2 * H, seed=seed + 2, std=H ** -0.5), bgu=randn(E, 2 * H, seed=seed + 3, std=0.2),
             dn=randn(E, H, H, seed=seed + 4, std=H ** -0.5), bd=randn(E, H, seed=seed + 5, std=0.2))
    block = types.SimpleNamespace(
        router=types.SimpleNamespace(weight=d["wr"].cuda(), bias=d["br"].cuda()),
        experts=types.SimpleNamespace(gate_up_proj=d["gu"].cuda(), gate_up_proj_bias=d["bgu"].cuda(), down_proj=d["dn"].cuda(),
                                      down_proj_bias=d["bd"].cuda()), top_k=K)
    return d, yamoe_b200.Fp8Yamoe.from_layer(block)


@pytest.mark.parametrize("B,S", [(1, 1), (2, 3), (4, 8), (1, 33), (2, 100)])
def test_fp8_layer_decode_and_prefill(B, S):
    H, E, K = 192, 12, 3
    d, layer = make_layer(H, E, K)
    x = randn(B, S, H, seed=B + S)
    T = B * S
    out, scores = layer(x.cuda())
    assert out.shape == (B, S, H) and scores.shape == (T, E)
    cap = -(-T * K // E)
    q = (layer.gate_up, layer.gate_up_scale, layer.down, layer.down_scale)
    if T <= 32:
        ref, _ = reference(dict(d, x=x.view(T, H)), K, cap, q)
        assert rel(out.view(T, H), ref) < BOUND
    else:
        import yamoe_b200
        idx, sc = yamoe_b200.router_forward(x.view(T, H).cuda(), d["wr"].cuda(), d["br"].cuda(), K)
        ref = experts_ref(x.view(T, H), idx.cpu(), sc.cpu().gather(1, idx.cpu()), q, (d["bgu"], d["bd"]), cap)
        assert rel(out.view(T, H), ref) < 2.0 ** -9 + 6e-4      # see test_gpu_fp8.test_experts


def test_state_dict_round_trip():
    import yamoe_b200
    _, layer = make_layer(64, 4, 2)
    x = randn(1, 5, 64, seed=9).cuda()
    other = make_layer(64, 4, 2, seed=50)[1]
    assert not torch.equal(other(x)[0], layer(x)[0])
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x)[0], layer(x)[0])
    assert isinstance(other, yamoe_b200.Fp8Yamoe)


def test_example_runs():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "fp8_layer.py")
    spec = importlib.util.spec_from_file_location("fp8_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(["--hidden", "256", "--experts", "8", "--top-k", "2", "--prompt", "100", "--classes", "50"])
    # e4m3 rounds a value by at most 2^-4 of it, 2^-4 / sqrt(3) in the 2-norm at worst; two products with both operands
    # rounded (prompt) sum four such errors: 4 * 0.036 = 0.144 at most, the decode step two: 0.072
    assert got["prompt"] < 0.144 and got["step"] < 0.144
    assert got["loss"][-1] < got["loss"][0]
