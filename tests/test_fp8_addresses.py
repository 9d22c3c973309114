"""C entry points of the 8-bit operators: addresses that the kernels cannot load from are refused on the host."""
import pytest

from test_fp8_cabi import BAD_ARG, BF16, F32, lib, matrix  # noqa: F401

T, H, E, K = 16, 128, 8, 2
# addresses that would pass: multiples of 16
GOOD = 4096


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name,off", [("gate_up_bias", 8), ("down_bias", 8), ("gate_up_bias", 2), ("router_indices", 4), ("routing_weights", 1)])
def test_experts(lib, dtype, name, off):  # noqa: F811
    ws = lib.yamoe_b200_experts_fp8_workspace_bytes(T, H, E, K, dtype)
    at = dict(router_indices=GOOD, routing_weights=GOOD, gate_up_bias=GOOD, down_bias=GOOD)
    at[name] += off
    assert lib.yamoe_b200_experts_fp8_forward(GOOD, at["router_indices"], at["routing_weights"], E, matrix(), at["gate_up_bias"], matrix(),
                                              at["down_bias"], GOOD, T, H, E, K, 4, dtype, GOOD, ws, None) == BAD_ARG


@pytest.mark.parametrize("name", ["router_bias", "scores"])
def test_layer(lib, name):  # noqa: F811
    ws = lib.yamoe_b200_moe_layer_workspace_bytes(T, H, E, K)
    at = dict(router_bias=GOOD, scores=GOOD)
    at[name] += 1
    assert lib.yamoe_b200_moe_layer(GOOD, GOOD, at["router_bias"], GOOD, None, GOOD, GOOD, None, GOOD, GOOD, at["scores"], T, H, E, K, 4, BF16,
                                    GOOD, ws, None) == BAD_ARG
