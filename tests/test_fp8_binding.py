"""Refusals of the C++ binding that one GPU cannot show: tensors of several devices.  The tensors here have a shape, a type and a
device, and no memory, so that no GPU is needed and nothing may be launched on them."""
import pytest
import torch

KEYS = torch._C.DispatchKeySet(torch._C.DispatchKey.Python) | torch._C.DispatchKeySet(torch._C.DispatchKey.PythonTLSSnapshot)
BF16, F32, F8, I64 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int64


@pytest.fixture(scope="module")
def ops():
    from yamoe_b200 import build
    build.build()
    import yamoe_b200
    assert yamoe_b200.ops.CPP_BINDING
    return yamoe_b200


class Shell(torch.Tensor):
    @staticmethod
    def __new__(cls, shape, dtype, device):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=torch.device(device))

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(func)


T, H, E, K = 4, 128, 8, 2
LAYER = [("hidden_states", (T, H), BF16), ("router_weight", (E, H), BF16), ("router_bias", (E,), BF16), ("gate_up", (E, 2 * H, H), F8),
         ("gate_up_bias", (E, 2 * H), BF16), ("down", (E, H, H), F8), ("down_bias", (E, H), BF16), ("gate_up_scale", (E, 2, 1), F32),
         ("down_scale", (E, 1, 1), F32)]
EXPERTS = [("hidden_states", (T, H), BF16), ("router_indices", (T, K), I64), ("routing_weights", (T, E), BF16)] + LAYER[3:]
MM = [("a", (T, H), F8), ("a_scale", (T, 1), F32), ("b", (H, H), F8), ("b_scale", (1, 1), F32)]
LINEAR = [("x", (T, H), BF16), ("weight", (H, H), BF16)]
CALLS = [(name, what, i) for name, what in (("moe_layer", LAYER), ("experts_fp8", EXPERTS), ("fp8_mm", MM), ("fp8_linear", LINEAR))
         for i in range(1, len(what))]


@pytest.mark.parametrize("name,what,i", CALLS, ids=["%s-%s" % (n, w[i][0]) for n, w, i in CALLS])
@pytest.mark.parametrize("device", ["cuda:1", "cpu"])
def test_a_tensor_of_another_device(ops, name, what, i, device):
    sizes = dict(expert_capacity=T, num_experts=E, top_k=K) if name in ("moe_layer", "experts_fp8") else {}
    tensors = {n: Shell(shape, dtype, device if j == i else "cuda:0") for j, (n, shape, dtype) in enumerate(what)}
    with torch._C._DisableTorchDispatch(), torch._C._ExcludeDispatchKeyGuard(KEYS):
        with pytest.raises(RuntimeError, match="device|on CUDA"):
            getattr(ops, name)(**tensors, **sizes)
