"""Refusals of the steps' binding that one GPU cannot show: tensors of several devices (see test_fp8_binding.py)."""
import pytest
import torch

from test_fp8_binding import KEYS, Shell, ops  # noqa: F401

T, H, E, K = 4, 128, 8, 2
BF16, F32, I8, I32, I64 = torch.bfloat16, torch.float32, torch.int8, torch.int32, torch.int64
WHAT = {"sort_tokens": [("hidden_states", (T, H), BF16), ("router_indices", (T, K), I64)],
        "combine_tokens": [("rows", (T * K, H), BF16), ("row_of", (T, K), I32), ("routing_weights", (T, E), BF16), ("router_indices", (T, K), I64)],
        "int8_mm": [("a", (T, H), I8), ("a_scale", (T,), F32), ("b", (E, H, H), I8), ("b_scale", (E, H), F32), ("offsets", (E + 1,), I32)]}
CALLS = [(name, i) for name in WHAT for i in range(1, len(WHAT[name]))]


@pytest.mark.parametrize("name,i", CALLS, ids=["%s-%s" % (n, WHAT[n][i][0]) for n, i in CALLS])
@pytest.mark.parametrize("device", ["cuda:1", "cpu"])
def test_a_tensor_of_another_device(ops, name, i, device):  # noqa: F811
    sizes = dict(num_experts=E) if name == "sort_tokens" else {}
    tensors = {n: Shell(shape, dtype, device if j == i else "cuda:0") for j, (n, shape, dtype) in enumerate(WHAT[name])}
    with torch._C._DisableTorchDispatch(), torch._C._ExcludeDispatchKeyGuard(KEYS):
        with pytest.raises(RuntimeError, match="device"):
            getattr(ops, name)(**tensors, **sizes)


def test_operators_have_no_cpu_form(ops):  # noqa: F811
    x = torch.zeros(4, 8)
    for call in (lambda: ops.sort_tokens(x, torch.zeros(4, 1, dtype=I64), 2), lambda: ops.combine_tokens(x, torch.zeros(4, 1, dtype=I32)),
                 lambda: ops.quantize_int8(x), lambda: ops.glu_fp8(x), lambda: ops.int8_mm(x.to(I8), x[:, 0], x.to(I8), x[:, 0])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
