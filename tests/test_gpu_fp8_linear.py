"""`fp8_linear` under autograd beyond one backward pass.
(Its values and gradients: test_gpu_fp8.py.)"""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from test_gpu_fp8 import randn

pytestmark = pytest.mark.gpu


def tensors(M=20, N=40, K=72, dtype=torch.bfloat16):
    return (randn(M, K, seed=1, dtype=dtype).cuda(), randn(N, K, seed=2, dtype=dtype, std=0.1).cuda(),
            randn(M, N, seed=3, dtype=dtype).cuda())


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(which, grad, no_grad):
    """A tangent is not dropped in silence, whether or not gradients are recorded beside it."""
    import yamoe_b200
    pair = list(tensors()[:2])
    if grad:
        pair[0].requires_grad_(True)
    with fwAD.dual_level(), torch.set_grad_enabled(not no_grad):
        pair[which] = fwAD.make_dual(pair[which], torch.ones_like(pair[which]))
        with pytest.raises(RuntimeError, match="forward"):
            yamoe_b200.fp8_linear(*pair)
        primal = [fwAD.unpack_dual(t).primal for t in pair]
        assert torch.equal(yamoe_b200.fp8_linear(*primal), yamoe_b200.fp8_linear(*[t.detach() for t in primal]))
