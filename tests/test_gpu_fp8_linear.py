"""`fp8_linear` under autograd beyond one backward pass, and with nothing to multiply.
(Its values and gradients: test_gpu_fp8.py.)"""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from test_gpu_fp8 import check_product, dequantised, randn

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


@pytest.mark.parametrize("wants", [(True, True), (True, False), (False, True)])
def test_second_order_is_refused(wants):
    """Gradients of a gradient do not exist: whoever asks for them gets an error, whoever does not is not disturbed by
    create_graph."""
    import yamoe_b200
    x, w, dy = tensors()
    x.requires_grad_(wants[0])
    w.requires_grad_(wants[1])
    leaves = [t for t in (x, w) if t.requires_grad]
    plain = torch.autograd.grad(yamoe_b200.fp8_linear(x, w), leaves, dy)
    first = torch.autograd.grad(yamoe_b200.fp8_linear(x, w), leaves, dy, create_graph=True)
    for a, b in zip(plain, first):
        assert torch.equal(a, b) and b.requires_grad
    # in a loss of its own, and beside a term that has a gradient
    for extra in (0.0, 1.0):
        y = yamoe_b200.fp8_linear(x, w)
        first = torch.autograd.grad(y, leaves, dy, create_graph=True)
        loss = sum((g.float() ** 2).sum() for g in first) + extra * sum((t.float() ** 2).sum() for t in leaves)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(loss, leaves, retain_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            loss.backward()
    # in the upstream gradient
    up = dy.clone().requires_grad_(True)
    first = torch.autograd.grad(yamoe_b200.fp8_linear(x, w), leaves, up, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(first[0].float().sum(), up)
    # a graph that other parts of a model need
    scale = torch.ones((), device="cuda", requires_grad=True)
    y = yamoe_b200.fp8_linear(x, w)
    loss = (y.float() * scale ** 2).sum()
    (ds,) = torch.autograd.grad(loss, scale, create_graph=True)
    (dds,) = torch.autograd.grad(ds, scale)
    assert torch.allclose(dds, 2 * y.detach().float().sum())


@pytest.mark.parametrize("M,N,K", [(20, 40, 72), (17, 33, 50), (1, 129, 9), (130, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_tensors_may_come_back_in_another_layout(M, N, K, dtype):
    import yamoe_b200
    x, w, dy = tensors(M, N, K, dtype)
    x.requires_grad_(True)
    w.requires_grad_(True)
    want = torch.autograd.grad(yamoe_b200.fp8_linear(x, w), (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = yamoe_b200.fp8_linear(x, w)
    got = torch.autograd.grad(y, (x, w), dy)

    def shifted(t):                        # one byte off
        if t.dtype != torch.float8_e4m3fn:
            return t.contiguous()
        room = torch.empty(t.numel() + 1, dtype=torch.uint8, device=t.device)[1:].view(t.shape)
        room.copy_(t.view(torch.uint8) if t.is_contiguous() else t.contiguous().view(torch.uint8))
        return room.view(t.dtype)
    with torch.autograd.graph.saved_tensors_hooks(shifted, lambda t: t):
        y = yamoe_b200.fp8_linear(x, w)
    odd = torch.autograd.grad(y, (x, w), dy)
    for a, b, c in zip(want, got, odd):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_saved_tensors_of_several_matrices():
    import yamoe_b200
    x, w, dy = (randn(3, *s, seed=i).cuda() for i, s in enumerate(((20, 72), (40, 72), (20, 40))))
    x.requires_grad_(True)
    w.requires_grad_(True)
    want = torch.autograd.grad(yamoe_b200.fp8_linear(x, w), (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = yamoe_b200.fp8_linear(x, w)
    for a, b in zip(want, torch.autograd.grad(y, (x, w), dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (0,), (2, 0), (0, 0), (2, 0, 3)])
@pytest.mark.parametrize("N,K", [(24, 40), (0, 40), (24, 0), (0, 0)])
def test_empty_sizes(lead, N, K):
    """No rows, outputs or inputs: what torch's linear gives, zeros where nothing is summed."""
    import yamoe_b200
    x, w = randn(*lead, K, seed=1).cuda().requires_grad_(True), randn(N, K, seed=2).cuda().requires_grad_(True)
    y = yamoe_b200.fp8_linear(x, w)
    assert y.shape == (*lead, N)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape
    with torch.no_grad():
        assert torch.equal(yamoe_b200.fp8_linear(x, w), y)
    if K == 0:
        assert not y.any()
    if N == 0:
        assert not dx.any()
    if x.numel() == 0:
        assert not dw.any()
    elif N > 0:
        flat = x.detach().reshape(-1, K).cpu()
        check_product(y.detach().reshape(-1, N), dequantised(flat, 1), dequantised(w.detach().cpu(), 128), "y")
