"""The steps on tensors of more than 2^31 values: the last rows are what a call on them alone gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
M, W = 400_000, 5760                          # 2.3e9 values, 4.6 GB in bf16


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def filled(*shape, dtype=BF16):
    x = torch.empty(*shape, device="cuda", dtype=dtype)
    x[:] = torch.randn(shape[-1], device="cuda")            # every row alike, but for the last ones
    x[-300:] = torch.randn(300, shape[-1], device="cuda", dtype=dtype)
    return x


def test_glu():
    import yamoe_b200
    x = filled(M, W).requires_grad_(True)
    y = yamoe_b200.glu_fp8(x)
    dy = torch.ones(1, W // 2, device="cuda", dtype=BF16).expand(M, -1)
    (d,) = torch.autograd.grad(y, x, dy)
    for part in (slice(M - 300, M), slice(0, 5)):
        leaf = x.detach()[part].clone().requires_grad_(True)
        z = yamoe_b200.glu_fp8(leaf)
        assert torch.equal(z, y[part]) and torch.equal(torch.autograd.grad(z, leaf, dy[part].contiguous())[0], d[part])


@pytest.mark.parametrize("transpose", [False, True])
def test_quantize(transpose):
    import yamoe_b200
    x = filled(M, W)
    q, s = yamoe_b200.quantize_int8(x, transpose)
    if not transpose:
        want = yamoe_b200.quantize_int8(x[-300:])
        assert torch.equal(q[-300:], want[0]) and torch.equal(s[-300:], want[1])
        return
    cols = slice(W - 70, W)
    want = yamoe_b200.quantize_int8(x[:, cols].contiguous(), True)
    assert torch.equal(s[cols], want[1]) and torch.equal(q[cols, -1000:], want[0][:, -1000:]) and torch.equal(q[cols, :1000], want[0][:, :1000])


@pytest.mark.parametrize("experts", [0, 4])
def test_product(experts):
    import yamoe_b200
    K = 32
    a = torch.randint(-127, 128, (M, K), device="cuda", dtype=torch.int8)
    b = torch.randint(-127, 128, (experts or 1, W, K), device="cuda", dtype=torch.int8)
    sa, sb = torch.rand(M, device="cuda"), torch.rand(experts or 1, W, device="cuda")
    off = torch.tensor([0, 5, M - 100, M - 100, M], dtype=torch.int32, device="cuda") if experts else None
    out = yamoe_b200.int8_mm(a, sa, b if experts else b[0], sb if experts else sb[0], BF16, off)
    last = yamoe_b200.int8_mm(a[-100:], sa[-100:], b[-1], sb[-1])
    assert torch.equal(out[-100:], last)
    assert torch.equal(out[:5], yamoe_b200.int8_mm(a[:5], sa[:5], b[0], sb[0]))


def test_sort_and_combine():
    import yamoe_b200
    E, C, H, T = 8, 100_000, 2880, 3000       # [E, C, H]: 2.3e9 values
    x = torch.randn(T, H, device="cuda", dtype=BF16).requires_grad_(True)
    idx = torch.stack([torch.full((T,), E - 1), torch.arange(T) % E], 1).cuda()
    rows, row_of, offsets = yamoe_b200.sort_tokens(x, idx, E, C)
    assert int(row_of.max()) == (E - 1) * C + T + T // E - 1 and offsets[-1] == 2 * T
    flat = rows.detach().view(E * C, H)
    assert torch.equal(flat[row_of[:, 0].long()], x.detach()) and torch.equal(flat[row_of[:, 1].long()], x.detach())
    assert not rows.detach()[E - 1, T + T // E:].any() and not rows.detach()[0, T // E:].any()
    out = yamoe_b200.combine_tokens(rows, row_of)
    assert torch.equal(out.detach(), (x.detach().float() * 2).to(BF16))
    (d,) = torch.autograd.grad(out, x, torch.ones_like(out))
    assert bool((d == 2).all())
