"""Products of quantised matrices at the sizes where the kernel changes its tiles: 128 x 256, 128 x 128 singly and in clusters of two,
three and four, several tiles to a CTA, rows that are and are not multiples of 16 bytes.  The bound is that of test_gpu_fp8.py."""
import pytest
import torch

from test_gpu_fp8 import GROUP

pytestmark = pytest.mark.gpu


def values(q, scale, block):
    s = scale.double().repeat_interleave(GROUP, -1)[..., : q.shape[-1]]
    return q.double() * (s if block == 1 else s.repeat_interleave(block, -2)[..., : q.shape[-2], :])


def check_product(out, a, b, what):
    """test_gpu_fp8.check_product on the GPU."""
    ref, size = a @ b.mT, a.abs() @ b.abs().mT
    kb = -(-a.shape[-1] // GROUP)
    bound = (6 * kb + 8) * 2.0 ** -23 * size + torch.finfo(out.dtype).eps / 2 * ref.abs()
    off = (out.double() - ref).abs() - bound
    assert out.shape == ref.shape and not torch.isnan(out).any(), what
    assert off.max() <= 0, (what, off.max().item(), (off > 0).sum().item())


def normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


#: tiles of 128 x 256 in one wave and in several (a CTA takes a second tile), of 128 x 128 in several, clusters of 2, 3 and 4
WIDE = [(2000, 2104, 700), (2000, 2101, 130), (4000, 2200, 264), (4096, 2050, 65), (2500, 4003, 200), (16000, 301, 640)]
NARROW = [(19300, 100, 300), (25700, 128, 129), (40000, 7, 64)]
CLUSTERS = [(333, 2048, 2000), (300, 2050, 2064), (700, 1100, 1500), (129, 2304, 4000), (65, 1030, 3000), (513, 640, 2400), (384, 1500, 1030)]


@pytest.mark.parametrize("M,N,K", WIDE + NARROW + CLUSTERS)
@pytest.mark.parametrize("block", [128, 1])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_tiles(M, N, K, block, out):
    import yamoe_b200
    gen = torch.Generator(device="cuda").manual_seed(M + N)
    a = normal(gen, M, K) * torch.logspace(-1, 1, K, device="cuda").bfloat16()
    b = normal(gen, N, K) * torch.logspace(0.5, -1, N, device="cuda").bfloat16()[:, None]
    (qa, sa), (qb, sb) = yamoe_b200.quantize_fp8(a, 1), yamoe_b200.quantize_fp8(b, block)
    c = yamoe_b200.fp8_mm(qa, sa, qb, sb, out)
    check_product(c, values(qa, sa, 1), values(qb, sb, block), (M, N, K))
    assert torch.equal(yamoe_b200.fp8_mm(qa, sa, qb, sb, out), c)        # no sum depends on the order of CTAs


@pytest.mark.parametrize("B,M,N,K", [(3, 1000, 2100, 400), (8, 600, 2048, 256), (2, 1500, 1999, 260), (40, 300, 250, 130), (200, 40, 90, 64)])
@pytest.mark.parametrize("block", [128, 1])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_tiles_of_several_matrices(B, M, N, K, block, out):
    import yamoe_b200
    gen = torch.Generator(device="cuda").manual_seed(B + M)
    (qa, sa), (qb, sb) = yamoe_b200.quantize_fp8(normal(gen, B, M, K), 1), yamoe_b200.quantize_fp8(normal(gen, B, N, K), block)
    check_product(yamoe_b200.fp8_mm(qa, sa, qb, sb, out), values(qa, sa, 1), values(qb, sb, block), (B, M, N, K))


@pytest.mark.parametrize("M,N,K", [(1531, 4096, 2048), (2100, 1900, 1500), (4000, 520, 700)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_large_products(M, N, K, dtype):
    import yamoe_b200
    gen = torch.Generator(device="cuda").manual_seed(M)
    x, w, dy = normal(gen, M, K, dtype=dtype), normal(gen, N, K, dtype=dtype), normal(gen, M, N, dtype=dtype)

    def rounded(t, block):
        return values(*yamoe_b200.quantize_fp8(t, block), block)         # bit by bit what the formula says: test_gpu_fp8.py
    xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = yamoe_b200.fp8_linear(xd, wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy)
    w8 = rounded(w, 128)
    check_product(y.detach(), rounded(x, 1), w8, "y")
    check_product(dx, rounded(dy, 1), w8.mT.contiguous(), "dx")
    check_product(dw, rounded(dy.mT, 1), rounded(x.mT, 1), "dw")


def test_shapes_of_empty_results():
    import yamoe_b200
    for shape in ((0, 128), (128, 0), (0, 4, 128), (3, 0, 129)):
        for block in (1, 128):
            q, s = yamoe_b200.quantize_fp8(torch.empty(*shape, device="cuda"), block)
            assert tuple(q.shape) == shape
            assert tuple(s.shape) == (*shape[:-2], -(-shape[-2] // block), -(-shape[-1] // 128))
