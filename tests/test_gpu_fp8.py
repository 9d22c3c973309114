"""Quantisation to e4m3, products of quantised matrices and their gradients, the expert forward on quantised weights.

References are plain torch in 64 bits.  Codes and scales have one definite value each (32-bit steps, see
include/yamoe_b200.h) and are compared bit by bit.  A product's bound: a block of 128 is four accumulations of 32 exact products,
then one multiplication by the scales and one addition per block; with n = 4 KB + 2 KB + 8 roundings of at most 2^-23 (the
tensor core may truncate) of sums that never exceed S = sum |a| |b|, the error stays below n 2^-23 S, plus half an ulp of
the output type (eps / 2 of the result)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

GROUP, FP8 = 128, torch.float8_e4m3fn


def quantise_ref(x, block):
    """(codes, scales) of a matrix [M, K] by the formula, 32-bit steps, on the CPU."""
    x = x.float().cpu()
    M, K = x.shape
    rb, cb = -(-M // block), -(-K // GROUP)
    p = torch.zeros(rb * block, cb * GROUP)
    p[:M, :K] = x
    g = p.view(rb, block, cb, GROUP)
    most = g.abs().amax(dim=(1, 3)).clamp(min=2.0 ** -100)
    most[torch.isnan(g).any(3).any(1)] = float("nan")
    top = torch.full_like(most, 448.0)
    q = (g * (top / most)[:, None, :, None]).reshape(p.shape)[:M, :K]
    return q.to(FP8), most / top


def values(q, scale, block):
    s = scale.double().cpu().repeat_interleave(GROUP, 1)[:, : q.shape[1]].repeat_interleave(block, 0)[: q.shape[0]]
    return q.cpu().double() * s


def same(a, b):
    """Bit by bit, any NaN like any other."""
    a, b = a.cpu().float(), b.cpu().float()
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def check_product(out, a, b, what):
    ref, size = a @ b.T, a.abs() @ b.abs().T
    kb = -(-a.shape[1] // GROUP)
    bound = (6 * kb + 8) * 2.0 ** -23 * size + torch.finfo(out.dtype).eps / 2 * ref.abs()
    off = (out.cpu().double() - ref).abs() - bound
    assert out.shape == ref.shape, what
    assert not torch.isnan(out).any(), what
    assert off.max() <= 0, (what, off.max().item(), (off > 0).sum().item())


def randn(*shape, seed=0, dtype=torch.bfloat16, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


# ---- quantisation ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 129), (5, 64), (130, 200), (128, 256), (257, 1000), (64, 2880), (129, 8)])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_bits(M, K, block, transpose, dtype):
    import yamoe_b200
    x = randn(M, K, seed=M + K, dtype=dtype) * torch.logspace(-3, 3, K).to(dtype)
    q, s = yamoe_b200.quantize_fp8(x.cuda(), block, transpose)
    rq, rs = quantise_ref(x.T if transpose else x, block)
    assert q.dtype == FP8 and q.shape == rq.shape and s.shape == rs.shape
    assert same(s, rs) and same(q, rq)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


@pytest.mark.parametrize("block,transpose", [(1, False), (1, True), (128, False), (128, True)])
def test_quantize_special_values(block, transpose):
    """Zeros, subnormals, the largest finite values, infinities and NaN; a group with one of the last two is all NaN (or
    zero times infinity), its neighbours are not touched."""
    import yamoe_b200
    x = randn(256, 384, seed=3, dtype=torch.float32)
    x[0:128, 0:128] = 0
    x[0:128, 128:256] = 1e-40
    x[128:256, 0:128] *= 3e38
    x[130, 300] = float("inf")
    x[140, 140] = float("nan")
    x[141, 141] = -float("inf")
    q, s = yamoe_b200.quantize_fp8(x.cuda(), block, transpose)
    rq, rs = quantise_ref(x.T if transpose else x, block)
    assert same(s, rs) and same(q, rq)
    assert torch.isnan(q.float()).any()


def test_quantize_batches_views_and_empty():
    import yamoe_b200
    x = randn(5, 70, 300, seed=1).cuda()
    for view in (x, x[1:4, 3:, 8:], x.transpose(1, 2), x.transpose(0, 1), x.expand(5, 70, 300)[:, :, :1]):
        for block, transpose in ((1, False), (1, True), (128, False), (128, True)):
            q, s = yamoe_b200.quantize_fp8(view, block, transpose)
            for i in range(view.shape[0]):
                rq, rs = quantise_ref(view[i].T if transpose else view[i], block)
                assert same(q[i], rq) and same(s[i], rs)
    for shape in ((0, 128), (128, 0), (0, 4, 128), (3, 0, 128)):
        q, s = yamoe_b200.quantize_fp8(torch.empty(*shape, device="cuda"))
        assert tuple(q.shape) == shape and s.numel() == 0 or 0 in shape


def test_quantize_experts_layout():
    import yamoe_b200
    gu, dn = randn(3, 72, 144, seed=5).cuda(), randn(3, 72, 72, seed=6).cuda()
    q1, s1, q2, s2 = yamoe_b200.quantize_experts(gu, dn)
    assert tuple(q1.shape) == (3, 144, 72) and tuple(s1.shape) == (3, 2, 1) and tuple(q2.shape) == (3, 72, 72)
    for e in range(3):
        rq, rs = quantise_ref(gu[e].T, 128)
        assert same(q1[e], rq) and same(s1[e], rs)


# ---- products -------------------------------------------------------------------------------------------------------

def operands(M, N, K, block, seed=0, std=1.0):
    import yamoe_b200
    a, b = randn(M, K, seed=seed).cuda(), randn(N, K, seed=seed + 1, std=std).cuda()
    # sizes that differ from group to group, so that a scale of another group would show
    a *= torch.logspace(-1, 1, K, device="cuda").to(a.dtype)
    b *= torch.logspace(0.5, -1, N, device="cuda").to(a.dtype)[:, None]
    return yamoe_b200.quantize_fp8(a, 1), yamoe_b200.quantize_fp8(b, block)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 128), (1, 5760, 2880), (2, 300, 100), (17, 64, 640), (33, 130, 257),
                                   (128, 256, 128), (129, 257, 129), (200, 2880, 2880), (256, 256, 4096), (300, 1000, 1000),
                                   (511, 16, 33), (1000, 520, 384), (64, 4096, 1024)])
@pytest.mark.parametrize("block", [128, 1])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product(M, N, K, block, out):
    import yamoe_b200
    (qa, sa), (qb, sb) = operands(M, N, K, block, seed=M + N + K)
    c = yamoe_b200.fp8_mm(qa, sa, qb, sb, out)
    assert c.dtype == out
    check_product(c, values(qa, sa, 1), values(qb, sb, block if sb.shape[0] != N else 1 if N > 1 else 128), f"{M}x{N}x{K}")


@pytest.mark.parametrize("B,M,N,K", [(3, 1, 200, 136), (5, 40, 128, 256), (2, 300, 264, 500), (8, 129, 64, 64)])
@pytest.mark.parametrize("block", [128, 1])
def test_product_of_several_matrices(B, M, N, K, block):
    import yamoe_b200
    a, b = randn(B, M, K, seed=1).cuda(), randn(B, N, K, seed=2).cuda()
    (qa, sa), (qb, sb) = yamoe_b200.quantize_fp8(a, 1), yamoe_b200.quantize_fp8(b, block)
    c = yamoe_b200.fp8_mm(qa, sa, qb, sb)
    for i in range(B):
        check_product(c[i], values(qa[i], sa[i], 1), values(qb[i], sb[i], block), i)


def test_product_strides_alignment_and_streams():
    """Operands in other layouts than the quantiser's: dense rows of odd width, offset, transposed and row-major scales."""
    import yamoe_b200
    (qa, sa), (qb, sb) = operands(70, 150, 201, 128)
    want = yamoe_b200.fp8_mm(qa, sa, qb, sb)
    odd = torch.empty(1 + 70 * 201, dtype=torch.uint8, device="cuda")[1:].view(70, 201)
    odd.copy_(qa.view(torch.uint8) if qa.is_contiguous() else qa.contiguous().view(torch.uint8))
    odd = odd.view(FP8)
    assert torch.equal(want, yamoe_b200.fp8_mm(odd, sa.contiguous(), qb, sb.contiguous()))
    tall = torch.empty(201, 150, dtype=torch.uint8, device="cuda")
    tall.copy_(qb.contiguous().view(torch.uint8).T)
    assert torch.equal(want, yamoe_b200.fp8_mm(qa, sa, tall.view(FP8).T, sb))
    rows = yamoe_b200.fp8_mm(qa[3:60:2], sa[3:60:2], qb, sb)
    assert torch.equal(rows, want[3:60:2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = yamoe_b200.fp8_mm(qa, sa, qb, sb)
    side.synchronize()
    assert torch.equal(got, want)


def test_product_nan_stays_in_its_row_and_empty_products():
    import yamoe_b200
    a, b = randn(40, 300, seed=1), randn(50, 300, seed=2)
    a[7, 290] = float("nan")
    (qa, sa), (qb, sb) = yamoe_b200.quantize_fp8(a.cuda(), 1), yamoe_b200.quantize_fp8(b.cuda(), 128)
    c = yamoe_b200.fp8_mm(qa, sa, qb, sb).cpu()
    bad = torch.isnan(c)
    assert bad[7].all() and not bad[:7].any() and not bad[8:].any()
    empty = torch.empty(0, 300, device="cuda").to(FP8), torch.empty(0, 3, device="cuda")
    assert tuple(yamoe_b200.fp8_mm(*empty, qb, sb).shape) == (0, 50)
    assert tuple(yamoe_b200.fp8_mm(qa, sa, *empty).shape) == (40, 0)
    none = yamoe_b200.fp8_mm(qa[:, :0], sa[:, :0], qb[:, :0], sb[:, :0])
    assert tuple(none.shape) == (40, 50) and not none.any()


def test_refusals():
    import yamoe_b200
    (qa, sa), (qb, sb) = operands(40, 50, 200, 128)
    x = torch.zeros(4, 8, device="cuda")
    bad = [
        (yamoe_b200.quantize_fp8, (x.half(),), "float32 or bfloat16"),
        (yamoe_b200.quantize_fp8, (x, 64), "block_rows"),
        (yamoe_b200.quantize_fp8, (x[0],), "2D"),
        (yamoe_b200.fp8_mm, (qa.float(), sa, qb, sb), "float8_e4m3fn"),
        (yamoe_b200.fp8_mm, (qa, sa.double(), qb, sb), "float32"),
        (yamoe_b200.fp8_mm, (qa, sa[:, :1], qb, sb), "one value per group"),
        (yamoe_b200.fp8_mm, (qa, sa[:1], qb, sb), "scale per row"),
        (yamoe_b200.fp8_mm, (qa[:, :136], sa, qb, sb), "K is"),
        (yamoe_b200.fp8_mm, (qa, sa, qb[None], sb[None]), "2D"),
        (yamoe_b200.fp8_mm, (qa, sa, qb, sb, torch.float16), "out_dtype"),
        (yamoe_b200.fp8_mm, (qa.cpu(), sa.cpu(), qb.cpu(), sb.cpu()), "CUDA|device|backend"),
        (yamoe_b200.fp8_linear, (x, x.bfloat16()), "dtype of x"),
        (yamoe_b200.fp8_linear, (x, x[:, :4]), "K is"),
    ]
    for fn, args, message in bad:
        with pytest.raises((RuntimeError, NotImplementedError), match=message):
            fn(*args)


# ---- gradients ------------------------------------------------------------------------------------------------------

def dequantised(x, block):
    return values(*quantise_ref(x, block), block)


@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (16, 128, 256), (100, 130, 72), (300, 257, 500), (129, 128, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_and_gradients(M, N, K, dtype):
    import yamoe_b200
    x, w, dy = randn(M, K, seed=1, dtype=dtype), randn(N, K, seed=2, dtype=dtype, std=0.1), randn(M, N, seed=3, dtype=dtype)
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = yamoe_b200.fp8_linear(xd, wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    assert y.dtype == dx.dtype == dw.dtype == dtype
    w8 = dequantised(w, 128)
    check_product(y.detach(), dequantised(x, 1), w8, "y")
    check_product(dx, dequantised(dy, 1), w8.T.contiguous(), "dx")
    check_product(dw, dequantised(dy.T, 1), dequantised(x.T, 1), "dw")
    with torch.no_grad():
        assert torch.equal(yamoe_b200.fp8_linear(xd, wd), y)
    # one gradient at a time is the same
    y1 = yamoe_b200.fp8_linear(xd, wd.detach())
    assert torch.equal(torch.autograd.grad(y1, xd, dy.cuda())[0], dx)
    y2 = yamoe_b200.fp8_linear(xd.detach(), wd)
    assert torch.equal(torch.autograd.grad(y2, wd, dy.cuda())[0], dw)


def test_linear_gradient_against_differences():
    """Where quantisation changes nothing (powers of two within each group's range), y is the plain product, and
    differences of a loss in x and w give the gradients: sums of small integers, exact in 32 bits."""
    import yamoe_b200
    gen = torch.Generator().manual_seed(7)

    def powers(*shape):
        v = torch.pow(2.0, torch.randint(-2, 3, shape, generator=gen).float()) * (torch.randint(0, 2, shape, generator=gen) * 2 - 1)
        v.view(-1, shape[-1])[:, 0] = 7.0      # 448 / 64: every group's scale is a power of two
        return v
    M, N, K = 6, 5, 8
    x, w = powers(M, K), powers(N, K)
    x[0], w[0] = 7.0, 7.0                      # and along the columns
    dy = powers(M, N)
    dy[0] = 7.0
    xd, wd = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = yamoe_b200.fp8_linear(xd, wd)
    assert torch.equal(y.detach().cpu().double(), x.double() @ w.double().T)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    h = 1.0
    for grad, base, other in ((dx, x, w), (dw, w, x)):
        for i, j in ((0, 0), (1, 3), (4, 7)):
            lo, hi = base.clone().double(), base.clone().double()
            lo[i, j] -= h
            hi[i, j] += h
            pair = [(v @ other.double().T if grad is dx else other.double() @ v.T) * dy.double() for v in (lo, hi)]
            assert (pair[1].sum() - pair[0].sum()) / (2 * h) == grad[i, j].cpu().double()


def test_linear_batched_and_leading_dimensions():
    import yamoe_b200
    x, w = randn(3, 20, 72, seed=1).cuda().requires_grad_(True), randn(3, 40, 72, seed=2).cuda().requires_grad_(True)
    dy = randn(3, 20, 40, seed=3).cuda()
    y = yamoe_b200.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for i in range(3):
        xi, wi = x[i].detach().requires_grad_(True), w[i].detach().requires_grad_(True)
        yi = yamoe_b200.fp8_linear(xi, wi)
        dxi, dwi = torch.autograd.grad(yi, (xi, wi), dy[i])
        assert torch.equal(y[i], yi) and torch.equal(dx[i], dxi) and torch.equal(dw[i], dwi)
    # a shared weight: its gradient sums over all leading dimensions; an expanded upstream gradient
    w2 = w[0].detach().requires_grad_(True)
    y = yamoe_b200.fp8_linear(x, w2)
    flat = yamoe_b200.fp8_linear(x.reshape(60, 72), w2)
    assert y.shape == (3, 20, 40) and torch.equal(y.view(60, 40), flat)
    g1 = torch.autograd.grad(y, (x, w2), torch.ones(1, 1, 1, device="cuda", dtype=y.dtype).expand_as(y))
    g2 = torch.autograd.grad(flat, (x, w2), torch.ones_like(flat))
    assert torch.equal(g1[0], g2[0]) and torch.equal(g1[1], g2[1])


# ---- expert forward -------------------------------------------------------------------------------------------------

def experts_ref(x, indices, weights, q, biases, cap, rows8=True):
    """The expert forward in 64 bits from the quantised weights; `rows8`: token rows and activations quantised too."""
    gu, gus, dn, dns = [t.cpu() for t in q]
    bgu, bd = biases
    out = torch.zeros(x.shape, dtype=torch.float64)
    size = torch.zeros_like(out)
    xr = dequantised(x, 1) if rows8 else x.double()
    for e in range(gu.shape[0]):
        token, slot = [v[:cap] for v in torch.nonzero(indices == e, as_tuple=True)]
        if token.numel() == 0:
            continue
        w1, w2 = values(gu[e], gus[e], 128), values(dn[e], dns[e], 128)
        pre = xr[token] @ w1.T + bgu[e].double()
        gate, up = pre[:, 0::2].clamp(max=7.0), pre[:, 1::2].clamp(-7.0, 7.0)
        act = (up + 1) * gate * torch.sigmoid(1.702 * gate)
        if rows8:
            act = dequantised(act.float(), 1)
        w = weights[token, slot, None].double()
        out.index_add_(0, token, (act @ w2.T + bd[e].double()) * w)
    return out


def rel(a, b):
    return ((a.cpu().double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("T,H,E,K,cap", [(1, 64, 4, 2, 1), (7, 136, 5, 3, 7), (40, 256, 8, 2, 6), (300, 128, 4, 2, 300),
                                         (700, 192, 3, 2, 500), (64, 2880, 8, 2, 64), (513, 512, 2, 1, 400), (33, 72, 40, 8, 33)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dense", [True, False])
def test_experts(T, H, E, K, cap, dtype, dense):
    """2-norm against 64 bits: half an ulp of the output, and codes of activations that fall to the other neighbour where
    32-bit sums differ (2^-4 of a value, for at most one in 10^4 of them: 6e-4)."""
    import yamoe_b200
    gen = torch.Generator().manual_seed(T + H)
    x = randn(T, H, seed=1, dtype=dtype).cuda()
    gate_up, down = randn(E, H, 2 * H, seed=2, std=H ** -0.5).cuda(), randn(E, H, H, seed=3, std=H ** -0.5).cuda()
    bgu, bd = randn(E, 2 * H, seed=4, dtype=dtype, std=0.2).cuda(), randn(E, H, seed=5, dtype=dtype, std=0.2).cuda()
    probs = torch.softmax(torch.randn(T, E, generator=gen), -1)
    best, indices = torch.topk(probs, K, dim=-1)
    weights = best.to(dtype)
    routing = torch.zeros(T, E, dtype=dtype).scatter_(1, indices, weights) if dense else weights
    if not dense and K == E:
        routing = torch.zeros(T, E, dtype=dtype).scatter_(1, indices, weights)
    q = yamoe_b200.quantize_experts(gate_up, down)
    out = yamoe_b200.experts_fp8(x, indices.cuda(), routing.cuda(), q[0], q[1], bgu, q[2], q[3], bd, cap, E, K)
    assert out.dtype == dtype and out.shape == x.shape
    ref = experts_ref(x.cpu(), indices, weights, q, (bgu.cpu(), bd.cpu()), cap)
    assert rel(out, ref) < (2.0 ** -9 if dtype == torch.bfloat16 else 0) + 6e-4
    dropped = ref.abs().sum(1) == 0
    assert not out.cpu()[dropped].any()


def test_experts_without_rows_and_ids_out_of_range():
    import yamoe_b200
    E, H, K = 4, 64, 2
    q = yamoe_b200.quantize_experts(randn(E, H, 2 * H, seed=2).cuda(), randn(E, H, H, seed=3).cuda())
    bgu, bd = torch.zeros(E, 2 * H, device="cuda").bfloat16(), torch.zeros(E, H, device="cuda").bfloat16()

    def call(x, idx, w, cap):
        return yamoe_b200.experts_fp8(x, idx, w, q[0], q[1], bgu, q[2], q[3], bd, cap, E, K)
    x = randn(6, H, seed=1).cuda()
    idx = torch.tensor([[0, 1], [-1, 2], [4, 3], [9, -5], [1, 2], [3, 0]]).cuda()
    w = torch.full((6, K), 0.5, device="cuda").bfloat16()
    out = call(x, idx, w, 6)
    assert not out[3].any() and out[0].any()
    keep = idx.clone()
    keep[1, 0], keep[2, 0] = 1, 1
    w2 = w.clone()
    w2[1, 0], w2[2, 0] = 0, 0
    again = call(x, keep, w2, 6)
    assert torch.equal(again[[0, 1, 2, 4, 5]], out[[0, 1, 2, 4, 5]])
    assert not call(x, idx, w, 0).any()
    assert call(x[:0], idx[:0], w[:0], 4).shape == (0, H)
    with pytest.raises(RuntimeError, match="gate_up must be"):
        yamoe_b200.experts_fp8(x, idx, w, q[2], q[3], bgu, q[2], q[3], bd, 4, E, K)
    with pytest.raises(RuntimeError, match="128 x 128"):
        yamoe_b200.experts_fp8(x, idx, w, q[0], q[1][:, :, :0], bgu, q[2], q[3], bd, 4, E, K)
