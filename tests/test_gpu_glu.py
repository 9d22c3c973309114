"""`glu_fp8` against the GLU and its derivative in 64 bits, and the steps of the expert layer run together."""
import pytest
import torch

from test_gpu_int8 import quantised as int8_of
from test_gpu_token_sort import choices, places, randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
ALPHA, LIMIT = 1.702, 7.0


def parts(pre):
    gate, up = pre.double()[..., 0::2], pre.double()[..., 1::2]
    g, u = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
    return gate, up, g, u, 1 / (1 + torch.exp(-ALPHA * g))


def own_error(g, dtype):
    """Relative error of the sigmoid in 32 bits: the argument's rounding and exp's.  fp32: at most 2 steps of exp, a rounding each of the sum,
    the quotient and the products behind; the approximate exp of bf16 is off by 2 + 1.16 |x| steps and the quotient by 2."""
    x = (ALPHA * g).abs()
    return (12 + x) * 2.0 ** -24 if dtype == F32 else (16 + 4 * x) * 2.0 ** -23


def values_of(pre):
    """What the e4m3 codes of pre [M, W] stand for, in fp32: the definition, with 32-bit divisions and products."""
    M, W = pre.shape
    g = torch.nn.functional.pad(pre.float(), (0, -W % 128)).view(M, -1, 128)
    a = g.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    top = torch.full_like(a, 448.0)
    return ((g * (top / a)).to(torch.float8_e4m3fn).float() * (a / top)).view(M, -1)[:, :W]


SIZES = [(1, 1), (1, 2880), (3, 4), (5, 63), (7, 64), (9, 65), (17, 500), (33, 512), (4, 1001), (300, 2880), (2, 4100)]


@pytest.mark.parametrize("M,N", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1])
def test_glu_and_gradient(M, N, dtype, shift):
    import yamoe_b200
    pre = randn(M, 2 * N, seed=1, dtype=F32).mul_(4).to(dtype)
    held = torch.cat([torch.zeros(shift, dtype=dtype), pre.reshape(-1)]).cuda()
    leaf = held[shift:].view(M, 2 * N).requires_grad_(True)
    y = yamoe_b200.glu_fp8(leaf)
    with torch.no_grad():
        assert torch.equal(yamoe_b200.glu_fp8(leaf), y)
    _, _, g, u, s = parts(pre)
    want = (u + 1) * g * s
    rel = own_error(g, dtype)
    bound = want.abs() * (rel + HALF[dtype] * (1 + rel)) + 1e-30
    assert y.shape == (M, N) and y.dtype == dtype
    assert ((y.detach().double().cpu() - want).abs() <= bound).all()
    dy = randn(M, N, seed=2, dtype=dtype)
    (got,) = torch.autograd.grad(y, leaf, dy.cuda())
    gate, up, g, u, s = parts(values_of(pre))
    d = dy.double()
    d_gate = torch.where(gate > LIMIT, 0.0, d * (u + 1) * s * (1 + ALPHA * g * (1 - s)))
    d_up = torch.where(up.abs() > LIMIT, 0.0, d * g * s)
    # the two terms of d_gate may cancel: their own errors, relative to the magnitudes
    most = (d * (u + 1)).abs() * s * (1 + ALPHA * g.abs())
    for have, want, size in ((got[:, 0::2], d_gate, most), (got[:, 1::2], d_up, d_up.abs())):
        own = 2 * own_error(g, dtype) * size
        off = (have.double().cpu() - want).abs()
        assert (off <= own + HALF[dtype] * (want.abs() + own) + 1e-30).all(), float(off.max())


def test_gradient_against_differences():
    """At values that the codes hold exactly the gradient is the slope of the GLU."""
    import yamoe_b200
    gen = torch.Generator().manual_seed(0)
    pre = torch.randint(-27, 28, (8, 128), generator=gen).float() / 4       # with 7 as the largest: a scale of 1 / 64
    pre[:, 0], pre[:, 1] = 7.0, -7.0
    exact = values_of(pre)
    leaf = pre.cuda().requires_grad_(True)
    y = yamoe_b200.glu_fp8(leaf)
    (grad,) = torch.autograd.grad(y.sum(), leaf)
    h = 1e-4
    inner = (exact.abs() < 6.9) & (exact == pre)

    def value(x):
        _, _, g, u, s = parts(x)
        return (u + 1) * g * s
    assert int(inner.sum()) > 100
    for column in range(0, 128, 5):
        step = torch.zeros_like(exact, dtype=torch.float64)
        step[:, column] = h
        slope = (value(exact.double() + step) - value(exact.double() - step)).sum(1) / (2 * h)
        ok = inner[:, column] & (exact[:, column ^ 1] == pre[:, column ^ 1])
        assert ((grad[:, column].double().cpu() - slope).abs()[ok] < 1e-4).all()


def test_clamps_zeros_and_values_that_are_no_numbers():
    import yamoe_b200
    inf, nan = float("inf"), float("nan")
    pre = torch.zeros(4, 256)
    pre[0, :6] = torch.tensor([8.0, 3.0, 2.0, 9.0, 2.0, -9.0])
    pre[1, 130], pre[2, 1] = nan, inf
    leaf = pre.cuda().requires_grad_(True)
    y = yamoe_b200.glu_fp8(leaf)
    _, _, g, u, s = parts(torch.nan_to_num(pre, nan=0.0))
    want = ((u + 1) * g * s).float()
    off = (y.detach().cpu() - want).abs()
    off[1, 65] = 0
    assert (off < 1e-5 * (1 + want.abs())).all() and y[1, 65].isnan() and int(y.isnan().sum()) == 1
    (d,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    d = d.cpu()
    assert d[0, 0] == 0 and d[0, 1] != 0 and d[0, 3] == 0 and d[0, 5] == 0 and d[0, 2] != 0
    assert d[1, 128:].isnan().all() and not d[1, :128].isnan().any()       # a group with a NaN or an infinity
    assert d[2, :128].isnan().all() and not d[2, 128:].isnan().any()
    assert not d[3].isnan().any() and bool((d[3, 0::2] == 0.5).all()) and not d[3, 1::2].any()


@pytest.mark.parametrize("shape", [(0, 8), (3, 0), (2, 0, 4), (2, 3, 0)])
def test_nothing(shape):
    import yamoe_b200
    x = torch.zeros(*shape).cuda().requires_grad_(True)
    y = yamoe_b200.glu_fp8(x)
    assert y.shape == (*shape[:-1], shape[-1] // 2)
    (d,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert d.shape == x.shape


def test_shapes_layouts_and_saved_tensors():
    import yamoe_b200
    x = randn(2, 5, 260, seed=1, dtype=BF16).cuda().requires_grad_(True)
    y = yamoe_b200.glu_fp8(x)
    up = randn(2, 5, 130, seed=2, dtype=BF16).cuda()
    want = torch.autograd.grad(y, x, up)[0]
    flat = x.detach().reshape(10, 260).requires_grad_(True)
    z = yamoe_b200.glu_fp8(flat)
    assert torch.equal(z.view(y.shape), y) and torch.equal(torch.autograd.grad(z, flat, up.view(10, 130))[0].view(x.shape), want)
    odd = x.detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
    z = yamoe_b200.glu_fp8(odd)
    assert torch.equal(torch.autograd.grad(z, odd, up.transpose(0, 1).contiguous().transpose(0, 1))[0], want)
    with torch.autograd.graph.save_on_cpu():
        z = yamoe_b200.glu_fp8(x)
    assert torch.equal(torch.autograd.grad(z, x, up)[0], want)
    with pytest.raises(RuntimeError, match="2 \\* N"):
        yamoe_b200.glu_fp8(torch.zeros(2, 3).cuda())
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        yamoe_b200.glu_fp8(torch.zeros(2, 4).half().cuda())


def test_checkpoint_takes_a_byte_per_value():
    """What lives between the two passes: codes and scales, not the inputs."""
    import yamoe_b200
    M, N = 4096, 2880
    x = torch.randn(M, 2 * N, device="cuda", dtype=BF16).requires_grad_(True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = yamoe_b200.glu_fp8(x)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert M * 2 * N <= kept <= M * 2 * N * 1.04


def test_captured_and_replayed():
    import yamoe_b200
    pre, dy = randn(40, 640, seed=1, dtype=BF16).cuda(), randn(40, 320, seed=2, dtype=BF16).cuda()

    def step():
        leaf = pre.detach().requires_grad_(True)
        y = yamoe_b200.glu_fp8(leaf)
        return (y.detach(), *torch.autograd.grad(y, leaf, dy))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(2):
        pre.copy_(randn(40, 640, seed=5 + turn, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


# ---- together --------------------------------------------------------------------------------------------------------------------

def layer_inputs(T, H, E, K):
    x = randn(T, H, seed=1, dtype=BF16)
    gate_up, down = randn(E, H, 2 * H, seed=2).mul_(H ** -0.5).to(BF16), randn(E, H, H, seed=3).mul_(H ** -0.5).to(BF16)
    logits = randn(T, E, seed=4)
    best, idx = torch.topk(logits, K, dim=-1)
    return x, gate_up, down, torch.softmax(best, -1), idx


@pytest.mark.parametrize("T,H,E,K", [(1, 128, 8, 2), (7, 256, 16, 4), (200, 128, 8, 2), (600, 192, 4, 2)])
def test_serving_in_integers(T, H, E, K):
    """sort -> quantise -> product -> GLU -> quantise -> product -> combine, against the same steps in 64 bits, each from what the step
    before it really gave."""
    import yamoe_b200
    x, gate_up, down, w, idx = layer_inputs(T, H, E, K)
    gu, dn = yamoe_b200.quantize_int8(gate_up.cuda(), True), yamoe_b200.quantize_int8(down.cuda(), True)
    rows, row_of, offsets = yamoe_b200.sort_tokens(x.cuda(), idx.cuda(), E)
    pre = yamoe_b200.int8_mm(*yamoe_b200.quantize_int8(rows), *gu, F32, offsets)
    act = yamoe_b200.glu_fp8(pre)
    y = yamoe_b200.int8_mm(*yamoe_b200.quantize_int8(act), *dn, F32, offsets)
    out = yamoe_b200.combine_tokens(y, row_of, w.cuda())

    def product(a, b):
        (qa, sa), (qb, sb) = int8_of(a), b
        return torch.cat([(qa[i:j].double() @ qb[e].double().T) * sa[i:j, None].double() * sb[e].double()
                          for e, (i, j) in enumerate(zip(off, off[1:]))])
    want_row, want_off = places(idx, E, None)
    off = want_off.tolist()
    weights = [tuple(t.cpu() for t in m) for m in (gu, dn)]
    for m, held in zip(weights, (gate_up, down)):
        want = int8_of(held.transpose(1, 2))
        assert torch.equal(m[0], want[0]) and torch.equal(m[1], want[1])
    assert torch.equal(row_of.cpu(), want_row) and torch.equal(rows.cpu()[want_row.long()], x[:, None].expand(-1, K, -1))
    want = product(rows.cpu(), weights[0])
    assert ((pre.double().cpu() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs() + 1e-37).all()
    _, _, g, u, s = parts(pre.cpu())
    want = (u + 1) * g * s
    assert ((act.double().cpu() - want).abs() <= want.abs() * (own_error(g, F32) + 2.0 ** -24) + 1e-30).all()
    want = product(act.cpu(), weights[1])
    assert ((y.double().cpu() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs() + 1e-37).all()
    each = y.double().cpu()[want_row.long()] * w.double()[..., None]
    assert ((out.double().cpu() - each.sum(1)).abs() <= (K + 1) * 2.0 ** -24 * 1.001 * each.abs().sum(1)).all()


def test_training_step():
    """sort with places -> fp8_linear -> GLU -> fp8_linear -> combine: the gradients are those of the same graph made of plain operations with the
    products' and the GLU's own backward passes in between."""
    import yamoe_b200
    T, H, E, K, C = 96, 128, 4, 2, 40
    x, gate_up, down, w, idx = layer_inputs(T, H, E, K)
    up = randn(T, H, seed=9, dtype=BF16).cuda()

    def leaves():
        return [t.cuda().requires_grad_(True) for t in (x, gate_up.transpose(1, 2).contiguous(), down.transpose(1, 2).contiguous(), w.to(BF16))]
    a = leaves()
    rows, row_of, _ = yamoe_b200.sort_tokens(a[0], idx.cuda(), E, C)
    assert int((row_of < 0).sum()) > 0                        # some are dropped
    act = yamoe_b200.glu_fp8(yamoe_b200.fp8_linear(rows, a[1]))
    out = yamoe_b200.combine_tokens(yamoe_b200.fp8_linear(act, a[2]), row_of, a[3])
    got = torch.autograd.grad(out, a, up)
    b = leaves()
    of = places(idx, E, C)[0].cuda().long()
    kept = (of >= 0)
    at = torch.where(kept, of, E * C)
    plain = torch.zeros(E * C + 1, H, device="cuda", dtype=BF16).index_put((at.reshape(-1),), b[0][:, None].expand(-1, K, -1).reshape(-1, H))
    act = yamoe_b200.glu_fp8(yamoe_b200.fp8_linear(plain[:-1].view(E, C, H), b[1]))
    y = yamoe_b200.fp8_linear(act, b[2]).view(E * C, H)
    y = torch.cat([y, torch.zeros(1, H, device="cuda", dtype=BF16)])[at].float()
    ref = (y * b[3].float()[..., None] * kept[..., None]).sum(1)
    want = torch.autograd.grad(ref.to(BF16), b, up)
    # out: one rounding of either side; gradients: what the sides round differently, as the order of sums, meets 8-bit quantisation again
    assert ((out.float() - ref).abs() <= 2.0 ** -8 * ref.abs() * 1.01 + 1e-6).all()
    for i, (g, r) in enumerate(zip(got, want)):
        assert g.shape == r.shape
        assert float((g.float() - r.float()).norm()) <= 2e-2 * float(r.float().norm()), i
