"""`quantize_int8` and `int8_mm` against plain forms in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def randn(*shape, seed, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def quantised(x):
    """Codes and scales of the rows by the definition: 32-bit division and product, nearest, ties to even; bad rows 0 and NaN."""
    x = x.float()
    most = x.abs().amax(-1)
    bad = ~torch.isfinite(most)
    a = torch.where(bad, 1.0, most).clamp(min=2.0 ** -100)
    inverse = torch.full_like(a, 127.0) / a
    q = torch.round(torch.where(bad[..., None], 0.0, x) * inverse[..., None]).to(torch.int8)
    return q, torch.where(bad, float("nan"), a / torch.full_like(a, 127.0))


def codes(*shape, seed, low=-128):
    return torch.randint(low, 128, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int8)


def scales(*shape, seed):
    return torch.rand(*shape, generator=torch.Generator().manual_seed(seed)) * 0.02 + 1e-3


def check(got, a, sa, b, sb, what=""):
    """The sum is exact; its conversion, the product with either scale and the rounding to the type are off by half a step each."""
    want = torch.matmul(a.double(), b.double().transpose(-1, -2)) * sa.double()[..., None] * sb.double()[..., None, :]
    fp32 = 3 * 2.0 ** -24 * 1.001 * want.abs()
    bound = (fp32 if got.dtype == F32 else fp32 + HALF[BF16] * (want.abs() + fp32)) + 1e-37
    assert got.shape == want.shape, what
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (what, float((off - bound).max()), int((off > bound).sum()))


@pytest.mark.parametrize("M,K", [(1, 1), (1, 2880), (7, 64), (33, 129), (130, 1024), (5, 1025), (300, 2048), (9, 5000), (3, 8192), (2, 8193),
                                 (2, 20000), (257, 40), (256, 63)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B", [0, 3])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize(M, K, dtype, B, transpose):
    import yamoe_b200
    x = randn(*((B,) if B else ()), M, K, seed=M + K, dtype=dtype)
    x[..., 0, :] = 0
    if M > 2:
        x[..., 1, K // 2] = 1000.0
        x[..., 2, :] *= 1e-30
    q, s = yamoe_b200.quantize_int8(x.cuda(), transpose)
    want_q, want_s = quantised(x.transpose(-1, -2) if transpose else x)
    assert q.dtype == torch.int8 and s.dtype == F32 and q.shape == want_q.shape and s.shape == want_s.shape
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    # a transposed view is quantised as it looks
    view = x.cuda().transpose(-1, -2).contiguous().transpose(-1, -2)
    again = yamoe_b200.quantize_int8(view, transpose)
    assert torch.equal(again[0], q) and torch.equal(again[1], s)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_that_are_no_numbers(transpose, dtype):
    import yamoe_b200
    x = randn(20, 300, seed=1, dtype=dtype)
    x[3, 5], x[4, 299], x[19, 0] = float("nan"), float("inf"), -float("inf")
    q, s = yamoe_b200.quantize_int8(x.cuda(), transpose)
    want_q, want_s = quantised(x.t() if transpose else x)
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(s.cpu().isnan(), want_s.isnan()) and int(s.isnan().sum()) == 3
    good = ~want_s.isnan()
    assert torch.equal(s.cpu()[good], want_s[good])
    # what is computed from such a row is NaN
    w, sw = codes(40, q.shape[-1], seed=2).cuda(), scales(40, seed=3).cuda()
    out = yamoe_b200.int8_mm(q, s, w, sw, F32).cpu()
    assert torch.equal(out.isnan().any(1), want_s.isnan()) and torch.equal(out.isnan().all(1), want_s.isnan())


def test_largest_values():
    import yamoe_b200
    x = torch.tensor([[3.0e38, -3.4e38, 1e38], [2.0 ** -126, -(2.0 ** -126), 1e-40], [2.0 ** -100, 2.0 ** -101, 0.0]])
    q, s = yamoe_b200.quantize_int8(x.cuda())
    want = quantised(x)
    assert torch.equal(q.cpu(), want[0]) and torch.equal(s.cpu(), want[1])


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (2, 0, 7), (0, 3, 4)])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_nothing(shape, transpose):
    import yamoe_b200
    q, s = yamoe_b200.quantize_int8(torch.zeros(*shape).cuda(), transpose)
    want = torch.empty(*shape).transpose(-1, -2).shape if transpose else torch.Size(shape)
    assert q.shape == want and s.shape == want[:-1] and bool((s == 2.0 ** -100 / 127).all())


# rows, outputs and inputs around the borders of both kernels, of tiles, chunks, k-blocks and the cluster's split
PRODUCTS = [(1, 1, 1), (1, 5760, 2880), (3, 17, 31), (8, 16, 64), (9, 100, 130), (16, 255, 1000), (17, 33, 16), (20, 256, 128), (31, 257, 129),
            (32, 512, 4000), (33, 64, 300), (64, 2880, 5760), (100, 300, 640), (255, 130, 257), (256, 256, 4096), (257, 770, 96), (333, 2048, 4095),
            (500, 31, 2000), (700, 1500, 1111), (1025, 2049, 520), (4100, 640, 384), (8192, 32, 33)]


@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_product(M, N, K, out):
    import yamoe_b200
    a, b, sa, sb = codes(M, K, seed=M), codes(N, K, seed=N + 1), scales(M, seed=2), scales(N, seed=3)
    got = yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out)
    check(got, a, sa, b, sb)


@pytest.mark.parametrize("B,M,N,K", [(1, 40, 50, 60), (3, 1, 40, 100), (5, 12, 100, 129), (4, 70, 300, 256), (16, 33, 257, 65), (2, 600, 1000, 384)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_several_products(B, M, N, K, out):
    import yamoe_b200
    a, b, sa, sb = codes(B, M, K, seed=1), codes(B, N, K, seed=2), scales(B, M, seed=3), scales(B, N, seed=4)
    check(yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out), a, sa, b, sb)


def bounds(counts, M):
    """Offsets of experts with these numbers of rows, somewhere among M."""
    first = (M - sum(counts)) // 2
    return torch.tensor([first + sum(counts[:e]) for e in range(len(counts) + 1)], dtype=torch.int32)


GROUPS = [(1, [1]), (4, [0, 1, 0, 2, 1, 0]), (8, [3, 0, 5]), (20, [0, 0, 20]), (32, [9, 0, 1, 22]), (32, [0] * 5), (31, [1] * 31),
          (33, [33]), (40, [0] * 7), (64, [1, 63, 0, 0]), (300, [257, 0, 31, 12]), (1000, [0, 512, 1, 255, 32, 200, 0]), (700, [100] * 5),
          (2048, [64] * 32), (1500, [3] * 500), (1100, [1] * 1024)]


@pytest.mark.parametrize("M,counts", GROUPS, ids=["%d-%d" % (m, len(c)) for m, c in GROUPS])
@pytest.mark.parametrize("N,K", [(48, 200), (300, 129)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_rows_sorted_by_expert(M, counts, N, K, out):
    """Also rows before the first and behind the last expert's, which are zero."""
    import yamoe_b200
    E, off = len(counts), bounds(counts, M)
    a, b, sa, sb = codes(M, K, seed=1), codes(E, N, K, seed=2), scales(M, seed=3), scales(E, N, seed=4)
    got = yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out, off.cuda())
    assert got.shape == (M, N) and got.dtype == out
    for e in range(E):
        i, j = int(off[e]), int(off[e + 1])
        check(got[i:j], a[i:j], sa[i:j], b[e], sb[e], e)
    assert not got[: int(off[0])].any() and not got[int(off[-1]):].any()
    assert torch.equal(yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out, off.long().cuda()), got)


def test_offsets_beyond_the_rows():
    """Offsets are kept within the rows that there are."""
    import yamoe_b200
    for M in (10, 100):
        a, b, sa, sb = codes(M, 64, seed=1), codes(3, 40, 64, seed=2), scales(M, seed=3), scales(3, 40, seed=4)
        off = torch.tensor([-5, 4, M + 9, 2 ** 31 - 1], dtype=torch.int32)
        got = yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), F32, off.cuda())
        check(got[:4], a[:4], sa[:4], b[0], sb[0])
        check(got[4:], a[4:], sa[4:], b[1], sb[1])


@pytest.mark.parametrize("M", [5, 200])
def test_largest_sums(M):
    """-128 x -128 over the longest rows: 2^31 - 2^14."""
    import yamoe_b200
    K = 2 ** 17 - 1
    a, b = torch.full((M, K), -128, dtype=torch.int8), torch.full((40, K), -128, dtype=torch.int8)
    b[1] = 127
    sa, sb = scales(M, seed=1), scales(40, seed=2)
    check(yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), F32), a, sa, b, sb)


@pytest.mark.parametrize("M", [6, 90])
@pytest.mark.parametrize("K", [50, 64])
def test_layouts(M, K):
    """Rows with a pitch of their own, garbage behind them, transposed and shifted codes, scales with strides."""
    import yamoe_b200
    N = 70
    a, b, sa, sb = codes(M, K, seed=1), codes(N, K, seed=2), scales(M, seed=3), scales(N, seed=4)
    want = yamoe_b200.int8_mm(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), F32)
    check(want, a, sa, b, sb)

    def wide(x, cols, shift=0):
        room = codes(x.shape[0], cols, seed=9).cuda()
        room[:, shift : shift + K] = x.cuda()
        return room[:, shift : shift + K]
    for make in (lambda x: wide(x, 96), lambda x: wide(x, 80, 16), lambda x: wide(x, 97), lambda x: wide(x, 96, 3),
                 lambda x: x.t().contiguous().cuda().t()):
        spread_a = torch.stack([sa, -sa], 1).cuda()[:, 0]
        spread_b = torch.stack([sb, -sb], 1).cuda()[:, 0]
        assert torch.equal(yamoe_b200.int8_mm(make(a), spread_a, make(b), spread_b, F32), want)
    one = scales(1, seed=5).cuda().expand(M)
    check(yamoe_b200.int8_mm(a.cuda(), one, b.cuda(), sb.cuda(), F32), a, one.cpu(), b, sb)


@pytest.mark.parametrize("shape", [(0, 4, 5), (4, 0, 5), (4, 5, 0), (0, 0, 0)])
def test_products_of_nothing(shape):
    import yamoe_b200
    M, N, K = shape
    a, b = torch.zeros(M, K, dtype=torch.int8).cuda(), torch.zeros(N, K, dtype=torch.int8).cuda()
    out = yamoe_b200.int8_mm(a, torch.ones(M).cuda(), b, torch.ones(N).cuda())
    assert out.shape == (M, N) and not out.any()
    out = yamoe_b200.int8_mm(a, torch.ones(M).cuda(), b[None].expand(2, N, K), torch.ones(2, N).cuda(), F32,
                             torch.tensor([0, M, M], dtype=torch.int32).cuda())
    assert out.shape == (M, N) and not out.any()


def test_captured_and_on_other_streams():
    import yamoe_b200
    cases = [(4, 256, 512, 0), (300, 256, 1024, 0), (200, 96, 256, 5)]
    for M, N, K, E in cases:
        x, w = randn(M, K, seed=1, dtype=BF16).cuda(), randn(*((E,) if E else ()), N, K, seed=2, dtype=BF16).cuda()
        off = bounds([M // E] * E, M).cuda() if E else None
        wq = yamoe_b200.quantize_int8(w)

        def step(x=x, wq=wq, off=off):
            return yamoe_b200.int8_mm(*yamoe_b200.quantize_int8(x), *wq, BF16, off)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        side.synchronize()
        assert torch.equal(other, step())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for turn in range(2):
            x.copy_(randn(M, K, seed=10 + turn, dtype=BF16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, step())


def test_refusals():
    import yamoe_b200
    f, q = yamoe_b200.int8_mm, yamoe_b200.quantize_int8
    a, b, sa, sb = codes(4, 32, seed=1).cuda(), codes(5, 32, seed=2).cuda(), scales(4, seed=3).cuda(), scales(5, seed=4).cuda()
    off = torch.tensor([0, 4], dtype=torch.int32).cuda()
    for bad, args in [("2D", (a[0], sa, b, sb)), ("int8", (a.float(), sa, b, sb)), ("float32", (a, sa.bfloat16(), b, sb)), ("2D", (a, sa, b[None], sb)),
                      ("one value per row", (a, sa[:3], b, sb)), ("K is", (a, sa, b[:, :16], sb)), ("one CUDA device", (a, sa.cpu(), b, sb)),
                      ("out_dtype", (a, sa, b, sb, torch.float16)), ("same number", (a[None], sa[None], b[None].expand(2, 5, 32), sb[None].expand(2, 5))),
                      ("3D", (a, sa, b, sb, F32, off)), ("2D", (a[None], sa[None], b[None], sb[None], F32, off)),
                      ("offsets", (a, sa, b[None], sb[None], F32, off[:1])), ("offsets", (a, sa, b[None], sb[None], F32, off.float())),
                      ("one CUDA device", (a, sa, b[None], sb[None], F32, off.cpu()))]:
        with pytest.raises(RuntimeError, match=bad):
            f(*args)
    long = torch.zeros(2, 2 ** 17, dtype=torch.int8).cuda()
    with pytest.raises(RuntimeError, match="2\\^17"):
        f(long, torch.ones(2).cuda(), long, torch.ones(2).cuda())
    many = torch.zeros(1025, 1, 32, dtype=torch.int8).cuda()
    with pytest.raises(RuntimeError, match="1024"):
        f(a, sa, many, torch.ones(1025, 1).cuda(), F32, torch.zeros(1026, dtype=torch.int32).cuda())
    for bad, args in [("2D", (sa,)), ("float32 or bfloat16", (a,)), ("float32 or bfloat16", (torch.zeros(2, 2).half().cuda(),))]:
        with pytest.raises(RuntimeError, match=bad):
            q(*args)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("K", [64, 250])
def test_values_between_two_codes(transpose, K):
    """A product with 127 / a is rounded to 32 bits before it is rounded to an integer: bf16 values of half the largest and the like."""
    import yamoe_b200
    gen = torch.Generator().manual_seed(1)
    top = (torch.randint(128, 256, (400, 1), generator=gen).float() * 2.0 ** -6)
    x = top * (torch.randint(-254, 255, (400, K), generator=gen).float() / 254)
    x = x.to(BF16)
    x[:, 0], x[:, 1] = top[:, 0].to(BF16), (top[:, 0] / 2).to(BF16)
    q, s = yamoe_b200.quantize_int8((x.t().contiguous() if transpose else x).cuda(), transpose)
    want = quantised(x)
    assert torch.equal(q.cpu(), want[0]) and torch.equal(s.cpu(), want[1])
