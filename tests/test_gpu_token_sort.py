"""`sort_tokens` and `combine_tokens` against plain forms in 64 bits: places, rows, sums and gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
#: half a step of a type, relative to the value
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def randn(*shape, seed, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def choices(T, K, E, seed, bad=0.0):
    gen = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, E, (T, K), generator=gen)
    skew = torch.rand(T, K, generator=gen) < 0.3
    idx[skew] = idx[skew] // 4
    if bad:
        off = torch.rand(T, K, generator=gen) < bad
        idx[off] = torch.tensor([-1, E, E + 7, -(2 ** 40), 2 ** 40])[torch.randint(0, 5, (T, K), generator=gen)][off]
    return idx


def places(indices, E, cap):
    """row_of and offsets by a loop over the experts."""
    flat = indices.reshape(-1)
    row_of, offsets = torch.full_like(flat, -1), [0]
    for e in range(E):
        mine = torch.nonzero(flat == e)[:, 0]
        mine = mine if cap is None else mine[:cap]
        row_of[mine] = torch.arange(len(mine)) + (offsets[-1] if cap is None else e * cap)
        offsets.append(offsets[-1] + len(mine))
    return row_of.view(indices.shape).int(), torch.tensor(offsets, dtype=torch.int32)


def spread(x, row_of, R):
    rows = torch.zeros(R, x.shape[1], dtype=x.dtype)
    t, k = torch.nonzero(row_of >= 0, as_tuple=True)
    rows[row_of[t, k].long()] = x[t]
    return rows


def sums(rows, row_of, w):
    """sum over k of w rows[row_of] in 64 bits, and of the magnitudes."""
    R = rows.shape[0]
    inside = (row_of >= 0) & (row_of < R)
    padded = torch.cat([rows.double(), torch.zeros(1, rows.shape[1], dtype=torch.float64)])
    each = padded[torch.where(inside, row_of, R).long()] * w.double()[..., None]
    return each.sum(1), each.abs().sum(1)


def check_sum(got, want, magnitude, terms, what):
    """`terms` roundings of partial sums in fp32, then one to the type."""
    want, magnitude = want.double(), magnitude.double()
    fp32 = terms * 2.0 ** -24 * 1.001 * magnitude
    bound = fp32 + HALF[got.dtype] * (want.abs() + fp32) + 1e-40
    assert got.shape == want.shape, what
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (what, float((off - bound).max()))


SIZES = [(0, 8, 4, 2), (1, 1, 1, 1), (1, 2880, 128, 4), (5, 7, 3, 2), (64, 33, 1024, 3), (333, 128, 64, 8), (1024, 24, 32, 4),
         (1025, 40, 32, 4), (4099, 8, 7, 1), (2000, 64, 1024, 32), (17, 8, 5, 0)]


@pytest.mark.parametrize("T,H,E,K", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("capacity", ["none", "small", "large", "zero"])
def test_sort(T, H, E, K, dtype, capacity):
    import yamoe_b200
    cap = {"none": None, "small": max(1, T * K // (2 * E)), "large": T + 3 if E <= 128 else 40, "zero": 0}[capacity]
    x, idx = randn(T, H, seed=1, dtype=dtype), choices(T, K, E, seed=2, bad=0.1)
    rows, row_of, offsets = yamoe_b200.sort_tokens(x.cuda(), idx.cuda(), E, cap)
    want_row, want_off = places(idx, E, cap)
    assert row_of.dtype == offsets.dtype == torch.int32
    assert torch.equal(row_of.cpu(), want_row) and torch.equal(offsets.cpu(), want_off)
    R = T * K if cap is None else E * cap
    assert rows.shape == ((R, H) if cap is None else (E, cap, H))
    assert torch.equal(rows.cpu().view(R, H), spread(x, want_row, R))


@pytest.mark.parametrize("T,K,E,cap", [(300000, 2, 5, None), (300000, 2, 1024, 100), (262144, 2, 32, None), (150001, 4, 1, 7)])
def test_sort_of_many(T, K, E, cap):
    """Blocks that rank several parts."""
    import yamoe_b200
    x, idx = randn(T, 1, seed=3), choices(T, K, E, seed=4, bad=0.01)
    rows, row_of, offsets = yamoe_b200.sort_tokens(x.cuda(), idx.cuda(), E, cap)
    want_row, want_off = places(idx, E, cap)
    assert torch.equal(row_of.cpu(), want_row) and torch.equal(offsets.cpu(), want_off)
    assert torch.equal(rows.cpu().view(-1, 1), spread(x, want_row, rows.numel()))


@pytest.mark.parametrize("shift", [1, 2, 4])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [40, 3000])
def test_addresses_off_the_wide_boundaries(T, dtype, shift):
    import yamoe_b200
    H, E, K = 24, 8, 2
    held = randn(T * H + shift, seed=5, dtype=dtype).cuda()
    x = held[shift:].view(T, H)
    idx = choices(T, K, E, seed=6)
    rows, row_of, _ = yamoe_b200.sort_tokens(x, idx.int().cuda(), E)
    assert torch.equal(rows.cpu(), spread(x.cpu(), places(idx, E, None)[0], T * K))
    moved = torch.cat([rows.new_zeros(shift), rows.reshape(-1)])[shift:].view(rows.shape)
    w = randn(T, K, seed=7).cuda()
    assert torch.equal(yamoe_b200.combine_tokens(moved, row_of, w), yamoe_b200.combine_tokens(rows, row_of, w))


@pytest.mark.parametrize("T,H,E,K", SIZES + [(2500, 512, 16, 2)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cap", [None, 9])
def test_gradient_of_sort(T, H, E, K, dtype, cap):
    import yamoe_b200
    x, idx = randn(T, H, seed=1, dtype=dtype).cuda().requires_grad_(True), choices(T, K, E, seed=2, bad=0.1)
    rows, row_of, offsets = yamoe_b200.sort_tokens(x, idx.cuda(), E, cap)
    assert rows.requires_grad and not row_of.requires_grad and not offsets.requires_grad
    up = randn(*rows.shape, seed=3, dtype=dtype)
    (dx,) = torch.autograd.grad(rows, x, up.cuda())
    want, most = sums(up.view(rows.numel() // H, H), row_of.cpu(), torch.ones(T, K))
    check_sum(dx, want, most, K, "d_hidden")


def weighted(kind, T, E, K, idx, dtype, seed):
    """(routing_weights, router_indices) as given, and the weight of each slot in 64 bits."""
    if kind == "none":
        return None, None, torch.ones(T, K, dtype=torch.float64)
    if kind == "slots":
        w = randn(T, K, seed=seed, dtype=dtype)
        return w, None, w.double()
    w = randn(T, E, seed=seed, dtype=dtype)
    inside = (idx >= 0) & (idx < E)
    return w, idx, torch.where(inside, w.double().gather(1, torch.where(inside, idx, 0)), 0.0)


@pytest.mark.parametrize("T,H,E,K", [s for s in SIZES] + [(2500, 520, 16, 2), (40, 12, 6, 11), (9, 16, 8, 600)])
@pytest.mark.parametrize("kind,dtype,wdtype", [("none", BF16, F32), ("none", F32, F32), ("slots", BF16, BF16), ("slots", BF16, F32),
                                               ("slots", F32, F32), ("dense", BF16, BF16), ("dense", BF16, F32), ("dense", F32, F32)])
@pytest.mark.parametrize("cap", [None, 9])
def test_combine_and_gradients(T, H, E, K, kind, dtype, wdtype, cap):
    import yamoe_b200
    idx = choices(T, K, E, seed=2, bad=0.1)
    row_of, offsets = places(idx, E, cap)
    R = T * K if cap is None else E * cap
    shape = (R, H) if cap is None else (E, cap, H)
    rows = randn(*shape, seed=4, dtype=dtype)
    w, given, each = weighted(kind, T, E, K, idx, wdtype, seed=5)
    leaves = [rows.cuda().requires_grad_(True)] + ([] if w is None else [w.cuda().requires_grad_(True)])
    out = yamoe_b200.combine_tokens(leaves[0], row_of.cuda(), leaves[1] if w is not None else None, None if given is None else given.cuda())
    flat = rows.view(R, H)
    want, most = sums(flat, row_of, each)
    check_sum(out.detach(), want, most, K, "out")
    with torch.no_grad():
        again = yamoe_b200.combine_tokens(leaves[0], row_of.cuda(), leaves[1] if w is not None else None, None if given is None else given.cuda())
    assert torch.equal(again, out)
    up = randn(T, H, seed=6, dtype=dtype)
    grads = torch.autograd.grad(out, leaves, up.cuda())
    t, k = torch.nonzero(row_of >= 0, as_tuple=True)
    d_rows = torch.zeros(R, H, dtype=torch.float64)
    d_rows[row_of[t, k].long()] = each[t, k, None] * up.double()[t]
    check_sum(grads[0].view(R, H), d_rows, d_rows.abs(), 1, "d_rows")
    if w is None:
        return
    each_dot = torch.zeros(T, K, dtype=torch.float64)
    each_most = torch.zeros(T, K, dtype=torch.float64)
    product = up.double()[t] * flat.double()[row_of[t, k].long()]
    each_dot[t, k], each_most[t, k] = product.sum(1), product.abs().sum(1)
    if given is None:
        check_sum(grads[1], each_dot, each_most, H + 16, "d_weights")
    else:
        d_w, most_w = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
        d_w.index_put_((t, given[t, k]), each_dot[t, k], accumulate=True)       # a token may have an expert twice
        most_w.index_put_((t, given[t, k]), each_most[t, k], accumulate=True)
        check_sum(grads[1], d_w, most_w, H + 16 + K, "d_weights")


def test_gradients_against_differences():
    """The combine is linear in rows and in weights: a difference of two outputs is what the gradient says, up to rounding."""
    import yamoe_b200
    T, H, E, K = 6, 10, 4, 3
    idx = choices(T, K, E, seed=1)
    row_of = places(idx, E, None)[0].cuda()
    rows, w, up = (randn(*s, seed=i).cuda() for i, s in enumerate(((T * K, H), (T, K), (T, H))))
    rows.requires_grad_(True)
    w.requires_grad_(True)
    g_rows, g_w = torch.autograd.grad(yamoe_b200.combine_tokens(rows, row_of, w), (rows, w), up)
    for leaf, grad, other in ((rows, g_rows, w), (w, g_w, rows)):
        step = randn(*leaf.shape, seed=9).cuda()
        with torch.no_grad():
            pair = [(leaf + s * step, other) if leaf is rows else (other, leaf + s * step) for s in (1.0, -1.0)]
            high, low = (yamoe_b200.combine_tokens(a, row_of, b).double() for a, b in pair)
        slope = float(((high - low) / 2 * up.double()).sum())
        assert abs(slope - float((grad.double() * step.double()).sum())) < 1e-4


def test_rows_that_several_assignments_share():
    """row_of may name a row as often as it likes, and rows that do not exist."""
    import yamoe_b200
    T, K, H, R = 50, 4, 40, 9
    gen = torch.Generator().manual_seed(0)
    row_of = torch.randint(-2, R + 2, (T, K), generator=gen).int()
    row_of[:, 3] = 2 ** 31 - 1
    row_of[row_of == 4] = 5                      # a row of nobody
    rows, w, up = (randn(*s, seed=i, dtype=F32) for i, s in enumerate(((R, H), (T, K), (T, H))))
    leaves = rows.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    out = yamoe_b200.combine_tokens(leaves[0], row_of.cuda(), leaves[1])
    want, most = sums(rows, row_of, w)
    check_sum(out.detach(), want, most, K, "out")
    d_rows, d_w = torch.autograd.grad(out, leaves, up.cuda())
    want, most = torch.zeros(2, R, H, dtype=torch.float64)
    for t in range(T):
        for k in range(K):
            r = int(row_of[t, k])
            if 0 <= r < R:
                want[r] += w[t, k].double() * up[t].double()
                most[r] += (w[t, k].double() * up[t].double()).abs()
    check_sum(d_rows, want, most, T * K, "d_rows")
    assert not d_rows[4].any()
    inside = (row_of >= 0) & (row_of < R)
    products = up.double()[:, None] * rows.double()[torch.where(inside, row_of, 0).long()] * inside[..., None]
    check_sum(d_w, products.sum(2), products.abs().sum(2), H + 16, "d_weights")


@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("H", [8, 33, 520])
@pytest.mark.parametrize("R", [12, 200, 1300])
def test_rows_that_many_share_are_summed_in_order(R, H, dense):
    """Weights of 24 bits: a product is rounded where it starts a sum and not where it joins one, so that the order of two shows already."""
    from yamoe_b200 import combine_tokens
    T, K, E = 1400, 2, 5
    row_of = torch.full((T * K,), -1, dtype=torch.int32)
    named = {0: 1, 1: 2, 2: 3, 3: 31, 4: 32, 5: 33, 6: 300, 9: 255, 10: 256, 11: 257, R - 1: 700}          # the others: nobody's
    free = torch.randperm(T * K, generator=torch.Generator().manual_seed(0))
    at = 0
    for r, n in named.items():
        row_of[free[at:at + n]] = r
        at += n
    row_of = row_of.view(T, K)
    idx = torch.randint(0, E, (T, K), generator=torch.Generator().manual_seed(1))
    w = randn(T, E if dense else K, seed=2)
    d = randn(T, H, seed=3)
    rows = torch.zeros(R, H, device="cuda", requires_grad=True)
    out = combine_tokens(rows, row_of.cuda(), w.cuda(), idx.cuda() if dense else None)
    grads = [torch.autograd.grad(out, rows, d.cuda(), retain_graph=True)[0].cpu() for _ in range(10)]
    for g in grads[1:]:
        assert torch.equal(g, grads[0])
    each = (w.gather(1, idx) if dense else w).double()
    assert not grads[0][torch.tensor([r not in named for r in range(R)])].any()
    for r in named:
        t, k = torch.nonzero(row_of == r, as_tuple=True)          # in the order of the assignments
        want, mag = torch.zeros(H, dtype=torch.float64), torch.zeros(H, dtype=torch.float64)
        for i, j in zip(t.tolist(), k.tolist()):
            want += each[i, j] * d[i].double()
            mag += (each[i, j] * d[i].double()).abs()
        check_sum(grads[0][r], want, mag, max(1, len(t)), f"row {r}")
    # 2^24 + 1 + 1 ... - 2^24: each one is lost to ties, in the order of the assignments; any that came after -2^24 or before 2^24 would show
    for n in (4, 40):
        of = torch.zeros(n, 1, dtype=torch.int32)
        d = torch.ones(n, H)
        d[0], d[-1] = 2.0 ** 24, -2.0 ** 24
        rows = torch.zeros(1, H, device="cuda", requires_grad=True)
        (g,) = torch.autograd.grad(combine_tokens(rows, of.cuda()), rows, d.cuda())
        assert not g.any()


def test_dropped_rows_do_not_spread_what_they_hold():
    """NaN and infinities in rows that nobody owns, and a weight of zero: as the formula has it."""
    import yamoe_b200
    rows = torch.tensor([[1.0, 2.0], [float("nan"), float("inf")], [3.0, 4.0]]).cuda()
    row_of = torch.tensor([[0, -1], [2, 0], [1, 0]], dtype=torch.int32).cuda()
    out = yamoe_b200.combine_tokens(rows, row_of, torch.tensor([[2.0, float("nan")], [1.0, 1.0], [0.0, 1.0]]).cuda()).cpu()
    assert out[:2].tolist() == [[2.0, 4.0], [4.0, 6.0]] and out[2].isnan().all()


@pytest.mark.parametrize("grads", ["rows", "weights"])
def test_one_gradient_alone(grads):
    import yamoe_b200
    T, H, E, K = 300, 48, 8, 2
    idx = choices(T, K, E, seed=1)
    row_of = places(idx, E, None)[0].cuda()
    rows, w, up = (randn(*s, seed=i).cuda() for i, s in enumerate(((T * K, H), (T, K), (T, H))))
    both = torch.autograd.grad(yamoe_b200.combine_tokens(rows.requires_grad_(True), row_of, w.requires_grad_(True)), (rows, w), up)
    rows, w = rows.detach().requires_grad_(grads == "rows"), w.detach().requires_grad_(grads == "weights")
    (one,) = torch.autograd.grad(yamoe_b200.combine_tokens(rows, row_of, w), rows if grads == "rows" else w, up)
    assert torch.equal(one, both[0 if grads == "rows" else 1])


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed on other contents; two graphs that share a pool, in turn."""
    import yamoe_b200
    E, K, H = 16, 4, 64
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for T in (30, 3000):
        x, idx, w = randn(T, H, seed=1).cuda(), choices(T, K, E, seed=2).cuda(), randn(T, K, seed=3).cuda()
        up = randn(T, H, seed=4).cuda()

        def step(x=x, idx=idx, w=w, up=up):
            x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            rows, row_of, _ = yamoe_b200.sort_tokens(x, idx, E)
            out = yamoe_b200.combine_tokens(rows * 2, row_of, w)
            return (out.detach(), *torch.autograd.grad(out, (x, w), up))
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            got = step()
        graphs.append((graph, got, step, (x, idx, w, up)))
    for turn in range(3):
        for graph, got, step, (x, idx, w, up) in graphs:
            x.copy_(randn(*x.shape, seed=10 + turn))
            idx.copy_(choices(x.shape[0], K, E, seed=20 + turn))
            w.copy_(randn(*w.shape, seed=30 + turn))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_on_a_stream_of_its_own():
    import yamoe_b200
    T, H, E, K = 700, 256, 16, 4
    x, idx = randn(T, H, seed=1, dtype=BF16).cuda(), choices(T, K, E, seed=2).cuda()
    want = yamoe_b200.sort_tokens(x, idx, E)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(yamoe_b200.sort_tokens(x, idx, E))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_refusals():
    import yamoe_b200
    x, idx = torch.zeros(4, 8).cuda(), torch.zeros(4, 2, dtype=torch.int64).cuda()
    sort, combine = yamoe_b200.sort_tokens, yamoe_b200.combine_tokens
    for bad, args in [("2D", (x[0], idx, 4)), ("float32 or bfloat16", (x.half(), idx, 4)), ("device", (x, idx.cpu(), 4)),
                      ("int64", (x, idx.float(), 4)), (r"\[T, K\]", (x, idx[:3], 4)), ("between 1 and 1024", (x, idx, 0)),
                      ("between 1 and 1024", (x, idx, 1025)), ("negative", (x, idx, 4, -1)), ("too many rows", (x, idx, 1024, 2 ** 21))]:
        with pytest.raises(RuntimeError, match=bad):
            sort(*args)
    rows, row_of, _ = sort(x, idx, 4)
    w = torch.zeros(4, 2).cuda()
    for bad, args in [("float32 or bfloat16", (rows.double(), row_of)), ("rows must be", (rows[0], row_of)), ("int32", (rows, row_of.long())),
                      ("device", (rows, row_of.cpu())), ("dtype", (rows, row_of, w.bfloat16())), ("dtype", (rows, row_of, w.double())),
                      (r"\[T, K\]", (rows, row_of, w[:3])), (r"\[T, K\]", (rows, row_of, torch.zeros(4, 5).cuda())),
                      ("belong", (rows, row_of, None, idx)), ("device", (rows, row_of, w, idx.cpu())), (r"\[T, K\]", (rows, row_of, w, idx[:, :1])),
                      ("1024", (rows, torch.zeros(1, 1025, dtype=torch.int32).cuda()))]:
        with pytest.raises(RuntimeError, match=bad):
            combine(*args)
        with pytest.raises(RuntimeError, match=bad):
            combine(args[0].detach().requires_grad_(True), *args[1:])


@pytest.mark.parametrize("name", ["sort", "combine", "glu"])
def test_derivatives_that_do_not_exist(name):
    import torch.autograd.forward_ad as fwAD
    import yamoe_b200
    x, idx = randn(6, 8, seed=1).cuda().requires_grad_(True), choices(6, 2, 3, seed=2).cuda()
    row_of = places(idx.cpu(), 3, None)[0].cuda()
    rows = randn(12, 8, seed=3).cuda().requires_grad_(True)
    call = {"sort": lambda t: yamoe_b200.sort_tokens(t, idx, 3)[0], "combine": lambda t: yamoe_b200.combine_tokens(t, row_of),
            "glu": yamoe_b200.glu_fp8}[name]
    leaf = rows if name == "combine" else x
    y = call(leaf)
    (first,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        first.sum().backward()
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward"):
        call(fwAD.make_dual(leaf.detach(), torch.ones_like(leaf)))
