"""NaN in a token, a weight or a bias reaches every result that depends on it and no other: the clamps of the GLU keep it, as
torch's do.  Which results those are is asked of the formulas (CPU, 32 bits); the others equal those of a run without it."""
import pytest
import torch

from oracle import experts_oracle as orc
from test_gpu_fp8 import randn
from test_gpu_moe_layer import call, make, quantised

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
GRADS = ["d_hidden", "d_routing", "d_wgu", "d_bgu", "d_wd", "d_bd"]
#: where: argument of `experts` and the element (expert 1 has 30 rows)
PLACES = {"token": (0, (7, 3)), "gate weight": (3, (1, 5, 20)), "up weight": (3, (1, 5, 21)), "gate bias": (4, (1, 20)),
          "up bias": (4, (1, 21))}


def problem(T, H, E, K, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    idx = torch.stack([torch.randperm(E, generator=gen)[:K] for _ in range(T)])
    w = (torch.rand(T, K, generator=gen) + 0.25).to(dtype)
    routing = torch.zeros(T, E, dtype=dtype).scatter_(1, idx, w)
    args = [randn(T, H, seed=seed, dtype=dtype), idx, routing, randn(E, H, 2 * H, seed=seed + 1, dtype=dtype, std=H ** -0.5),
            randn(E, 2 * H, seed=seed + 2, dtype=dtype, std=0.2), randn(E, H, H, seed=seed + 3, dtype=dtype, std=H ** -0.5),
            randn(E, H, seed=seed + 4, dtype=dtype, std=0.2)]
    return args, randn(T, H, seed=seed + 5, dtype=dtype)


def with_nan(args, place):
    i, at = PLACES[place]
    changed = [a.clone() for a in args]
    changed[i][at] = NAN
    return changed


PATHS = [(torch.bfloat16, "tcgen05", 90), (torch.bfloat16, "simt", 90), (torch.bfloat16, "gemv", 8), (torch.bfloat16, "auto", 400),
         (torch.float32, "auto", 90), (torch.float32, "simt", 90)]


@pytest.mark.parametrize("place", sorted(PLACES))
@pytest.mark.parametrize("dtype,path,T", PATHS)
def test_experts_forward(dtype, path, T, place):
    import yamoe_b200
    H, E, K = 128, 6, 2
    args, _ = problem(T, H, E, K, dtype)
    bad = with_nan(args, place)
    ref = torch.isnan(orc.experts_forward_oracle(*bad, T, E, K))
    assert ref.any() and not ref.all()
    yamoe_b200.set_path(path)
    try:
        clean, got = [yamoe_b200.experts(*[a.cuda() for a in v], T, E, K).cpu() for v in (args, bad)]
    finally:
        yamoe_b200.set_path("auto")
    assert torch.equal(torch.isnan(got), ref)
    assert torch.equal(got[~ref], clean[~ref])


@pytest.mark.parametrize("place", sorted(PLACES))
@pytest.mark.parametrize("dtype,path", [(d, p) for d, p, t in PATHS if t == 90])
@pytest.mark.parametrize("saved", [False, True])
def test_experts_gradients(dtype, path, place, saved):
    import yamoe_b200
    T, H, E, K = 90, 128, 6, 2
    args, grad = problem(T, H, E, K, dtype)
    bad = with_nan(args, place)
    ref = [torch.isnan(g) for g in orc.experts_backward_oracle(grad, *bad, T, E, K)]
    assert all(r.any() and not r.all() for r in ref[:4])
    dev = [a.cuda() for a in bad]
    yamoe_b200.set_path(path)
    try:
        if saved:
            _, kept = yamoe_b200.ops.experts_forward_saving(*dev, T, E, K)
            got = yamoe_b200.ops.experts_backward_saved(grad.cuda(), kept, dev[2], dev[3], dev[5], dev[6], T, E, K)
        else:
            got = yamoe_b200.experts_backward(grad.cuda(), *dev, T, E, K)
        got = [g.cpu() for g in got]
    finally:
        yamoe_b200.set_path("auto")
    for g, r, name in zip(got, ref, GRADS):
        assert torch.equal(torch.isnan(g), r), name


@pytest.mark.parametrize("T,H,E,K", [(90, 128, 6, 2), (40, 200, 5, 2), (300, 256, 3, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_experts_fp8_token(T, H, E, K, dtype, value):
    """A group of 128 with such a value is all NaN, and with it the token."""
    import yamoe_b200
    args, _ = problem(T, H, E, K, dtype, seed=T)
    q = yamoe_b200.quantize_experts(args[3].cuda(), args[5].cuda())

    def run(x):
        return yamoe_b200.experts_fp8(x.cuda(), args[1].cuda(), args[2].cuda(), q[0], q[1], args[4].cuda(), q[2], q[3], args[6].cuda(),
                                      T, E, K).cpu()
    bad = args[0].clone()
    bad[7, 3] = value
    clean, got = run(args[0]), run(bad)
    others = torch.arange(T) != 7
    assert torch.isfinite(clean).all() and torch.isnan(got[7]).all()
    assert torch.equal(got[others], clean[others])


@pytest.mark.parametrize("place", ["gate weight", "up weight", "gate bias", "up bias"])
@pytest.mark.parametrize("T,H,E,K", [(90, 128, 6, 2), (40, 328, 5, 2), (300, 256, 3, 1)])
def test_experts_fp8_weights(T, H, E, K, place):
    import yamoe_b200
    args, _ = problem(T, H, E, K, torch.bfloat16, seed=T)

    def run(a):
        q = yamoe_b200.quantize_experts(a[3].cuda(), a[5].cuda())
        return yamoe_b200.experts_fp8(a[0].cuda(), a[1].cuda(), a[2].cuda(), q[0], q[1], a[4].cuda(), q[2], q[3], a[6].cuda(), T, E, K).cpu()
    clean, got = run(args), run(with_nan(args, place))
    hit = (args[1] == 1).any(1)
    assert hit.any() and not hit.all()
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("place", ["gate weight", "up weight", "gate bias", "up bias"])
@pytest.mark.parametrize("T,H,E,K", [(1, 2880, 8, 4), (4, 256, 8, 2), (20, 512, 6, 2), (32, 136, 3, 1)])
@pytest.mark.parametrize("fp8", [False, True])
def test_moe_layer(T, H, E, K, fp8, place):
    """The routing does not depend on the experts' weights, so that its own weights stay finite."""
    d = make(T, H, E, K, seed=T + H)
    if T == 1:
        d["br"][1] = 30.0                # the one token is expert 1's
    bad = {k: v.clone() for k, v in d.items()}
    bad["gu" if "weight" in place else "bgu"][(1, 5, 20 + ("up" in place)) if "weight" in place else (1, 20 + ("up" in place))] = NAN
    (clean, scores), (got, same) = [call(v, K, T, quantised(v) if fp8 else None) for v in (d, bad)]
    assert torch.equal(scores, same) and torch.isfinite(scores).all()
    hit = (scores[:, 1] != 0).cpu()
    assert hit.any()
    assert torch.isnan(got.cpu()[hit]).all() and torch.equal(got.cpu()[~hit], clean.cpu()[~hit])
