"""`moe_layer` with more experts than a warp holds logits of, and than a CTA has threads.  Bounds: test_gpu_moe_layer.py."""
import pytest
import torch

from test_gpu_moe_layer import BOUND, call, make, quantised, reference, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H,E,K", [(5, 64, 129, 4), (1, 64, 200, 8), (32, 72, 289, 8), (13, 64, 300, 6), (32, 64, 577, 8),
                                     (8, 64, 1024, 32), (32, 64, 1024, 8)])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("drop", [False, True])
def test_layer(T, H, E, K, fp8, drop):
    d = make(T, H, E, K, seed=T + E)
    if drop:
        d["br"][::7] += 4.0              # some experts get more tokens than they keep
    cap = 2 if drop else T
    q = quantised(d) if fp8 else None
    out, scores = call(d, K, cap, q)
    ref, ref_scores = reference(d, K, cap, q)
    assert torch.equal(scores.cpu() != 0, ref_scores > 1e-38)
    assert rel(scores, ref_scores) < BOUND and rel(out, ref) < BOUND
    assert not out.cpu()[ref.abs().sum(1) == 0].any()
    again = call(d, K, cap, q)
    assert torch.equal(again[0], out) and torch.equal(again[1], scores)


@pytest.mark.parametrize("E", [64, 128, 129, 300, 1024])
def test_equal_logits(E):
    """Equal logits go to the lower expert, whatever lane or pass they fall to."""
    T, H, K = 4, 64, 5
    d = make(T, H, E, K, seed=3)
    d["wr"] = torch.zeros_like(d["wr"])
    d["br"] = torch.zeros(E).bfloat16()
    places = sorted({E - 1, E // 2, E // 2 + 32 if E // 2 + 32 < E else 40, 33, 1})[:4]
    d["br"][places] = 2.0
    out, scores = call(d, K, T)
    want = set(places) | {0}
    assert all(set(torch.nonzero(r)[:, 0].tolist()) == want for r in scores.cpu())
    ref, _ = reference(d, K, T)
    assert rel(out, ref) < BOUND


@pytest.mark.parametrize("E", [129, 1024])
def test_masked_experts_and_nan(E):
    T, H, K = 6, 64, 3
    d = make(T, H, E, K, seed=4)
    d["wr"] = torch.zeros_like(d["wr"])
    d["br"] = torch.full((E,), -float("inf")).bfloat16()
    d["br"][[E - 1, 70]] = 1.0
    out, scores = call(d, K, T)
    assert (scores.cpu()[:, [70, E - 1]] == 0.5).all() and (scores.cpu() > 0).sum() == 2 * T
    assert rel(out, reference(d, K, T)[0]) < BOUND
    d["br"] = torch.zeros(E).bfloat16()
    d["br"][[E - 2, 100]] = float("nan")
    out, scores = call(d, K, T)
    assert torch.isnan(out).all() and torch.equal(torch.nonzero(torch.isnan(scores[0]))[:, 0].cpu(), torch.tensor([0, 100, E - 2]))
