"""The layer for a few tokens against plain torch in 64 bits.

2-norm bounds, bf16 results: rounding to bf16 is at most half an ulp, 2^-9 in the 2-norm (eps / 2 / sqrt(3) = 2.3e-3 at the worst
spread of mantissas, 1.7e-3 on average); before it all sums are fp32, activations have 11 (e4m3 weights: 2^-12 / sqrt(3) =
1.4e-4) or 16 bits; 2^-8 / sqrt(3) + 2^-12 is the bound.  Scores are bf16 numbers of fp32 weights: the same bound."""
import pytest
import torch

from test_gpu_fp8 import randn, values

pytestmark = pytest.mark.gpu
BOUND = 2.0 ** -8 / 3 ** 0.5 + 2.0 ** -12


def make(T, H, E, K, seed=0, bias=None):
    d = dict(x=randn(T, H, seed=seed), wr=randn(E, H, seed=seed + 1, std=H ** -0.5), br=randn(E, seed=seed + 2, std=0.1),
             gu=randn(E, H, 2 * H, seed=seed + 3, std=H ** -0.5), bgu=randn(E, 2 * H, seed=seed + 4, std=0.2),
             dn=randn(E, H, H, seed=seed + 5, std=H ** -0.5), bd=randn(E, H, seed=seed + 6, std=0.2))
    if bias is not None:
        d["br"] = bias.to(torch.bfloat16)
    return d


def reference(d, K, cap, q=None):
    x = d["x"].double()
    E = d["wr"].shape[0]
    logits = x @ d["wr"].double().T + (d["br"].double() if d["br"] is not None else 0)
    best, idx = torch.sort(torch.nan_to_num(logits, nan=float("inf"), posinf=float("inf"), neginf=-float("inf")), dim=1,
                           descending=True, stable=True)
    idx = idx[:, :K]
    best = logits.gather(1, idx)
    w = torch.exp(best - best[:, :1])
    w = w / w.sum(1, keepdim=True)
    out = torch.zeros_like(x)
    for e in range(E):
        token, slot = [v[:cap] for v in torch.nonzero(idx == e, as_tuple=True)]
        if token.numel() == 0:
            continue
        if q is None:
            w1, w2 = d["gu"][e].double().T, d["dn"][e].double().T
        else:
            w1, w2 = values(q[0][e], q[1][e], 128), values(q[2][e], q[3][e], 128)
        pre = x[token] @ w1.T + d["bgu"][e].double()
        gate, up = pre[:, 0::2].clamp(max=7.0), pre[:, 1::2].clamp(-7.0, 7.0)
        act = (up + 1) * gate * torch.sigmoid(1.702 * gate)
        out.index_add_(0, token, (act @ w2.T + d["bd"][e].double()) * w[token, slot, None])
    return out, torch.zeros_like(logits).scatter_(1, idx, w)


def call(d, K, cap, q=None):
    import yamoe_b200
    c = {k: v.cuda() if v is not None else None for k, v in d.items()}
    E = d["wr"].shape[0]
    if q is None:
        return yamoe_b200.moe_layer(c["x"], c["wr"], c["br"], c["gu"], c["bgu"], c["dn"], c["bd"], cap, E, K)
    return yamoe_b200.moe_layer(c["x"], c["wr"], c["br"], q[0], c["bgu"], q[2], c["bd"], cap, E, K, q[1], q[3])


def quantised(d):
    import yamoe_b200
    return yamoe_b200.quantize_experts(d["gu"].cuda(), d["dn"].cuda())


def rel(a, b):
    return ((a.cpu().double() - b).norm() / b.norm()).item()


SHAPES = [(1, 64, 4, 2), (1, 2880, 8, 4), (2, 136, 5, 3), (3, 72, 40, 8), (5, 8, 3, 1), (7, 256, 16, 4), (8, 1024, 32, 4),
          (13, 200, 6, 6), (16, 512, 128, 4), (17, 64, 2, 1), (31, 192, 24, 8), (32, 320, 33, 5), (32, 128, 1, 1), (4, 2048, 64, 32)]


@pytest.mark.parametrize("T,H,E,K", SHAPES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("drop", [False, True])
def test_layer(T, H, E, K, fp8, drop):
    d = make(T, H, E, K, seed=T + H)
    cap = max(1, -(-T * K // E) - 1) if drop else T
    q = quantised(d) if fp8 else None
    out, scores = call(d, K, cap, q)
    ref, ref_scores = reference(d, K, cap, q)
    assert out.dtype == scores.dtype == torch.bfloat16 and out.shape == ref.shape and scores.shape == ref_scores.shape
    assert torch.equal(scores.cpu() != 0, ref_scores > 1e-38)
    assert rel(scores, ref_scores) < BOUND
    assert rel(out, ref) < BOUND
    assert not out.cpu()[ref.abs().sum(1) == 0].any()
    again = call(d, K, cap, q)
    assert torch.equal(again[0], out) and torch.equal(again[1], scores)      # no sum depends on the order of CTAs


@pytest.mark.parametrize("fp8", [False, True])
def test_all_tokens_on_few_experts(fp8):
    """More rows of an expert than one pass over its weights takes."""
    T, H, E, K = 32, 264, 9, 3
    bias = torch.zeros(E)
    bias[[1, 4, 8]] = 30.0
    d = make(T, H, E, K, seed=5, bias=bias)
    q = quantised(d) if fp8 else None
    for cap in (32, 17, 16, 3):
        out, scores = call(d, K, cap, q)
        ref, ref_scores = reference(d, K, cap, q)
        assert rel(out, ref) < BOUND and rel(scores, ref_scores) < BOUND
        assert not out.cpu()[cap:].any()


@pytest.mark.parametrize("fp8", [False, True])
def test_capacity_zero_no_bias_no_tokens(fp8):
    d = make(6, 96, 8, 2, seed=9)
    d["br"] = None
    q = quantised(d) if fp8 else None
    out, scores = call(d, 2, 0, q)
    assert not out.any() and rel(scores, reference(d, 2, 0, q)[1]) < BOUND
    assert rel(call(d, 2, 6, q)[0], reference(d, 2, 6, q)[0]) < BOUND
    d["x"] = d["x"][:0]
    out, scores = call(d, 2, 6, q)
    assert out.shape == (0, 96) and scores.shape == (0, 8)


def test_equal_logits_and_masked_experts():
    """Equal logits go to the lower expert; -inf keeps an expert out while K others are left, and beyond that its weight
    is zero; a token all of whose experts are masked has no weights (NaN), like the softmax of such a row."""
    T, H, E, K = 4, 64, 8, 3
    d = make(T, H, E, K, seed=3)
    d["wr"] = torch.zeros_like(d["wr"])
    d["br"] = torch.tensor([1, 2, 2, 1, 2, 2, 1, 1.0]).bfloat16()
    out, scores = call(d, K, T)
    assert torch.equal(scores.cpu()[0] != 0, torch.tensor([False, True, True, False, True, False, False, False]))
    inf = float("inf")
    d["br"] = torch.tensor([-inf, 0, -inf, -inf, 1, -inf, -inf, -inf]).bfloat16()
    out, scores = call(d, K, T)
    ref, ref_scores = reference(d, K, T)
    assert rel(out, ref) < BOUND and (scores.cpu()[:, [1, 4]] > 0).all() and (scores.cpu() > 0).sum() == 2 * T
    d["br"] = torch.full((E,), -inf).bfloat16()
    out, scores = call(d, K, T)
    assert torch.isnan(out).all() and (torch.isnan(scores).sum(1) == K).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_large_small_and_special_activations(fp8):
    T, H, E, K = 6, 128, 4, 2
    d = make(T, H, E, K, seed=11)
    d["wr"] = torch.zeros_like(d["wr"])
    d["br"] = torch.tensor([3.0, 2.0, 1.0, 0.0]).bfloat16()
    d["bgu"], d["bd"] = torch.zeros_like(d["bgu"]), torch.zeros_like(d["bd"])
    d["x"][0] *= 1e30
    d["x"][1] *= 1e-30
    d["x"][2] = 0
    d["x"][3, 5] = 1e20
    q = quantised(d) if fp8 else None
    out, _ = call(d, K, T, q)
    ref, _ = reference(d, K, T, q)
    for t in (0, 1, 3, 4, 5):
        assert rel(out[t], ref[t]) < BOUND, t
    assert not out[2].any()
    d["x"][4, 7] = float("nan")
    out2, _ = call(d, K, T, q)
    assert torch.isnan(out2[4]).all() and torch.equal(out2[[0, 1, 2, 3, 5]], out[[0, 1, 2, 3, 5]])


def test_streams_graphs_and_strides():
    import yamoe_b200
    T, H, E, K = 4, 256, 8, 2
    d = {k: v.cuda() for k, v in make(T, H, E, K, seed=1).items()}
    args = (d["wr"], d["br"], d["gu"], d["bgu"], d["dn"], d["bd"], T, E, K)
    want = yamoe_b200.moe_layer(d["x"], *args)[0]
    wide = torch.zeros(T, 2 * H + 1, device="cuda", dtype=torch.bfloat16)
    wide[:, 1:H + 1] = d["x"]
    assert torch.equal(yamoe_b200.moe_layer(wide[:, 1:H + 1], *args)[0], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = yamoe_b200.moe_layer(d["x"], *args)[0]
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = yamoe_b200.moe_layer(d["x"], *args)[0]
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_layer_refusals():
    import yamoe_b200
    d = {k: v.cuda() for k, v in make(4, 64, 8, 2, seed=1).items()}
    q = quantised(d)
    good = dict(hidden_states=d["x"], router_weight=d["wr"], router_bias=d["br"], gate_up=d["gu"], gate_up_bias=d["bgu"],
                down=d["dn"], down_bias=d["bd"], expert_capacity=4, num_experts=8, top_k=2)
    yamoe_b200.moe_layer(**good)
    for change, message in ((dict(hidden_states=d["x"].float()), "bfloat16"), (dict(hidden_states=d["x"].repeat(9, 1)), "at most 32"),
                            (dict(router_weight=d["wr"][:4]), "router_weight"), (dict(gate_up=q[0]), "scales"),
                            (dict(gate_up=q[0], gate_up_scale=q[1]), "both"), (dict(gate_up_scale=q[1], down_scale=q[3]), "scales"),
                            (dict(gate_up=d["dn"]), "gate_up must be"), (dict(top_k=9), "top_k"),
                            (dict(expert_capacity=-1), "bad argument"), (dict(down_bias=d["bd"].float()), "down_bias")):
        with pytest.raises(RuntimeError, match=message):
            yamoe_b200.moe_layer(**{**good, **change})
