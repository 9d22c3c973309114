"""Workloads of the 8-bit operators and of the layer for a few tokens: inputs, plain forms, exact results.

A case is a dict of plain values:
  op     "quantize"  `yamoe_b200.quantize_fp8`: groups of 1 x 128 or blocks of 128 x 128, as stored or transposed
         "mm"        `yamoe_b200.fp8_mm`: the product of two quantised matrices
         "linear"    `yamoe_b200.fp8_linear`, forward and backward: quantisation and three products
         "experts"   `yamoe_b200.experts_fp8`: the expert forward on quantised weights
         "layer"     `yamoe_b200.moe_layer`: router and experts for a few tokens, weights in bf16 or in 8 bits
  quantize, mm, linear: B matrices (0: one, without a leading dimension) of M rows; mm and linear with N outputs, K inputs
  experts, layer: T tokens, hidden size H, E experts, K of them per token, rows per expert `cap`

Shapes are those of perf/cases.py (one set of weights: H, E, K), the gate_up and down projections of its layers as plain
matrices, and odd sizes between.  Weights and biases are N(0, 0.02), activations and upstream gradients N(0, 1), router
logits N(0, 1).
"""
import math

import torch

own = False

#: (H, E, K) of the repository's own configurations
OSS_20B, OSS_120B = (2880, 32, 4), (2880, 128, 4)
HALF, SMALL, SMALL_16, WIDE, README = (2880, 16, 2), (1024, 32, 4), (1024, 16, 2), (2048, 64, 8), (2880, 8, 2)

STD, GROUP, E4M3_MAX, LEAST = 0.02, 128, 448.0, 2.0 ** -100
GLU_LIMIT, GLU_ALPHA = 7.0, 1.702
BF16, FP32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _quantize(M, K, B=0, dtype="bf16", block=1, transpose=False):
    return dict(op="quantize", B=B, M=M, K=K, dtype=dtype, block=block, transpose=transpose)


def _mm(M, N, K, B=0, out="bf16", block=128):
    return dict(op="mm", B=B, M=M, N=N, K=K, out=out, block=block)


def _linear(M, N, K, B=0, dtype="bf16"):
    return dict(op="linear", B=B, M=M, N=N, K=K, dtype=dtype)


def _experts(T, shape, cap=None):
    H, E, K = shape
    return dict(op="experts", T=T, H=H, E=E, K=K, cap=cap if cap is not None else min(T, 2 * -(-T * K // E)))


def _layer(T, shape, weights, cap=None):
    H, E, K = shape
    return dict(op="layer", T=T, H=H, E=E, K=K, cap=cap if cap is not None else T, weights=weights)


def listed():
    named = {
        # activations of a prompt on their way into a product
        "quantize_rows_4096": _quantize(4096, 2880),
        # a checkpoint's gate_up weights, once at load time: transposed, 128 x 128 blocks
        "quantize_experts": _quantize(2880, 5760, B=32, block=128, transpose=True),
        # one token through one projection
        "mm_1": _mm(1, 5760, 2880),
        # a ragged batch, sums kept in 32 bits, one scale per row of either operand (a weight gradient)
        "mm_333_rows": _mm(333, 2048, 4095, out="fp32", block=1),
        # a long prompt through the widest projection
        "mm_8192": _mm(8192, 5760, 2880),
        # a training step of a projection on a ragged batch, and of eight experts' projections at once
        "linear_1531": _linear(1531, 4096, 2048),
        "linear_8x600": _linear(600, 2048, 1024, B=8),
        # prefill of one prompt: the weights of all experts are read for some 64 rows each; and of 16 prompts
        "experts_512": _experts(512, OSS_20B),
        "experts_4096": _experts(4096, OSS_20B),
        # one user, one token at a time, in both kinds of weights; a small batch
        "layer_1": _layer(1, OSS_120B, "bf16"),
        "layer_1_fp8": _layer(1, OSS_120B, "fp8"),
        "layer_16_fp8": _layer(16, WIDE, "fp8"),
    }
    return [dict(c, name=n) for n, c in named.items()]


SHAPES = (OSS_20B, OSS_120B, HALF, SMALL, SMALL_16, WIDE, README)


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("quantize", "mm", "linear", "experts", "layer"))
        B = rng.choice((0, 0, 0, rng.randint(1, 16)))
        if op == "quantize":
            case = _quantize(_log(rng, 1, 8192), _log(rng, 64, 5760), B, rng.choice(("bf16", "bf16", "fp32")),
                             rng.choice((1, 128)), rng.random() < 0.4)
        elif op == "mm":
            case = _mm(_log(rng, 1, 8192), _log(rng, 64, 5760), _log(rng, 64, 5760), B, rng.choice(("bf16", "bf16", "fp32")),
                       rng.choice((128, 128, 1)))
        elif op == "linear":
            case = _linear(_log(rng, 16, 4096), _log(rng, 64, 5760), _log(rng, 64, 5760), B, rng.choice(("bf16", "bf16", "fp32")))
        elif op == "experts":
            T, shape = _log(rng, 1, 4096), rng.choice(SHAPES)
            case = _experts(T, shape, rng.choice((None, None, max(1, T * shape[2] // shape[1]))))
        else:
            T, shape = _log(rng, 1, 32), rng.choice(SHAPES)
            case = _layer(T, shape, rng.choice(("bf16", "fp8")), rng.choice((None, None, -(-T * shape[2] // shape[1]))))
        if _cost(case) <= most:
            return case


def _ceil(a, b):
    return -(-a // b)


def _experts_hit(case):
    """Expected number of experts that at least one of T tokens chooses (uniform routing)."""
    E, K, T = case["E"], case["K"], case["T"]
    return E * (1 - (1 - K / E) ** T)


def work(case):
    op = case["op"]
    if op in ("experts", "layer"):
        T, H, E, K = (case[k] for k in "THEK")
        size = 2 if case.get("weights") == "bf16" else 1
        nbytes = _experts_hit(case) * (3 * H * H * size + 6 * H) + 2 * T * H * 2
        nbytes += T * K * 8 + T * E * 2 if op == "experts" else E * H * 2 + E * 2 + T * E * 2
        if size == 1:
            nbytes += _experts_hit(case) * 3 * _ceil(H, GROUP) ** 2 * 4
        return {"bytes": nbytes, "flops": 6 * T * K * H * H + (2 * T * E * H if op == "layer" else 0)}
    B, M, K = max(1, case["B"]), case["M"], case["K"]
    size = 2 if case.get("dtype", case.get("out")) == "bf16" else 4
    if op == "quantize":
        rows, cols = (K, M) if case["transpose"] else (M, K)
        return {"bytes": B * (M * K * (size + 1) + 4 * _ceil(rows, case["block"]) * _ceil(cols, GROUP)), "flops": 2 * B * M * K}
    N = case["N"]
    if op == "mm":
        scales = 4 * _ceil(K, GROUP) * (M + _ceil(N, case["block"]))
        return {"bytes": B * (M * K + N * K + M * N * size + scales), "flops": 2 * B * M * N * K}
    return {"bytes": B * size * 2 * (M * K + N * K + M * N), "flops": 6 * B * M * N * K}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1.6e15)


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _pad_last2(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % cols, 0, -x.shape[-2] % rows))


def _quantized(x, block):
    """(q, scale) of x [..., M, K] in groups of `block` rows x 128 columns."""
    x = x.to(FP32)
    M, K = x.shape[-2:]
    p = _pad_last2(x, block, GROUP)
    g = p.view(*p.shape[:-2], p.shape[-2] // block, block, p.shape[-1] // GROUP, GROUP)
    most = g.abs().amax(dim=(-3, -1)).clamp(min=LEAST)
    top = torch.full_like(most, E4M3_MAX)
    scale, inverse = most / top, top / most
    q = (g * inverse[..., :, None, :, None]).view(p.shape)[..., :M, :K].to(FP8)
    return q, scale


def _values(q, scale):
    """The fp32 values that q [..., M, K] with its scales stands for."""
    block = 1 if scale.shape[-2] == q.shape[-2] else GROUP
    s = scale.repeat_interleave(GROUP, -1)[..., : q.shape[-1]]
    return q.to(FP32) * (s if block == 1 else s.repeat_interleave(GROUP, -2)[..., : q.shape[-2], :])


def _rounded(x, block):
    return _values(*_quantized(x, block))


def _t(x):
    return x.transpose(-1, -2)


def _glu(pre):
    gate, up = pre[..., 0::2].clamp(max=GLU_LIMIT), pre[..., 1::2].clamp(-GLU_LIMIT, GLU_LIMIT)
    return (up + 1) * gate * torch.sigmoid(GLU_ALPHA * gate)


def _plain_experts(x, indices, weights, gate_up, gate_up_bias, down, down_bias, cap, act_form):
    """x [T, H] and weights [T, K] in 32 bits; gate_up(e), down(e): the fp32 matrices [.., 2H, H], [.., H, H] of experts e."""
    T, K = indices.shape
    E, H = gate_up_bias.shape[0], x.shape[1]
    flat = indices.reshape(-1)
    mine = flat[:, None] == torch.arange(E, device=x.device)
    place = (mine.cumsum(0) * mine).sum(1) - 1              # stable place of an assignment among its expert's
    kept = place < cap
    if T * K <= E:                                          # few rows: an expert's matrices for each
        act = _glu(torch.bmm(gate_up(flat), x.repeat_interleave(K, 0)[:, :, None])[:, :, 0] + gate_up_bias[flat].to(FP32))
        y = torch.bmm(down(flat), act_form(act)[:, :, None])[:, :, 0] + down_bias[flat].to(FP32)
    else:                                                   # an expert's rows side by side, the surplus in a last row
        every = torch.arange(E, device=x.device)
        row = torch.where(kept, flat * cap + place, E * cap)
        rows = torch.zeros(E * cap + 1, H, device=x.device)
        rows[row] = x.repeat_interleave(K, 0)
        act = _glu(torch.bmm(rows[:-1].view(E, cap, H), _t(gate_up(every))) + gate_up_bias[:, None].to(FP32))
        y = torch.bmm(act_form(act), _t(down(every))) + down_bias[:, None].to(FP32)
        y = torch.cat([y.view(E * cap, H), torch.zeros(1, H, device=x.device)])[row]
    w = torch.where(kept, weights.reshape(-1), 0.0)
    return torch.where(kept[:, None], y * w[:, None], 0.0).view(T, K, H).sum(1)


def _plain(s):
    op = s["op"]
    if op == "quantize":
        return _quantized(_t(s["x"]) if s["transpose"] else s["x"], s["block"])
    if op == "mm":
        return torch.matmul(_values(*s["a"]), _t(_values(*s["b"]))).to(s["out"])
    if op == "linear":
        x, w, dy = s["x"].detach(), s["w"].detach(), s["dy"]
        w8 = _rounded(w, GROUP)
        y = torch.matmul(_rounded(x, 1), _t(w8))
        dx = torch.matmul(_rounded(dy, 1), w8)
        dw = torch.matmul(_rounded(_t(dy), 1), _t(_rounded(_t(x), 1)))
        return [v.to(x.dtype) for v in (y, dx, dw)]
    x = s["x"].to(FP32)
    gate_up, gate_up_bias, down, down_bias = s["experts"]
    if op == "experts":
        routing = s["routing"].to(FP32).gather(1, s["indices"])
        out = _plain_experts(_rounded(x, 1), s["indices"], routing, lambda e: _values(gate_up[0][e], gate_up[1][e]), gate_up_bias,
                             lambda e: _values(down[0][e], down[1][e]), down_bias, s["cap"], lambda act: _rounded(act, 1))
        return out.to(s["x"].dtype)
    logits = torch.matmul(x, _t(s["router"][0].to(FP32))) + s["router"][1].to(FP32)
    best, indices = torch.topk(logits, s["K"], dim=-1)
    weights = torch.softmax(best, dim=-1)
    scores = torch.zeros_like(logits).scatter(1, indices, weights)
    of = [(lambda e, m=m: _values(m[0][e], m[1][e]) if isinstance(m, tuple) else m[e].to(FP32)) for m in (gate_up, down)]
    out = _plain_experts(x, indices, weights, of[0], gate_up_bias, of[1], down_bias, s["cap"], lambda act: act)
    return out.to(s["x"].dtype), scores.to(s["x"].dtype)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _operand(gen, shape, std, block):
    """A quantised matrix as the framework's quantiser leaves it: rows padded to 16 bytes, scales with the rows side by side."""
    *lead, rows, cols = shape
    held = torch.empty(*lead, rows, _ceil(cols, 16) * 16, dtype=FP8, device="cuda")[..., :cols]
    scale = torch.empty(*lead, _ceil(cols, GROUP), _ceil(rows, block), device="cuda").transpose(-1, -2)
    flat_q, flat_s = [held], [scale]
    if lead:                                                # one matrix at a time: bounds the fp32 temporaries
        flat_q, flat_s = held.unbind(0), scale.unbind(0)
    for q, s in zip(flat_q, flat_s):
        got = _quantized(torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(0, std, generator=gen), block)
        q.copy_(got[0])
        s.copy_(got[1])
    return held, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def normal(*shape, std=1.0, dtype=BF16):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)

    if op in ("quantize", "mm", "linear"):
        lead = (case["B"],) if case["B"] else ()
        M, K = case["M"], case["K"]
        dtype = BF16 if case.get("dtype", case.get("out")) == "bf16" else FP32
        if op == "quantize":
            return dict(op=op, x=normal(*lead, M, K, dtype=dtype), block=case["block"], transpose=case["transpose"])
        N = case["N"]
        if op == "mm":
            return dict(op=op, a=_operand(gen, (*lead, M, K), 1.0, 1), b=_operand(gen, (*lead, N, K), STD, case["block"]), out=dtype)
        return dict(op=op, x=normal(*lead, M, K, dtype=dtype).requires_grad_(True),
                    w=normal(*lead, N, K, std=STD, dtype=dtype).requires_grad_(True), dy=normal(*lead, M, N, dtype=dtype))
    T, H, E, K = (case[k] for k in "THEK")
    if op == "experts" or case["weights"] == "fp8":
        gate_up, down = _operand(gen, (E, 2 * H, H), STD, GROUP), _operand(gen, (E, H, H), STD, GROUP)
    else:
        gate_up, down = normal(E, H, 2 * H, std=STD), normal(E, H, H, std=STD)
    state = dict(op=op, x=normal(T, H), K=K, cap=case["cap"])
    biases = normal(E, 2 * H, std=STD), normal(E, H, std=STD)
    if op == "experts":
        best, indices = torch.topk(torch.softmax(torch.randn(T, E, generator=gen, device="cuda"), dim=-1), K, dim=-1)
        state["indices"] = indices
        state["routing"] = torch.zeros(T, E, device="cuda").scatter_(1, indices, best).to(BF16)
    else:
        state["router"] = normal(E, H, std=H ** -0.5), normal(E, std=STD)
        if case["weights"] == "bf16":                       # the plain form takes matrices [.., outputs, inputs]
            state["native"] = gate_up, down
            gate_up, down = _t(gate_up), _t(down)
    state["experts"] = gate_up, biases[0], down, biases[1]
    return state


def run(state):
    if not own:
        return _plain(state)
    import yamoe_b200
    s, op = state, state["op"]
    if op == "quantize":
        return yamoe_b200.quantize_fp8(s["x"], s["block"], s["transpose"])
    if op == "mm":
        return yamoe_b200.fp8_mm(*s["a"], *s["b"], s["out"])
    if op == "linear":
        y = yamoe_b200.fp8_linear(s["x"], s["w"])
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])]
    gate_up, gate_up_bias, down, down_bias = s["experts"]
    E = gate_up_bias.shape[0]
    if op == "experts":
        return yamoe_b200.experts_fp8(s["x"], s["indices"], s["routing"], *gate_up, gate_up_bias, *down, down_bias, s["cap"], E, s["K"])
    if "native" in s:
        gate_up, down = s["native"]
        return yamoe_b200.moe_layer(s["x"], *s["router"], gate_up, gate_up_bias, down, down_bias, s["cap"], E, s["K"])
    return yamoe_b200.moe_layer(s["x"], *s["router"], gate_up[0], gate_up_bias, down[0], down_bias, s["cap"], E, s["K"],
                                gate_up[1], down[1])


# ---- in 64 bits -----------------------------------------------------------------------------------------------------

def _codes64(v):
    """The e4m3 value nearest to v (ties to even): 3 bits behind the first, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.pow(2.0, (e - 4).clamp(min=-9).double())
    return torch.round(v / step) * step


def _groups64(x, block):
    """Quantised values and scales of a matrix [M, K] in 64 bits, but for 448 / max and its product with a value, which by
    definition are 32-bit numbers: bf16 inputs often lie on the very middle between two codes, or next to it."""
    x = x.double()
    most = torch.stack([torch.stack([c.abs().max() for c in r.split(block, 0)]) if block > 1 else r.abs().amax(1)
                        for r in x.split(GROUP, 1)], 1).clamp(min=LEAST)

    def spread(v):
        return v.repeat_interleave(GROUP, 1)[:, : x.shape[1]].repeat_interleave(block, 0)[: x.shape[0]]

    scale = most / E4M3_MAX
    return _codes64((x * spread((E4M3_MAX / most).float().double())).float().double()), scale, spread(scale)


def _back64(x, block):
    q, _, each = _groups64(x, block)
    return q * each


def _held64(q, scale):
    each = scale.double().repeat_interleave(GROUP, 1)[:, : q.shape[1]]
    if scale.shape[0] != q.shape[0]:
        each = each.repeat_interleave(GROUP, 0)[: q.shape[0]]
    return q.double() * each


def _matrices(*tensors):
    return zip(*(t.unbind(0) if t.dim() == 3 else [t] for t in tensors))


def _stacked(parts, like):
    return torch.stack(parts) if like.dim() == 3 else parts[0]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].transpose(-1, -2) if case["transpose"] else s["x"]
        got = [_groups64(m, case["block"])[:2] for (m,) in _matrices(x)]
        return _stacked([q for q, _ in got], x), _stacked([c for _, c in got], x)
    if op == "mm":
        return _stacked([_held64(a, c) @ _held64(b, d).T for a, c, b, d in _matrices(*s["a"], *s["b"])], s["a"][0])
    if op == "linear":
        parts = []
        for x, w, dy in _matrices(s["x"].detach(), s["w"].detach(), s["dy"]):
            w8 = _back64(w, GROUP)
            parts.append((_back64(x, 1) @ w8.T, _back64(dy, 1) @ w8, _back64(dy.T, 1) @ _back64(x.T, 1).T))
        return [_stacked(list(p), s["dy"]) for p in zip(*parts)]
    x = s["x"].double()
    T, K = case["T"], case["K"]
    if op == "layer":
        logits = x @ s["router"][0].double().T + s["router"][1].double()
        best, indices = torch.sort(logits, dim=1, descending=True, stable=True)
        best, indices = best[:, :K], indices[:, :K]
        weights = torch.exp(best - best[:, :1])
        weights = weights / weights.sum(1, keepdim=True)
    else:
        x, indices = _back64(x, 1), s["indices"]
        weights = s["routing"].double().gather(1, indices)
    gate_up, gate_up_bias, down, down_bias = s["experts"]
    out = torch.zeros_like(x)
    for e in torch.unique(indices).tolist():
        token, slot = [v[: case["cap"]] for v in torch.nonzero(indices == e, as_tuple=True)]
        w1, w2 = (_held64(m[0][e], m[1][e]) if isinstance(m, tuple) else m[e].double() for m in (gate_up, down))
        pre = x[token] @ w1.T + gate_up_bias[e].double()
        gate, up = pre[:, 0::2].clamp(max=7.0), pre[:, 1::2].clamp(-7.0, 7.0)
        act = (up + 1) * gate / (1 + torch.exp(-1.702 * gate))
        if op == "experts":
            act = _back64(act, 1)
        out.index_add_(0, token, (act @ w2.T + down_bias[e].double()) * weights[token, slot, None])
    if op == "experts":
        return out
    return out, torch.zeros_like(logits).scatter_(1, indices, weights)
