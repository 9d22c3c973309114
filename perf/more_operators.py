"""Workloads of the expert layer's steps: tokens sorted by expert and back, products of 8-bit integers, the GLU with an
8-bit checkpoint.  Inputs, plain forms, exact results.

A case is a dict of plain values:
  op     "sort"      `yamoe_b200.sort_tokens`: the rows of T tokens, K experts each, in the experts' order
         "combine"   `yamoe_b200.combine_tokens`: the rows of each token, weighted and added
         "quantize"  `yamoe_b200.quantize_int8`: 8-bit integers with a scale per row, as stored or transposed
         "mm"        `yamoe_b200.int8_mm`: the product of two quantised matrices; E > 0: rows sorted by expert, a matrix each
         "glu"       `yamoe_b200.glu_fp8`: the clamped GLU, whose backward pass reads its inputs from 8 bits
  sort, combine: T tokens of H values, E experts, K per token, rows per expert `cap` (-1: all, one expert's behind the other's),
                 `idle` tokens at the end that belong to no expert, `train`: with the backward pass
  quantize, mm:  B matrices (0: one, without a leading dimension) of M rows; mm with N outputs, K inputs
  glu:           M rows of 2 N values

Shapes are those of perf/cases.py (one set of weights: H, E, K), the gate_up and down projections of its layers as plain
matrices, and odd sizes between.  Weights are N(0, 0.02), activations and upstream gradients N(0, 1), router logits N(0, 1)
with a popularity N(0, 0.5) of each expert.
"""
import math

import torch

own = False

#: (H, E, K) of the repository's own configurations
OSS_20B, OSS_120B = (2880, 32, 4), (2880, 128, 4)
HALF, SMALL, SMALL_16, WIDE, README = (2880, 16, 2), (1024, 32, 4), (1024, 16, 2), (2048, 64, 8), (2880, 8, 2)
SHAPES = (OSS_20B, OSS_120B, HALF, SMALL, SMALL_16, WIDE, README)

STD, GROUP, E4M3_MAX, INT8_MAX, LEAST = 0.02, 128, 448.0, 127.0, 2.0 ** -100
GLU_LIMIT, GLU_ALPHA = 7.0, 1.702
BF16, FP32, FP64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp32": FP32}


def _sort(T, shape, cap=-1, dtype="bf16", train=False, idle=0):
    H, E, K = shape
    return dict(op="sort", T=T, H=H, E=E, K=K, cap=cap, dtype=dtype, train=train, idle=idle)


def _combine(T, shape, weights, cap=-1, dtype="bf16", train=False, idle=0):
    H, E, K = shape
    return dict(op="combine", T=T, H=H, E=E, K=K, cap=cap, dtype=dtype, train=train, idle=idle, weights=weights)


def _quantize(M, K, B=0, dtype="bf16", transpose=False):
    return dict(op="quantize", B=B, M=M, K=K, dtype=dtype, transpose=transpose)


def _mm(M, N, K, B=0, E=0, out="bf16"):
    return dict(op="mm", B=B, E=E, M=M, N=N, K=K, out=out)


def _glu(M, N, dtype="bf16", train=False):
    return dict(op="glu", M=M, N=N, dtype=dtype, train=train)


def _share(T, shape):
    """Twice an expert's mean number of rows."""
    return min(T, 2 * -(-T * shape[2] // shape[1]))


def listed():
    named = {
        # 16 users, a token each, on their way to the experts; a training step's tokens, in places for twice the mean
        "sort_16": _sort(16, OSS_120B),
        "sort_8192_train": _sort(8192, OSS_20B, cap=_share(8192, OSS_20B), train=True),
        # the results of an odd batch on their way back; a training step's, with the router's dense weights
        "combine_333": _combine(333, WIDE, "slots", dtype="fp32"),
        "combine_8192_train": _combine(8192, OSS_20B, "dense", train=True),
        # activations of a prompt on their way into a product; a checkpoint's gate_up weights, once at load time
        "quantize_4096": _quantize(4096, 2880),
        "quantize_experts": _quantize(2880, 5760, B=32, transpose=True),
        # one token through one projection; a ragged batch, sums kept in 32 bits; a long prompt through the widest projection
        "mm_1": _mm(1, 5760, 2880),
        "mm_333": _mm(333, 2048, 4095, out="fp32"),
        "mm_8192": _mm(8192, 5760, 2880),
        # the sorted rows of a prompt of 512 tokens through 32 experts' gate_up projections
        "mm_experts_2048": _mm(2048, 5760, 2880, E=32),
        # the activations of such a prompt; of a training step, forward and backward
        "glu_2048": _glu(2048, 2880),
        "glu_32768_train": _glu(32768, 2880, train=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("sort", "combine", "quantize", "mm", "glu")}
    while True:
        op = rng.choice(tuple(most))
        B = rng.choice((0, 0, 0, rng.randint(1, 16)))
        dtype = rng.choice(("bf16", "bf16", "fp32"))
        if op in ("sort", "combine"):
            T, shape = _log(rng, 1, 8192), rng.choice(SHAPES)
            if rng.random() < 0.3:
                shape = (_log(rng, 8, 4096), *shape[1:])
            cap = rng.choice((-1, -1, _share(T, shape), -(-T * shape[2] // shape[1])))
            args = dict(cap=cap, dtype=dtype, train=rng.random() < 0.5, idle=rng.choice((0, 0, rng.randint(0, T // 2))))
            case = _sort(T, shape, **args) if op == "sort" else _combine(T, shape, rng.choice(("none", "slots", "dense")), **args)
        elif op == "quantize":
            case = _quantize(_log(rng, 1, 8192), _log(rng, 64, 5760), B, dtype, rng.random() < 0.4)
        elif op == "mm":
            case = _mm(_log(rng, 1, 8192), _log(rng, 64, 5760), _log(rng, 64, 5760), B, 0, dtype)
            if rng.random() < 0.4:
                case.update(B=0, E=rng.choice(SHAPES)[1])
        else:
            case = _glu(_log(rng, 1, 32768), _log(rng, 32, 2880), dtype, rng.random() < 0.5)
        if _cost(case) <= most[op]:
            return case


def _ceil(a, b):
    return -(-a // b)


def _n_rows(case):
    return case["T"] * case["K"] if case["cap"] < 0 else case["E"] * case["cap"]


def _matrices_hit(E, M):
    """Expected number of experts that at least one of M rows belongs to (uniform routing)."""
    return E * (1 - (1 - 1 / E) ** M)


def work(case):
    op = case["op"]
    if op in ("sort", "combine"):
        size, S, R = (2 if case["dtype"] == "bf16" else 4), (case["T"] - case["idle"]) * case["K"], _n_rows(case)
        token, moved, held = case["T"] * case["H"] * size, min(S, R) * case["H"] * size, R * case["H"] * size
        if op == "sort":
            nbytes = token + held + 12 * case["T"] * case["K"] + 4 * case["E"] + (moved + token if case["train"] else 0)
            return {"bytes": nbytes, "flops": S * case["H"] * case["train"]}
        n_weights = {"none": 0, "slots": case["T"] * case["K"], "dense": case["T"] * case["E"]}[case["weights"]]
        nbytes = moved + token + 4 * case["T"] * case["K"] + 4 * n_weights
        if case["train"]:
            nbytes += token + moved + held + 4 * n_weights
        return {"bytes": nbytes, "flops": 2 * S * case["H"] * (3 if case["train"] else 1)}
    M = case["M"]
    size = 2 if case.get("dtype", case.get("out")) == "bf16" else 4
    if op == "glu":
        nbytes = M * case["N"] * size * 3
        if case["train"]:
            nbytes += M * (case["N"] * size * 3 + 2 * (2 * case["N"] + 4 * _ceil(2 * case["N"], GROUP)))
        return {"bytes": nbytes, "flops": M * case["N"] * (30 if case["train"] else 10)}
    B, K = max(1, case["B"]), case["K"]
    if op == "quantize":
        return {"bytes": B * (M * K * (size + 1) + 4 * (K if case["transpose"] else M)), "flops": 2 * B * M * K}
    N, weights = case["N"], _matrices_hit(case["E"], M) if case["E"] else 1
    return {"bytes": B * (M * K + weights * N * (K + 4) + M * N * size + 4 * M), "flops": 2 * B * M * N * K}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1.6e15)


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _placed(indices, E, cap):
    """row_of [T, K] and offsets [E + 1] of assignments sorted by expert: those of one in the order of their places."""
    flat = indices.reshape(-1)
    mine = flat[:, None] == torch.arange(E, device=flat.device)
    place = (mine.cumsum(0) * mine).sum(1) - 1
    counts = mine.sum(0)
    if cap >= 0:
        counts = counts.clamp(max=cap)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    first = offsets[:-1] if cap < 0 else torch.arange(E, device=flat.device) * cap
    kept = (place >= 0) & (place < cap) if cap >= 0 else place >= 0
    row = torch.where(kept, first[flat.clamp(min=0)] + place, -1)
    return row.view(indices.shape).to(torch.int32), offsets.to(torch.int32)


def _at(rows, row_of):
    """rows [R, H] at row_of [T, K], zeros where that is -1."""
    with_zero = torch.cat([rows, rows.new_zeros(1, rows.shape[1])])
    return with_zero[torch.where(row_of < 0, rows.shape[0], row_of).long()]


def _spread(values, row_of, R):
    """[R, H] with values [T, K, H] at row_of, zeros elsewhere."""
    out = values.new_zeros(R + 1, values.shape[-1])
    out[torch.where(row_of < 0, R, row_of).long().reshape(-1)] = values.reshape(-1, values.shape[-1])
    return out[:R]


def _int8(x, transpose):
    x = x.to(FP32)
    if transpose:
        x = x.transpose(-1, -2)
    most = x.abs().amax(dim=-1).clamp(min=LEAST)
    top = torch.full_like(most, INT8_MAX)
    return torch.round(x * (top / most)[..., None]).to(torch.int8), most / top


def _fp8_values(x):
    """The fp32 values that x [M, W] has in e4m3 with a scale per group of 128 columns."""
    M, W = x.shape
    g = torch.nn.functional.pad(x.to(FP32), (0, -W % GROUP)).view(M, -1, GROUP)
    most = g.abs().amax(dim=-1, keepdim=True).clamp(min=LEAST)
    top = torch.full_like(most, E4M3_MAX)
    return ((g * (top / most)).to(FP8).to(FP32) * (most / top)).view(M, -1)[:, :W]


def _glu_parts(pre):
    gate, up = pre[:, 0::2], pre[:, 1::2]
    g, u = gate.clamp(max=GLU_LIMIT), up.clamp(-GLU_LIMIT, GLU_LIMIT)
    return gate, up, g, u, torch.sigmoid(GLU_ALPHA * g)


def _plain(s):
    op = s["op"]
    if op == "sort":
        x = s["x"].detach()
        row_of, offsets = _placed(s["indices"], s["E"], s["cap"])
        R = row_of.numel() if s["cap"] < 0 else s["E"] * s["cap"]
        rows = _spread(x[:, None].expand(-1, row_of.shape[1], -1), row_of, R)
        shape = (R, x.shape[1]) if s["cap"] < 0 else (s["E"], s["cap"], x.shape[1])
        if not s["train"]:
            return rows.view(shape), row_of, offsets
        d_x = _at(s["d_rows"].reshape(R, -1).to(FP32), row_of).sum(1).to(x.dtype)
        return rows.view(shape), row_of, offsets, d_x
    if op == "combine":
        rows, row_of = s["rows"].detach().reshape(-1, s["rows"].shape[-1]), s["row_of"]
        each = _at(rows.to(FP32), row_of)
        w = None if s["weights"] is None else s["weights"].detach().to(FP32)
        if w is not None and s["indices"] is not None:
            w = torch.where(s["indices"] >= 0, w.gather(1, s["indices"].clamp(min=0)), 0.0)
        out = (each if w is None else each * w[..., None]).sum(1).to(rows.dtype)
        if not s["train"]:
            return out
        d_out = s["d_out"].to(FP32)[:, None].expand_as(each)
        d_rows = _spread(d_out if w is None else d_out * w[..., None], row_of, rows.shape[0]).to(rows.dtype).view(s["rows"].shape)
        if w is None:
            return out, d_rows
        d_w = (d_out * each).sum(2)
        if s["indices"] is not None:
            wide = d_w.new_zeros(d_w.shape[0], s["weights"].shape[1] + 1)
            d_w = wide.scatter(1, torch.where(s["indices"] < 0, wide.shape[1] - 1, s["indices"]), d_w)[:, :-1]
        return out, d_rows, d_w.to(s["weights"].dtype)
    if op == "quantize":
        return _int8(s["x"], s["transpose"])
    if op == "mm":                             # the sums of whole numbers pass 24 bits
        (a, sa), (b, sb) = s["a"], s["b"]
        if s["offsets"] is None:
            return (torch.matmul(a.to(FP64), b.to(FP64).transpose(-1, -2)) * sa[..., None] * sb[..., None, :]).to(s["out"])
        M, place = a.shape[0], torch.arange(s["most"], device=a.device)
        out = torch.zeros(M + 1, b.shape[1], dtype=s["out"], device=a.device)
        for e in range(b.shape[0]):
            row = s["offsets"][e] + place
            row = torch.where(row < s["offsets"][e + 1], row, M)
            inside = row.clamp(max=M - 1)
            out[row] = (torch.matmul(a[inside].to(FP64), b[e].to(FP64).T) * sa[inside, None] * sb[e]).to(s["out"])
        return out[:M]
    pre = s["pre"].detach()
    _, _, g, u, sig = _glu_parts(pre.to(FP32))
    act = ((u + 1) * g * sig).to(pre.dtype)
    if not s["train"]:
        return act
    gate, up, g, u, sig = _glu_parts(_fp8_values(pre))
    dy = s["dy"].to(FP32)
    d_gate = torch.where(gate > GLU_LIMIT, 0.0, dy * (u + 1) * sig * (1 + GLU_ALPHA * g * (1 - sig)))
    d_up = torch.where(up.abs() > GLU_LIMIT, 0.0, dy * g * sig)
    return act, torch.stack([d_gate, d_up], dim=2).view(pre.shape).to(pre.dtype)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _operand(gen, shape, std):
    """A quantised matrix as the framework's quantiser leaves it: rows padded to 16 bytes, a scale per row."""
    *lead, rows, cols = shape
    held = torch.empty(*lead, rows, _ceil(cols, 16) * 16, dtype=torch.int8, device="cuda")[..., :cols]
    scale = torch.empty(*lead, rows, device="cuda")
    for q, s in zip(held.unbind(0), scale.unbind(0)) if lead else ((held, scale),):     # bounds the fp32 temporaries
        got = _int8(torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(0, std, generator=gen), False)
        q.copy_(got[0])
        s.copy_(got[1])
    return held, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    dtype = TYPES[case.get("dtype", case.get("out"))]

    def normal(*shape, std=1.0, dtype=dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)

    def routed(T, E, K):
        logits = normal(T, E, dtype=FP32) + normal(E, std=0.5, dtype=FP32)
        return torch.topk(logits, K, dim=-1)

    if op in ("sort", "combine"):
        T, H, E, K, train = (case[k] for k in ("T", "H", "E", "K", "train"))
        best, indices = routed(T, E, K)
        indices[T - case["idle"]:] = -1
        shape = (T * K, H) if case["cap"] < 0 else (E, case["cap"], H)
        if op == "sort":
            state = dict(op=op, x=normal(T, H), indices=indices, E=E, cap=case["cap"], train=train)
            if train:
                state["x"].requires_grad_(True)
                state["d_rows"] = normal(*shape)
            return state
        state = dict(op=op, rows=normal(*shape), row_of=_placed(indices, E, case["cap"])[0], indices=None, weights=None, train=train)
        weights = torch.softmax(best, dim=-1)
        if case["weights"] == "slots":
            state["weights"] = weights.to(dtype)
        elif case["weights"] == "dense":
            state["weights"] = torch.zeros(T, E, device="cuda").scatter_(1, indices.clamp(min=0), weights).to(dtype)
            state["indices"] = indices
        if train:
            state["rows"].requires_grad_(True)
            state["d_out"] = normal(T, H)
            if state["weights"] is not None:
                state["weights"].requires_grad_(True)
        return state
    if op == "glu":                            # some values lie beyond the clamps
        state = dict(op=op, pre=normal(case["M"], 2 * case["N"], std=2.5), train=case["train"])
        if case["train"]:
            state["pre"].requires_grad_(True)
            state["dy"] = normal(case["M"], case["N"])
        return state
    lead = (case["B"],) if case["B"] else ()
    M, K = case["M"], case["K"]
    if op == "quantize":
        return dict(op=op, x=normal(*lead, M, K), transpose=case["transpose"])
    N, E = case["N"], case["E"]
    state = dict(op=op, a=_operand(gen, (*lead, M, K), 1.0), out=dtype, offsets=None)
    if E:
        experts = routed(M, E, 1)[1]
        state["offsets"] = _placed(experts, E, -1)[1]
        state["most"] = int(state["offsets"].diff().max())
        lead = (E,)
    state["b"] = _operand(gen, (*lead, N, K), STD)
    return state


def run(state):
    if not own:
        return _plain(state)
    import yamoe_b200
    s, op = state, state["op"]
    if op == "sort":
        rows, row_of, offsets = yamoe_b200.sort_tokens(s["x"], s["indices"], s["E"], s["cap"] if s["cap"] >= 0 else None)
        if not s["train"]:
            return rows, row_of, offsets
        return rows.detach(), row_of, offsets, *torch.autograd.grad(rows, s["x"], s["d_rows"])
    if op == "combine":
        out = yamoe_b200.combine_tokens(s["rows"], s["row_of"], s["weights"], s["indices"])
        if not s["train"]:
            return out
        leaves = (s["rows"],) if s["weights"] is None else (s["rows"], s["weights"])
        return out.detach(), *torch.autograd.grad(out, leaves, s["d_out"])
    if op == "quantize":
        return yamoe_b200.quantize_int8(s["x"], s["transpose"])
    if op == "mm":
        return yamoe_b200.int8_mm(*s["a"], *s["b"], s["out"], s["offsets"])
    act = yamoe_b200.glu_fp8(s["pre"])
    if not s["train"]:
        return act
    return act.detach(), *torch.autograd.grad(act, s["pre"], s["dy"])


# ---- in 64 bits -----------------------------------------------------------------------------------------------------

def _order64(indices, E, cap):
    """Row of each assignment and the rows before each expert's, expert by expert."""
    flat = indices.reshape(-1)
    row_of, offsets = torch.full_like(flat, -1), [0]
    for e in range(E):
        mine = torch.nonzero(flat == e)[:, 0]
        if cap >= 0:
            mine = mine[:cap]
        row_of[mine] = torch.arange(len(mine), device=flat.device) + (offsets[-1] if cap < 0 else e * cap)
        offsets.append(offsets[-1] + len(mine))
    return row_of.view(indices.shape).int(), torch.tensor(offsets, dtype=torch.int32, device=flat.device)


def _e4m3(v):
    """The e4m3 value nearest to v (ties to even): 3 bits behind the first, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.pow(2.0, (e - 4).clamp(min=-9).double())
    return torch.round(v / step) * step


def _silu64(gate):
    """g sigmoid(1.702 g) of the clamped gate and its derivative."""
    g = gate.clamp(max=7.0)
    s = 1 / (1 + torch.exp(-1.702 * g))
    return g * s, (s + 1.702 * g * s * (1 - s)) * (gate <= 7.0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sort":
        x = s["x"].detach().double()
        row_of, offsets = _order64(s["indices"], case["E"], case["cap"])
        token, slot = torch.nonzero(row_of >= 0, as_tuple=True)
        at = row_of[token, slot].long()
        shape = (_n_rows(case), case["H"]) if case["cap"] < 0 else (case["E"], case["cap"], case["H"])
        rows = torch.zeros(_n_rows(case), case["H"], dtype=FP64, device="cuda")
        rows[at] = x[token]
        if not case["train"]:
            return rows.view(shape), row_of, offsets
        d_x = torch.zeros_like(x)
        for k in range(case["K"]):
            here = slot == k
            d_x[token[here]] += s["d_rows"].reshape(-1, case["H"])[at[here]].double()
        return rows.view(shape), row_of, offsets, d_x
    if op == "combine":
        rows, row_of = s["rows"].detach().reshape(-1, case["H"]), s["row_of"]
        out = torch.zeros(case["T"], case["H"], dtype=FP64, device="cuda")
        d_rows = torch.zeros(rows.shape, dtype=FP64, device="cuda")
        weights = None if s["weights"] is None else s["weights"].detach().double()
        d_w = None if weights is None else torch.zeros_like(weights)
        for k in range(case["K"]):
            token = torch.nonzero(row_of[:, k] >= 0)[:, 0]
            at, column = row_of[token, k].long(), k if s["indices"] is None else s["indices"][token, k]
            w = 1.0 if weights is None else weights[token, column][:, None]
            r = rows[at].double()
            out[token] += w * r
            if case["train"]:
                d = s["d_out"][token].double()
                d_rows[at] = w * d
                if d_w is not None:
                    d_w[token, column] = (d * r).sum(1)
        if not case["train"]:
            return out
        d_rows = d_rows.view(s["rows"].shape)
        return (out, d_rows) if d_w is None else (out, d_rows, d_w)
    if op == "quantize":                       # 127 / most and its product with a value are 32-bit numbers by definition
        x = s["x"].transpose(-1, -2) if case["transpose"] else s["x"]
        codes, scales = [], []
        for m in x.unbind(0) if x.dim() == 3 else [x]:
            most = m.abs().amax(1).double().clamp(min=LEAST)
            codes.append(torch.round((m.double() * (127.0 / most).float().double()[:, None]).float()).to(torch.int8))
            scales.append(most / 127.0)
        return (torch.stack(codes), torch.stack(scales)) if x.dim() == 3 else (codes[0], scales[0])
    if op == "mm":
        (a, sa), (b, sb) = s["a"], s["b"]
        if s["offsets"] is None:
            parts = [(p.double() @ q.double().T) * sp.double()[:, None] * sq.double()
                     for p, sp, q, sq in (zip(a, sa, b, sb) if a.dim() == 3 else [(a, sa, b, sb)])]
            return torch.stack(parts) if a.dim() == 3 else parts[0]
        bounds = s["offsets"].tolist()
        return torch.cat([(a[i:j].double() @ b[e].double().T) * sa[i:j, None].double() * sb[e].double()
                          for e, (i, j) in enumerate(zip(bounds, bounds[1:]))])
    pre = s["pre"].detach().double()
    act = _silu64(pre[:, 0::2])[0] * (pre[:, 1::2].clamp(-7.0, 7.0) + 1)
    if not case["train"]:
        return act
    kept = torch.empty_like(pre)
    for i in range(0, pre.shape[1], GROUP):
        g = pre[:, i : i + GROUP]
        most = g.abs().amax(1, keepdim=True).clamp(min=LEAST)
        # 448 / most, its product with a value, and the scale are 32-bit numbers by definition
        q = _e4m3((g * (E4M3_MAX / most).float().double()).float().double())
        kept[:, i : i + GROUP] = q * (most / E4M3_MAX).float().double()
    gate, up = kept[:, 0::2], kept[:, 1::2]
    value, slope = _silu64(gate)
    d_pre = torch.empty_like(pre)
    d_pre[:, 0::2] = s["dy"].double() * (up.clamp(-7.0, 7.0) + 1) * slope
    d_pre[:, 1::2] = s["dy"].double() * value * (up.abs() <= 7.0)
    return act, d_pre
