"""The expert layer's steps where a call's size or arguments lie at a border of the host code around the kernels."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32 = torch.bfloat16, torch.float32

SORTS = """
import sys
import torch
sys.path.insert(0, "tests")
import yamoe_b200
from test_gpu_token_sort import choices, places
E, K, sizes = %r
for T in sizes:
    idx = choices(T, K, E, seed=T)
    x = torch.arange(T, dtype=torch.float32)[:, None]
    rows, row_of, offsets = yamoe_b200.sort_tokens(x.cuda(), idx.cuda(), E)
    want = places(idx, E, None)
    assert torch.equal(row_of.cpu(), want[0]) and torch.equal(offsets.cpu(), want[1]), T
    assert torch.equal(rows.cpu()[want[0].reshape(-1).long(), 0], x.expand(T, K).reshape(-1)), T
"""


@pytest.mark.parametrize("E,K,sizes", [(256, 8, list(range(474, 481))), (320, 8, list(range(211, 217))), (360, 4, list(range(93, 103)))])
def test_sorts_around_48_KB_of_shared_memory(E, K, sizes):
    """What a launch may have without being allowed more counts its static arrays too.  In a process of its own, where no larger sort came before."""
    run = subprocess.run([sys.executable, "-c", SORTS % ((E, K, sizes),)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


THREADS = """
import sys
import threading
import torch
sys.path.insert(0, "tests")
import yamoe_b200
from test_gpu_token_sort import choices, places
sizes = [(40, 1024, 4), (900, 300, 4), (500, 1024, 8), (460, 512, 8), (8, 700, 2), (1000, 256, 4)]
inputs = [(torch.arange(T, dtype=torch.float32)[:, None].cuda(), choices(T, K, E, seed=T)) for T, E, K in sizes]
given = [idx.cuda() for _, idx in inputs]
streams = [torch.cuda.Stream() for _ in sizes]
torch.cuda.synchronize()
start, results, wrong = threading.Barrier(len(sizes)), [None] * len(sizes), []


def work(i):
    try:
        with torch.cuda.stream(streams[i]):
            start.wait(60)
            for _ in range(20):
                results[i] = yamoe_b200.sort_tokens(inputs[i][0], given[i], sizes[i][1])
    except Exception as e:
        wrong.append(e)


threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert not wrong, wrong
for (T, E, K), (_, idx), (rows, row_of, offsets) in zip(sizes, inputs, results):
    want = places(idx, E, None)
    assert torch.equal(row_of.cpu(), want[0]) and torch.equal(offsets.cpu(), want[1]), (T, E, K)
"""


def test_sorts_from_several_host_threads():
    """First calls of different sizes at the same time, each on a stream of its own."""
    run = subprocess.run([sys.executable, "-c", THREADS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr


# ---- 8-bit integers
def quantised_by_entry(x, batch, M, K, transpose):
    """yamoe_b200_int8_quantize itself: its status, codes and scales of `batch` matrices [M, K]."""
    from yamoe_b200 import _lib
    rows, cols = (K, M) if transpose else (M, K)
    ld = max(16, -(-cols // 16) * 16)
    q = torch.full((batch, rows, ld), 77, dtype=torch.int8, device="cuda")
    s = torch.full((batch, rows), -1.0, device="cuda")
    out = _lib.Int8Matrix(q=q.data_ptr(), scale=s.data_ptr(), ld=ld, q_batch=rows * ld, scale_row=1, scale_batch=rows)
    import ctypes
    status = _lib.lib().yamoe_b200_int8_quantize(x.data_ptr() or None, ctypes.byref(out), batch, M, K, int(transpose), 1 if x.dtype == BF16 else 0,
                                                 torch.cuda.current_stream().cuda_stream)
    return status, q, s


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,rows", [(1, 5), (3, 200)])
def test_rows_without_values_through_the_C_entry(batch, rows, dtype, transpose):
    """Rows of no values have the scale of a row of zeros and no codes; those of x^T are the columns of an x without rows."""
    M, K = (0, rows) if transpose else (rows, 0)
    status, q, s = quantised_by_entry(torch.empty(batch, M, K, dtype=dtype, device="cuda"), batch, M, K, transpose)
    assert status == 0
    assert bool((s == 2.0 ** -100 / 127).all()) and bool((q == 77).all())
    assert torch.ones(4, device="cuda").sum().item() == 4          # nothing is left for the next call to report


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("B", [65535, 65536, 140001])
def test_more_matrices_than_a_grid_has_rows(B, transpose):
    import yamoe_b200
    x = torch.randn(B, 2, 3, generator=torch.Generator().manual_seed(B)).cuda()
    x[-1, 0, 0], x[0, 1, 1] = 40.0, float("inf")
    q, s = yamoe_b200.quantize_int8(x, transpose)
    flat = (x.transpose(1, 2) if transpose else x).reshape(-1, 2 if transpose else 3)
    want_q, want_s = yamoe_b200.quantize_int8(flat)
    assert torch.equal(q.reshape(flat.shape), want_q)
    assert torch.equal(s.reshape(-1).nan_to_num(-1.0), want_s.nan_to_num(-1.0)) and bool(s.isnan().any())


def test_numbers_of_matrices_that_are_refused():
    import ctypes
    from yamoe_b200 import _lib
    out = ctypes.byref(_lib.Int8Matrix(q=4096, scale=4096, ld=16, q_batch=32, scale_row=1, scale_batch=2))
    assert _lib.lib().yamoe_b200_int8_quantize(4096, out, 1 << 31, 2, 3, 0, 1, None) == -5


@pytest.mark.parametrize("M", [6, 200])
@pytest.mark.parametrize("table", [[0, 4, 2 ** 40], [-(2 ** 35), 3, 2 ** 31], [0, 2 ** 32, 2 ** 32 + 5], [2 ** 33] * 3, [1, 3, 5]])
def test_offsets_of_64_bits(M, table):
    """They are kept within the rows as the numbers that they are."""
    import yamoe_b200
    gen = torch.Generator().manual_seed(1)
    a, b = torch.randint(-127, 128, (M, 64), generator=gen), torch.randint(-127, 128, (2, 40, 64), generator=gen)
    off = [min(max(o, 0), M) for o in table]
    want = torch.zeros(M, 40)
    for e in range(2):
        want[off[e] : off[e + 1]] = (a[off[e] : off[e + 1]] @ b[e].T).float()
    for given in (torch.tensor(table), torch.tensor(table).repeat_interleave(2)[::2]):
        got = yamoe_b200.int8_mm(a.to(torch.int8).cuda(), torch.ones(M, device="cuda"), b.to(torch.int8).cuda(), torch.ones(2, 40, device="cuda"), F32, given.cuda())
        assert torch.equal(got.cpu(), want)


# ---- derivatives that the integer operators do not have
def integer_calls():
    import yamoe_b200
    a, b = torch.ones(4, 32, dtype=torch.int8, device="cuda"), torch.ones(5, 32, dtype=torch.int8, device="cuda")
    sa, sb = torch.ones(4, device="cuda"), torch.ones(5, device="cuda")
    x = torch.randn(4, 32, generator=torch.Generator().manual_seed(0)).cuda()
    return {"quantize": (x, lambda t: yamoe_b200.quantize_int8(t)[1]), "quantize_transposed": (x, lambda t: yamoe_b200.quantize_int8(t, True)[1]),
            "a_scale": (sa, lambda t: yamoe_b200.int8_mm(a, t, b, sb, F32)), "b_scale": (sb, lambda t: yamoe_b200.int8_mm(a, sa, b, t, F32)),
            "chain": (x, lambda t: yamoe_b200.int8_mm(*yamoe_b200.quantize_int8(t), b, sb))}


CALLS = ["quantize", "quantize_transposed", "a_scale", "b_scale", "chain"]


@pytest.mark.parametrize("name", CALLS)
def test_integers_have_no_gradient(name):
    """The result is that of a tensor that wants none; a backward pass that reaches the operator raises, and one that does not goes through."""
    leaf, call = integer_calls()[name]
    want = call(leaf)
    assert not want.requires_grad
    leaf = leaf.clone().requires_grad_(True)
    out = call(leaf)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.float().sum().backward()
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad((call(leaf).float().sum() + leaf.sum()), leaf)
    assert leaf.grad is None
    (g,) = torch.autograd.grad(call(leaf).detach().float().sum() + leaf.sum(), leaf)
    assert torch.equal(g, torch.ones_like(leaf))
    with torch.no_grad():
        assert not call(leaf).requires_grad
    with torch.inference_mode():
        assert torch.equal(call(leaf), want)


@pytest.mark.parametrize("name", CALLS)
def test_integers_refuse_forward_mode(name):
    import torch.autograd.forward_ad as fwAD
    leaf, call = integer_calls()[name]
    with fwAD.dual_level():
        for t in (fwAD.make_dual(leaf, torch.ones_like(leaf)), fwAD.make_dual(leaf.clone().requires_grad_(True), torch.ones_like(leaf))):
            with pytest.raises(RuntimeError, match="forward"):
                call(t)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
                call(t)
