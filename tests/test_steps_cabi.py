"""C entry points of the expert layer's steps: refusals that need no GPU."""
import ctypes

import pytest

OK, BAD_ARG, WORKSPACE, DTYPE, UNSUPPORTED = 0, -1, -2, -3, -5
F32, BF16 = 0, 1
P = 4096                                     # an address that would pass


@pytest.fixture(scope="module")
def lib():
    from yamoe_b200 import build
    build.build()
    from yamoe_b200 import _lib
    return _lib.lib()


def matrix(**change):
    from yamoe_b200 import _lib
    good = dict(q=P, scale=P, ld=128, q_batch=128 * 64, scale_row=1, scale_batch=64)
    return ctypes.byref(_lib.Int8Matrix(**{**good, **change}))


def test_sort_refusals(lib):
    f, n = lib.yamoe_b200_sort_tokens, lib.yamoe_b200_sort_tokens_workspace_bytes
    T, H, E, K = 16, 64, 8, 2
    assert 0 < n(T, E, K) <= n(1 << 20, E, K) and n(0, E, K) > 0
    for bad in ((-1, E, K), (T, 0, K), (T, 1025, K), (T, E, -1), (1 << 29, E, 2), (1 << 40, E, 1)):
        assert n(*bad) == 0, bad

    def call(x=P, idx=P, rows=P, row_of=P, offsets=P, t=T, h=H, e=E, k=K, cap=-1, dtype=BF16, work=P, size=n(T, E, K)):
        return f(x, idx, rows, row_of, offsets, t, h, e, k, cap, dtype, work, size, None)
    assert call(dtype=2) == DTYPE
    for bad in (dict(x=None), dict(idx=None), dict(rows=None), dict(row_of=None), dict(offsets=None), dict(t=-1), dict(h=-1), dict(e=0),
                dict(k=-1), dict(x=P + 1), dict(rows=P + 1), dict(dtype=F32, x=P + 2), dict(idx=P + 4), dict(row_of=P + 2), dict(offsets=P + 1)):
        assert call(**bad) == BAD_ARG, bad
    for bad in (dict(e=1025), dict(t=1 << 30), dict(t=1 << 40), dict(h=1 << 41), dict(cap=1 << 31), dict(cap=1 << 28)):
        assert call(**bad) == UNSUPPORTED, bad
    assert call(work=None) == call(work=P + 128) == call(size=n(T, E, K) - 1) == WORKSPACE


def test_combine_refusals(lib):
    f = lib.yamoe_b200_combine_tokens
    T, H, E, K, R = 16, 64, 8, 2, 32

    def call(rows=P, r=R, row_of=P, w=P, wd=BF16, idx=None, out=P, t=T, h=H, e=E, k=K, dtype=BF16):
        return f(rows, r, row_of, w, wd, idx, out, t, h, e, k, dtype, None)
    assert call(dtype=3) == call(wd=7) == call(dtype=F32, wd=BF16) == DTYPE
    for bad in (dict(rows=None), dict(row_of=None), dict(out=None), dict(t=-1), dict(r=-1), dict(h=-1), dict(k=-1), dict(rows=P + 1),
                dict(row_of=P + 2), dict(w=P + 1), dict(wd=F32, w=P + 2), dict(idx=P + 4), dict(out=P + 1), dict(dtype=F32, wd=F32, out=P + 2)):
        assert call(**bad) == BAD_ARG, bad
    assert call(t=1 << 30) == call(r=1 << 31) == call(h=1 << 32) == call(t=1 << 40) == UNSUPPORTED
    assert call(t=0, rows=None, row_of=None, out=None) == call(h=0, rows=None, out=None) == OK


def test_combine_backward_refusals(lib):
    f, n = lib.yamoe_b200_combine_tokens_backward, lib.yamoe_b200_combine_tokens_backward_workspace_bytes
    T, H, E, K, R = 16, 64, 8, 2, 32
    assert n(R, T, K) >= 4 * (R + T * K) and n(-1, T, K) == n(R, -1, K) == n(R, T, -1) == n(R, 1 << 30, 2) == 0

    def call(d=P, rows=P, r=R, row_of=P, w=P, wd=BF16, idx=None, dr=P, dw=P, t=T, h=H, e=E, k=K, dtype=BF16, work=P, size=n(R, T, K)):
        return f(d, rows, r, row_of, w, wd, idx, dr, dw, t, h, e, k, dtype, work, size, None)
    assert call(dtype=3) == call(wd=7) == DTYPE
    for bad in (dict(d=None), dict(d=P + 1), dict(rows=None), dict(row_of=None), dict(w=None), dict(dr=P + 1), dict(dw=P + 1), dict(r=-1),
                dict(t=-1), dict(idx=P + 2)):
        assert call(**bad) == BAD_ARG, bad
    assert call(k=1025, t=1) == call(r=1 << 31) == call(t=1 << 30) == UNSUPPORTED
    assert call(work=None) == call(work=P + 64) == call(size=n(R, T, K) - 1) == WORKSPACE
    assert call(dr=None, dw=None) == OK


def test_quantize_refusals(lib):
    f = lib.yamoe_b200_int8_quantize
    assert f(P, matrix(), 1, 64, 128, 0, 2, None) == DTYPE
    assert f(P, matrix(), -1, 64, 128, 0, BF16, None) == f(P, None, 1, 64, 128, 0, BF16, None) == f(None, matrix(), 1, 64, 128, 0, BF16, None) == BAD_ARG
    assert f(P + 1, matrix(), 1, 64, 128, 0, BF16, None) == f(P + 2, matrix(), 1, 64, 128, 0, F32, None) == BAD_ARG
    for bad in (dict(q=0), dict(scale=0), dict(q=P + 4), dict(scale=P + 2), dict(ld=112), dict(ld=136)):
        assert f(P, matrix(**bad), 1, 64, 128, 0, BF16, None) == BAD_ARG, bad
    assert f(P, matrix(q_batch=100), 2, 64, 128, 0, BF16, None) == BAD_ARG
    assert f(P, matrix(ld=48), 1, 64, 128, 1, BF16, None) == BAD_ARG                # x^T has 64 columns
    assert f(None, matrix(), 1, 0, 128, 0, BF16, None) == f(None, None, 0, 64, 128, 0, BF16, None) == OK
    assert f(P, matrix(ld=1 << 33), 1, 64, 1 << 32, 0, BF16, None) == UNSUPPORTED


def test_product_refusals(lib):
    f, n = lib.yamoe_b200_int8_mm, lib.yamoe_b200_int8_mm_workspace_bytes
    ws = n(1, 64, 64, 128)
    assert 0 < ws <= 4096 and n(1, -1, 64, 128) == 0

    def call(a=matrix(), b=matrix(), offsets=None, out=P, batch=1, M=64, N=64, K=128, dtype=BF16, work=P, size=ws):
        return f(a, b, offsets, out, batch, M, N, K, dtype, work, size, None)
    assert call(dtype=7) == DTYPE
    for bad in (dict(M=-1), dict(out=None), dict(out=P + 1), dict(a=None), dict(b=None), dict(a=matrix(ld=64)), dict(b=matrix(q=P + 8)),
                dict(batch=2, b=matrix(q_batch=0)), dict(batch=2, a=matrix(q_batch=128 * 63)), dict(batch=2, b=matrix(q_batch=128 * 64 + 16)),
                dict(dtype=F32, out=P + 2), dict(offsets=P + 2), dict(a=matrix(scale=P + 1))):
        assert call(**bad) == BAD_ARG, bad
    assert call(work=None) == call(work=P + 1) == call(size=ws - 1) == WORKSPACE
    assert call(M=1 << 30) == call(K=1 << 17) == call(batch=1025, offsets=P) == UNSUPPORTED
    assert call(M=0, a=None, b=None, out=None, work=None) == OK


def test_glu_refusals(lib):
    fwd, bwd = lib.yamoe_b200_glu_forward, lib.yamoe_b200_glu_backward

    def forward(x=P, out=P, q=P, s=P, ld=128, M=4, N=64, dtype=BF16):
        return fwd(x, out, q, s, ld, M, N, dtype, None)

    def backward(d=P, q=P, s=P, ld=128, out=P, M=4, N=64, dtype=BF16):
        return bwd(d, q, s, ld, out, M, N, dtype, None)
    for f in (forward, backward):
        assert f(dtype=9) == DTYPE
        for bad in (dict(out=None), dict(out=P + 1), dict(q=P + 8), dict(s=None), dict(s=P + 1), dict(ld=112), dict(ld=136), dict(M=-1), dict(N=-1)):
            assert f(**bad) == BAD_ARG, bad
        assert f(N=1 << 30, ld=1 << 31) == UNSUPPORTED
        assert f(M=0, out=None) == f(N=0, out=None) == OK
    assert forward(x=None) == forward(x=P + 1) == backward(d=None) == backward(q=None) == BAD_ARG


def test_operators_need_the_binding():
    """Without the C++ binding the operators exist and say what they need."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import yamoe_b200\nfor n in ('sort_tokens', 'combine_tokens', 'quantize_int8', 'int8_mm', 'glu_fp8'):\n"
            "    try:\n        getattr(yamoe_b200, n)(1)\n    except RuntimeError as e:\n        print(e)\n")
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         env=dict(os.environ, YAMOE_B200_PY_BINDING="1"), timeout=300)
    assert out.returncode == 0 and out.stdout.count("C++ binding") == 5, out.stdout + out.stderr
