"""C entry points of the 8-bit operators and of the layer for a few tokens: refusals that need no GPU."""
import ctypes

import pytest

OK, BAD_ARG, WORKSPACE, DTYPE, UNSUPPORTED = 0, -1, -2, -3, -5
F32, BF16 = 0, 1


@pytest.fixture(scope="module")
def lib():
    from yamoe_b200 import build
    build.build()
    from yamoe_b200 import _lib
    return _lib.lib()


def matrix(**change):
    from yamoe_b200 import _lib
    good = dict(q=4096, scale=4096, ld=128, q_batch=128 * 64, scale_row=1, scale_group=64, scale_batch=64)
    return ctypes.byref(_lib.Fp8Matrix(**{**good, **change}))


def test_quantize_refusals(lib):
    f = lib.yamoe_b200_fp8_quantize
    assert f(4096, matrix(), None, 1, 64, 128, 1, 2, None) == DTYPE
    assert f(4096, matrix(), None, 1, 64, 128, 64, BF16, None) == BAD_ARG           # groups of 1 or 128 rows
    assert f(4096, None, None, 1, 64, 128, 1, BF16, None) == BAD_ARG                # no output
    assert f(None, matrix(), None, 1, 64, 128, 1, BF16, None) == BAD_ARG
    assert f(4097, matrix(), None, 1, 64, 128, 1, BF16, None) == BAD_ARG            # odd address of bf16
    assert f(4096, matrix(), None, -1, 64, 128, 1, BF16, None) == BAD_ARG
    for bad in (dict(q=0), dict(scale=0), dict(q=4100), dict(scale=4098), dict(ld=112), dict(ld=136)):
        assert f(4096, matrix(**bad), None, 1, 64, 128, 1, BF16, None) == BAD_ARG, bad
    assert f(4096, matrix(q_batch=100), None, 2, 64, 128, 1, BF16, None) == BAD_ARG
    assert f(4096, None, matrix(ld=48), 1, 64, 128, 128, F32, None) == BAD_ARG      # x^T has 64 columns
    assert f(None, matrix(), None, 1, 0, 128, 1, BF16, None) == OK                  # nothing to do
    assert f(4096, matrix(ld=1 << 33), None, 1, 64, 1 << 32, 1, BF16, None) == UNSUPPORTED


def test_product_refusals(lib):
    f, n = lib.yamoe_b200_fp8_mm, lib.yamoe_b200_fp8_mm_workspace_bytes
    ws = n(1, 64, 64, 128)
    assert 0 < ws <= 4096 and n(1, -1, 64, 128) == 0

    def call(a=matrix(), b=matrix(), block=128, out=4096, batch=1, M=64, N=64, K=128, dtype=BF16, work=4096, size=ws):
        return f(a, b, block, out, batch, M, N, K, dtype, work, size, None)
    assert call(dtype=7) == DTYPE
    for bad in (dict(block=2), dict(M=-1), dict(out=None), dict(out=4097), dict(a=None), dict(b=None), dict(a=matrix(ld=64)),
                dict(b=matrix(q=4104)), dict(batch=2, b=matrix(q_batch=0)), dict(dtype=F32, out=4098)):
        assert call(**bad) == BAD_ARG, bad
    assert call(work=None) == call(work=4097) == call(size=ws - 1) == WORKSPACE
    assert call(M=1 << 30) == UNSUPPORTED
    assert call(M=0, a=None, b=None, out=None, work=None) == OK


def test_experts_refusals(lib):
    f, n = lib.yamoe_b200_experts_fp8_forward, lib.yamoe_b200_experts_fp8_workspace_bytes
    T, H, E, K = 16, 128, 8, 2
    ws = n(T, H, E, K, BF16)
    assert ws > 0 and n(T, H, E, K, F32) >= ws
    assert n(T, 130, E, K, BF16) == n(T, H, 2000, K, BF16) == n(T, H, E, K, 5) == 0

    def call(x=4096, cols=E, gate_up=matrix(), down=matrix(), cap=4, h=H, dtype=BF16, work=4096, size=ws, out=4096, experts=E):
        return f(x, 4096, 4096, cols, gate_up, 4096, down, 4096, out, T, h, experts, K, cap, dtype, work, size, None)
    assert call(dtype=9) == DTYPE
    for bad in (dict(x=None), dict(x=4104), dict(cols=3), dict(gate_up=None), dict(down=matrix(ld=64)), dict(cap=-1), dict(h=132),
                dict(out=None), dict(out=4104), dict(gate_up=matrix(q_batch=8))):
        assert call(**bad) == BAD_ARG, bad
    assert call(work=None) == call(work=4128) == call(size=ws - 1) == WORKSPACE
    assert call(experts=2000, cols=K) == UNSUPPORTED


def test_layer_refusals(lib):
    f, n = lib.yamoe_b200_moe_layer, lib.yamoe_b200_moe_layer_workspace_bytes
    T, H, E, K = 4, 128, 8, 2
    ws = n(T, H, E, K)
    assert ws > 0 and n(32, H, E, 8) > 0
    for bad in ((33, H, E, K), (32, H, 16, 9), (T, 100, E, K), (T, H, E, 9), (T, H, 1025, K), (T, H, 64, 33), (T, 1 << 17, E, K)):
        assert n(*bad) == 0, bad

    def call(x=4096, wr=4096, gu=4096, gu8=None, dn=4096, dn8=None, bias=4096, t=T, h=H, e=E, k=K, cap=4, dtype=BF16, work=4096,
             size=ws, out=4096, scores=4096):
        return f(x, wr, None, gu, gu8, bias, dn, dn8, bias, out, scores, t, h, e, k, cap, dtype, work, size, None)
    assert call(dtype=F32) == DTYPE
    for bad in (dict(x=None), dict(x=4104), dict(wr=None), dict(gu=None), dict(dn=None), dict(gu8=matrix()), dict(dn8=matrix()),
                dict(gu=None, dn=None, gu8=matrix(ld=64), dn8=matrix()), dict(bias=None), dict(bias=4097), dict(cap=-1), dict(k=9),
                dict(h=100), dict(out=None), dict(scores=None), dict(t=-1)):
        assert call(**bad) == BAD_ARG, bad
    assert call(t=33) == call(e=2000) == UNSUPPORTED
    assert call(work=None) == call(work=4128) == call(size=ws - 1) == WORKSPACE
    assert call(t=0, x=None, out=None, scores=None) == OK


def test_operators_need_the_binding():
    """Without the C++ binding the operators exist and say what they need."""
    import subprocess
    import sys
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = "import torch, yamoe_b200\ntry:\n    yamoe_b200.fp8_mm(1)\nexcept RuntimeError as e:\n    print(e)\n"
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         env=dict(os.environ, YAMOE_B200_PY_BINDING="1"), timeout=300)
    assert out.returncode == 0 and "C++ binding" in out.stdout, out.stdout + out.stderr
