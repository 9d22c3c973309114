"""Layouts of quantised matrices: what tensor maps cannot describe by their documented rules (a matrix pitch that is a whole number of
row pitches, and no less than the matrix's rows) is refused by the C entries and copied by the torch operators."""
import pytest
import torch

from test_fp8_cabi import BAD_ARG, BF16, lib, matrix  # noqa: F401

P = 4096


def codes(rows, **change):
    return matrix(**{**dict(ld=128, q_batch=rows * 128), **change})


@pytest.mark.parametrize("bad", [dict(q_batch=64 * 128 - 128), dict(q_batch=64 * 128 + 16), dict(ld=64 * 128, q_batch=128)])
def test_product(lib, bad):  # noqa: F811
    ws = lib.yamoe_b200_fp8_mm_workspace_bytes(2, 64, 64, 128)

    def call(a, b, batch):
        return lib.yamoe_b200_fp8_mm(a, b, 128, P, batch, 64, 64, 128, BF16, P, ws, None)
    assert call(codes(64, **bad), codes(64), 2) == call(codes(64), codes(64, **bad), 2) == BAD_ARG


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("by", [-128, 16])
def test_experts_and_layer(lib, which, by):  # noqa: F811
    T, H, E, K = 4, 128, 8, 2
    m = [codes(2 * H), codes(H)]
    m[which] = codes((2 * H, H)[which], q_batch=(2 * H, H)[which] * 128 + by)
    ws = lib.yamoe_b200_experts_fp8_workspace_bytes(T, H, E, K, BF16)
    assert lib.yamoe_b200_experts_fp8_forward(P, P, P, E, m[0], P, m[1], P, P, T, H, E, K, 4, BF16, P, ws, None) == BAD_ARG
    ws = lib.yamoe_b200_moe_layer_workspace_bytes(T, H, E, K)
    assert lib.yamoe_b200_moe_layer(P, P, None, None, m[0], P, None, m[1], P, P, P, T, H, E, K, 4, BF16, P, ws, None) == BAD_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("B,M,N,K", [(3, 70, 150, 256), (5, 1, 200, 136), (2, 33, 1, 64), (1, 40, 50, 208), (4, 129, 128, 200)])
def test_matrices_in_other_layouts(B, M, N, K):
    """Rows of the matrices among one another, every second row, overlapping matrices, one matrix for all."""
    import yamoe_b200
    gen = torch.Generator(device="cuda").manual_seed(B + M)
    a, b = [torch.randn(B, r, K, device="cuda", generator=gen).bfloat16() for r in (M, N)]
    (qa, sa), (qb, sb) = yamoe_b200.quantize_fp8(a), yamoe_b200.quantize_fp8(b, 128)
    want = yamoe_b200.fp8_mm(qa, sa, qb, sb)

    # memory for q's codes and a view of it
    layouts = {
        "rows among one another": lambda q: ((q.shape[1], B, 512), lambda r: r.transpose(0, 1)[:, :, :K]),
        "every second row": lambda q: ((B, 2 * q.shape[1] + 1, 256), lambda r: r[:, 1::2][:, :, :K]),
        "matrices part of a row more apart": lambda q: ((B, q.shape[1] * 256 + 48),
                                                        lambda r: r.as_strided((B, q.shape[1], K), (q.shape[1] * 256 + 48, 256, 1)))}
    for name, layout in layouts.items():
        views = []
        for q in (qa, qb):
            shape, of = layout(q)
            room = torch.zeros(shape, dtype=torch.uint8, device="cuda")
            of(room).copy_(q.contiguous().view(torch.uint8))
            views.append(of(room.view(torch.float8_e4m3fn)))
        assert torch.equal(yamoe_b200.fp8_mm(views[0], sa, views[1], sb), want), name
    same = yamoe_b200.fp8_mm(qa, sa, qb[:1].expand(B, N, K), sb[:1].expand(B, *sb.shape[1:]))
    for i in range(B):
        assert torch.equal(same[i], yamoe_b200.fp8_mm(qa[i], sa[i], qb[0], sb[0]))
