"""Quantisation of rows whose length is near 2^31, where offsets and the rounding up of sizes pass 31 bits."""
import pytest
import torch

from test_gpu_fp8 import quantise_ref, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [2 ** 31 - 8, 2 ** 31 - 1024, 2 ** 31 - 1])
def test_two_rows(K):
    import yamoe_b200
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.zeros(2, K, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(1)
    last = (K - 1) // 128 * 128
    spots = sorted({0, 1024, (1 << 30) - 128, 1 << 30, K // 2048 * 1024, last - 1024, last - 128, last})
    for m in range(2):
        for k in spots:
            n = min(128, K - k)
            x[m, k:k + n] = torch.randn(n, generator=gen).bfloat16()
    q, s = yamoe_b200.quantize_fp8(x)
    assert q.shape == x.shape and s.shape == (2, -(-K // 128))
    found = 0
    for m in range(2):
        for k in spots:
            rq, rs = quantise_ref(x[m:m + 1, k:k + 128], 1)
            assert same(q[m:m + 1, k:k + 128], rq) and same(s[m:m + 1, k // 128:k // 128 + 1], rs), (m, k)
            found += int((rq.view(torch.uint8) != 0).sum())
    # all other codes are zero and all other scales the least one
    assert sum(int(torch.count_nonzero(part)) for m in range(2) for part in q.view(torch.uint8)[m].split(1 << 28)) == found
    least = torch.full((), 2.0 ** -100) / torch.full((), 448.0)
    assert int((s != least.cuda()).sum()) == 2 * len(spots)
