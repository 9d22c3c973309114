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
