"""Attention over chosen blocks and rotary positions in the modes around them."""
import pytest
import torch

from sfast.hip import functional as F
from sfast.hip import lib as L
from test_video_attention_gpu import BF16, make, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H, D", [(24, 64), (12, 64), (24, 128), (12, 80)])
def test_batch_invariant_mode_on_whole_query_blocks(H, D, monkeypatch):
    """240 (120) workgroups a sample: one sample and the reference batch, or the reference batch and eight samples, lie on either side of 256."""
    B, S = 8, 1280
    q, k, v, blocks = make((B, S, S, H, H, D, 128, 64, 16, None, None), BF16, 2)
    go = randn(q.shape, BF16, 3)

    def rows(n):
        leaves = [t[:n].detach().requires_grad_() for t in (q, k, v)]
        out, lse = F.block_sparse_attention(*leaves, blocks[:n])
        return (out.detach(), lse.detach()) + torch.autograd.grad(out, leaves, go[:n])
    lib = L.load()
    monkeypatch.setenv("SFAST_BATCH_INVARIANT", "1")
    try:
        assert lib.sfast_hip_init() == 0
        whole = rows(B)
        for n in (1, 2, 3):
            for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), rows(n), whole):
                assert torch.equal(a, b[:n]), (n, name)
    finally:
        monkeypatch.undo()
        assert lib.sfast_hip_init() == 0
