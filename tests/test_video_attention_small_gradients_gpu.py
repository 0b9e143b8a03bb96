"""Gradients of any magnitude: they are linear in what comes in. bf16 has fp32's range, so a power of two changes nothing but exponents."""
import pytest
import torch

import video_attention_ref as R
from sfast.hip import functional as F
from test_video_attention_gpu import BF16, F32, lens, make, randn

pytestmark = pytest.mark.gpu

CASES = [
    # one query block (a single rounding), a clip's shape in small, blocks of 128 keys, a padded batch
    (2, 60, 900, 4, 2, 64, 64, 64, 6, None, None), (1, 300, 900, 4, 2, 64, 128, 64, 6, None, None), (2, 200, 700, 4, 2, 128, 64, 128, 4, [700, 300], [200, 60]),
    (2, 900, 900, 24, 24, 96, 128, 64, 3, None, None),
]


def run(case, q, k, v, blocks, go, gl):
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out, lse = F.block_sparse_attention(*leaves, blocks, bq, bk, lens(kl), lens(ql))
    if go is None:
        return torch.autograd.grad(lse, leaves, torch.where(torch.isfinite(lse.detach()), gl, 0.0))
    finite = torch.isfinite(lse.detach())
    return torch.autograd.grad((out, torch.where(finite, lse, 0.0)), leaves, (go, gl))


@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("power", [20, 30, 60])
@pytest.mark.parametrize("case", CASES)
def test_gradients_of_a_small_loss(case, power, alone):
    """The mean over 10^8 elements gives gradients of 2^-27 and below. `alone`: lse carries the gradient alone."""
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v, blocks = make(case, BF16)
    go, gl = None if alone else randn((B, Sq, H, D), BF16, 77), randn((B, H, Sq), F32, 78)
    s = 2.0 ** -power
    got = run(case, q, k, v, blocks, None if alone else go * s, gl * s)
    small = torch.zeros((B, Sq, H, D), dtype=BF16, device="cuda") if alone else go * s
    want = R.attention(q, k, v, blocks, bq, bk, kl, ql, None, small, gl * s)
    for name, g, whole in zip(("dq", "dk", "dv"), got, run(case, q, k, v, blocks, go, gl)):
        R.check(name, g, *want[name])
        assert torch.equal(g, whole * s), f"{name} is not linear"
