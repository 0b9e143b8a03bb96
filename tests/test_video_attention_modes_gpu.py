"""Attention over chosen blocks and rotary positions in the modes around them, and what a turn leaves alone."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import video_attention_ref as R
from sfast.hip import functional as F
from sfast.hip import lib as L
from test_video_attention_gpu import BF16, F16, F32, grid, make, randn

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


def test_there_are_no_derivatives_in_forward_mode():
    """A tangent that is not carried on would count as zero."""
    q, k, v, blocks = make((1, 100, 300, 2, 2, 64, 128, 64, 3, None, None), BF16)
    pos = grid(1, 1, 300, 1, F32)
    out, lse = F.block_sparse_attention(q, k, v, blocks)
    calls = {
        "rotary, query": lambda d: F.rotary_nd(d(k), None, pos, [64]),
        "rotary, key": lambda d: F.rotary_nd(k, d(v), pos, [64]),
        "rotary, positions": lambda d: F.rotary_nd(k, v, d(pos), [64]),
        "means": lambda d: F.block_means(d(q), 64),
        "query": lambda d: F.block_sparse_attention(d(q), k, v, blocks),
        "key": lambda d: F.block_sparse_attention(q, d(k), v, blocks),
        "value": lambda d: F.block_sparse_attention(q, k, d(v), blocks),
        "backward, gradient": lambda d: F.block_sparse_attention_backward(d(out), None, q, k, v, blocks, out, lse),
        "backward, gradient of lse": lambda d: F.block_sparse_attention_backward(out, d(lse), q, k, v, blocks, out, lse),
        "backward, value": lambda d: F.block_sparse_attention_backward(out, None, q, k, d(v), blocks, out, lse),
    }
    for name, call in calls.items():
        with fwd.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
            call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
            raise AssertionError(name)
        call(lambda t: t)   # the same call without a tangent
    for f, x in ((lambda t: F.rotary_nd(t, None, pos, [64])[0], k), (lambda t: F.block_sparse_attention(t, k, v, blocks)[0], q)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        with fwd.dual_level(), pytest.raises(RuntimeError):
            f(fwd.make_dual(x.detach().requires_grad_(), torch.ones_like(x)))


def test_gradients_that_were_called_for_are_not_differentiated_again():
    """Leaves that want gradients go into the call as they are; only differentiating its results is refused."""
    q, k, v, blocks = make((1, 100, 300, 2, 2, 64, 128, 64, 3, None, None), BF16)
    out, lse = F.block_sparse_attention(q, k, v, blocks)
    want = F.block_sparse_attention_backward(out, None, q, k, v, blocks, out, lse)
    q.requires_grad_()
    got = F.block_sparse_attention_backward(out, None, q, k, v, blocks, out, lse)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="second derivative"):
        got[1].sum().backward()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D, sections", [(64, [16, 24]), (80, [30, 20]), (256, [128, 64]), (10, [2, 4])])
def test_elements_behind_the_sections_are_copied_bit_by_bit(D, sections, interleaved, dtype):
    """Infinities, NaN and negative zeros among them: a neighbour is not touched by them."""
    used = sum(sections)
    x = randn((2, 12, 3, D), dtype, 1)
    tail = x[..., used:]
    gen = torch.Generator().manual_seed(3)
    odd = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 0.0], dtype=dtype)
    pick = torch.randint(0, 10, tail.shape, generator=gen)
    tail.copy_(torch.where(pick < 5, odd[pick.clamp(max=4)], tail.cpu()))
    assert not torch.isfinite(x[..., used:]).all()
    bits = torch.int32 if dtype == F32 else torch.int16
    pos = grid(1, 3, 4, 2, F32, 3, 0.7)
    want, bound = R.rope(x[..., :used], pos, sections, 10000.0, interleaved)
    for a in F.rotary_nd(x, x, pos, sections, interleaved=interleaved):
        assert torch.equal(a[..., used:].contiguous().view(bits), x[..., used:].contiguous().view(bits))
        R.check("turned", a[..., :used], want, bound)
