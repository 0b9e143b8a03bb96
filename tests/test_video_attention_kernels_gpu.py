"""Every kernel that the rules of attention over chosen blocks can pick, on small shapes with many workgroups, against the plain 64-bit form.

A clip runs kernels that a handful of short sequences never reaches: 128-row query blocks on a full chip, 64- and 128-key blocks with all their
rows in one wave, lists and query blocks in more than one round. Each case below names the kernel that it is there for, and the test fails if
another one ran."""
import itertools

import pytest
import torch

import video_attention_ref as R
from sfast.hip import functional as F
from sfast.hip import lib as L
from test_video_attention_gpu import BF16, F16, F32, lens, make, randn

pytestmark = pytest.mark.gpu

# (kernel: padded head dim, rows of a workgroup, LDS stages, packed), case: B, Sq, Sk, H, Hk, D, block_q, block_k, topk, key lengths, query lengths
FORWARD = [
    ((64, 32, 2, True), (2, 1, 700, 8, 2, 40, 128, 64, 6, [700, 333], None)),
    ((64, 64, 2, True), (2, 16, 700, 6, 2, 64, 64, 128, 3, [700, 333], [16, 5])),
    ((64, 64, 4, False), (1, 300, 700, 4, 2, 64, 64, 64, 5, None, [290])),
    ((64, 128, 4, False), (1, 300, 700, 4, 2, 40, 128, 64, 5, None, [290])),
    ((64, 64, 2, False), (1, 900, 900, 24, 24, 64, 64, 64, 3, [870], None)),
    ((64, 128, 2, False), (2, 900, 900, 24, 24, 64, 128, 64, 3, [900, 555], [900, 700])),
    ((64, 128, 2, False), (2, 900, 900, 24, 12, 40, 128, 128, 3, [900, 555], None)),
    ((128, 32, 2, True), (2, 1, 700, 8, 2, 128, 128, 64, 6, [700, 333], None)),
    ((128, 64, 2, True), (2, 16, 700, 6, 2, 96, 64, 128, 3, [700, 333], [16, 5])),
    ((128, 64, 4, False), (1, 300, 700, 4, 2, 128, 64, 64, 5, None, [290])),
    ((128, 128, 4, False), (1, 300, 700, 4, 2, 80, 128, 64, 5, None, [290])),
    ((128, 64, 2, False), (1, 900, 900, 24, 24, 128, 64, 64, 3, [870], None)),
    ((128, 128, 2, False), (2, 900, 900, 24, 24, 128, 128, 64, 3, [900, 555], [900, 700])),
    ((128, 128, 2, False), (2, 900, 900, 24, 12, 80, 128, 128, 3, [900, 555], None)),
]

# (kernels: padded head dim, keys of a workgroup, waves that share a tile's rows, single rounding), case
BACKWARD = [
    ((64, 64, 2, False), (2, 900, 900, 24, 24, 64, 128, 64, 3, [900, 555], [900, 700])),
    ((64, 64, 2, False), (1, 200, 700, 4, 2, 40, 64, 128, 3, [650], None)),
    ((64, 64, 2, True), (2, 100, 900, 24, 24, 40, 128, 64, 3, [900, 555], None)),
    ((64, 64, 2, True), (2, 64, 900, 4, 2, 64, 64, 128, 3, None, [64, 7])),
    ((64, 128, 1, False), (2, 900, 900, 24, 24, 64, 128, 128, 3, [900, 555], [900, 700])),
    ((64, 128, 1, False), (2, 300, 1100, 24, 24, 40, 64, 128, 4, None, None)),
    ((64, 128, 1, True), (2, 100, 900, 24, 24, 64, 128, 128, 3, [900, 555], None)),
    ((64, 128, 1, True), (2, 64, 900, 24, 24, 64, 64, 128, 3, None, [64, 9])),
    ((128, 64, 1, False), (2, 900, 900, 24, 24, 128, 128, 64, 3, [900, 555], [900, 700])),
    ((128, 64, 1, False), (2, 300, 900, 24, 12, 80, 64, 64, 3, None, None)),
    ((128, 64, 1, True), (2, 100, 900, 24, 24, 96, 128, 64, 3, [900, 555], None)),
    ((128, 64, 1, True), (2, 64, 900, 24, 24, 128, 64, 64, 3, None, [64, 9])),
    ((128, 64, 2, False), (1, 300, 700, 4, 2, 128, 128, 64, 5, [650], [290])),
    ((128, 64, 2, False), (1, 300, 700, 4, 2, 80, 64, 128, 5, None, None)),
    ((128, 64, 2, True), (1, 100, 700, 4, 2, 128, 128, 128, 3, [650], None)),
    ((128, 64, 2, True), (1, 64, 700, 4, 2, 96, 64, 64, 3, None, [60])),
    ((128, 128, 1, False), (2, 900, 900, 24, 24, 128, 128, 128, 3, [900, 555], [900, 700])),
    ((128, 128, 1, False), (2, 300, 1100, 24, 12, 80, 64, 128, 4, None, None)),
    ((128, 128, 1, True), (2, 100, 900, 24, 24, 96, 128, 128, 3, [900, 555], None)),
    ((128, 128, 1, True), (2, 64, 900, 24, 24, 128, 64, 128, 3, None, [64, 9])),
]


def check_forward(case, q, k, v, blocks, want):
    bq, bk, kl, ql = case[6], case[7], case[9], case[10]
    out, lse = F.block_sparse_attention(q, k, v, blocks, bq, bk, lens(kl), lens(ql))
    name = L.last_kernel()
    R.check("out", out, *want["out"])
    R.check("lse", lse, *want["lse"])
    return name, out, lse


def gradients(case, q, k, v, blocks, go, gl):
    """The gradients through autograd, and again by the call that a captured step makes (whose kernels' names this thread sees)."""
    bq, bk, kl, ql = case[6], case[7], case[9], case[10]
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out, lse = F.block_sparse_attention(*leaves, blocks, bq, bk, lens(kl), lens(ql))
    finite = torch.isfinite(lse.detach())
    got = torch.autograd.grad((out, torch.where(finite, lse, 0.0)), leaves, (go, gl))
    direct = F.block_sparse_attention_backward(go, torch.where(finite, gl, 0.0), q, k, v, blocks, out.detach(), lse.detach(), bq, bk, lens(kl), lens(ql))
    return out, got, direct, L.last_kernel()


def check_backward(case, dtype, blocks=None, seed=0):
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v, chosen = make(case, dtype, seed)
    blocks = chosen if blocks is None else blocks
    go, gl = randn((B, Sq, H, D), dtype, 77), randn((B, H, Sq), F32, 78)
    want = R.attention(q, k, v, blocks, bq, bk, kl, ql, None, go, gl)
    out, got, direct, name = gradients(case, q, k, v, blocks, go, gl)
    R.check("out", out.detach(), *want["out"])
    for n, g in zip(("dq", "dk", "dv"), got):
        R.check(n, g, *want[n])
    # without what out's rounding left, delta keeps that rounding's error: half a step of out a product (dV has no delta in it)
    assert torch.equal(direct[2], got[2])
    return name


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel, case", FORWARD)
def test_forward(kernel, case, dtype):
    q, k, v, blocks = make(case, dtype)
    name, _, _ = check_forward(case, q, k, v, blocks, R.attention(q, k, v, blocks, case[6], case[7], case[9], case[10]))
    dp, rows, stages, packed = kernel
    assert name.startswith(f"block_attn_fwd[DP={dp},rows={rows},stages={stages},") and name.endswith(",packed]") == packed, name


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel, case", BACKWARD)
def test_backward(kernel, case, dtype):
    name = check_backward(case, dtype)
    dp, keys, halves, fine = kernel
    assert name.startswith(f"block_attn_bwd[DP={dp},rows={case[6]},keys={keys},halves={halves},") and name.endswith(",fine]") == fine, name


def test_no_kernel_is_left_out():
    forward = set(itertools.product((64, 128), (64, 128), (2, 4), (False,))) | set(itertools.product((64, 128), (32, 64), (2,), (True,)))
    assert {kernel for kernel, _ in FORWARD} == forward
    dkv = {(64, 64, 2), (64, 128, 1), (128, 64, 1), (128, 64, 2), (128, 128, 1)}
    assert {kernel for kernel, _ in BACKWARD} == {k + (fine,) for k in dkv for fine in (False, True)}
    dq = set(itertools.product((64, 128), (64, 128), (False, True)))
    assert {(kernel[0], case[6], kernel[3]) for kernel, case in BACKWARD} == dq


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D, bq", [(64, 64), (128, 128)])
def test_a_list_longer_than_a_round_on_a_full_chip(D, bq, dtype):
    """More entries than a workgroup holds at a time (1024) where nothing is cut: dQ takes its list in rounds, the forward joins two parts."""
    H, nQ, nK, topk = 33, 8, 20, 1100
    case = (1, nQ * bq - 5, nK * 64 - 10, H, H, D, bq, 64, topk, None, None)
    blocks = torch.randint(-1, nK + 1, (1, H, nQ, topk), generator=torch.Generator().manual_seed(5), dtype=torch.int32).cuda()   # with repeats
    q, k, v, _ = make(case, dtype)
    name, _, _ = check_forward(case, q, k, v, blocks, R.attention(q, k, v, blocks, bq, 64))
    assert ",split=2]" in name, name
    name = check_backward(case, dtype, blocks)
    assert ",parts=1+1]" in name, name


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [(1, 19150, 640, 13, 13, 64, 64, 64, 6, None, [19140]), (1, 19150, 640, 26, 26, 64, 64, 64, 6, None, None),
                                  (1, 19150, 640, 13, 13, 128, 64, 64, 6, [630], None), (1, 19150, 1200, 26, 26, 96, 64, 128, 6, None, None)])
def test_more_query_blocks_than_a_round(case, dtype):
    """300 query blocks: dK and dV take their names (256 at a time) in two rounds."""
    name = check_backward(case, dtype)
    assert ",parts=1+1]" in name, name
