"""Rotary positions over several axes, block means, the choice of key blocks and attention over chosen blocks on the MI355X, against plain
64-bit forms (video_attention_ref.py) with bounds that count the roundings."""
import math

import pytest
import torch

import sfast  # noqa: F401  registers the operators
import video_attention_ref as R
from sfast.hip import functional as F
from sfast.libs.xformers.sparse_attention import sparse_attention

pytestmark = pytest.mark.gpu
OPS, ATT = torch.ops.sfast, torch.ops.sfast_xformers
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def randn(shape, dtype, seed, spread=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).cuda()


def lens(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- rotary ----------------------------------------------------------------------------------------------------------------------------
def grid(t, y, x, axes, dtype=torch.int64, start=0, step=1.0):
    p = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(y), torch.arange(x), indexing="ij"), -1).reshape(-1, 3)
    p = torch.cat([p, p[:, :1]], 1)[:, :axes] + start
    return (p.double() * step if dtype.is_floating_point else p).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("case", [
    # B, (t, y, x), H, Hk, D, sections
    (1, (1, 1, 1), 1, 1, 2, [2]), (2, (3, 5, 7), 6, 2, 80, [16, 24, 24]), (1, (2, 16, 16), 24, 24, 128, [16, 56, 56]), (3, (1, 4, 33), 5, 5, 64, [22, 42]),
    (1, (4, 3, 2), 8, 1, 256, [64, 64, 64, 64]), (2, (1, 1, 77), 3, 3, 40, [40]), (1, (2, 3, 5), 2, 2, 96, [2, 6, 10, 14]), (1, (5, 1, 1), 20, 4, 128, [128]),
])
def test_rotary(case, interleaved, dtype):
    B, (t, y, x), H, Hk, D, sections = case
    S = t * y * x
    q, k = randn((B, S, H, D), dtype, 1), randn((B, S, Hk, D), dtype, 2)
    pos = grid(t, y, x, len(sections))
    qo, ko = OPS.rotary_embedding_nd(q, k, pos, sections, 10000.0, interleaved)
    for name, got, src in (("q", qo, q), ("k", ko, k)):
        R.check(name, got, *R.rope(src, pos, sections, 10000.0, interleaved))
        assert torch.equal(got[..., sum(sections):], src[..., sum(sections):])


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_positions_of_every_type_far_negative_and_per_sequence(ptype, interleaved):
    B, S, H, D, sections = 2, 30, 3, 64, [20, 20, 24]
    q, k = randn((B, S, H, D), F32, 3), randn((B, S, 1, D), F32, 4)
    pos = torch.stack([grid(2, 3, 5, 3, ptype, 0, 0.37), grid(2, 3, 5, 3, ptype, 1000000, 1.0)])
    pos[0] = -pos[0]
    qo, ko = OPS.rotary_embedding_nd(q, k, pos, sections, 500.0, interleaved)
    R.check("q", qo, *R.rope(q, pos, sections, 500.0, interleaved))
    R.check("k", ko, *R.rope(k, pos, sections, 500.0, interleaved))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotary_strides(interleaved, dtype):
    B, S, H, D, sections = 2, 21, 4, 64, [24, 40]
    pos = grid(1, 3, 7, 2)
    packed = randn((B, S, 3, H, D), dtype, 5)                       # views of a packed projection
    heads_first = randn((B, H, S, D), dtype, 6).transpose(1, 2)     # [B, H, S, D] in memory
    shifted = randn((B * S * H * D + 1,), dtype, 7)[1:].view(B, S, H, D)  # an odd address
    odd_rows = randn((B, S, H, D + 1), dtype, 8)[..., :D]           # odd strides
    other = randn((B, D, S, H), dtype, 9).permute(0, 2, 3, 1)       # head dim not innermost
    wide_pos = torch.cat([pos, pos], 1)[:, ::2]
    for x in (packed[:, :, 0], heads_first, shifted, odd_rows, other, packed[:, :, 1].expand(B, S, H, D), packed[:1, :, 2].expand(B, S, H, D)):
        qo, ko = OPS.rotary_embedding_nd(x, packed[:, :, 2], pos, sections, 10000.0, interleaved)
        R.check("q", qo, *R.rope(x, pos, sections, 10000.0, interleaved))
        R.check("k", ko, *R.rope(packed[:, :, 2], pos, sections, 10000.0, interleaved))
    got = OPS.rotary_embedding_nd(heads_first, heads_first, wide_pos, sections, 10000.0, interleaved)[0]
    R.check("strided positions", got, *R.rope(heads_first, wide_pos, sections, 10000.0, interleaved))


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_gradient_is_the_turn_back(interleaved):
    B, S, H, Hk, D, sections = 2, 12, 4, 2, 48, [8, 16, 20]
    pos = grid(1, 3, 4, 3, torch.float32, 5, 0.7)
    q, k = randn((B, S, H, D), F32, 1).requires_grad_(), randn((B, S, Hk, D), F32, 2).requires_grad_()
    gq, gk = randn((B, S, H, D), F32, 3), randn((B, S, Hk, D), F32, 4)
    qo, ko = OPS.rotary_embedding_nd(q, k, pos, sections, 10000.0, interleaved)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk), retain_graph=True)
    R.check("dq", dq, *R.rope(gq, pos, sections, 10000.0, interleaved, inverse=True))
    R.check("dk", dk, *R.rope(gk, pos, sections, 10000.0, interleaved, inverse=True))
    dk_only, = torch.autograd.grad(ko, k, gk, retain_graph=True)   # only one of the two results is used
    assert torch.equal(dk_only, dk)
    dq_only, = torch.autograd.grad(qo, q, gq)
    assert torch.equal(dq_only, dq)
    # differences: the operator is linear, so a difference quotient has rounding errors only
    e = randn((B, S, H, D), F32, 5)
    plus, minus = [OPS.rotary_embedding_nd((q + s * e).detach(), k.detach(), pos, sections, 10000.0, interleaved)[0].double() for s in (1, -1)]
    lhs, rhs = ((plus - minus) / 2 * gq.double()).sum(), (dq.double() * e.double()).sum()
    assert abs(lhs - rhs) <= 16 * R.U32 * (e.abs().double() * gq.abs().double()).sum() * 4


def test_rotary_one_tensor_and_empty():
    pos = grid(1, 1, 6, 1)
    q = randn((1, 6, 2, 32), BF16, 1)
    got, none = F.rotary_nd(q, None, pos, [32])
    assert none is None
    R.check("q", got, *R.rope(q, pos, [32], 10000.0, True))
    a, b = OPS.rotary_embedding_nd(q[:, :0], q[:, :0], pos[:0], [32])
    assert a.shape == (1, 0, 2, 32) and b.shape == (1, 0, 2, 32)


# ---- block means -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("case", [
    # B, S, H, D, block, lengths
    (1, 1, 1, 8, 64, None), (2, 64, 3, 64, 64, None), (2, 65, 3, 40, 64, [65, 1]), (3, 300, 2, 128, 128, [0, 129, 300]), (1, 1000, 5, 7, 33, None),
    (2, 129, 4, 96, 128, [128, -5]), (2, 200, 1, 12, 1, [200, 10000]), (1, 2500, 2, 64, 1024, [2049]),
])
def test_block_means(case, dtype):
    B, S, H, D, block, lengths = case
    x = randn((B, S, H, D), dtype, 1)
    if lengths is not None:
        for b, n in enumerate(lengths):
            x[b, max(0, min(n, S)):] = float("nan")   # behind the sequence: not read
    want = R.means(x, block, lengths)
    # one rounding to fp32; the 64-bit sums lose 2^-53 a step
    R.check("means", ATT.block_means(x, block, lens(lengths)), want, R.U32 * want.abs() + 2.0 ** -40)
    if lengths is not None:
        R.check("int64 lengths", ATT.block_means(x, block, lens(lengths).long()), want, R.U32 * want.abs() + 2.0 ** -40)


def test_block_means_strides():
    x = randn((2, 3, 100, 64), BF16, 1).transpose(1, 2)
    packed = randn((2, 100, 3, 4, 36), F16, 2)
    odd = randn((2 * 100 * 3 * 64 + 1,), BF16, 3)[1:].view(2, 100, 3, 64)
    for t in (x, packed[:, :, 1], odd, randn((2, 64, 100, 3), F16, 4).permute(0, 2, 3, 1), x[:1].expand(2, -1, -1, -1)):
        want = R.means(t, 64)
        R.check("means", ATT.block_means(t, 64), want, R.U32 * want.abs() + 2.0 ** -40)


# ---- choice of blocks --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("case", [
    # B, nQ, nK, H, Hk, D, topk, lengths (keys), block_k
    (1, 1, 1, 1, 1, 4, 1, None, 64), (2, 3, 5, 4, 2, 40, 2, [5 * 64, 65], 64), (1, 16, 64, 2, 2, 64, 64, None, 64), (1, 17, 65, 3, 1, 64, 7, None, 64),
    (2, 40, 129, 2, 1, 128, 16, [129 * 128, 0], 128), (1, 1, 256, 8, 2, 80, 31, None, 64), (1, 2, 257, 2, 2, 64, 300, [100 * 64 + 1], 64),
    (1, 33, 1025, 1, 1, 64, 100, None, 64), (2, 1, 2049, 2, 1, 64, 64, [2049 * 64, 700], 64), (1, 1, 9000, 1, 1, 32, 128, None, 128), (1, 5, 900, 6, 2, 128, 90, None, 64),
    (1, 2, 30000, 1, 1, 16, 5, None, 64), (1, 70, 8, 4, 4, 20, 3, None, 64),
])
def test_block_topk(case):
    B, nQ, nK, H, Hk, D, k, lengths, block_k = case
    qm, km = randn((B, nQ, H, D), F32, 1), randn((B, nK, Hk, D), F32, 2)
    if lengths is not None:
        for b, n in enumerate(lengths):
            km[b, -(-n // block_k):] = float("nan")   # behind the sequence: not read
    got = ATT.block_topk(qm, km, k, block_k, lens(lengths)).cpu()
    assert torch.equal(got, R.topk(qm, km, k, block_k, lengths))


def test_block_topk_ties_zeros_nan_and_infinities():
    qm = torch.zeros((1, 1, 1, 8), device="cuda")
    qm[..., 0] = 1.0

    def choose(values, k):
        km = torch.zeros((1, len(values), 1, 8), device="cuda")
        km[0, :, 0, 0] = torch.tensor(values, device="cuda")
        return ATT.block_topk(qm, km, k).flatten().tolist()

    inf, nan = math.inf, math.nan
    assert choose([1.0] * 100, 3) == [0, 1, 2]
    assert choose([0.0, -0.0, 0.0, -1.0, -0.0], 3) == [0, 1, 2]
    assert choose([-1.0, 2.0, 2.0, 3.0, 2.0], 3) == [1, 2, 3]
    assert choose([-3.0, -1.0, -2.0, -1.0], 2) == [1, 3]
    assert choose([nan, 5.0, nan, 6.0], 2) == [0, 2]          # (0 * nan in the other elements does not occur: they are zero)
    assert choose([5.0, nan, 6.0], 2) == [1, 2]
    for values in ([1e-300, 2e-300, 0.0], [2.0, 2.0 + 2.0 ** -22, 2.0]):
        assert choose(values, 1) == [max(range(3), key=lambda i: torch.tensor(values[i]).item())]
    # scores alike in their upper bits: 2^-22 apart in a product of two fp32 numbers, in every width of the search
    for n in (40, 200, 1000, 2000, 2049, 9000):
        qm2 = torch.full((1, 1, 1, 8), 1.0 + 2.0 ** -12, device="cuda")
        km = torch.full((1, n, 1, 8), 1.0, device="cuda")
        gen = torch.Generator().manual_seed(n)
        km[0, :, 0, 0] += (torch.randint(0, 4, (n,), generator=gen) * 2.0 ** -23).cuda()
        for k in (1, 7, n // 2):
            assert torch.equal(ATT.block_topk(qm2, km, k).cpu(), R.topk(qm2, km, k, 64))
    big = torch.zeros((1, 3000, 1, 8), device="cuda")          # sixteen waves, all alike, ties over the waves' borders
    assert ATT.block_topk(qm, big, 2500).flatten().tolist() == list(range(2500))


def test_block_topk_takes_strided_means_and_no_blocks():
    qm, km = randn((2, 4, 6, 32), F32, 1).transpose(1, 2), randn((2, 9, 3, 32), F32, 2)   # nQ = 6, H = 4
    km = km[:, :, :2]
    assert torch.equal(ATT.block_topk(qm, km, 3).cpu(), R.topk(qm, km, 3, 64))
    assert (ATT.block_topk(qm, km[:, :0], 3) == -1).all()
    assert ATT.block_topk(qm[:, :0], km, 3).shape == (2, 2, 0, 3)


# ---- attention over chosen blocks ----------------------------------------------------------------------------------------------------------
CASES = [
    # B, Sq, Sk, H, Hk, D, block_q, block_k, topk, key lengths, query lengths
    (1, 1, 1, 1, 1, 8, 64, 64, 1, None, None),
    (1, 1, 64, 1, 1, 64, 128, 64, 1, None, None),
    (2, 1, 1000, 8, 2, 128, 128, 64, 12, [1000, 130], None),
    (4, 1, 5000, 32, 8, 64, 64, 128, 30, [5000, 1, 0, 129], None),
    (1, 5, 3000, 12, 1, 128, 64, 64, 40, None, [4]),
    (1, 16, 777, 4, 2, 80, 128, 128, 5, None, None),
    (2, 64, 64, 2, 2, 64, 64, 64, 1, None, None),
    (2, 65, 63, 2, 1, 40, 64, 64, 1, [63, 5], [65, 64]),
    (1, 128, 129, 3, 3, 128, 128, 128, 2, None, None),
    (2, 300, 500, 6, 3, 80, 64, 64, 5, [500, 257], [300, 0]),
    (1, 513, 1029, 4, 2, 96, 128, 128, 4, None, None),
    (3, 200, 450, 2, 1, 64, 128, 64, 3, [450, 64, 0], [200, 199, 7]),
    (1, 1000, 1000, 2, 2, 64, 128, 64, 16, None, None),
    (1, 257, 4000, 1, 1, 128, 64, 128, 32, None, None),
    (1, 33, 2000, 1, 1, 16, 128, 64, 32, None, None),
]


def make(case, dtype, seed=0, spread=1.0):
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v = [randn(s, dtype, seed + i, spread) for i, s in enumerate(((B, Sq, H, D), (B, Sk, Hk, D), (B, Sk, Hk, D)))]
    blocks = R.choose(B, Hk, -(-Sq // bq), -(-Sk // bk), topk, torch.Generator().manual_seed(seed + 9))
    return q, k, v, blocks.cuda()


def attend(case, q, k, v, blocks, scale=None, grads=False, dtype=None):
    """Runs the case and checks every result against the plain form."""
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    if not grads:
        out, lse = ATT.block_sparse_attention(q, k, v, blocks, bq, bk, lens(kl), lens(ql), scale)
        want = R.attention(q, k, v, blocks, bq, bk, kl, ql, scale)
        R.check("out", out, *want["out"])
        R.check("lse", lse, *want["lse"])
        return out, lse
    go, gl = randn((B, Sq, H, D), q.dtype, 77), randn((B, H, Sq), F32, 78)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out, lse = ATT.block_sparse_attention(*leaves, blocks, bq, bk, lens(kl), lens(ql), scale)
    want = R.attention(q, k, v, blocks, bq, bk, kl, ql, scale, go, gl)
    finite = torch.isfinite(lse.detach())
    got = torch.autograd.grad((out, torch.where(finite, lse, 0.0)), leaves, (go, gl))
    R.check("out", out.detach(), *want["out"])
    for name, g in zip(("dq", "dk", "dv"), got):
        assert g.dtype == q.dtype
        R.check(name, g, *want[name])
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", CASES)
def test_block_attention(case, dtype):
    attend(case, *make(case, dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", CASES)
def test_block_attention_gradients(case, dtype):
    attend(case, *make(case, dtype), grads=True)


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("case", [(1, 1, 700, 4, 1, 64, 128, 64, 8, None, None), (2, 300, 700, 4, 2, 64, 128, 64, 8, [700, 650], None), (1, 100, 600, 2, 2, 128, 64, 128, 4, None, None)])
def test_block_attention_odd_lists(case, grads):
    """Entries that name nothing, the same block several times, a list without any block, in no order."""
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v, blocks = make(case, BF16, 3)
    nK = -(-Sk // bk)
    blocks = blocks.flip(-1).contiguous()
    blocks[..., 1] = blocks[..., 0]
    blocks[..., 2] = blocks[..., 0]
    blocks[..., 3] = torch.tensor([-1, nK, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")[torch.arange(blocks.shape[2], device="cuda") % 4]
    attend(case, q, k, v, blocks, grads=grads)
    blocks[0, 0, 0] = -1
    attend(case, q, k, v, blocks, grads=grads)
    blocks[:] = -1
    got = attend(case, q, k, v, blocks, grads=grads)
    if grads:
        assert all((g == 0).all() for g in got)


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("case", [CASES[3], CASES[9], CASES[11]])
def test_block_attention_does_not_read_behind_the_sequences(case, grads):
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v, blocks = make(case, F16, 5)
    attend(case, q, k, v, blocks, grads=grads)
    go = randn((B, Sq, H, D), F16, 77)

    def results():
        leaves = [t.detach().requires_grad_(grads) for t in (q, k, v)]
        out, lse = ATT.block_sparse_attention(*leaves, blocks, bq, bk, lens(kl), lens(ql))
        if not grads:
            return out, lse
        gl = torch.where(torch.isfinite(lse.detach()), randn((B, H, Sq), F32, 78), 0.0)
        return torch.autograd.grad((out, torch.where(torch.isfinite(lse.detach()), lse, 0.0)), leaves, (go, gl))
    want = results()
    for b in range(B):
        k[b, R.clip(kl, b, Sk):] = float("nan")
        v[b, R.clip(kl, b, Sk):] = float("inf")
        q[b, R.clip(ql, b, Sq):] = float("nan")
        go[b, R.clip(ql, b, Sq):] = float("nan")
    for g, w in zip(results(), want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [(1, 1, 900, 4, 2, 64, 64, 64, 10, None, None), (1, 200, 900, 2, 1, 128, 128, 64, 10, None, None)])
def test_block_attention_scales_peaks_and_far_scores(case, dtype):
    """Peaked rows (the reference maximum moves often), scores far below and above zero, a given scale."""
    q, k, v, blocks = make(case, dtype, 11, spread=4.0)
    attend(case, q, k, v, blocks)
    attend(case, q, k, v, blocks, scale=0.7)
    attend(case, q, k, v, blocks, scale=1e-3, grads=True)
    ramp = torch.linspace(-6, 6, k.shape[1], device="cuda")[None, :, None, None]
    for sign in (1.0, -1.0):
        qq = q.abs()
        kk = (k.abs() * 0.1 + ramp * sign).to(dtype)
        attend(case, qq, kk, v, blocks)
    attend(case, q.abs() + 1, (-(k.abs() + 4)).to(dtype), v, blocks, grads=True)


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_block_attention_strides(dtype, grads):
    case = (2, 140, 260, 4, 2, 64, 64, 64, 3, [260, 200], None)
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    _, _, _, blocks = make(case, dtype)
    heads_first = randn((B, H, Sq, D), dtype, 1).transpose(1, 2)
    kv = randn((B, Sk, 2, Hk, D), dtype, 2)
    padded = randn((B, Sk, Hk, D + 8), dtype, 3)[..., :D]
    odd = randn((B * Sk * Hk * D + 1,), dtype, 4)[1:].view(B, Sk, Hk, D)
    inner = randn((B, D, Sk, Hk), dtype, 5).permute(0, 2, 3, 1)
    shared = randn((1, Sk, 1, D), dtype, 6).expand(B, Sk, Hk, D)
    long = randn((B, 2 * Sk, Hk, D), dtype, 7)[:, ::2]
    for k, v in ((kv[:, :, 0], kv[:, :, 1]), (padded, odd), (inner, padded), (shared, shared), (long, long)):
        attend(case, heads_first, k, v, blocks, grads=grads)
    wide = torch.cat([blocks, blocks], -1)[..., :topk]          # a list that is a view
    assert not wide.is_contiguous()
    attend(case, heads_first, kv[:, :, 0], kv[:, :, 1], wide, grads=grads)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_block_attention_gradients_of_far_scores_under_a_tiny_scale(dtype):
    """q . k of -3 * 10^9 (D elements of magnitude 5000 each way) with a scale that makes it -3: f16 has no way to hold -lse / scale, which
    is said with a NaN, not with a zero; bf16 does it."""
    D = 128
    q = torch.full((1, 1, 1, D), 5000.0, dtype=dtype, device="cuda")
    k = torch.full((1, 2, 1, D), -5000.0, dtype=dtype, device="cuda")
    v = torch.ones(1, 2, 1, D, dtype=dtype, device="cuda")
    blocks = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device="cuda")
    out, lse = F.block_sparse_attention(q, k, v, blocks, scale=1e-9)
    dq, dk, dv = F.block_sparse_attention_backward(torch.ones_like(out), None, q, k, v, blocks, out, lse, scale=1e-9)
    if dtype == F16:
        assert torch.isnan(dv).all()
    else:
        assert torch.equal(dv, torch.full_like(dv, 0.5))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("Sq, Sk, H, Hk, D, bq, bk, topk", [(1, 900, 64, 16, 64, 64, 64, 9), (30, 300, 16, 8, 96, 128, 64, 3), (64, 500, 12, 12, 40, 64, 128, 4), (500, 3, 20, 10, 80, 64, 128, 1)])
def test_gradients_of_one_block_keep_one_rounding(Sq, Sk, H, Hk, D, bq, bk, topk, dtype):
    """A rounding is off by at most half a step, evenly: the root of the mean square is at most half a step / sqrt(3) of the value (5 % more for
    the few thousand samples). Probabilities and dS that entered as rounded numbers would come to sqrt(2) of it."""
    case = (2, Sq, Sk, H, Hk, D, bq, bk, topk, None, None)
    q, k, v, blocks = make(case, dtype)
    gen = torch.Generator().manual_seed(9)
    go = torch.randn(q.shape, generator=gen).to(dtype).cuda()
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out, _ = F.block_sparse_attention(*leaves, blocks, bq, bk)
    got = torch.autograd.grad(out, leaves, go)
    want = R.attention(q.cpu().double(), k.cpu().double(), v.cpu().double(), blocks.cpu(), bq, bk, None, None, None, go.cpu().double(), None)
    for name, g in zip(("dq", "dk", "dv"), got):
        w = want[name][0]
        assert ((g.cpu().double() - w).norm() / w.norm()).item() <= 1.05 * R.half_step(dtype) / 3 ** 0.5, name


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [
    (1, 50, 3000, 4, 2, 64, 64, 64, 40, None, None), (2, 130, 2900, 2, 2, 80, 128, 128, 20, [2900, 900], [130, 70]), (1, 1, 2500, 8, 1, 128, 128, 64, 39, None, None),
    (1, 4000, 100, 4, 2, 64, 64, 64, 2, None, None), (2, 3000, 130, 2, 1, 40, 128, 128, 2, [130, 60], [3000, 1111]), (1, 2500, 200, 2, 2, 128, 128, 128, 1, None, [2400]),
    (2, 2100, 1, 3, 3, 96, 64, 64, 1, None, [2100, 0]),
])
def test_block_attention_gradients_in_parts(case, dtype):
    """Few query blocks with long lists, few key blocks that many query blocks name: the chain of tiles is cut, parts are added."""
    attend(case, *make(case, dtype), grads=True)


def test_block_attention_rows_that_overlap():
    """Rows that share memory (windows over a line of numbers), the last one with an infinity: it stays in its own column."""
    D, S = 16, 5
    gen = torch.Generator().manual_seed(3)
    lines = [torch.randn(8 * (S - 1) + D, generator=gen).to(F16) for _ in range(3)]
    lines[2][-1] = float("inf")
    got = [t.cuda().as_strided((1, S, 1, D), (128, 8, 16, 1)) for t in lines]
    want = [t.as_strided((1, S, 1, D), (128, 8, 16, 1)).contiguous().cuda() for t in lines]
    blocks = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device="cuda")
    out, lse = F.block_sparse_attention(*got, blocks)
    assert torch.isfinite(out[..., :-1]).all() and torch.isinf(out[..., -1]).all()
    same, lse2 = F.block_sparse_attention(*want, blocks)
    assert torch.equal(out, same) and torch.equal(lse, lse2)


def test_block_attention_gradient_of_an_expanded_and_of_an_unused_result():
    case = CASES[9]
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v, blocks = make(case, BF16, 2)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out, lse = ATT.block_sparse_attention(*leaves, blocks, bq, bk, lens(kl), lens(ql))
    got = torch.autograd.grad(out.sum(), leaves, retain_graph=True)   # the gradient of out is one value, expanded
    ones = torch.ones_like(out)
    want = R.attention(q.detach(), k.detach(), v.detach(), blocks, bq, bk, kl, ql, None, ones)
    for name, g in zip(("dq", "dk", "dv"), got):
        R.check(name, g, *want[name])
    gl = torch.where(torch.isfinite(lse.detach()), randn(lse.shape, F32, 8), 0.0)
    got = torch.autograd.grad(lse, leaves, gl)
    want = R.attention(q.detach(), k.detach(), v.detach(), blocks, bq, bk, kl, ql, None, torch.zeros_like(out), gl)
    for name, g in zip(("dq", "dk", "dv"), got):
        R.check(name, g, *want[name])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_row_with_one_key_has_no_score_gradient(dtype):
    """One key: P = 1 and dP = delta, so dq = dk = 0 but for what rowsum(dO O) is off: the step of out's rest (u^2) and the fp32 sums. A rounded
    out alone would leave u."""
    B, Sq, Sk, H, D = 2, 70, 129, 2, 64
    q, k, v, go = [randn((B, n, H, D), dtype, i) for i, n in enumerate((Sq, Sk, Sk, Sq))]
    blocks = torch.full((B, H, 1, 1), 2, dtype=torch.int32, device="cuda")   # the block that holds key 128 alone
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out, lse = ATT.block_sparse_attention(*leaves, blocks)
    dq, dk, dv = torch.autograd.grad(out, leaves, go)
    last_k, last_v = k.detach()[:, 128:].double(), v.detach()[:, 128:].double()
    assert torch.equal(out.detach(), v.detach()[:, 128:].expand_as(out))
    u = R.half_step(dtype)
    off = (go.double().abs() * last_v.abs()).sum(-1, keepdim=True) * (u * u + (2 * D + 8) * R.U32) * (1 + u) * D ** -0.5
    R.check("dq", dq, torch.zeros_like(dq, dtype=torch.float64), off * last_k.abs() + R.tiny(dtype))
    assert (dk[:, :128] == 0).all() and (dv[:, :128] == 0).all()
    R.check("dk", dk[:, 128:], torch.zeros_like(last_k), (off * q.detach().double().abs()).sum(1, keepdim=True) + R.tiny(dtype))
    total = go.double().sum(1, keepdim=True)
    R.check("dv", dv[:, 128:], total, u * total.abs() + Sq * R.U32 * 2 * go.double().abs().sum(1, keepdim=True))


def test_there_is_no_second_derivative():
    q, k, v, blocks = make(CASES[1], BF16)
    q.requires_grad_()
    out, _ = ATT.block_sparse_attention(q, k, v, blocks, 128, 64)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), q, create_graph=True)
    x = randn((1, 6, 1, 8), F32, 1).requires_grad_()          # a turn has one: it is linear in what it turns
    y, none = OPS.rotary_embedding_nd(x, None, grid(1, 2, 3, 1), [8])
    assert none is None
    g, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
    h, = torch.autograd.grad(g.sum(), x)
    assert torch.isfinite(h).all() and (h != 0).any()
    assert not ATT.block_means(x, 64).requires_grad


def test_block_attention_gradients_against_differences():
    """The derivative of the loss along a direction, from gradients and from a central difference of the 64-bit plain form."""
    case = (1, 70, 150, 2, 1, 32, 64, 64, 2, None, None)
    q, k, v, blocks = make(case, F16, 21)
    go = randn(q.shape, F16, 5)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(ATT.block_sparse_attention(*leaves, blocks, 64, 64)[0], leaves, go)
    for i, name in enumerate(("dq", "dk", "dv")):
        direction = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        h, values = 1e-4, []
        for s in (1, -1):
            moved = [t.detach().double() for t in leaves]
            moved[i] = moved[i] + s * h * direction
            # (the plain form only takes the type's half step from its inputs)
            values.append((R.attention(*moved, blocks, 64, 64)["out"][0] * go.double()).sum())
        slope = (values[0] - values[1]) / (2 * h)
        want = R.attention(*[t.detach() for t in leaves], blocks, 64, 64, grad_out=go)[name]
        bound = (want[1] * direction.abs()).sum() + 1e-6 * want[0].abs().sum()   # h^2 times third derivatives of order one
        assert abs((got[i].double() * direction).sum() - slope) <= bound


@pytest.mark.parametrize("case", [CASES[3], CASES[12]])
def test_block_attention_gives_the_same_bits_again(case):
    B, Sq, Sk, H, Hk, D, bq, bk, topk, kl, ql = case
    q, k, v, blocks = make(case, BF16, 4)
    go = randn(q.shape, BF16, 5)
    results = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out, lse = ATT.block_sparse_attention(*leaves, blocks, bq, bk, lens(kl))
        results.append((out.detach(), lse.detach()) + torch.autograd.grad(out, leaves, go))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_block_attention_over_a_cache_longer_than_32_bits():
    """Rows behind 4 GB of a key cache (64-bit tile addresses), means and choice included."""
    B, Sk, Hk, D, H = 1, 2200000, 8, 128, 8                      # 2.2 M rows x 2 KB = 4.5 GB each of K and V
    k = torch.zeros((B, Sk, Hk, D), dtype=BF16, device="cuda")
    v = torch.zeros((B, Sk, Hk, D), dtype=BF16, device="cuda")
    at = [0, Sk // 64 // 2, Sk // 64 - 1, -(-Sk // 64) - 1]
    rows = torch.cat([torch.arange(j * 64, min(Sk, j * 64 + 64)) for j in at]).cuda()
    k[0, rows], v[0, rows] = randn((len(rows), Hk, D), BF16, 1), randn((len(rows), Hk, D), BF16, 2)
    q = randn((B, 1, H, D), BF16, 3)
    blocks = torch.tensor(at, dtype=torch.int32).expand(B, Hk, 1, len(at)).contiguous().cuda()
    out, lse = ATT.block_sparse_attention(q, k, v, blocks)
    small = torch.arange(len(at), dtype=torch.int32).expand(B, Hk, 1, len(at)).contiguous().cuda()
    want = R.attention(q, k[:, rows], v[:, rows], small, 128, 64)
    R.check("out", out, *want["out"])
    R.check("lse", lse, *want["lse"])
    km = ATT.block_means(k, 64)
    want = R.means(k[:, at[-1] * 64:], 64)
    R.check("means", km[:, -1:], want, R.U32 * want.abs() + 2.0 ** -40)


def test_a_long_list_is_cut_into_parts():
    """More entries than one workgroup holds: forward in parts, gradients in rounds."""
    case = (1, 70, 64 * 1500, 1, 1, 64, 64, 64, 1500, None, None)
    q, k, v, blocks = make(case, BF16, 1)
    attend(case, q, k, v, blocks)
    attend(case, q, k, v, blocks, grads=True)


# ---- together -------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_clip_through_positions_choice_and_attention(dtype):
    """As a transformer over video makes the calls: positions, means, choice, attention; then the same through sparse_attention, and a
    training step through all of it."""
    B, (t, y, x), H, Hk, D, sections, topk = 2, (5, 9, 16), 4, 2, 64, [16, 24, 24], 4
    S = t * y * x
    q, k, v = [randn((B, S, h, D), dtype, i) for i, h in enumerate((H, Hk, Hk))]
    pos = grid(t, y, x, 3)
    kl = [S, 500]
    leaves = [a.requires_grad_() for a in (q, k, v)]
    qr, kr = OPS.rotary_embedding_nd(leaves[0], leaves[1], pos, sections)
    qd, kd = qr.detach(), kr.detach()
    R.check("q", qd, *R.rope(q.detach(), pos, sections, 10000.0, True))
    qm, km = ATT.block_means(qd, 128), ATT.block_means(kd, 64, lens(kl))
    blocks = ATT.block_topk(qm, km, topk, 64, lens(kl))
    assert torch.equal(blocks.cpu(), R.topk(qm, km, topk, 64, kl))
    out, lse = ATT.block_sparse_attention(qr, kr, leaves[2], blocks, 128, 64, lens(kl))
    want = R.attention(qd, kd, v.detach(), blocks, 128, 64, kl)
    R.check("out", out.detach(), *want["out"])
    assert torch.equal(sparse_attention(qr, kr, leaves[2], topk, key_lengths=lens(kl)).detach(), out.detach())
    go = randn(q.shape, dtype, 9)
    got = torch.autograd.grad(out, leaves, go)
    want = R.attention(qd, kd, v.detach(), blocks, 128, 64, kl, grad_out=go)
    R.check("dv", got[2], *want["dv"])
    # the turn back of the gradients that attention gave
    alone = [a.detach().requires_grad_() for a in (qd, kd, v)]
    d = torch.autograd.grad(ATT.block_sparse_attention(*alone, blocks, 128, 64, lens(kl))[0], alone, go)
    back = OPS.rotary_embedding_nd(d[0], d[1], pos, sections, 10000.0, True, True)
    assert torch.equal(got[0], back[0]) and torch.equal(got[1], back[1])


def test_every_block_chosen_is_dense_attention():
    B, S, H, D = 1, 500, 2, 64
    q, k, v = [randn((B, S, H, D), F16, i) for i in range(3)]
    out = sparse_attention(q, k, v, topk=-(-S // 64))
    dense = ATT.memory_efficient_attention(q, k, v)
    blocks = torch.arange(8, dtype=torch.int32).expand(B, H, 4, 8).contiguous().cuda()
    want, bound = R.attention(q, k, v, blocks, 128, 64)["out"]
    R.check("sparse", out, want, bound)
    # the dense operator also rounds the scaled q once to f16: scores move by up to one half step of their reach
    reach = (q.double().abs().amax() * k.double().abs().sum(-1).amax()) * D ** -0.5
    R.check("dense", dense, want, bound + 4 * R.half_step(F16) * reach * v.double().abs().amax())


def test_a_token_at_a_time_over_a_kept_cache():
    """Serving: a preallocated cache and its block means grow by a token; each step's result is the plain form over the valid part."""
    B, cap, H, Hk, D, topk = 2, 512, 4, 2, 64, 3
    k, v = [torch.full((B, cap, Hk, D), float("nan"), dtype=BF16, device="cuda") for _ in range(2)]
    k[:, :190], v[:, :190] = randn((B, 190, Hk, D), BF16, 1), randn((B, 190, Hk, D), BF16, 2)
    km = ATT.block_means(k, 64, lens([190, 190]))
    for step in range(190, 197):
        kl = [step + 1, step + 1]
        k[:, step], v[:, step] = randn((B, Hk, D), BF16, 3 * step), randn((B, Hk, D), BF16, 3 * step + 1)
        j = step // 64
        km[:, j:j + 1] = ATT.block_means(k[:, j * 64:(j + 1) * 64], 64, lens([step + 1 - j * 64] * B))
        q = randn((B, 1, H, D), BF16, 3 * step + 2)
        blocks = ATT.block_topk(ATT.block_means(q, 128), km, topk, 64, lens(kl))
        out, lse = ATT.block_sparse_attention(q, k, v, blocks, 128, 64, lens(kl))
        n = step + 1
        want = R.attention(q, k[:, :n], v[:, :n], blocks, 128, 64)
        R.check("out", out, *want["out"])
        assert torch.equal(blocks.cpu(), R.topk(q.float(), R.means(k[:, :n], 64).float(), topk, 64))


@pytest.mark.parametrize("Sq", [1, 300])
def test_captured_calls_replay_on_new_inputs(Sq):
    B, H, Hk, D, Sk = 2, 4, 2, 64, 300
    pos = torch.arange(Sk, device="cuda")[:, None].repeat(1, 3)

    def one(q, k, v, kl):
        qr, kr = OPS.rotary_embedding_nd(k if Sq == 1 else q, k, pos, [16, 24, 24])
        qr = q if Sq == 1 else qr
        blocks = ATT.block_topk(ATT.block_means(qr, 128), ATT.block_means(kr, 64, kl), 4, 64, kl)
        out, lse = ATT.block_sparse_attention(qr, kr, v, blocks, 128, 64, kl)
        d = ATT.block_sparse_attention_backward(out, lse.clamp(min=-1.0), qr, kr, v, blocks, out, lse, 128, 64, kl)
        return (blocks, out, lse) + d

    def inputs(seed):
        return (randn((B, Sq, H, D), BF16, seed), randn((B, Sk, Hk, D), BF16, seed + 1), randn((B, Sk, Hk, D), BF16, seed + 2), lens([300 - seed % 7, 200]))

    static, other = inputs(0), inputs(50)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        one(*static)
    torch.cuda.current_stream().wait_stream(stream)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        got1 = one(*static)
    with torch.cuda.graph(g2):       # a second graph of the same calls: workspaces of its own
        got2 = one(*other)
    for seed in (3, 17, 31):
        fresh, fresh2 = inputs(seed), inputs(seed + 100)
        for a, b in zip(static + other, fresh + fresh2):
            a.copy_(b)
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        for got, ins in ((got1, fresh), (got2, fresh2)):
            for a, b in zip(got, one(*ins)):
                assert torch.equal(a, b)
    # a graph lives as long as the tensors of its pool are used: keep both to the end
    del g1, g2


def test_a_captured_training_step():
    """Forward and gradients in one graph (no eager graph of the same leaves is alive: that is what torch asks of any captured backward)."""
    case = (1, 200, 300, 4, 2, 64, 128, 64, 3, None, None)
    q, k, v, blocks = make(case, BF16, 1)
    pos = torch.arange(300, device="cuda")[:, None].repeat(1, 3)
    go = randn(q.shape, BF16, 9)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        kr = OPS.rotary_embedding_nd(leaves[1], None, pos, [16, 24, 24])[0]
        out, lse = ATT.block_sparse_attention(leaves[0], kr, leaves[2], blocks)
        return (out.detach(), lse.detach()) + torch.autograd.grad(out, leaves, go)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6, 7):
        with torch.no_grad():
            for i, t in enumerate(leaves):
                t.copy_(randn(t.shape, BF16, 10 * seed + i))
        graph.replay()
        torch.cuda.synchronize()
        got_now = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(got_now, step()))
    del graph


def test_a_nan_key_reaches_the_rows_that_name_it_only():
    case = (1, 300, 500, 2, 2, 64, 64, 64, 2, None, None)
    q, k, v, blocks = make(case, F16, 4)
    want = R.attention(q, k, v, blocks, 64, 64)["out"]
    for bad in (math.nan, math.inf):
        kk = k.clone()
        kk[0, 70, 1, 3] = bad                         # block 1 of the second head
        out, lse = ATT.block_sparse_attention(q, kk, v, blocks, 64, 64)
        names = (blocks[0, 1] == 1).any(-1).repeat_interleave(64)[:300]
        clean = torch.ones((300, 2), dtype=torch.bool, device="cuda")
        clean[:, 1] = ~names
        assert names.any() and not names.all()
        assert torch.isfinite(out[0][clean]).all()
        if math.isnan(bad):
            assert torch.isnan(out[0, :, 1][names]).all()
        else:                                          # a score of +inf leaves no number, one of -inf takes the key out
            up = names & (q[0, :, 1, 3] > 0)
            down = names & (q[0, :, 1, 3] < 0)
            assert torch.isnan(out[0, :, 1][up]).all() and torch.isfinite(out[0, :, 1][down]).all()
        off = (out.double() - want[0]).abs() > want[1]
        assert not off[0][clean].any()


def test_batch_invariant_mode_cuts_lists_alike_for_every_batch(monkeypatch):
    """SFAST_BATCH_INVARIANT=1: a sample's bits do not depend on how many ride with it (the parts of its lists are those of the reference batch)."""
    from sfast.hip import lib as L
    lib = L.load()
    B, Sq, Sk, H, Hk, D = 24, 1, 4000, 8, 2, 128
    q, k, v, blocks = make((B, Sq, Sk, H, Hk, D, 128, 64, 40, None, None), BF16, 2)

    def rows(n):
        return ATT.block_sparse_attention(q[:n], k[:n], v[:n], blocks[:n])
    monkeypatch.setenv("SFAST_BATCH_INVARIANT", "1")
    try:
        assert lib.sfast_hip_init() == 0
        a, b, c = rows(1), rows(2), rows(B)
        for x, y in ((a, b), (a, c), (b, c)):
            n = min(len(x[0]), len(y[0]))
            assert torch.equal(x[0][:n], y[0][:n]) and torch.equal(x[1][:n], y[1][:n])
    finally:
        monkeypatch.undo()
        assert lib.sfast_hip_init() == 0
    want = R.attention(q, k, v, blocks, 128, 64)
    R.check("out", c[0], *want["out"])
    R.check("out", rows(B)[0], *want["out"])


def test_two_streams_at_once():
    case = (1, 300, 600, 4, 2, 64, 128, 64, 4, None, None)
    ins = [make(case, BF16, s) for s in (1, 100)]
    want = [ATT.block_sparse_attention(*x, 128, 64) for x in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ATT.block_sparse_attention(*ins[i], 128, 64))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_empty_calls():
    q, k = randn((2, 10, 4, 64), BF16, 1), randn((2, 20, 2, 64), BF16, 2)
    blocks = torch.zeros((2, 2, 1, 1), dtype=torch.int32, device="cuda")
    out, lse = ATT.block_sparse_attention(q[:, :0], k, k, blocks[:, :, :0])
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    for kk, bb in ((k[:, :0], blocks), (k, blocks[..., :0])):
        leaves = [q.detach().requires_grad_(), kk.detach().requires_grad_(), kk.detach().requires_grad_()]
        out, lse = ATT.block_sparse_attention(*leaves, bb)
        assert (out == 0).all() and (lse == -math.inf).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out, leaves, torch.ones_like(out)))
    assert ATT.block_means(k[:, :0], 64).shape == (2, 0, 2, 64)


def test_refusals():
    q, k = randn((2, 70, 4, 64), BF16, 1), randn((2, 130, 2, 64), BF16, 2)
    blocks = torch.zeros((2, 2, 1, 1), dtype=torch.int32, device="cuda")
    pos = torch.zeros((70, 1), dtype=torch.int64, device="cuda")
    bad = [
        lambda: ATT.block_sparse_attention(q.float(), k.float(), k.float(), blocks),
        lambda: ATT.block_sparse_attention(q, k.half(), k.half(), blocks),
        lambda: ATT.block_sparse_attention(q, k, k[:, :1], blocks),
        lambda: ATT.block_sparse_attention(q[:, :, :3], k, k, blocks),
        lambda: ATT.block_sparse_attention(q[0], k[0], k[0], blocks),
        lambda: ATT.block_sparse_attention(q[..., :60], k[..., :60], k[..., :60], blocks),
        lambda: ATT.block_sparse_attention(q.repeat(1, 1, 1, 3), k.repeat(1, 1, 1, 3), k.repeat(1, 1, 1, 3), blocks),
        lambda: ATT.block_sparse_attention(q, k, k, blocks.long()),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, 64),             # two query blocks of 64
        lambda: ATT.block_sparse_attention(q, k, k, blocks, 96),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, 128, 32),
        lambda: ATT.block_sparse_attention(q, k, k, blocks[:1]),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, key_lengths=lens([1])),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, key_lengths=torch.ones(2, device="cuda")),
        lambda: ATT.block_sparse_attention(q, k, k, blocks.cpu()),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, scale=0.0),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, scale=-1.0),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, scale=math.inf),
        lambda: ATT.block_sparse_attention(q, k, k, blocks, scale=math.nan),
        lambda: ATT.block_sparse_attention_backward(q[:, :1], None, q, k, k, blocks, q, torch.zeros((2, 4, 70), device="cuda")),
        lambda: ATT.block_sparse_attention_backward(q, None, q, k, k, blocks, q, torch.zeros((2, 4, 71), device="cuda")),
        lambda: ATT.block_means(q[0], 64),
        lambda: ATT.block_means(q, 0),
        lambda: ATT.block_means(q, 1025),
        lambda: ATT.block_means(q.double(), 64),
        lambda: ATT.block_topk(q.float(), k, 1),
        lambda: ATT.block_topk(q.float(), k.float(), 0),
        lambda: ATT.block_topk(q.float()[..., :62], k.float()[..., :62], 1),
        lambda: ATT.block_topk(q.float()[:, :, :3], k.float(), 1),
        lambda: ATT.block_topk(torch.zeros((1, 1, 1, 4), device="cuda"), torch.zeros((1, 32769, 1, 4), device="cuda"), 1),
        lambda: OPS.rotary_embedding_nd(q, k, pos, [64]),                    # k of another length
        lambda: OPS.rotary_embedding_nd(q, q, pos, [63]),
        lambda: OPS.rotary_embedding_nd(q, q, pos, [66]),
        lambda: OPS.rotary_embedding_nd(q, q, pos, [32, 32]),
        lambda: OPS.rotary_embedding_nd(q, q, pos, []),
        lambda: OPS.rotary_embedding_nd(q, q, pos[:3], [64]),
        lambda: OPS.rotary_embedding_nd(q, q, pos.half(), [64]),
        lambda: OPS.rotary_embedding_nd(q, q.half(), pos, [64]),
        lambda: OPS.rotary_embedding_nd(q, q, pos, [64], -1.0),
        lambda: OPS.rotary_embedding_nd(q, q, pos, [64], math.inf),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(f"call {i} was not refused")
