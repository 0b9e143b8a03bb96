"""Video-attention operators without a GPU: the C structs, what the entry points refuse before they launch anything, the workspaces they ask
for, and the plain forms that the GPU tests compare with."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import video_attention_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sfast_hip.h")


def test_structs_match_the_header(built_lib):
    from sfast.hip import lib as L
    structs = {"sfast_rope_params": L.RopeParams, "sfast_block_means_params": L.BlockMeansParams, "sfast_block_topk_params": L.BlockTopkParams,
               "sfast_block_attn_params": L.BlockAttnParams}
    fields = [(n, f[0]) for n, st in structs.items() for f in st._fields_]
    body = "".join(f'printf("%zu\\n", sizeof({n}));' for n in structs) + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for n, f in fields)
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "abi.c"), os.path.join(d, "abi")
        with open(src, "w") as f:
            f.write(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(){{{body}return 0;}}\n')
        subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", src, "-o", exe])
        out = [int(x) for x in subprocess.check_output([exe]).split()]
    assert out[:len(structs)] == [C.sizeof(st) for st in structs.values()]
    assert out[len(structs):] == [getattr(structs[n], f).offset for n, f in fields]


def attn_params(L, **over):
    p = L.BlockAttnParams()
    p.dtype, p.B, p.H, p.Hk, p.Sq, p.Sk, p.D, p.block_q, p.block_k, p.topk, p.scale = L.BF16, 2, 4, 2, 300, 500, 64, 128, 64, 4, 0.125
    for n, (s, h) in (("qs", (300, 4)), ("ks", (500, 2)), ("vs", (500, 2)), ("os", (300, 4)), ("dos", (300, 4)), ("dqs", (300, 4)), ("dks", (500, 2)), ("dvs", (500, 2))):
        setattr(p, n, (C.c_int64 * 3)(s * h * 64, h * 64, 64))
    for n, v in over.items():
        setattr(p, n, (C.c_int64 * 3)(*v) if isinstance(v, tuple) else v)
    return p


@pytest.mark.parametrize("over, code", [
    ({"B": 0}, -2), ({"Sq": -1}, -2), ({"Sk": 0}, -2), ({"topk": 0}, -2), ({"Hk": 3}, -2), ({"Hk": 0}, -2), ({"D": 0}, -2),
    ({"dtype": 2}, -1), ({"D": 60}, -1), ({"D": 136}, -1), ({"block_q": 96}, -1), ({"block_k": 32}, -1), ({"scale": 0.0}, -1), ({"scale": -1.0}, -1),
    ({"scale": float("inf")}, -1), ({"scale": float("nan")}, -1), ({"ks": (0, 130, 64)}, -1), ({"vs": (4, 128, 64)}, -1), ({"qs": (-8, 256, 64)}, -1),
    ({"ks": (0, 1 << 23, 64)}, -1), ({"os": (0, 2, 64)}, -1),
])
def test_block_attention_refuses_before_it_launches(built_lib, over, code):
    from sfast.hip import lib as L
    lib = L.load()
    p = attn_params(L, **over)
    ptr = 4096   # an aligned address that nothing reads
    assert lib.sfast_hip_block_attention(ptr, ptr, ptr, ptr, None, None, ptr, ptr, None, C.byref(p), ptr, 1 << 40, None) == code
    assert b"block_attention" in lib.sfast_hip_last_error()
    assert lib.sfast_hip_block_attention_backward(ptr, ptr, ptr, ptr, None, None, ptr, None, ptr, ptr, None, ptr, ptr, ptr, C.byref(p), ptr, 1 << 40, None) == code


def test_block_attention_refuses_addresses_and_workspaces(built_lib):
    from sfast.hip import lib as L
    lib = L.load()
    p = attn_params(L, Sq=1, topk=8)   # a split call: it needs a workspace
    need = lib.sfast_hip_block_attention_workspace_bytes(C.byref(p))
    assert need > 0 and need % 4 == 0
    good = [4096] * 8
    for at in (0, 1, 2, 3, 6, 7):      # q, k, v, blocks, out, lse
        args = [4096, 4096, 4096, 4096, None, None, 4096, 4096, None]
        args[at] = None
        assert lib.sfast_hip_block_attention(*args, C.byref(p), 4096, need, None) == -2
    for at in (0, 1, 2):
        args = [4096, 4096, 4096, 4096, None, None, 4096, 4096, None]
        args[at] = 4098
        assert lib.sfast_hip_block_attention(*args, C.byref(p), 4096, need, None) == -1
    args = good[:4] + [None, None, 4096, 4096, None]
    assert lib.sfast_hip_block_attention(*args, C.byref(p), None, 0, None) == -3
    assert lib.sfast_hip_block_attention(*args, C.byref(p), 4096, need - 1, None) == -3
    need = lib.sfast_hip_block_attention_backward_workspace_bytes(C.byref(p))
    assert need >= (2 * 4 * 1 + 2 * 2 * 1 * 8) * 4
    back = [4096, 4096, 4096, 4096, None, None, 4096, None, 4096, 4096, None, 4096, 4096, 4096]
    assert lib.sfast_hip_block_attention_backward(*back, C.byref(p), 4096, need - 1, None) == -3
    for at in (0, 3, 6, 8, 9, 11, 12, 13):
        args = list(back)
        args[at] = None
        assert lib.sfast_hip_block_attention_backward(*args, C.byref(p), 4096, need, None) == -2


def test_rotary_means_and_choice_refuse_before_they_launch(built_lib):
    from sfast.hip import lib as L
    lib = L.load()

    def rope(sections=(16, 24, 24), **over):
        s = (C.c_int64 * 3)(64 * 4 * 10, 64 * 4, 64)
        p = L.RopeParams(L.BF16, 2, 10, 4, 4, 64, len(sections), (C.c_int32 * 4)(*sections), 1, 0, L.POS_I64, 10000.0, s, s, s, s, (C.c_int64 * 2)(0, 3))
        for n, v in over.items():
            setattr(p, n, v)
        return lib.sfast_hip_rope_nd(4096, 4096, 4096, 4096, 4096, C.byref(p), None)
    assert rope(sections=(16, 24, 26)) == -2 and rope(sections=(15,)) == -2 and rope(sections=(0, 2)) == -2
    assert rope(n_axes=0) == -1 and rope(n_axes=5) == -1 and rope(D=63) == -1 and rope(D=258) == -1 and rope(dtype=7) == -1 and rope(pos_type=4) == -1
    assert rope(theta=0.0) == -2 and rope(theta=float("inf")) == -2 and rope(theta=float("nan")) == -2 and rope(B=0) == -2 and rope(S=-3) == -2
    assert rope(qs=(C.c_int64 * 3)(1, 1, 1)) == -1    # neighbouring pairs at odd elements

    def means(**over):
        p = L.BlockMeansParams(L.BF16, 2, 100, 4, 64, 64, (C.c_int64 * 3)(64 * 4 * 100, 64 * 4, 64))
        for n, v in over.items():
            setattr(p, n, v)
        return lib.sfast_hip_block_means(4096, None, 4096, C.byref(p), None)
    assert means(B=0) == -2 and means(block=0) == -2 and means(block=1025) == -2 and means(dtype=3) == -1

    def topk(ws=4096, nb=1 << 40, **over):
        p = L.BlockTopkParams(2, 3, 9, 4, 2, 64, 3, 64)
        for n, v in over.items():
            setattr(p, n, v)
        return lib.sfast_hip_block_topk(4096, 4096, None, 4096, C.byref(p), ws, nb, None)
    assert topk(Hk=3) == -2 and topk(topk=0) == -2 and topk(nK=0) == -2 and topk(D=62) == -1 and topk(nK=32769) == -1 and topk(block_k=0) == -2
    assert topk(ws=None) == -3 and topk(nb=2 * 2 * 3 * 9 * 8 - 1) == -3


@pytest.mark.parametrize("name", ["qs", "ks", "vs", "dos"])
def test_block_attention_refuses_rows_that_overlap(built_lib, name):
    from sfast.hip import lib as L
    lib = L.load()
    p = attn_params(L, **{name: (300 * 64 * 4, 56, 64)})
    args = [4096, 4096, 4096, 4096, None, None, 4096, 4096, None]
    if name != "dos":
        assert lib.sfast_hip_block_attention(*args, C.byref(p), 4096, 1 << 40, None) == -1
    back = [4096, 4096, 4096, 4096, None, None, 4096, None, 4096, 4096, None, 4096, 4096, 4096]
    assert lib.sfast_hip_block_attention_backward(*back, C.byref(p), 4096, 1 << 40, None) == -1


def test_calls_beyond_a_launch_are_refused(built_lib):
    """A grid has fewer than 2^32 threads along an axis."""
    from sfast.hip import lib as L
    lib = L.load()
    s = (C.c_int64 * 3)(1 << 40, 64, 64)
    p = L.RopeParams(L.BF16, 2, 1 << 29, 1, 1, 64, 1, (C.c_int32 * 4)(64), 1, 0, L.POS_I64, 10000.0, s, s, s, s, (C.c_int64 * 2)(0, 1))
    assert lib.sfast_hip_rope_nd(4096, 4096, 4096, 4096, 4096, C.byref(p), None) == -1
    p = L.BlockMeansParams(L.BF16, 1, (1 << 31) - 1, 1, 64, 64, s)
    assert lib.sfast_hip_block_means(4096, None, 4096, C.byref(p), None) == -1
    p = L.BlockTopkParams(8, 1 << 20, 4096, 1, 1, 64, 8, 64)
    assert lib.sfast_hip_block_topk(4096, 4096, None, 4096, C.byref(p), 4096, 1 << 60, None) == -1
    p = attn_params(L, Sq=1 << 30, H=4, Hk=4, B=2, topk=1)
    args = [4096, 4096, 4096, 4096, None, None, 4096, 4096, None]
    assert lib.sfast_hip_block_attention(*args, C.byref(p), 4096, 1 << 60, None) == -1
    p = attn_params(L, Sq=1 << 27, H=4, topk=2000)      # lists that are cut: a second launch has a wave for every row
    assert lib.sfast_hip_block_attention(*args, C.byref(p), 4096, 1 << 60, None) == -1
    back = [4096, 4096, 4096, 4096, None, None, 4096, None, 4096, 4096, None, 4096, 4096, 4096]
    p = attn_params(L, Sq=1 << 28, topk=1)
    assert lib.sfast_hip_block_attention_backward(*back, C.byref(p), 4096, 1 << 60, None) == -1


def test_block_attention_refuses_a_scale_that_lse_cannot_be_divided_by(built_lib):
    from sfast.hip import lib as L
    lib = L.load()
    p = attn_params(L, scale=2.0 ** -101)
    assert lib.sfast_hip_block_attention(4096, 4096, 4096, 4096, None, None, 4096, 4096, None, C.byref(p), 4096, 1 << 40, None) == -1
    back = [4096, 4096, 4096, 4096, None, None, 4096, None, 4096, 4096, None, 4096, 4096, 4096]
    assert lib.sfast_hip_block_attention_backward(*back, C.byref(p), 4096, 1 << 40, None) == -1


def test_the_choice_refuses_lists_longer_than_any_row(built_lib):
    """(the entries behind the last block are filled with -1 in steps of 32-bit indexes)"""
    from sfast.hip import lib as L
    lib = L.load()
    for topk in (32769, (1 << 31) - 1):
        p = L.BlockTopkParams(1, 1, 9, 1, 1, 64, topk, 64)
        assert lib.sfast_hip_block_topk_workspace_bytes(C.byref(p)) == 0
        assert lib.sfast_hip_block_topk(4096, 4096, None, 4096, C.byref(p), 4096, 1 << 40, None) == -1
        assert b"block_topk" in lib.sfast_hip_last_error()


def test_operators_take_no_cpu_tensors(built_lib):
    import sfast  # noqa: F401
    from sfast.hip import functional as F
    x = torch.zeros(1, 64, 1, 64, dtype=torch.float16)
    for call in (lambda: F.rotary_nd(x, x, torch.zeros(64, 1), [64]), lambda: F.block_means(x, 64), lambda: F.block_topk(x.float(), x.float(), 1),
                 lambda: F.block_sparse_attention(x, x, x, torch.zeros(1, 1, 1, 1, dtype=torch.int32)),
                 lambda: torch.ops.sfast_xformers.block_means(x, 64), lambda: torch.ops.sfast.rotary_embedding_nd(x, x, torch.zeros(64, 1), [64])):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


@pytest.mark.parametrize("Sq, Sk, H, Hk, bq, bk, kl, ql", [(70, 150, 4, 2, 64, 64, [150, 70], [70, 3]), (1, 130, 2, 1, 128, 128, None, None), (64, 64, 1, 1, 64, 64, [0, 64], None)])
def test_the_plain_form_is_its_own_gradient(Sq, Sk, H, Hk, bq, bk, kl, ql):
    """dq, dk, dv of the plain form against autograd through a gather of the listed keys, in 64 bits, with entries named twice and none."""
    B, D = 2, 8
    gen = torch.Generator().manual_seed(0)
    q, k, v = [torch.randn(s, generator=gen, dtype=torch.float64) for s in ((B, Sq, H, D), (B, Sk, Hk, D), (B, Sk, Hk, D))]
    nQ, nK = -(-Sq // bq), -(-Sk // bk)
    blocks = R.choose(B, Hk, nQ, nK, 3, gen)
    blocks[0, 0, 0, :2] = 0
    go, gl = torch.randn((B, Sq, H, D), generator=gen, dtype=torch.float64), torch.randn((B, H, Sq), generator=gen, dtype=torch.float64)
    want = R.attention(q, k, v, blocks, bq, bk, kl, ql, None, go, gl)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    loss = 0.0
    for b in range(B):
        n, m = R.clip(kl, b, Sk), R.clip(ql, b, Sq)
        for h in range(H):
            for i in range(m):
                keys = [x for j in blocks[b, h // (H // Hk), i // bq].tolist() if 0 <= j < nK for x in range(j * bk, min(n, (j + 1) * bk))]
                if not keys:
                    assert (want["out"][0][b, i, h] == 0).all() and want["lse"][0][b, h, i] == float("-inf")
                    continue
                s = k[b, keys, h // (H // Hk)] @ q[b, i, h] * D ** -0.5
                o = torch.softmax(s, 0) @ v[b, keys, h // (H // Hk)]
                assert torch.allclose(o, want["out"][0][b, i, h], atol=1e-12) and torch.allclose(s.logsumexp(0), want["lse"][0][b, h, i], atol=1e-12)
                loss = loss + (o * go[b, i, h]).sum() + s.logsumexp(0) * gl[b, h, i]
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(loss, leaves)):
        assert torch.allclose(g, want[name][0], atol=1e-11), name


def test_the_plain_turn_keeps_lengths_and_turns_back():
    x = torch.randn(1, 12, 2, 20, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    pos = torch.arange(24).reshape(12, 2)
    for interleaved in (True, False):
        y, _ = R.rope(x, pos, [8, 10], 100.0, interleaved)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and not torch.allclose(y[:, 1:], x[:, 1:])
        assert torch.allclose(R.rope(y, pos, [8, 10], 100.0, interleaved, inverse=True)[0], x) and torch.equal(y[..., 18:], x[..., 18:])
        assert torch.allclose(y[:, :1, :, :8], x[:, :1, :, :8])   # position 0 of the first axis
