"""64-bit plain forms of the video-attention operators, with elementwise bounds on what a kernel may be off.

Bounds count roundings: u = finfo(T).eps / 2 for each value rounded to T (outputs; probabilities and dS, which enter the second products as T),
2^-24 for each fp32 operation of a sum, 2^-25 as the half step of f16's subnormals."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130


def rope(x, positions, sections, theta, interleaved, inverse=False):
    """Returns (turned x, bound)."""
    y = x.double().clone()
    mass = torch.zeros_like(y)
    pos = positions.double()
    if pos.ndim == 2:
        pos = pos[None]
    at = 0
    for axis, size in enumerate(sections):
        i = torch.arange(size // 2, device=x.device)
        lo, hi = (at + 2 * i, at + 2 * i + 1) if interleaved else (at + i, at + i + size // 2)
        angle = pos[..., axis, None] * theta ** (-2.0 * i.double() / size)
        c, s = angle.cos()[:, :, None, :], angle.sin()[:, :, None, :] * (-1.0 if inverse else 1.0)
        a, b = x.double()[..., lo], x.double()[..., hi]
        y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
        mass[..., lo] = mass[..., hi] = a.abs() + b.abs()
        at += size
    # cosine and sine are rounded once to fp32 (2^-24 each), two fp32 products / sums (2^-24 each); the angle itself is good to
    # 2^-52 * |turns|: 10^6 * 2^-52 turns is far below 2^-24
    return y, half_step(x.dtype) * y.abs() + 4 * U32 * mass + tiny(x.dtype)


def means(x, block, lengths=None):
    B, S, H, D = x.shape
    out = torch.zeros((B, -(-S // block), H, D), dtype=torch.float64, device=x.device)
    for b in range(B):
        n = S if lengths is None else max(0, min(S, int(lengths[b])))
        for j in range(-(-n // block)):
            out[b, j] = x[b, j * block:min(n, (j + 1) * block)].double().mean(dim=0)
    return out


def topk(qm, km, k, block_k, lengths=None):
    """Python's own sort: by descending score (NaN first), then ascending index."""
    B, nQ, H, D = qm.shape
    nK, Hk = km.shape[1], km.shape[2]
    g = H // Hk
    out = torch.full((B, Hk, nQ, k), -1, dtype=torch.int32)
    qd, kd = qm.double().cpu(), km.double().cpu()
    for b in range(B):
        n = nK if lengths is None else min(nK, -(-max(0, int(lengths[b])) // block_k))
        for hk in range(Hk):
            q = qd[b, :, hk * g:(hk + 1) * g].sum(dim=1)
            score = (q @ kd[b, :n, hk].t()).tolist()
            for i in range(nQ):
                row = score[i] if n else []
                order = sorted(range(n), key=lambda j: (0.0 if math.isnan(row[j]) else 1.0, 0.0 if math.isnan(row[j]) else -row[j], j))[:k]
                out[b, hk, i, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
    return out


def clip(lengths, b, size):
    return size if lengths is None else max(0, min(size, int(lengths[b])))


def attention(q, k, v, blocks, block_q, block_k, key_lengths=None, query_lengths=None, scale=None, grad_out=None, grad_lse=None):
    """Dense form: key j weighs as often for row s as the list of s's query block names j's block. Returns a dict name -> (value, bound) of
    out, lse and, with grad_out, dq, dk, dv."""
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    g, nK = H // Hk, -(-Sk // block_k)
    scale = D ** -0.5 if scale is None else scale
    u, small, dev = half_step(q.dtype), tiny(q.dtype), q.device
    new = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=dev)  # noqa: E731
    out, out_e, lse, lse_e = new(B, Sq, H, D), new(B, Sq, H, D), new(B, H, Sq) - math.inf, new(B, H, Sq)
    dq, dq_e, dk, dk_e, dv, dv_e = new(B, Sq, H, D), new(B, Sq, H, D), new(B, Sk, Hk, D), new(B, Sk, Hk, D), new(B, Sk, Hk, D), new(B, Sk, Hk, D)
    for b in range(B):
        n, m = clip(key_lengths, b, Sk), clip(query_lengths, b, Sq)
        if n == 0 or m == 0:
            continue
        for h in range(H):
            hk = h // g
            lists = blocks[b, hk].long().to(dev)
            names = new(lists.shape[0], nK + 1)
            names.scatter_add_(1, torch.where((lists < 0) | (lists >= nK), nK, lists), torch.ones_like(lists, dtype=torch.float64))
            w = names[torch.arange(m, device=dev) // block_q][:, torch.arange(n, device=dev) // block_k]
            Q, K, V = q[b, :m, h].double(), k[b, :n, hk].double(), v[b, :n, hk].double()
            s = Q @ K.t() * scale
            s = torch.where(w > 0, s, -math.inf)
            top = s.amax(dim=1, keepdim=True)
            ref = torch.where(torch.isinf(top), 0.0, top)
            e = w * torch.exp(s - ref)
            e = torch.where(w > 0, e, 0.0)
            z = e.sum(dim=1, keepdim=True)
            p = torch.where(z > 0, e / z, 0.0)
            o = p @ V
            out[b, :m, h] = o
            lse[b, h, :m] = torch.where(z > 0, ref + torch.log(z), -math.inf)[:, 0]
            count = w.sum(dim=1, keepdim=True)
            # a score: D fp32 products and sums, the scaling, the exponent (whose argument is as large as the score), exp2 itself
            reach = (Q.abs() @ K.abs().t() * scale).amax(dim=1, keepdim=True)
            d = U32 * (2 * D + 8) * reach + U32 * 16
            mass = p @ V.abs()
            # probabilities: rounded to T (subnormal f16 steps relative to a largest one of at least 1), their sum in fp32; then the output
            out_e[b, :m, h] = (u + 2 * d + U32 * (count + 8)) * mass + small * count * V.abs().amax() + u * o.abs() + small
            lse_e[b, h, :m] = (d + U32 * (count + 8))[:, 0] + 4 * U32 * torch.nan_to_num(lse[b, h, :m], neginf=0.0).abs()
            if grad_out is None:
                continue
            G = grad_out[b, :m, h].double()
            gl = new(m, 1) if grad_lse is None else grad_lse[b, h, :m].double()[:, None]
            gl = torch.where(z > 0, gl, 0.0)
            dP = G @ V.t()
            delta = (G * o).sum(dim=1, keepdim=True) - gl
            dS = p * (dP - delta)
            # P again from lse: the errors of the score and of lse; delta from the rounded out; dP summed in fp32
            dp_rel = 2 * d + U32 * (count + 8) + 8 * U32 * torch.nan_to_num(lse[b, h, :m, None], neginf=0.0).abs()
            d_delta = (G.abs() * (out_e[b, :m, h] + U32 * D * o.abs())).sum(dim=1, keepdim=True) + U32 * 4 * gl.abs()
            d_dP = U32 * 2 * D * (G.abs() @ V.abs().t())
            dS_e = p * (d_dP + d_delta) + (u + dp_rel) * dS.abs() + p * (dP.abs() + delta.abs()) * 4 * U32 + small * (w > 0)
            p_e = (u + dp_rel) * p + small * (w > 0)
            rows = U32 * 2 * max(m * g, n)
            dq[b, :m, h] = dS @ K * scale
            dq_e[b, :m, h] = (dS_e @ K.abs() + rows * (dS.abs() @ K.abs())) * scale
            dk[b, :n, hk] += dS.t() @ Q * scale
            dk_e[b, :n, hk] += (dS_e.t() @ Q.abs() + rows * (dS.abs().t() @ Q.abs())) * scale
            dv[b, :n, hk] += p.t() @ G
            dv_e[b, :n, hk] += p_e.t() @ G.abs() + rows * (p.t() @ G.abs())
    r = {"out": (out, out_e), "lse": (lse, lse_e)}
    if grad_out is not None:
        for name, x, x_e in (("dq", dq, dq_e), ("dk", dk, dk_e), ("dv", dv, dv_e)):
            r[name] = (x, x_e + u * x.abs() + small)
    return r


def check(name, got, want, bound):
    """got within bound of want everywhere; infinities equal."""
    got = got.double().to(want.device)
    assert got.shape == want.shape, f"{name}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got) & (got == want), inf), f"{name}: infinities differ"
    off = torch.where(inf, 0.0, (got - want).abs())
    assert not torch.isnan(off).any(), f"{name}: NaN"
    bad = off > bound
    if bad.any():
        i = int((off - bound).flatten().argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off; worst at {i}: got {got.flatten()[i].item():.6g}, want "
                             f"{want.flatten()[i].item():.6g}, bound {bound.expand_as(want).flatten()[i].item():.3g}")


def choose(B, Hk, nQ, nK, topk, gen):
    """Ascending random choices of `topk` blocks (all, then -1, where there are fewer)."""
    score = torch.rand((B, Hk, nQ, nK), generator=gen)
    k = min(topk, nK)
    lists = score.topk(k, dim=-1).indices.sort(dim=-1).values.to(torch.int32)
    pad = torch.full((B, Hk, nQ, topk - k), -1, dtype=torch.int32)
    return torch.cat([lists, pad], dim=-1)
