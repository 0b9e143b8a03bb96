"""What is measured of the video-attention operators: rotary positions over several axes, block means, the choice of key blocks, and
attention over the chosen blocks, forward and backward.

`run` computes an operator in its plain form (elementary torch operations, 32 bits, one rounding at the end) or, with `own` set, through
the framework's entry points; `exact` computes the same from the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_DEVICE = "cuda"


def _ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    package = os.path.join(root, "stable-fast_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import sfast  # noqa: F401  registers the operators
    return torch.ops.sfast, torch.ops.sfast_xformers


# ---- cases ---------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one new token of four conversations, far into its sequence: latency
        {"name": "rope_token", "kind": "rope", "B": 4, "T": 1, "Y": 1, "X": 1, "H": 24, "Hk": 8, "D": 128, "sections": "16,56,56", "dtype": "bf16",
         "interleaved": True, "grad": False, "start": 1000000, "step": 0.0},
        # q and k of all tokens of a clip: 25 frames of 36 x 64 latents
        {"name": "rope_video", "kind": "rope", "B": 1, "T": 25, "Y": 36, "X": 64, "H": 24, "Hk": 24, "D": 128, "sections": "44,42,42", "dtype": "bf16",
         "interleaved": True, "grad": False, "start": 0, "step": 0.0},
        # fine-tuning in 32 bits: odd grid, fractional positions (a resolution the model was not trained on), a part of the head is not rotated
        {"name": "rope_grad_odd", "kind": "rope", "B": 2, "T": 3, "Y": 17, "X": 23, "H": 6, "Hk": 3, "D": 80, "sections": "16,24,24", "dtype": "f32",
         "interleaved": False, "grad": True, "start": 0, "step": 0.63},
        # block means of a padded batch's key cache
        {"name": "means_cache", "kind": "means", "B": 4, "S": 8191, "H": 8, "D": 128, "block": 64, "dtype": "bf16", "ragged": True},
        # block means of a clip's queries
        {"name": "means_video", "kind": "means", "B": 1, "S": 57600, "H": 10, "D": 64, "block": 128, "dtype": "f16", "ragged": False},
        # one token's choice among the blocks of a long cache
        {"name": "topk_token", "kind": "topk", "B": 8, "nQ": 1, "nK": 2048, "H": 32, "Hk": 8, "D": 128, "topk": 64, "block": 64, "ragged": True},
        # every query block of a clip chooses a tenth of the key blocks
        {"name": "topk_video", "kind": "topk", "B": 1, "nQ": 450, "nK": 900, "H": 10, "Hk": 10, "D": 64, "topk": 90, "block": 64, "ragged": False},
        # one new token against a long cache, grouped heads, a padded batch
        {"name": "attend_token", "kind": "attend", "B": 4, "Sq": 1, "Sk": 65536, "H": 32, "Hk": 8, "D": 128, "block_q": 128, "block_k": 64, "topk": 64,
         "dtype": "bf16", "ragged": True, "grad": False},
        # a small image beside a prompt: odd lengths, grouped heads, a head dimension that fills no tile
        {"name": "attend_ragged", "kind": "attend", "B": 2, "Sq": 1000, "Sk": 1337, "H": 6, "Hk": 3, "D": 80, "block_q": 64, "block_k": 64, "topk": 8,
         "dtype": "f16", "ragged": True, "grad": False},
        # a clip of 21 frames of 30 x 52 latents, an eighth of the key blocks
        {"name": "attend_video", "kind": "attend", "B": 1, "Sq": 32760, "Sk": 32760, "H": 24, "Hk": 24, "D": 128, "block_q": 128, "block_k": 64, "topk": 64,
         "dtype": "bf16", "ragged": False, "grad": False},
        # a training step's attention on small odd sizes
        {"name": "attend_grad_ragged", "kind": "attend", "B": 2, "Sq": 777, "Sk": 1029, "H": 8, "Hk": 4, "D": 64, "block_q": 128, "block_k": 128, "topk": 4,
         "dtype": "f16", "ragged": True, "grad": True},
        # a training step's attention over 25 frames of 18 x 32 latents
        {"name": "attend_grad_video", "kind": "attend", "B": 1, "Sq": 14400, "Sk": 14400, "H": 20, "Hk": 20, "D": 64, "block_q": 128, "block_k": 64, "topk": 32,
         "dtype": "bf16", "ragged": False, "grad": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    hk = rng.randint(1, most)
    return hk * rng.randint(1, max(1, min(4, most // hk))), hk


def _draw(rng):
    kind = rng.choice(["rope", "rope", "means", "topk", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "rope":
        h, hk = _heads(rng, 24)
        d = rng.choice([40, 64, 80, 96, 128])
        axes = rng.randint(1, 4)
        sections = [2 * rng.randint(1, d // (2 * axes)) for _ in range(axes)]
        return {"kind": kind, "B": rng.randint(1, 4), "T": _log_int(rng, 1, 25), "Y": _log_int(rng, 1, 64), "X": _log_int(rng, 1, 64), "H": h, "Hk": hk, "D": d,
                "sections": ",".join(map(str, sections)), "dtype": rng.choice(["bf16", "f16", "f32"]), "interleaved": rng.random() < 0.5,
                "grad": rng.random() < 0.5, "start": rng.choice([0, _log_int(rng, 1, 1000000)]), "step": rng.choice([0.0, rng.uniform(0.1, 2.0)])}
    if kind == "means":
        return {"kind": kind, "B": rng.randint(1, 4), "S": _log_int(rng, 1, 57600), "H": rng.randint(1, 24), "D": rng.choice([40, 64, 80, 96, 128]),
                "block": rng.choice([64, 128]), "dtype": rng.choice(["bf16", "f16", "f32"]), "ragged": rng.random() < 0.5}
    if kind == "topk":
        h, hk = _heads(rng, 24)
        nk = _log_int(rng, 1, 2048)
        return {"kind": kind, "B": rng.randint(1, 8), "nQ": _log_int(rng, 1, 450), "nK": nk, "H": h, "Hk": hk, "D": rng.choice([40, 64, 80, 96, 128]),
                "topk": _log_int(rng, 1, min(128, nk)), "block": rng.choice([64, 128]), "ragged": rng.random() < 0.5}
    h, hk = _heads(rng, 24)
    grad = rng.random() < 0.4
    bk = rng.choice([64, 128])
    sk = _log_int(rng, 1, 32768)
    sq = rng.choice([1, _log_int(rng, 1, 32768)])
    return {"kind": kind, "B": rng.randint(1, 4), "Sq": sq, "Sk": sk, "H": h, "Hk": hk, "D": rng.choice([40, 64, 80, 96, 128]), "block_q": rng.choice([64, 128]),
            "block_k": bk, "topk": _log_int(rng, 1, min(64, -(-sk // bk))), "dtype": dtype, "ragged": rng.random() < 0.5, "grad": grad}


def draw(rng):
    most = {}
    for case in listed():
        key = (case["kind"], case.get("grad", False))
        w = work(case)
        most[key] = (max(most.get(key, (0, 0))[0], w["bytes"]), max(most.get(key, (0, 0))[1], w["flops"]))
    most[("rope", True)] = most[("rope", False)]
    while True:
        case = _draw(rng)
        w = work(case)
        top = most[(case["kind"], case.get("grad", False))]
        if w["bytes"] <= top[0] and w["flops"] <= top[1]:
            return case


# ---- inputs --------------------------------------------------------------------------------------------------------------------------
def _lengths(batch, size, ragged):
    """Valid rows of each sequence: the first is full, the others fall off; the last of four or more is a free slot of the batch."""
    if not ragged:
        return [size] * batch
    out = [size - (size * b) // (batch + 1) - (b & 1) for b in range(batch)]
    if batch >= 4:
        out[-1] = 0
    return [max(0, n) for n in out]


def _randn(shape, dtype, gen, spread=1.0):
    x = torch.randn(shape, generator=gen, device=_DEVICE, dtype=torch.float32 if dtype is torch.float32 else dtype)
    return x.mul_(spread) if spread != 1.0 else x


def _positions(case):
    """[S, A]: the first axis counts frames (or tokens), the next rows, columns; a fourth repeats the frame."""
    axes = len(case["sections"].split(","))
    t, y, x = torch.meshgrid(torch.arange(case["T"]), torch.arange(case["Y"]), torch.arange(case["X"]), indexing="ij")
    grid = torch.stack([t, y, x, t], dim=-1).reshape(-1, 4)[:, :axes] + case["start"]
    if case["step"]:
        grid = grid.to(torch.float32) * case["step"]
    return grid.to(_DEVICE).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    state = {"case": case}
    kind = case["kind"]
    if kind == "rope":
        dt = _DTYPES[case["dtype"]]
        s = case["T"] * case["Y"] * case["X"]
        state["positions"] = _positions(case)
        state["q"] = _randn((case["B"], s, case["H"], case["D"]), dt, gen)
        state["k"] = _randn((case["B"], s, case["Hk"], case["D"]), dt, gen)
        if case["grad"]:
            state["dq"] = _randn((case["B"], s, case["H"], case["D"]), dt, gen)
            state["dk"] = _randn((case["B"], s, case["Hk"], case["D"]), dt, gen)
            state["q"].requires_grad_(True)
            state["k"].requires_grad_(True)
    elif kind == "means":
        state["x"] = _randn((case["B"], case["S"], case["H"], case["D"]), _DTYPES[case["dtype"]], gen)
        state["lengths"] = torch.tensor(_lengths(case["B"], case["S"], True), dtype=torch.int32, device=_DEVICE) if case["ragged"] else None
    elif kind == "topk":
        # means of 64 and more rows, neighbours alike
        state["qm"] = _randn((case["B"], case["nQ"], case["H"], case["D"]), torch.float32, gen, 0.2)
        state["km"] = _randn((case["B"], case["nK"], case["Hk"], case["D"]), torch.float32, gen, 0.2)
        state["lengths"] = torch.tensor(_lengths(case["B"], case["nK"] * case["block"], True), dtype=torch.int32, device=_DEVICE) if case["ragged"] else None
    else:
        dt = _DTYPES[case["dtype"]]
        b, sq, sk, h, hk, d = (case[n] for n in ("B", "Sq", "Sk", "H", "Hk", "D"))
        state["q"] = _randn((b, sq, h, d), dt, gen)
        state["k"] = _randn((b, sk, hk, d), dt, gen)
        state["v"] = _randn((b, sk, hk, d), dt, gen)
        lens = _lengths(b, sk, case["ragged"])
        state["lengths"] = torch.tensor(lens, dtype=torch.int32, device=_DEVICE) if case["ragged"] else None
        # a choice as block_topk makes it: the nearest blocks and some far ones, ascending, -1 where a sequence has no more
        nq, nk = -(-sq // case["block_q"]), -(-sk // case["block_k"])
        score = torch.randn((b, hk, nq, nk), generator=gen, device=_DEVICE)
        at = torch.arange(nq, device=_DEVICE)[:, None] * (nk / nq)
        score += 4.0 * torch.exp(-(torch.arange(nk, device=_DEVICE)[None, :] - at).abs() / 4.0)
        first = torch.arange(nk, device=_DEVICE) * case["block_k"]
        outside = first[None, :] >= torch.tensor(lens, device=_DEVICE)[:, None]
        score.masked_fill_(outside[:, None, None, :], -math.inf)
        top, index = torch.topk(score, case["topk"], dim=-1)
        index = torch.where(torch.isinf(top), nk, index).sort(dim=-1).values
        state["blocks"] = torch.where(index == nk, -1, index).to(torch.int32).contiguous()
        if case["grad"]:
            state["do"] = _randn((b, sq, h, d), dt, gen)
            for n in ("q", "k", "v"):
                state[n].requires_grad_(True)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    case = state["case"]
    sfast_ops, attn = _ops()
    kind = case["kind"]
    if kind == "rope":
        sections = [int(n) for n in case["sections"].split(",")]
        q, k = sfast_ops.rotary_embedding_nd(state["q"], state["k"], state["positions"], sections, 10000.0, case["interleaved"])
        if not case["grad"]:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (state["q"], state["k"]), (state["dq"], state["dk"]))
    if kind == "means":
        return attn.block_means(state["x"], case["block"], state["lengths"])
    if kind == "topk":
        return attn.block_topk(state["qm"], state["km"], case["topk"], case["block"], state["lengths"])
    out, lse = attn.block_sparse_attention(state["q"], state["k"], state["v"], state["blocks"], case["block_q"], case["block_k"], state["lengths"])
    if not case["grad"]:
        return out, lse
    return (out.detach(), lse.detach()) + torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"])


def _run_plain(state):
    with torch.no_grad():
        return {"rope": _plain_rope, "means": _plain_means, "topk": _plain_topk, "attend": _plain_attend}[state["case"]["kind"]](state)


def _plain_rope(state):
    case = state["case"]
    sections = [int(n) for n in case["sections"].split(",")]
    cos, sin = [], []
    for axis, size in enumerate(sections):
        freq = 10000.0 ** (-torch.arange(0, size, 2, device=_DEVICE, dtype=torch.float64) / size)
        angle = state["positions"][:, axis, None].double() * freq
        cos.append(angle.cos().float()[None, :, None, :])
        sin.append(angle.sin().float()[None, :, None, :])

    def rotate(x, sign):
        y, at = x.float(), 0
        parts = []
        for axis, size in enumerate(sections):
            p = y[..., at:at + size]
            a, b = (p[..., 0::2], p[..., 1::2]) if case["interleaved"] else (p[..., :size // 2], p[..., size // 2:])
            c, s = cos[axis], sign * sin[axis]
            pair = (a * c - b * s, a * s + b * c)
            parts.append(torch.stack(pair, dim=-1).flatten(-2) if case["interleaved"] else torch.cat(pair, dim=-1))
            at += size
        parts.append(y[..., at:])
        return torch.cat(parts, dim=-1).to(x.dtype)

    out = (rotate(state["q"], 1.0), rotate(state["k"], 1.0))
    return out + (rotate(state["dq"], -1.0), rotate(state["dk"], -1.0)) if case["grad"] else out


def _plain_means(state):
    case = state["case"]
    b, s, h, d, block = (case[n] for n in ("B", "S", "H", "D", "block"))
    n = -(-s // block)
    lengths = state["lengths"] if state["lengths"] is not None else torch.full((b,), s, device=_DEVICE)
    valid = torch.arange(n * block, device=_DEVICE)[None, :] < lengths[:, None]
    x = torch.nn.functional.pad(state["x"], (0, 0, 0, 0, 0, n * block - s))
    x = torch.where(valid[:, :, None, None], x.float(), 0.0).reshape(b, n, block, h, d)
    count = valid.reshape(b, n, block).sum(dim=2).clamp(min=1)
    return (x.sum(dim=2, dtype=torch.float64) / count[:, :, None, None]).float()


def _choose(score, topk, counts):
    """The topk best of the last axis among the first `counts`, ties to the lowest index; ascending, then -1."""
    nk = score.shape[-1]
    at = torch.arange(nk, device=score.device)
    valid = (at[None, :] < counts[:, None])[:, None, None, :]
    order = torch.where(valid, score, -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., :topk]
    order = torch.where(torch.gather(valid.expand_as(score), -1, order), order, nk).sort(dim=-1).values
    return torch.where(order == nk, -1, order).to(torch.int32)


def _plain_topk(state):
    case = state["case"]
    b, nq, nk, h, hk, d = (case[n] for n in ("B", "nQ", "nK", "H", "Hk", "D"))
    # in 64 bits: a choice stands next to a border
    q = state["qm"].double().reshape(b, nq, hk, h // hk, d).sum(dim=3).permute(0, 2, 1, 3)
    score = torch.matmul(q, state["km"].double().permute(0, 2, 3, 1).contiguous())
    counts = torch.full((b,), nk, device=_DEVICE) if state["lengths"] is None else (state["lengths"] + case["block"] - 1) // case["block"]
    out = _choose(score, case["topk"], counts)
    return out


def _plain_attend(state):
    case = state["case"]
    b, sq, sk, h, hk, d, bq, bk, topk = (case[n] for n in ("B", "Sq", "Sk", "H", "Hk", "D", "block_q", "block_k", "topk"))
    g, nq, scale = h // hk, -(-case["Sq"] // case["block_q"]), case["D"] ** -0.5
    lengths = state["lengths"] if state["lengths"] is not None else torch.full((b,), sk, device=_DEVICE)
    k = state["k"].permute(0, 2, 1, 3).reshape(b * hk * sk, d)
    v = state["v"].permute(0, 2, 1, 3).reshape(b * hk * sk, d)

    def rows(x):   # [B, Sq, H, D] -> [B * Hk * nQ, G * block_q, D]
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nq * bq - sq)).reshape(b, nq, bq, hk, g, d)
        return x.permute(0, 3, 1, 4, 2, 5).reshape(b * hk * nq, g * bq, d)

    def back(x):   # [B * Hk * nQ, G * block_q, E] -> [B, Sq, H, E]
        e = x.shape[-1]
        return x.reshape(b, hk, nq, g, bq, e).permute(0, 2, 4, 1, 3, 5).reshape(b, nq * bq, h, e)[:, :sq]

    q = rows(state["q"])
    do = rows(state["do"]) if case["grad"] else None
    base = torch.arange(b * hk, device=_DEVICE).repeat_interleave(nq) * sk
    limit = lengths.repeat_interleave(hk * nq)
    lists = state["blocks"].reshape(b * hk * nq, topk).long()
    out = torch.empty(q.shape, dtype=torch.float32, device=_DEVICE)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=_DEVICE)
    if case["grad"]:
        dq = torch.empty_like(out)
        dk = torch.zeros((b * hk * sk, d), dtype=torch.float32, device=_DEVICE)
        dv = torch.zeros_like(dk)
    step = max(1, (1 << 29) // (topk * bk * max(d, g * bq)))
    for at in range(0, q.shape[0], step):
        end = slice(at, at + step)
        place = lists[end, :, None] * bk + torch.arange(bk, device=_DEVICE)
        place = place.reshape(place.shape[0], -1)
        valid = (place >= 0) & (place < limit[end, None]) & (lists[end] >= 0).repeat_interleave(bk, dim=1)
        place = torch.where(valid, place, 0) + base[end, None]
        kg, vg, qg = k[place].float(), torch.where(valid[..., None], v[place].float(), 0.0), q[end].float()
        s = torch.where(valid[:, None, :], torch.matmul(qg, kg.transpose(1, 2)) * scale, -math.inf)
        top = s.amax(dim=-1, keepdim=True)
        top = torch.where(torch.isinf(top), 0.0, top)
        p = torch.exp(s - top)
        total = p.sum(dim=-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        o = torch.matmul(p, vg)
        out[end] = o
        lse[end] = (torch.log(total) + top)[..., 0]
        if case["grad"]:
            dog = do[end].float()
            dp = torch.matmul(dog, vg.transpose(1, 2))
            ds = p * (dp - (dog * o).sum(dim=-1, keepdim=True)) * scale
            dq[end] = torch.matmul(ds, torch.where(valid[..., None], kg, 0.0))
            dkg, dvg = torch.matmul(ds.transpose(1, 2), qg), torch.matmul(p.transpose(1, 2), dog)
            dk.index_add_(0, place.reshape(-1), dkg.reshape(-1, d))
            dv.index_add_(0, place.reshape(-1), dvg.reshape(-1, d))
    result = (back(out).to(state["q"].dtype), back(lse[..., None])[..., 0].permute(0, 2, 1).contiguous())
    if case["grad"]:
        dt = state["q"].dtype
        result += (back(dq).to(dt),) + tuple(x.reshape(b, hk, sk, d).permute(0, 2, 1, 3).to(dt) for x in (dk, dv))
    return result


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "rope":
        e = 4 if case["dtype"] == "f32" else 2
        s = case["T"] * case["Y"] * case["X"]
        values = case["B"] * s * (case["H"] + case["Hk"]) * case["D"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * 2 * values * e + s * len(case["sections"].split(",")) * 8, "flops": passes * 3 * values}
    if kind == "means":
        e = 4 if case["dtype"] == "f32" else 2
        rows = sum(_lengths(case["B"], case["S"], case["ragged"]))
        n = -(-case["S"] // case["block"])
        return {"bytes": rows * case["H"] * case["D"] * e + case["B"] * n * case["H"] * case["D"] * 4, "flops": rows * case["H"] * case["D"]}
    if kind == "topk":
        blocks = [-(-n // case["block"]) for n in _lengths(case["B"], case["nK"] * case["block"], case["ragged"])]
        size = case["B"] * case["nQ"] * case["H"] * case["D"] * 4 + sum(blocks) * case["Hk"] * case["D"] * 4
        return {"bytes": size + case["B"] * case["Hk"] * case["nQ"] * case["topk"] * 4, "flops": 2 * sum(blocks) * case["nQ"] * case["Hk"] * case["D"]}
    b, sq, h, hk, d, bk = (case[n] for n in ("B", "Sq", "H", "Hk", "D", "block_k"))
    nq = -(-sq // case["block_q"])
    lens = _lengths(b, case["Sk"], case["ragged"])
    keys = [min(case["topk"] * bk, n) for n in lens]                       # keys a row attends to
    read = [min(nq * case["topk"] * bk, n) for n in lens]                  # keys a head reads at least once
    rows = b * sq * h * d * 2
    size = 2 * rows + 2 * sum(read) * hk * d * 2 + b * h * sq * 4 + b * hk * nq * case["topk"] * 4
    flops = 4 * sq * h * d * sum(keys)
    if case["grad"]:
        size += 2 * rows + 2 * b * case["Sk"] * hk * d * 2
        flops += 10 * sq * h * d * sum(keys)
    return {"bytes": size, "flops": flops}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _exact_rope, "means": _exact_means, "topk": _exact_topk, "attend": _exact_attend}[case["kind"]](state)


def _exact_rope(state):
    """Each pair as a complex number times exp(i angle)."""
    case = state["case"]

    def turn(x, conjugate):
        y, at = x.double().clone(), 0
        for axis, size in enumerate(int(n) for n in case["sections"].split(",")):
            i = torch.arange(size // 2, device=_DEVICE)
            lo, hi = (at + 2 * i, at + 2 * i + 1) if case["interleaved"] else (at + i, at + i + size // 2)
            angle = state["positions"][:, axis].double()[:, None] * torch.exp(-2.0 * i.double() / size * math.log(10000.0))[None, :]
            unit = torch.polar(torch.ones_like(angle), -angle if conjugate else angle)[None, :, None, :]
            z = torch.complex(y[..., lo], y[..., hi]) * unit
            y[..., lo], y[..., hi] = z.real, z.imag
            at += size
        return y

    out = (turn(state["q"], False), turn(state["k"], False))
    return out + (turn(state["dq"], True), turn(state["dk"], True)) if case["grad"] else out


def _exact_means(state):
    case = state["case"]
    x, block = state["x"].double(), case["block"]
    n = -(-case["S"] // block)
    out = torch.zeros((case["B"], n, case["H"], case["D"]), dtype=torch.float64, device=_DEVICE)
    for b, length in enumerate(_lengths(case["B"], case["S"], case["ragged"])):
        full = length // block
        if full:
            out[b, :full] = x[b, :full * block].reshape(full, block, case["H"], case["D"]).mean(dim=1)
        if length % block:
            out[b, full] = x[b, full * block:length].mean(dim=0)
    return out


def _exact_topk(state):
    case = state["case"]
    g = case["H"] // case["Hk"]
    out = torch.full((case["B"], case["Hk"], case["nQ"], case["topk"]), -1, dtype=torch.int32, device=_DEVICE)
    lens = _lengths(case["B"], case["nK"] * case["block"], case["ragged"])
    for b in range(case["B"]):
        n = -(-lens[b] // case["block"])
        for hk in range(case["Hk"]):
            keys = state["km"][b, :n, hk].double()
            score = sum(torch.matmul(state["qm"][b, :, hk * g + i].double(), keys.t()) for i in range(g))
            rank = (-score).argsort(dim=-1, stable=True)[:, :case["topk"]].sort(dim=-1).values
            out[b, hk, :, :rank.shape[1]] = rank.to(torch.int32)
    return out


def _exact_attend(state):
    """Dense attention in which key j counts as often for row s as the list of s's block names j's block."""
    case = state["case"]
    b, sq, sk, h, hk, d, bq, bk = (case[n] for n in ("B", "Sq", "Sk", "H", "Hk", "D", "block_q", "block_k"))
    g, scale = h // hk, d ** -0.5
    lens = _lengths(b, sk, case["ragged"])
    nq, nk = -(-sq // bq), -(-sk // bk)
    out = torch.zeros((b, sq, h, d), dtype=torch.float64, device=_DEVICE)
    lse = torch.full((b, h, sq), -math.inf, dtype=torch.float64, device=_DEVICE)
    dq = torch.zeros_like(out)
    dk = torch.zeros((b, sk, hk, d), dtype=torch.float64, device=_DEVICE)
    dv = torch.zeros_like(dk)
    rows = max(bq, ((1 << 26) // max(sk, 1)) // bq * bq)
    for ib in range(b):
        n = lens[ib]
        for head in range(h if n else 0):
            ik = head // g
            keys, values = state["k"][ib, :n, ik].double(), state["v"][ib, :n, ik].double()
            names = torch.zeros((nq, nk + 1), dtype=torch.float64, device=_DEVICE)
            lists = state["blocks"][ib, ik].long()
            names.scatter_add_(1, torch.where(lists < 0, nk, lists), torch.ones_like(lists, dtype=torch.float64))
            for at in range(0, sq, rows):
                q = state["q"][ib, at:at + rows, head].double()
                r = torch.arange(at, at + q.shape[0], device=_DEVICE) // bq
                w = names[r][:, torch.arange(n, device=_DEVICE) // bk]
                s = torch.matmul(q, keys.t()) * scale
                top = torch.where(w > 0, s, -math.inf).amax(dim=1, keepdim=True)
                e = torch.where(w > 0, w * torch.exp(s - top), 0.0)
                z = e.sum(dim=1, keepdim=True)
                p = torch.where(z > 0, e / z, 0.0)
                o = torch.matmul(p, values)
                out[ib, at:at + rows, head] = o
                lse[ib, head, at:at + rows] = torch.where(z > 0, top + torch.log(z), -math.inf)[:, 0]
                if case["grad"]:
                    do = state["do"][ib, at:at + rows, head].double()
                    dv[ib, :n, ik] += torch.matmul(p.t(), do)
                    ds = p * (torch.matmul(do, values.t()) - (do * o).sum(dim=1, keepdim=True)) * scale
                    dq[ib, at:at + rows, head] = torch.matmul(ds, keys)
                    dk[ib, :n, ik] += torch.matmul(ds.t(), q)
    return (out, lse, dq, dk, dv) if case["grad"] else (out, lse)
