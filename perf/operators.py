"""What is measured of the transformer-block operators: packed attention and axial rotary positions.

``listed()`` and ``draw()`` give cases, ``prepare()`` the tensors a user's program holds before the
call, ``run()`` one pass (the plain form in elementary float32 torch operations, or the package's
own calls where ``own`` is set), ``work()`` what a pass cannot do without and ``exact()`` the
result from the definition in float64.

Attention lengths are written as text: comma-separated counts of tokens, ``CxN`` standing for C
sequences of N.  An empty ``keys`` means that queries and keys are the same tokens.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"


# ---- cases -----------------------------------------------------------------------------------
def listed():
    return [
        # One image at inference: the decoder's self-attention over its 300 queries, 8 heads of 32
        # channels (hidden 256).  Latency is what counts.
        {"name": "queries_fwd", "op": "attention", "train": False, "lengths": "300", "keys": "", "heads": 8,
         "kv_heads": 8, "dim": 32, "causal": False, "lse": False},
        # The same layer in a training step: 8 images x 13 detection groups, each group of 300
        # queries attending within itself, forward and gradients.
        {"name": "groups_train", "op": "attention", "train": True, "lengths": "104x300", "keys": "", "heads": 8,
         "kv_heads": 8, "dim": 32, "causal": False, "lse": False},
        # The windowed ViT backbone (6 heads of 64): 8 images of 24 x 24 patches in 2 x 2 windows
        # of 144 patches and a class token.
        {"name": "windows_fwd", "op": "attention", "train": False, "lengths": "32x145", "keys": "", "heads": 6,
         "kv_heads": 6, "dim": 64, "causal": False, "lse": False},
        # The backbone's unwindowed blocks in training on images of unequal size, packed without
        # padding: from a single token to a 40 x 40 map.
        {"name": "images_train", "op": "attention", "train": True,
         "lengths": "577,1601,1,241,1025,37,785,1297,900,577,128,129,401,1157,677,311", "keys": "", "heads": 6,
         "kv_heads": 6, "dim": 64, "causal": False, "lse": False},
        # Decoder queries of 8 images over feature tokens of unequal count, one image without any
        # (its rows are empty), channels that fill no tile; the log-sum-exp is returned too.
        {"name": "cross_fwd", "op": "attention", "train": False, "lengths": "8x300",
         "keys": "576,2304,0,1600,33,1,900,4000", "heads": 8, "kv_heads": 8, "dim": 80, "causal": False, "lse": True},
        # Text prompts of unequal length packed in one call, causal, 4 query heads to a key head.
        {"name": "prompt_fwd", "op": "attention", "train": False, "lengths": "4096,1,777,2048,130,3000", "keys": "",
         "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "lse": True},
        # Training on long causal sequences with grouped heads: the largest case.
        {"name": "prompt_train", "op": "attention", "train": True, "lengths": "8192,3001,130", "keys": "", "heads": 8,
         "kv_heads": 2, "dim": 128, "causal": True, "lse": False},
        # Serving: one new token of each of 8 sequences over all its keys.
        {"name": "one_token_fwd", "op": "attention", "train": False, "lengths": "8x1",
         "keys": "16384,9000,1,12345,4096,16000,777,13001", "heads": 16, "kv_heads": 4, "dim": 128, "causal": True,
         "lse": False},
        # One image's 24 x 24 patches, two axes: the smallest call.
        {"name": "rotary_image_fwd", "op": "rotary", "train": False, "tokens": 576, "heads": 6, "kv_heads": 6,
         "dim": 64, "rotary": 64, "axes": 2, "extent": 24, "interleaved": False, "type": "bf16", "real": False},
        # Video tokens with time, height and width, grouped heads of 128 channels.
        {"name": "rotary_video_fwd", "op": "rotary", "train": False, "tokens": 32768, "heads": 16, "kv_heads": 4,
         "dim": 128, "rotary": 128, "axes": 3, "extent": 512, "interleaved": False, "type": "bf16", "real": False},
        # A float32 training step of the backbone, coordinates as real numbers.
        {"name": "rotary_image_train", "op": "rotary", "train": True, "tokens": 8 * 577, "heads": 6, "kv_heads": 6,
         "dim": 64, "rotary": 64, "axes": 2, "extent": 24, "interleaved": False, "type": "f32", "real": True},
        # Odd everything: interleaved pairs over part of the channels, an odd count of tokens and
        # heads, a single key head.
        {"name": "rotary_part_train", "op": "rotary", "train": True, "tokens": 20011, "heads": 7, "kv_heads": 1,
         "dim": 80, "rotary": 48, "axes": 3, "extent": 100, "interleaved": True, "type": "bf16", "real": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.3:
        kv = rng.choice([1, 2, 3, 4, 6, 8])
        group = rng.choice([1, 1, 2, 4, 7])
        dim = rng.choice([32, 64, 72, 80, 128])
        kind = rng.choice(["bf16", "bf16", "f32"])
        axes = rng.choice([1, 2, 3])
        # Bounded by the largest listed rotation's bytes.
        most = 300_000_000 // (4 * kv * (group + 1) * dim * (4 if kind == "f32" else 2))
        return {"op": "rotary", "train": rng.random() < 0.5, "tokens": _spread(rng, 1, most), "heads": kv * group,
                "kv_heads": kv, "dim": dim, "rotary": dim if rng.random() < 0.6 else 2 * rng.randint(axes, dim // 2),
                "axes": axes, "extent": _spread(rng, 2, 64 if kind == "f32" else 4000),
                "interleaved": rng.random() < 0.4, "type": kind, "real": rng.random() < 0.3}
    kv = rng.choice([1, 2, 4, 6, 8])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8]) if kv <= 4 else 1
    dim = rng.choice([32, 64, 64, 80, 128, 128])
    longest = _spread(rng, 1, 6000)
    form = rng.choice(["self", "self", "self", "cross", "token"])
    # Bounded by the largest listed case: sum of squared longest lengths times heads.
    most = max(1, min(64, int(8 * 3 * 8192 ** 2 / (max(1, longest) ** 2 * kv * group * 2))))
    count = _spread(rng, 1, most)
    some = lambda hi: [hi] + [rng.randint(0 if rng.random() < 0.1 else 1, hi) for _ in range(count - 1)]  # noqa: E731
    keys = some(longest)
    lengths = keys if form == "self" else [1] * count if form == "token" else some(_spread(rng, 1, 900))
    return {"op": "attention", "train": form != "token" and rng.random() < 0.5,
            "lengths": ",".join(map(str, lengths)), "keys": "" if form == "self" else ",".join(map(str, keys)),
            "heads": kv * group, "kv_heads": kv, "dim": dim, "causal": form != "cross" and rng.random() < 0.6,
            "lse": rng.random() < 0.3}


def _lengths(text):
    out = []
    for part in text.split(","):
        count, _, n = part.rpartition("x")
        out += [int(n)] * (int(count) if count else 1)
    return out


# ---- inputs ----------------------------------------------------------------------------------
def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV)


def _places(lengths):
    """Sequence and place of every packed row, and the packed row of every padded place."""
    n = torch.tensor(lengths, dtype=torch.int64, device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=DEV), n)
    start = n.cumsum(0) - n
    place = torch.arange(int(n.sum()), device=DEV) - start[seq]
    rows = start[:, None] + torch.arange(max(1, int(n.max())), device=DEV)
    return {"n": n, "seq": seq, "place": place, "rows": rows.clamp_(max=max(0, int(n.sum()) - 1))}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV)  # noqa: E731
    heads, kv, dim, train = case["heads"], case["kv_heads"], case["dim"], case["train"]
    state = {"case": case}
    if case["op"] == "attention":
        lengths = _lengths(case["lengths"])
        keys = _lengths(case["keys"]) if case["keys"] else lengths
        # Activations as a fused projection leaves them: rows of [heads | key heads | value heads].
        if case["keys"]:
            q = normal(sum(lengths), heads, dim).to(torch.bfloat16)
            k, v = normal(sum(keys), 2 * kv, dim).to(torch.bfloat16).split((kv, kv), 1)
        else:
            q, k, v = normal(sum(lengths), heads + 2 * kv, dim).to(torch.bfloat16).split((heads, kv, kv), 1)
        state.update(q=q, k=k, v=v, offsets=_offsets(lengths), at=_places(lengths))
        state.update(key_offsets=_offsets(keys) if case["keys"] else None,
                     key_at=_places(keys) if case["keys"] else state["at"])
        if train:
            state["g"] = normal(sum(lengths), heads, dim).to(torch.bfloat16)
            for name in ("q", "k", "v"):
                state[name] = state[name].detach().requires_grad_(True)
        return state
    dtype = torch.float32 if case["type"] == "f32" else torch.bfloat16
    tokens, axes, half = case["tokens"], case["axes"], case["rotary"] // 2
    q, k = normal(tokens, heads + kv, dim).to(dtype).split((heads, kv), 1)
    if case["real"]:
        positions = torch.rand((tokens, axes), generator=gen, device=DEV) * case["extent"]
    else:
        positions = torch.randint(0, case["extent"], (tokens, axes), generator=gen, device=DEV, dtype=torch.int32)
    sections = [half // axes + (1 if a < half % axes else 0) for a in range(axes)]
    inv_freq = torch.cat([100.0 ** (-torch.arange(n, device=DEV, dtype=torch.float32) / max(1, n)) for n in sections])
    state.update(q=q, k=k, positions=positions, inv_freq=inv_freq, sections=sections,
                 axis=torch.repeat_interleave(torch.arange(axes, device=DEV), torch.tensor(sections, device=DEV)))
    if train:
        state["gq"], state["gk"] = normal(tokens, heads, dim).to(dtype), normal(tokens, kv, dim).to(dtype)
        state["q"], state["k"] = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    return state


# ---- one pass --------------------------------------------------------------------------------
def run(state):
    if state["case"]["op"] == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    return _own_rotary(state) if own else _plain_rotary(state)


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own_attention(state):
    case = state["case"]
    got = _package().packed_attention(state["q"], state["k"], state["v"], state["offsets"], state["key_offsets"],
                                      causal=case["causal"], return_lse=case["lse"])
    out, lse = got if case["lse"] else (got, None)
    answer = {"out": out}
    if case["lse"]:
        answer["lse"] = lse
    if case["train"]:
        answer["dq"], answer["dk"], answer["dv"] = torch.autograd.grad(out, (state["q"], state["k"], state["v"]),
                                                                       state["g"])
    return answer


def _own_rotary(state):
    case = state["case"]
    q, k = _package().axial_rotary(state["q"], state["k"], state["positions"], state["inv_freq"], state["sections"],
                                   interleaved=case["interleaved"])
    answer = {"q": q, "k": k}
    if case["train"]:
        answer["dq"], answer["dk"] = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["gq"], state["gk"]))
    return answer


@torch.no_grad()
def _plain_attention(state):
    """Sequences padded to the longest, all scores formed, masked and normalised."""
    case, at, key_at = state["case"], state["at"], state["key_at"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    batch, lq, lk = at["rows"].shape[0], at["rows"].shape[1], key_at["rows"].shape[1]
    group, scale = heads // kv, dim ** -0.5

    def queries(x):  # packed [T, H, D] -> [B, Hkv, G * Lq, D]
        return x.float()[at["rows"]].reshape(batch, lq, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(
            batch, kv, group * lq, dim)

    def keys(x):
        return x.float()[key_at["rows"]].transpose(1, 2)

    def unpad(x):
        return x.reshape(batch, kv, group, lq, -1).permute(0, 3, 1, 2, 4).reshape(batch, lq, heads, -1)[
            at["seq"], at["place"]]

    q, k = queries(state["q"]), keys(state["k"])
    i = torch.arange(lq, device=DEV)[:, None]
    j = torch.arange(lk, device=DEV)[None, :]
    nq, nk = at["n"][:, None, None], key_at["n"][:, None, None]
    allowed = (i < nq) & (j < nk)
    if case["causal"]:
        allowed &= j <= i + nk - nq
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(batch, kv, group, lq, lk)
    scores.masked_fill_(~allowed[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    p = p.view(batch, kv, group * lq, lk)
    v = keys(state["v"])
    answer = {"out": unpad(torch.matmul(p, v)).to(torch.bfloat16)}
    if case["lse"]:
        answer["lse"] = unpad(top + total.log()).squeeze(-1).t()
    if case["train"]:
        g = queries(state["g"])
        dv = torch.matmul(p.transpose(-1, -2), g)
        ds = torch.matmul(g, v.transpose(-1, -2))
        ds = ds.sub_((ds * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        answer["dq"] = unpad(torch.matmul(ds, k)).to(torch.bfloat16)
        dk = torch.matmul(ds.transpose(-1, -2), q)
        answer["dk"], answer["dv"] = (
            x.transpose(1, 2)[key_at["seq"], key_at["place"]].to(torch.bfloat16) for x in (dk, dv))
    return answer


@torch.no_grad()
def _plain_rotary(state):
    case = state["case"]
    angle = state["positions"].float()[:, state["axis"]] * state["inv_freq"]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    turn = 2 * cos.shape[-1]

    def rotated(x, sin):
        part, rest = x.float()[..., :turn], x[..., turn:]
        if case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = part[..., :turn // 2], part[..., turn // 2:]
            part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((part.to(x.dtype), rest), -1)

    answer = {"q": rotated(state["q"], sin), "k": rotated(state["k"], sin)}
    if case["train"]:
        answer["dq"], answer["dk"] = rotated(state["gq"], -sin), rotated(state["gk"], -sin)
    return answer


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    heads, kv, dim, train = case["heads"], case["kv_heads"], case["dim"], case["train"]
    if case["op"] == "rotary":
        size = 4 if case["type"] == "f32" else 2
        values = case["tokens"] * (heads + kv) * dim
        turned = case["tokens"] * (heads + kv) * case["rotary"]
        # q and k in and out, their cotangents in and gradients out, positions once; a rotated
        # pair takes four products and two sums.
        return {"bytes": (4 if train else 2) * values * size + case["tokens"] * case["axes"] * 4,
                "flops": 3 * turned * (2 if train else 1)}
    lengths = _lengths(case["lengths"])
    keys = _lengths(case["keys"]) if case["keys"] else lengths
    if case["causal"]:
        # Row i of n sees min(m, max(0, i + 1 + m - n)) of m keys.
        pairs = sum(n * m - n * (n - 1) // 2 if m >= n else m * (m + 1) // 2 for n, m in zip(lengths, keys))
    else:
        pairs = sum(n * m for n, m in zip(lengths, keys))
    rows, key_rows = sum(lengths), sum(keys)
    moved = 2 * rows * heads * dim + 2 * key_rows * kv * dim  # q, out; k, v
    if train:
        moved += 2 * rows * heads * dim + 2 * key_rows * kv * dim  # g, dq; dk, dv
    # Two products forward; four more for the gradients, the scores kept.
    return {"bytes": 2 * moved + (4 * rows * heads if case["lse"] else 0),
            "flops": (12 if train else 4) * pairs * heads * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_attention(state) if case["op"] == "attention" else _exact_rotary(state)


def _exact_attention(state):
    """One sequence and one head at a time, from the sums of the definition."""
    case = state["case"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    lengths = _lengths(case["lengths"])
    keys = _lengths(case["keys"]) if case["keys"] else lengths
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    out, lse = torch.zeros_like(q), torch.full((case["heads"], q.shape[0]), -math.inf, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    r = c = 0
    for n, m in zip(lengths, keys):
        for h in range(case["heads"] if n and m else 0):
            rows, cols = slice(r, r + n), slice(c, c + m)
            kh, vh = k[cols, h // group], v[cols, h // group]
            s = scale * (q[rows, h] @ kh.T)
            if case["causal"]:
                s[torch.ones_like(s, dtype=torch.bool).triu(m - n + 1)] = -math.inf
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(z == -math.inf, 0.0, z)[:, None])
            out[rows, h], lse[h, rows] = p @ vh, z
            if case["train"]:
                g = state["g"][rows, h].double()
                dp = g @ vh.T
                ds = scale * p * (dp - (g * out[rows, h]).sum(-1, keepdim=True))
                dq[rows, h] = ds @ kh
                dk[cols, h // group] += ds.T @ q[rows, h]
                dv[cols, h // group] += p.T @ g
        r, c = r + n, c + m
    answer = {"out": out}
    if case["lse"]:
        answer["lse"] = lse
    if case["train"]:
        answer.update(dq=dq, dk=dk, dv=dv)
    return answer


def _exact_rotary(state):
    """As products of complex numbers: x1 + i x2 times exp(i theta)."""
    case, half = state["case"], state["inv_freq"].numel()
    theta = state["positions"].double()[:, state["axis"]] * state["inv_freq"].double()
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)

    def rotated(x, turn):
        y = x.detach().double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    answer = {"q": rotated(state["q"], turn), "k": rotated(state["k"], turn)}
    if case["train"]:
        answer.update(dq=rotated(state["gq"], turn.conj()), dk=rotated(state["gk"], turn.conj()))
    return answer
