"""What is measured of the operators around an attention layer and its training step: packed attention whose
scores are capped, lean on distance or have a prefix mask; norms of queries and keys with the axial rotation in the
same pass; and the global gradient norm with clipping.

``listed()`` and ``draw()`` give cases, ``prepare()`` the tensors a user's program holds before the
call, ``run()`` one pass (the plain form in elementary float32 torch operations, or the package's
own calls where ``own`` is set), ``work()`` what a pass cannot do without and ``exact()`` the
result from the definition in float64.

Counts are written as text: comma-separated numbers, ``CxN`` standing for C times N.  An empty
``keys`` means that queries and keys are the same tokens; an empty ``prefix`` that there is none.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"


# ---- cases -----------------------------------------------------------------------------------
def listed():
    return [
        # Serving with capped scores: one new token of each of 6 sequences over all its keys.
        {"name": "capped_token_fwd", "op": "attention", "train": False, "lengths": "6x1",
         "keys": "12000,7,5003,16001,900,8192", "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "cap": 30.0,
         "slopes": False, "prefix": "", "lse": False},
        # Text prompts of unequal length with capped scores, grouped heads.
        {"name": "capped_prompt_fwd", "op": "attention", "train": False, "lengths": "3500,1,611,2048,97", "keys": "",
         "heads": 16, "kv_heads": 4, "dim": 128, "causal": True, "cap": 50.0, "slopes": False, "prefix": "",
         "lse": True},
        # Long causal sequences in training, capped and leaning on distance: the largest case.
        {"name": "capped_long_train", "op": "attention", "train": True, "lengths": "7000,2501,66", "keys": "",
         "heads": 8, "kv_heads": 2, "dim": 128, "causal": True, "cap": 30.0, "slopes": True, "prefix": "",
         "lse": False},
        # An image's 576 patches and a class token, seen by every token, then a caption that is causal.
        {"name": "prefix_train", "op": "attention", "train": True, "lengths": "877,600,1200,577,705,640", "keys": "",
         "heads": 6, "kv_heads": 6, "dim": 64, "causal": True, "cap": 0.0, "slopes": False, "prefix": "6x577",
         "lse": False},
        # One image's decoder queries in order of their score, leaning on distance both ways: latency counts.
        {"name": "sloped_queries_fwd", "op": "attention", "train": False, "lengths": "300", "keys": "", "heads": 8,
         "kv_heads": 8, "dim": 32, "causal": False, "cap": 0.0, "slopes": True, "prefix": "", "lse": False},
        # One image's 24 x 24 patches, two axes: the smallest call.
        {"name": "normed_image_fwd", "op": "rotary", "train": False, "tokens": 576, "heads": 6, "kv_heads": 6,
         "dim": 64, "rotary": 64, "axes": 2, "extent": 24, "interleaved": False, "type": "bf16"},
        # Video tokens with time, height and width, grouped heads of 128 channels, forward and gradients.
        {"name": "normed_video_train", "op": "rotary", "train": True, "tokens": 32768, "heads": 16, "kv_heads": 4,
         "dim": 128, "rotary": 128, "axes": 3, "extent": 512, "interleaved": False, "type": "bf16"},
        # A float32 training step of the backbone.
        {"name": "normed_backbone_train", "op": "rotary", "train": True, "tokens": 8 * 577, "heads": 6, "kv_heads": 6,
         "dim": 64, "rotary": 64, "axes": 2, "extent": 24, "interleaved": False, "type": "f32"},
        # Odd everything: interleaved pairs over part of the channels, an odd count of tokens and
        # heads, a single key head.
        {"name": "normed_part_fwd", "op": "rotary", "train": False, "tokens": 20011, "heads": 7, "kv_heads": 1,
         "dim": 80, "rotary": 48, "axes": 3, "extent": 100, "interleaved": True, "type": "bf16"},
        # The gradients of a backbone of 12 layers of 384 channels and its decoder, each a tensor by
        # itself, clipped in float32 into the optimizer's buffer; the tensors stay from step to step.
        {"name": "clip_model", "op": "clip", "counts": "48x147456,24x589824,12x1536,133x384,226944,221184,"
         "36x65536,6x524288,6x2048,90x256,3x23296,91", "type": "f32", "out": "f32", "flat": False, "kept": True,
         "limit": 0.1},
        # The same gradients in one flat buffer, as a data-parallel step reduces them, in bf16, clipped into
        # the float32 buffer that the optimizer reads.
        {"name": "clip_flat", "op": "clip", "counts": "27361627", "type": "bf16", "out": "f32", "flat": True,
         "kept": False, "limit": 0.1},
        # One decoder layer's gradients, views of a flat buffer at odd places; the norm is below the limit.
        {"name": "clip_layer", "op": "clip", "counts": "196608,768,65536,256,16384,64,8192,32,65536,256,65536,256,"
         "262144,1024,262144,256,6x256,91", "type": "bf16", "out": "bf16", "flat": True, "kept": False, "limit": 2.0},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.25:
        return _draw_rotary(rng)
    if kind < 0.45:
        return _draw_clip(rng)
    kv = rng.choice([1, 2, 4, 6, 8])
    group = rng.choice([1, 1, 2, 3, 4, 7, 8]) if kv <= 4 else 1
    dim = rng.choice([32, 64, 64, 80, 128, 128])
    # Bounded by the largest listed case: pairs of query and key times heads.
    most = (7000 ** 2 + 2501 ** 2) // 2 * 8 // (kv * group)
    longest = _spread(rng, 1, min(5000, math.isqrt(most)))
    form = rng.choice(["self", "self", "self", "cross", "token"])
    count = _spread(rng, 1, max(1, min(64, most // longest ** 2)))
    some = lambda hi: [hi] + [rng.randint(0 if rng.random() < 0.1 else 1, hi) for _ in range(count - 1)]  # noqa: E731
    keys = some(longest)
    lengths = keys if form == "self" else [1] * count if form == "token" else some(_spread(rng, 1, 900))
    causal = form != "cross" and rng.random() < 0.7
    prefix = ",".join(str(rng.randint(0, n)) for n in keys) if causal and rng.random() < 0.35 else ""
    cap = round(math.exp(rng.uniform(math.log(8.0), math.log(60.0))), 1) if rng.random() < 0.6 else 0.0
    return {"op": "attention", "train": form != "token" and rng.random() < 0.5,
            "lengths": ",".join(map(str, lengths)), "keys": "" if form == "self" else ",".join(map(str, keys)),
            "heads": kv * group, "kv_heads": kv, "dim": dim, "causal": causal, "cap": cap,
            "slopes": rng.random() < 0.5 or (cap == 0.0 and not prefix), "prefix": prefix,
            "lse": rng.random() < 0.3}


def _draw_rotary(rng):
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
            "interleaved": rng.random() < 0.4, "type": kind}


def _draw_clip(rng):
    total, counts = _spread(rng, 1, 28_000_000), []
    tensors = _spread(rng, 1, 400)
    while total > 0 and len(counts) < tensors:
        counts.append(total if len(counts) == tensors - 1 else min(total, _spread(rng, 1, max(1, total // 4))))
        total -= counts[-1]
    rng.shuffle(counts)
    kind, out = rng.choice([("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
    return {"op": "clip", "counts": ",".join(map(str, counts)), "type": kind, "out": out, "flat": rng.random() < 0.5,
            "kept": rng.random() < 0.5, "limit": rng.choice([0.01, 0.1, 0.5, 2.0])}


def _numbers(text):
    out = []
    for part in text.split(",") if text else ():
        count, _, n = part.rpartition("x")
        out += [int(n)] * (int(count) if count else 1)
    return out


# ---- inputs ----------------------------------------------------------------------------------
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


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
    state = {"case": case}
    {"attention": _prepare_attention, "rotary": _prepare_rotary, "clip": _prepare_clip}[case["op"]](
        state, case, gen, normal)
    return state


def _prepare_attention(state, case, gen, normal):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    lengths = _numbers(case["lengths"])
    keys = _numbers(case["keys"]) if case["keys"] else lengths
    # Activations as a fused projection leaves them: rows of [heads | key heads | value heads]; queries are three
    # times as large, so that scores spread over +-10 and more, where a cap tells.
    if case["keys"]:
        q = normal(sum(lengths), heads, dim).mul_(3.0).to(torch.bfloat16)
        k, v = normal(sum(keys), 2 * kv, dim).to(torch.bfloat16).split((kv, kv), 1)
    else:
        qkv = normal(sum(lengths), heads + 2 * kv, dim)
        qkv[:, :heads] *= 3.0
        q, k, v = qkv.to(torch.bfloat16).split((heads, kv, kv), 1)
    state.update(q=q, k=k, v=v, offsets=_offsets(lengths), at=_places(lengths))
    state.update(key_offsets=_offsets(keys) if case["keys"] else None,
                 key_at=_places(keys) if case["keys"] else state["at"])
    # Each head's slope half an octave, or a little less, below the one before.
    state["slopes"] = (torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEV) / heads) if case["slopes"] else None)
    state["prefix"] = (torch.tensor(_numbers(case["prefix"]), dtype=torch.int32, device=DEV) if case["prefix"]
                       else None)
    if case["train"]:
        state["g"] = normal(sum(lengths), heads, dim).to(torch.bfloat16)
        for name in ("q", "k", "v"):
            state[name] = state[name].detach().requires_grad_(True)


def _prepare_rotary(state, case, gen, normal):
    heads, kv, dim, dtype = case["heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
    tokens, axes, half = case["tokens"], case["axes"], case["rotary"] // 2
    q, k = normal(tokens, heads + kv, dim).mul_(1.7).to(dtype).split((heads, kv), 1)
    positions = torch.randint(0, case["extent"], (tokens, axes), generator=gen, device=DEV, dtype=torch.int32)
    sections = [half // axes + (1 if a < half % axes else 0) for a in range(axes)]
    inv_freq = torch.cat([100.0 ** (-torch.arange(n, device=DEV, dtype=torch.float32) / max(1, n)) for n in sections])
    state.update(q=q, k=k, positions=positions, inv_freq=inv_freq, sections=sections, eps=1e-6,
                 wq=1.0 + 0.3 * normal(dim), wk=1.0 + 0.3 * normal(dim),
                 axis=torch.repeat_interleave(torch.arange(axes, device=DEV), torch.tensor(sections, device=DEV)))
    if case["train"]:
        state["gq"], state["gk"] = normal(tokens, heads, dim).to(dtype), normal(tokens, kv, dim).to(dtype)
        for name in ("q", "k", "wq", "wk"):
            state[name] = state[name].detach().requires_grad_(True)


def _prepare_clip(state, case, gen, normal):
    counts = _numbers(case["counts"])
    # Gradients' sizes differ by some powers of ten from one part of a model to another, of 16,384 values here.
    sizes = 10.0 ** (torch.rand(sum(counts) // 16384 + 1, generator=gen, device=DEV) * 3 - 5)
    flat = normal(sum(counts)).mul_(sizes.repeat_interleave(16384)[:sum(counts)]).to(TYPES[case["type"]])
    state["gradients"] = [x if case["flat"] else x.clone() for x in flat.split(counts)]
    # The results go to views of the optimizer's one buffer.
    state["out"] = torch.empty(sum(counts), device=DEV, dtype=TYPES[case["out"]])
    state["outs"] = list(state["out"].split(counts))
    # The limit as a part of what the norm will be, about: sizes' mean square is (10^-4 - 10^-10) / (6 ln 10).
    expected = math.sqrt(sum(counts) * (1e-4 - 1e-10) / (6 * math.log(10.0)))
    state["max_norm"] = case["limit"] * expected
    if own and case["kept"]:
        state["clipper"] = _package().GradientClipper(state["gradients"], out=state["outs"])


# ---- one pass --------------------------------------------------------------------------------
def run(state):
    forms = {"attention": (_plain_attention, _own_attention), "rotary": (_plain_rotary, _own_rotary),
             "clip": (_plain_clip, _own_clip)}
    return forms[state["case"]["op"]][1 if own else 0](state)


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own_attention(state):
    case = state["case"]
    got = _package().packed_attention(state["q"], state["k"], state["v"], state["offsets"], state["key_offsets"],
                                      causal=case["causal"], return_lse=case["lse"], score_cap=case["cap"] or None,
                                      distance_slopes=state["slopes"], prefix=state["prefix"])
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
    q, k = _package().normed_axial_rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                                          state["sections"], state["wq"], state["wk"], eps=state["eps"],
                                          interleaved=case["interleaved"])
    answer = {"q": q, "k": k}
    if case["train"]:
        names = ("q", "k", "wq", "wk")
        grads = torch.autograd.grad((q, k), [state[n] for n in names], (state["gq"], state["gk"]))
        answer.update({"d" + n: g for n, g in zip(names, grads)})
    return answer


def _own_clip(state):
    if state["case"]["kept"]:
        norm = state["clipper"].clip(state["max_norm"])
    else:
        norm = _package().clip_gradients(state["gradients"], state["max_norm"], out=state["outs"])
    return {"norm": norm, "out": state["out"]}


@torch.no_grad()
def _plain_attention(state):
    """Sequences padded to the longest, all scores formed, changed, masked and normalised."""
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
    ahead = j - (i + nk - nq)
    allowed = (i < nq) & (j < nk)
    if case["causal"]:
        before = ahead <= 0
        if state["prefix"] is not None:
            before |= j < state["prefix"][:, None, None]
        allowed &= before
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(batch, kv, group, lq, lk)
    slope = None
    if case["cap"]:
        scores.div_(case["cap"]).tanh_()
        if case["train"]:
            slope = 1 - scores.square()  # of the capped score
        scores.mul_(case["cap"])
    if state["slopes"] is not None:
        far = ahead.abs().float()
        for h in range(heads):  # head by head: a bias for all at once would be as large as the scores
            scores[:, h // group, h % group] -= state["slopes"][h] * far
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
        if slope is not None:
            ds *= slope.view(ds.shape)
        answer["dq"] = unpad(torch.matmul(ds, k)).to(torch.bfloat16)
        dk = torch.matmul(ds.transpose(-1, -2), q)
        answer["dk"], answer["dv"] = (
            x.transpose(1, 2)[key_at["seq"], key_at["place"]].to(torch.bfloat16) for x in (dk, dv))
    return answer


@torch.no_grad()
def _plain_rotary(state):
    case = state["case"]
    angle = state["positions"].double()[:, state["axis"]] * state["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turn = 2 * cos.shape[-1]

    def rotated(x, sin):
        part, rest = x[..., :turn], x[..., turn:]
        if case["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = part[..., :turn // 2], part[..., turn // 2:]
            part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((part, rest), -1)

    answer = {}
    for name in ("q", "k"):
        x, w = state[name].float(), state["w" + name]
        inv = (x.square().mean(-1, keepdim=True) + state["eps"]).rsqrt()
        unit = x * inv
        answer[name] = rotated(unit * w, sin).to(state[name].dtype)
        if case["train"]:
            g = rotated(state["g" + name].float(), -sin)
            answer["dw" + name] = (g * unit).double().sum((0, 1)).float()
            g = g * w
            answer["d" + name] = (inv * (g - unit * (g * unit).mean(-1, keepdim=True))).to(state[name].dtype)
    return answer


@torch.no_grad()
def _plain_clip(state):
    total = 0.0
    for x in state["gradients"]:
        total = total + x.float().square().sum(dtype=torch.float64)
    norm = total.sqrt()
    factor = torch.where(norm <= state["max_norm"], 1.0, state["max_norm"] / norm).float()
    for x, y in zip(state["gradients"], state["outs"]):
        y.copy_(x.float() * factor)
    return {"norm": norm.float(), "out": state["out"]}


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    if case["op"] == "clip":
        size = {"f32": 4, "bf16": 2}
        n = sum(_numbers(case["counts"]))
        # A square and a sum for the norm, a product for the result.
        return {"bytes": n * (size[case["type"]] + size[case["out"]]), "flops": 3 * n}
    heads, kv, dim, train = case["heads"], case["kv_heads"], case["dim"], case["train"]
    if case["op"] == "rotary":
        size = 4 if case["type"] == "f32" else 2
        values = case["tokens"] * (heads + kv) * dim
        turned = case["tokens"] * (heads + kv) * case["rotary"]
        # Forward x in and y out; the gradients read x and y's cotangent and write x's.  Square, sum and two
        # products for the norm and a rotated pair's four products and two sums; for the gradients about twice that.
        return {"bytes": (5 if train else 2) * values * size + case["tokens"] * case["axes"] * 4,
                "flops": (4 * values + 3 * turned) * (3 if train else 1)}
    lengths = _numbers(case["lengths"])
    keys = _numbers(case["keys"]) if case["keys"] else lengths
    pairs = 0
    for x, (n, m) in enumerate(zip(lengths, keys)):
        if not case["causal"]:
            pairs += n * m
            continue
        # Row i of n sees min(m, max(0, i + 1 + m - n, prefix)) of m keys.
        least = min(m, _numbers(case["prefix"])[x]) if case["prefix"] else 0
        first = min(n, max(0, least - 1 - m + n))  # rows that see the prefix alone
        i = n - first
        pairs += first * least + i * (first + 1 + m - n + m) // 2 if i else n * least
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
    return {"attention": _exact_attention, "rotary": _exact_rotary, "clip": _exact_clip}[case["op"]](state)


def _exact_attention(state):
    """One sequence and one head at a time, from the sums of the definition."""
    case, cap = state["case"], state["case"]["cap"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    lengths = _numbers(case["lengths"])
    keys = _numbers(case["keys"]) if case["keys"] else lengths
    prefix = _numbers(case["prefix"]) or [0] * len(lengths)
    group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    out, lse = torch.zeros_like(q), torch.full((case["heads"], q.shape[0]), -math.inf, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    r = c = 0
    for n, m, p in zip(lengths, keys, prefix):
        place = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] + (m - n)
        key = torch.arange(m, device=DEV, dtype=torch.float64)[None, :]
        hidden = (key > place) & (key >= p) if case["causal"] else None
        for h in range(case["heads"] if n and m else 0):
            rows, cols = slice(r, r + n), slice(c, c + m)
            kh, vh = k[cols, h // group], v[cols, h // group]
            s = scale * (q[rows, h] @ kh.T)
            turn = 1.0
            if cap:
                turn = torch.cosh(s / cap).square_().reciprocal_()
                s = cap * torch.tanh(s / cap)
            if state["slopes"] is not None:
                s = s - float(state["slopes"][h]) * (place - key).abs()
            if hidden is not None:
                s[hidden] = -math.inf
            z = torch.logsumexp(s, -1)
            p_ij = torch.exp(s - torch.where(z == -math.inf, 0.0, z)[:, None])
            out[rows, h], lse[h, rows] = p_ij @ vh, z
            if case["train"]:
                g = state["g"][rows, h].double()
                dp = g @ vh.T
                ds = turn * scale * p_ij * (dp - (g * out[rows, h]).sum(-1, keepdim=True))
                dq[rows, h] = ds @ kh
                dk[cols, h // group] += ds.T @ q[rows, h]
                dv[cols, h // group] += p_ij.T @ g
        r, c = r + n, c + m
    answer = {"out": out}
    if case["lse"]:
        answer["lse"] = lse
    if case["train"]:
        answer.update(dq=dq, dk=dk, dv=dv)
    return answer


def _exact_rotary(state):
    """As products of complex numbers, x1 + i x2 times exp(i theta), and the norm's derivative as a projection."""
    case, half = state["case"], state["inv_freq"].numel()
    theta = state["positions"].double()[:, state["axis"]] * state["inv_freq"].double()
    turn = torch.polar(torch.ones_like(theta), theta)[:, None]
    i = torch.arange(half, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)

    def rotated(x, turn):
        y = x.clone()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    answer = {}
    for name in ("q", "k"):
        x, w = state[name].detach().double(), state["w" + name].detach().double()
        power = (x * x).sum(-1, keepdim=True) / case["dim"] + state["eps"]
        unit = x / power.sqrt()
        answer[name] = rotated(unit * w, turn)
        if case["train"]:
            g = rotated(state["g" + name].double(), turn.conj())
            answer["dw" + name] = torch.einsum("thd,thd->d", g, unit)
            dot = torch.einsum("thd,d,thd->th", g, w, x)[..., None]
            answer["d" + name] = (g * w) / power.sqrt() - x * dot / (case["dim"] * power ** 1.5)
    return answer


def _exact_clip(state):
    gradients = [x.double() for x in state["gradients"]]
    norm = torch.stack([torch.dot(x, x) for x in gradients]).sum().sqrt()
    factor = min(1.0, state["max_norm"] / float(norm))
    return {"norm": norm, "out": torch.cat(gradients) * factor}
