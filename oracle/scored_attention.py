"""Oracle of the packed attention whose scores are capped, lean on distance or see a prefix, and of its gradients: in
float64, one sequence and one head at a time, with elementwise bounds on what an implementation may be off that forms
scores and sums in float32 and rounds the softmax weights, dS and its results to bf16."""

from __future__ import annotations

import numpy as np

U = 2.0 ** -8 * 1.05  # bf16 round to nearest: 2^-8 relative; 5% for second-order terms
F = 2.0 ** -20        # float32 dot products of up to 128 terms: a few units of 2^-23
CAP = 2.0 ** -20      # a capped score, relative: its polynomial's 6.5e-7 and a few roundings of 2^-24
E = 2.0 ** -21        # products and sums of a few float32 numbers


def scored_attention(q, k, v, offsets, key_offsets=None, causal=False, scale=None, cap=None, slopes=None, prefix=None,
                     grad=None, grad_lse=None):
    """``q [T, H, D]``, ``k, v [Tk, Hkv, D]``; offsets, cap, slopes ``[H]`` and prefix as the operator takes them.

    Returns a dict of ``out``, ``lse`` and, with ``grad``, ``dq``, ``dk``, ``dv``, and of the bounds under the same
    names + ``_bound``.  A score is off by e: the product's F sum |scale q k|, the cap's CAP |s'| + E cap (its far form
    subtracts from the cap), and E of the distance's part and of the result, which is also how far lse is off.  P is
    then off by P (e + sum P e) beside its rounding U P; dS by that of its P, delta by what o is off, and the
    cap's derivative, 1 - t^2, by 2 t times t's error.

    out may be divided by the sum of the rounded weights rather than of the exact ones: with P_j (1 + d_j), |d_j| <= U,
    sum P d v / (1 + sum P d) - o sum P d / (1 + sum P d) is U (sum P |v| + |o|) at most, and the result's own rounding
    U |o| more: U (sum P |v| + 2 |o|) in all.
    """
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    T, H, D = q.shape
    group = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    off = np.asarray(offsets)
    koff = off if key_offsets is None else np.asarray(key_offsets)
    names = ["out"] + (["dq", "dk", "dv"] if grad is not None else [])
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    r = {n: np.zeros_like(like[n]) for n in names}
    r.update({n + "_bound": np.zeros_like(like[n]) for n in names})
    r["lse"] = np.full((H, T), -np.inf)
    r["lse_bound"] = np.zeros((H, T))
    for s in range(len(off) - 1):
        rows, cols = slice(off[s], off[s + 1]), slice(koff[s], koff[s + 1])
        n, m = off[s + 1] - off[s], koff[s + 1] - koff[s]
        if n <= 0 or m <= 0:
            continue
        ahead = np.arange(m)[None] - (np.arange(n)[:, None] + m - n)
        seen = np.ones((n, m), bool)
        if causal:
            seen = ahead <= 0
            if prefix is not None:
                seen |= np.arange(m)[None] < prefix[s]
        some = seen.any(1)
        for h in range(H):
            qh, kh, vh = q[rows, h], k[cols, h // group], v[cols, h // group]
            x = scale * qh @ kh.T
            size = scale * np.abs(qh) @ np.abs(kh).T
            e = F * size
            turn, turn_off = 1.0, 0.0
            if cap is not None:
                t = np.tanh(x / cap)
                x = cap * t
                turn = 1.0 - t * t
                e = e * turn + CAP * np.abs(x) + E * cap
                turn_off = 2.0 * np.abs(t) * e / cap + E
            if slopes is not None:
                bias = float(slopes[h]) * np.abs(ahead)
                x = x - bias
                e = e + E * np.abs(bias)
            e = np.where(seen, e + E * (1.0 + np.abs(x)), 0.0)
            x = np.where(seen, x, -np.inf)
            top = np.where(some, x.max(1), 0.0)
            w = np.exp(x - top[:, None])
            z = w.sum(1)
            p = w / np.where(some, z, 1.0)[:, None]
            pe = p * e
            p_off = pe + p * pe.sum(1)[:, None]  # beside the rounding
            o = p @ vh
            a = p @ np.abs(vh)
            r["out"][rows, h] = o
            o_off = p_off @ np.abs(vh)
            r["out_bound"][rows, h] = U * (a + 2.0 * np.abs(o)) + o_off
            with np.errstate(divide="ignore"):
                r["lse"][h, rows] = np.where(some, top + np.log(z), -np.inf)
            r["lse_bound"][h, rows] = np.where(some, F + E * np.abs(top) + pe.sum(1), 0.0)
            if grad is None:
                continue
            g = np.asarray(grad, np.float64)[rows, h]
            delta = (g * o).sum(1)
            if grad_lse is not None:
                delta = delta - np.asarray(grad_lse, np.float64)[h, rows]
            raw = p * (g @ vh.T - delta[:, None])
            ds = raw * turn
            off_delta = (np.abs(g) * (U * (np.abs(o) + a) + o_off)).sum(1)
            off_ds = (U * np.abs(ds) + turn * (p * off_delta[:, None] + F * p * (np.abs(g) @ np.abs(vh).T)
                                               + np.abs(raw) * (e + pe.sum(1)[:, None] + F))
                      + turn_off * np.abs(raw))
            r["dq"][rows, h] = scale * ds @ kh
            r["dq_bound"][rows, h] = scale * off_ds @ np.abs(kh)
            r["dk"][cols, h // group] += scale * ds.T @ qh
            r["dk_bound"][cols, h // group] += scale * off_ds.T @ np.abs(qh)
            r["dv"][cols, h // group] += p.T @ g
            r["dv_bound"][cols, h // group] += (U * p + p_off).T @ np.abs(g)
    for n in names[1:]:
        r[n + "_bound"] += U * np.abs(r[n])
    return r
