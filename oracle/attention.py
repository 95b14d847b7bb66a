"""Oracle of the packed softmax attention and its gradients, in float64, one sequence and one head
at a time from the sums of the definition -- with elementwise bounds on what an implementation may
be off that forms scores and sums in float32 and rounds the softmax weights, dS and its results to
bf16 (see :func:`attention`)."""

from __future__ import annotations

import numpy as np

U = 2.0 ** -8 * 1.05  # bf16 round to nearest: 2^-8 relative; 5% for second-order and float32 terms
F = 2.0 ** -20        # float32 dot products of up to 128 terms: a few units of 2^-23


def attention(q, k, v, offsets, key_offsets=None, causal=False, scale=None, grad=None, grad_lse=None):
    """``q [T, H, D]``, ``k, v [Tk, Hkv, D]``; offsets as the operator takes them.

    Returns a dict of ``out [T, H, D]``, ``lse [H, T]`` and, with ``grad [T, H, D]`` (and
    ``grad_lse [H, T]``), ``dq``, ``dk``, ``dv``; and under the same names + ``_bound`` the largest
    elementwise error.  With P off by U P (its rounding to bf16):

    * out:  U sum_j P |v_j| + U |out|;
    * lse:  F (1 + largest sum_d |scale q_d k_d|), the float32 score's error;
    * dv:   U sum_i P |g_i| + U |dv|;
    * delta = sum_d g o is off by U sum_d |g| (|o| + sum_j P |v_j|), so dS by U |dS| + P times
      that, and dq and dk by those times scale |k| and scale |q|, plus U of themselves.
      (With the part that o's rounding lost kept beside it, the |o| term is slack.)
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
        seen = np.ones((n, m), bool)
        if causal:
            seen = np.arange(m)[None] <= np.arange(n)[:, None] + m - n
        some = seen.any(1)
        for h in range(H):
            qh, kh, vh = q[rows, h], k[cols, h // group], v[cols, h // group]
            x = np.where(seen, scale * qh @ kh.T, -np.inf)
            top = np.where(some, x.max(1), 0.0)
            e = np.exp(x - top[:, None])
            z = e.sum(1)
            p = e / np.where(some, z, 1.0)[:, None]
            o = p @ vh
            a = p @ np.abs(vh)
            r["out"][rows, h] = o
            r["out_bound"][rows, h] = U * (a + np.abs(o))
            with np.errstate(divide="ignore"):
                r["lse"][h, rows] = np.where(some, top + np.log(z), -np.inf)
            size = scale * np.abs(qh) @ np.abs(kh).T
            r["lse_bound"][h, rows] = F * (1.0 + np.where(seen, size, 0.0).max(1))
            if grad is None:
                continue
            g = np.asarray(grad, np.float64)[rows, h]
            delta = (g * o).sum(1)
            if grad_lse is not None:
                delta = delta - np.asarray(grad_lse, np.float64)[h, rows]
            ds = p * (g @ vh.T - delta[:, None])
            off_delta = U * (np.abs(g) * (np.abs(o) + a)).sum(1)
            # The float32 products behind dP and S: F of their absolute sums.
            off_ds = (U * np.abs(ds) + p * off_delta[:, None] + F * p * (np.abs(g) @ np.abs(vh).T)
                      + F * np.abs(ds) * (1.0 + size))
            r["dq"][rows, h] = scale * ds @ kh
            r["dq_bound"][rows, h] = scale * off_ds @ np.abs(kh)
            r["dk"][cols, h // group] += scale * ds.T @ qh
            r["dk_bound"][cols, h // group] += scale * off_ds.T @ np.abs(qh)
            r["dv"][cols, h // group] += p.T @ g
            r["dv_bound"][cols, h // group] += U * p.T @ np.abs(g)
    for n in names[1:]:
        r[n + "_bound"] += U * np.abs(r[n])
    return r
