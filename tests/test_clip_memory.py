"""Results of a clipping that share memory with one another, or with a gradient that is not their own, are refused before
any launch, by their addresses and sizes alone: the kernel would read what it has written already.  A call that
fits goes on to its next check, that of the workspace, which none of these has."""

from __future__ import annotations

import ctypes
import random

import pytest

F32, BF16 = 0, 1


def _refused(pkg, ins, outs=None):
    """Of ``(address, type, count)`` triples."""
    N = pkg._native
    outs = ins if outs is None else outs
    (a, t, n), (b, u, m) = zip(*ins), zip(*outs)
    assert n == m
    p = lambda kind, v: (kind * len(v))(*v)  # noqa: E731
    status = N.lib().rfdetr_clip_gradients(None, p(ctypes.c_void_p, a), p(ctypes.c_int32, t), p(ctypes.c_void_p, b),
                                           p(ctypes.c_int32, u), p(ctypes.c_int64, n), len(n), 1.0, 4096, None, 0)
    assert status in (N.ERR_SHAPE, N.ERR_WORKSPACE)
    return status == N.ERR_SHAPE


@pytest.mark.parametrize(("ins", "outs", "want"), [
    ([(64, F32, 4), (80, F32, 4)], None, False),                                    # in place, side by side
    ([(80, F32, 4), (64, F32, 4)], None, False),                                    # in any order
    ([(64, F32, 4), (64, F32, 4)], None, True),                                     # twice
    ([(64, F32, 4), (76, F32, 4)], None, True),                                     # one value in common
    ([(64, F32, 40), (80, F32, 1)], None, True),                                    # one inside another
    ([(64, F32, 4), (70, BF16, 0), (80, F32, 4)], None, False),                     # a tensor of no values
    ([(64, F32, 0), (64, F32, 0)], None, False),
    ([(64, F32, 4), (80, F32, 4)], [(640, F32, 4), (656, F32, 4)], False),          # into others
    ([(64, F32, 4), (64, F32, 4)], [(640, F32, 4), (656, F32, 4)], False),          # gradients may be alike
    ([(64, F32, 4), (80, F32, 4)], [(64, F32, 4), (656, F32, 4)], False),           # one in place
    ([(64, F32, 4), (80, F32, 4)], [(80, F32, 4), (64, F32, 4)], True),             # each other's
    ([(64, F32, 4), (80, F32, 4)], [(640, F32, 4), (64, F32, 4)], True),            # another's
    ([(64, F32, 4)], [(68, F32, 4)], True),                                         # its own, one value on
    ([(64, F32, 4)], [(60, F32, 4)], True),
    ([(64, BF16, 4)], [(72, F32, 4)], False),                                       # right behind it
    ([(64, BF16, 4), (72, BF16, 4)], [(640, F32, 4), (652, F32, 4)], True)])        # results
def test_ranges(pkg, ins, outs, want):
    assert _refused(pkg, ins, outs) is want


def test_against_every_byte(pkg):
    rng = random.Random(0)
    seen = []
    for _ in range(3000):
        n = rng.randint(1, 5)
        counts = [rng.choice([0, 1, 2, 3, 8]) for _ in range(n)]
        ins = [(4 * rng.randint(1, 60), rng.choice([F32, BF16]), c) for c in counts]
        # (A result at its gradient's own address has its type, or another check refuses it.)
        outs = [i if rng.random() < 0.4 else (4 * rng.randint(61, 64) if rng.random() < 0.3 else i[0] + 4 * rng.choice(
            [-1, 1, 2, 3, 9]), rng.choice([F32, BF16]), i[2]) for i in ins]
        outs = [(p or 400, t, c) for p, t, c in outs]
        cover = [set(range(p, p + c * (2 if t == BF16 else 4))) for p, t, c in ins]
        out_cover = [set(range(p, p + c * (2 if t == BF16 else 4))) for p, t, c in outs]
        want = any(out_cover[a] & out_cover[b] for a in range(n) for b in range(a))
        want |= any(out_cover[a] & cover[b] and not (a == b and ins[a] == outs[a]) for a in range(n) for b in range(n))
        assert _refused(pkg, ins, outs) is want
        seen.append(want)
    assert 300 < sum(seen) < 2700
