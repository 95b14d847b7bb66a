"""Packed attention on the device against the float64 oracle, elementwise within the bounds that
the oracle derives from the operator's roundings (bf16 weights and results, float32 sums)."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle import attention as OA

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _bf16(rng, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(torch.bfloat16)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _offsets(lengths, first=0):
    return torch.tensor(np.cumsum([first, *lengths]), dtype=torch.int32, device=DEV)


def _close(name, got, want, bound):
    got = _f64(got)
    assert got.shape == want.shape
    same = got == want  # infinities
    off = np.where(same, 0.0, np.abs(got - np.where(same, 0.0, want)))
    bad = ~(off <= bound + 1e-30)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.size} outside the bound; first at {np.argwhere(bad)[0]}, " \
                          f"{got[bad][0]} for {want[bad][0]} within {bound[bad][0]:.3e}"


def _fault_free(pkg):
    assert pkg._native.lib().rfdetr_take_device_fault(torch.cuda.current_stream().cuda_stream) == 0


def _check(pkg, lengths, keys=None, heads=2, kv=2, dim=64, causal=False, scale=None, seed=0, grad=True,
           with_lse_grad=False):
    rng = np.random.default_rng(seed)
    own = keys is None
    tk = sum(lengths if own else keys)
    q, k, v = _bf16(rng, sum(lengths), heads, dim), _bf16(rng, tk, kv, dim), _bf16(rng, tk, kv, dim)
    g = _bf16(rng, sum(lengths), heads, dim)
    gl = torch.tensor(rng.standard_normal((heads, sum(lengths))).astype(np.float32), device=DEV)
    off, koff = _offsets(lengths), None if own else _offsets(keys)
    r = OA.attention(_f64(q), _f64(k), _f64(v), off.cpu().numpy(), None if own else koff.cpu().numpy(), causal, scale,
                     _f64(g) if grad else None, _f64(gl) if with_lse_grad else None)
    plain = pkg.packed_attention(q, k, v, off, koff, causal=causal, scale=scale, check=True)
    _close("out", plain, r["out"], r["out_bound"])
    if not grad:
        _fault_free(pkg)
        return
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out, lse = pkg.packed_attention(*leaves, off, koff, causal=causal, scale=scale, return_lse=True)
    _close("out", out, r["out"], r["out_bound"])
    _close("lse", lse, r["lse"], r["lse_bound"])
    outs, gs = ((out, lse), (g, gl)) if with_lse_grad else ((out,), (g,))
    for name, d in zip(("dq", "dk", "dv"), torch.autograd.grad(outs, leaves, gs)):
        _close(name, d, r[name], r[name + "_bound"])
    _fault_free(pkg)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("lengths", [(1,), (7,), (64,), (128,), (129,), (300, 300), (5, 0, 257, 1, 130)])
def test_lengths(pkg, lengths, dim, causal):
    _check(pkg, lengths, dim=dim, causal=causal, seed=sum(lengths) + dim)


@pytest.mark.parametrize("dim", [8, 16, 40, 72, 80, 96, 120])
def test_channels_that_fill_no_tile(pkg, dim):
    _check(pkg, (70, 200), dim=dim, causal=True, seed=dim)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize(("heads", "kv"), [(1, 1), (4, 1), (6, 2), (7, 1), (8, 2), (5, 5), (64, 1), (71, 1), (96, 1)])
def test_grouped_heads(pkg, heads, kv, causal):
    _check(pkg, (33, 150, 2), heads=heads, kv=kv, dim=64, causal=causal, seed=heads * 10 + kv)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize(("lengths", "keys"), [((300, 300, 4), (576, 0, 1)), ((1, 1, 1, 1), (700, 1, 0, 129)),
                                               ((200, 10), (30, 200)), ((3,), (0,)), ((0, 5), (3, 64)),
                                               ((1000, 2), (129, 2000))])
def test_queries_of_other_tokens(pkg, lengths, keys, causal):
    """Rows whose mask leaves nothing among them: no keys at all, or (causal) more queries than keys."""
    _check(pkg, lengths, keys, heads=4, kv=2, dim=64, causal=causal, seed=len(lengths) + sum(keys))


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_long(pkg, dim, causal):
    _check(pkg, (1700, 900), heads=4, kv=2, dim=dim, causal=causal, seed=dim)


def test_many_short_sequences(pkg):
    lengths = [int(n) for n in np.random.default_rng(1).integers(0, 9, 2500)]
    _check(pkg, lengths, heads=2, kv=1, dim=32, causal=True)


def test_lse_gradient(pkg):
    _check(pkg, (100, 190), heads=4, kv=2, dim=64, causal=True, with_lse_grad=True)
    _check(pkg, (100, 3), (40, 200), heads=2, kv=2, dim=128, with_lse_grad=True)


def test_lse_gradient_alone(pkg):
    rng = np.random.default_rng(3)
    q, k, v = (_bf16(rng, 50, 2, 32).requires_grad_(True) for _ in range(3))
    gl = rng.standard_normal((2, 50))
    off = _offsets((50,))
    _, lse = pkg.packed_attention(q, k, v, off, return_lse=True)
    dq, dk, dv = torch.autograd.grad(lse, (q, k, v), torch.tensor(gl, device=DEV, dtype=torch.float32))
    r = OA.attention(_f64(q), _f64(k), _f64(v), [0, 50], grad=np.zeros((50, 2, 32)), grad_lse=gl)
    _close("dq", dq, r["dq"], r["dq_bound"])
    _close("dk", dk, r["dk"], r["dk_bound"])
    assert not dv.any()


@pytest.mark.parametrize("scale", [0.02, 1.0, 3.0])
def test_scales(pkg, scale):
    """Flat and sharp softmax: with scale 3 the running maximum moves far and often."""
    _check(pkg, (400, 77), heads=2, kv=1, dim=64, scale=scale, causal=True)


def test_rising_scores(pkg):
    """Keys whose scores rise along the sequence, so the running maximum grows at every tile, and
    fall, so it never does."""
    for sign in (1, -1):
        n, dim = 900, 64
        ramp = (np.arange(n) / 20.0)[:, None, None] * sign
        k = torch.tensor(np.broadcast_to(ramp, (n, 1, dim)).copy(), device=DEV).to(torch.bfloat16)
        q = torch.full((n, 2, dim), 0.25, device=DEV, dtype=torch.bfloat16)
        v = _bf16(np.random.default_rng(5), n, 1, dim)
        off = _offsets((n,))
        for causal in (False, True):
            out, lse = pkg.packed_attention(q, k, v, off, causal=causal, return_lse=True)
            r = OA.attention(_f64(q), _f64(k), _f64(v), [0, n], causal=causal)
            _close("out", out, r["out"], r["out_bound"])
            _close("lse", lse, r["lse"], r["lse_bound"])


def test_views_of_a_fused_projection(pkg):
    """Token strides of the whole projection, head strides of heads-first storage, sliced cotangents."""
    rng = np.random.default_rng(7)
    off = _offsets((100, 130))
    fused = _bf16(rng, 230, 8, 64)
    q, k, v = fused.split((4, 2, 2), 1)
    want = pkg.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), off)
    assert torch.equal(pkg.packed_attention(q, k, v, off), want)
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]  # heads outermost
    assert torch.equal(pkg.packed_attention(*turned, off), want)
    odd = torch.empty(230, 4, 65, device=DEV, dtype=torch.bfloat16)[..., 1:]  # unaligned: copied
    odd.copy_(q)
    assert torch.equal(pkg.packed_attention(odd, k, v, off), want)
    a = [x.detach().requires_grad_(True) for x in (q, k, v)]
    b = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    g = _bf16(rng, 230, 9, 64)[:, 2:6]
    for x, y in zip(torch.autograd.grad(pkg.packed_attention(*a, off), a, g),
                    torch.autograd.grad(pkg.packed_attention(*b, off), b, g.contiguous())):
        assert torch.equal(x, y)
    # A cotangent broadcast over everything (stride 0).
    for x, y in zip(torch.autograd.grad(pkg.packed_attention(*a, off).sum(), a),
                    torch.autograd.grad(pkg.packed_attention(*b, off), b, torch.ones_like(want))):
        assert torch.equal(x, y)


def test_one_key_has_no_score_gradient(pkg):
    """A softmax over one key is 1 whatever the score: its query's and key's gradients are exactly 0."""
    rng = np.random.default_rng(8)
    q, k, v = (_bf16(rng, 40, 2, 64).requires_grad_(True) for _ in range(3))
    g = _bf16(rng, 40, 2, 64)
    off = _offsets([1] * 40)
    for causal in (False, True):
        out = pkg.packed_attention(q, k, v, off, causal=causal)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), g)
        assert torch.equal(out, v) and torch.equal(dv, g) and not dq.any() and not dk.any()


def test_rows_outside_all_sequences(pkg):
    """A packed buffer with unused rows before, after: output and gradients 0, log-sum-exp -inf,
    whatever they hold."""
    rng = np.random.default_rng(9)
    n, first, used = 700, 37, (300, 150)
    q, k, v = (_bf16(rng, n, 2, 64) for _ in range(3))
    last = first + sum(used)
    for x in (q, k, v):
        x[:first] = float("nan")
        x[last:] = float("inf")
    off = _offsets(used, first)
    g = _bf16(rng, n, 2, 64)
    g[last:] = float("nan")
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out, lse = pkg.packed_attention(*leaves, off, return_lse=True)
    grads = torch.autograd.grad(out, leaves, g)
    inner = [x.detach()[first:last].clone().requires_grad_(True) for x in (q, k, v)]
    want, want_lse = pkg.packed_attention(*inner, _offsets(used), return_lse=True)
    want_grads = torch.autograd.grad(want, inner, g[first:last])
    for got, ref in zip((out, *grads), (want, *want_grads)):
        assert not got[:first].any() and not got[last:].any()
        assert torch.equal(got[first:last], ref)
    assert torch.equal(lse[:, first:last], want_lse) and torch.isneginf(lse[:, :first]).all()


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_sequences_do_not_reach_each_other(pkg, poison):
    """Non-finite rows of one sequence leave every other sequence's outputs and gradients as they are."""
    rng = np.random.default_rng(10)
    lengths = (70, 90, 131, 5)
    q, k, v, g = (_bf16(rng, sum(lengths), 4, 64) for _ in range(4))
    off = _offsets(lengths)

    def run(q, k, v, g):
        leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
        out = pkg.packed_attention(*leaves, off, causal=True)
        return (out, *torch.autograd.grad(out, leaves, g))

    want = run(q, k, v, g)
    bad = slice(70, 160)
    for x in (q, k, v, g):
        x[bad] = poison
    for got, ref in zip(run(q, k, v, g), want):
        assert torch.equal(got[:70], ref[:70]) and torch.equal(got[160:], ref[160:])


def test_same_bits_each_time_and_on_another_stream(pkg):
    rng = np.random.default_rng(11)
    off = _offsets((900, 333))
    q, k, v = (_bf16(rng, 1233, h, 128).requires_grad_(True) for h in (8, 2, 2))
    g = _bf16(rng, 1233, 8, 128)

    def run():
        out = pkg.packed_attention(q, k, v, off, causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), g))

    want = run()
    for _ in range(5):
        for a, b in zip(run(), want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_thread_that_has_made_no_other_call(pkg):
    """A new thread has no current context of the device until some call gives it one."""
    rng = np.random.default_rng(8)
    q, k, v, g = (_bf16(rng, 40, 2, 64) for _ in range(4))
    off = _offsets((40,))
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    want = pkg.packed_attention(q, k, v, off)
    loss = (pkg.packed_attention(*leaves, off).float() * g.float()).sum()
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    out, status = torch.empty_like(q), []
    lib = pkg._native.lib()
    args = [stream]
    for x in (q, k, v):
        args += [x.data_ptr(), *x.stride()[:2]]
    args += [off.data_ptr(), None, out.data_ptr(), None, None, None, 0, 1, 40, 40, 2, 2, 64, 0, 0.125]
    thread = threading.Thread(target=lambda: status.append(lib.rfdetr_packed_attention(*args)))
    thread.start()
    thread.join()
    assert status == [pkg._native.OK]
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    loss.backward()
    assert all(torch.isfinite(x.grad).all() for x in leaves)


def test_empty_tensors(pkg):
    e = torch.empty((0, 4, 64), device=DEV, dtype=torch.bfloat16)
    out, lse = pkg.packed_attention(e, e, e, _offsets((0, 0)), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    rng = np.random.default_rng(12)
    q = _bf16(rng, 9, 4, 64).requires_grad_(True)
    k = e.clone().requires_grad_(True)
    out, lse = pkg.packed_attention(q, k, k, _offsets((9,)), _offsets((0,)), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()
    dq, dk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
    assert not dq.any() and dk.shape == k.shape
    # No queries: the keys' gradients are 0.
    dk, dv = (_bf16(rng, 9, 4, 64).requires_grad_(True) for _ in range(2))
    q0 = e.clone().requires_grad_(True)
    out = pkg.packed_attention(q0, dk, dv, _offsets((0,)), _offsets((9,)))
    for x in torch.autograd.grad(out, (dk, dv), torch.ones_like(out)):
        assert not x.any()
    # No sequences at all.
    out = pkg.packed_attention(q, q, q, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert not out.any()


def test_offsets_are_clamped(pkg):
    """Offsets past the tensors are cut at their ends; `check` refuses them."""
    rng = np.random.default_rng(13)
    q, k, v = (_bf16(rng, 100, 2, 32) for _ in range(3))
    far = torch.tensor([0, 60, 5000], dtype=torch.int32, device=DEV)
    want = pkg.packed_attention(q, k, v, _offsets((60, 40)))
    assert torch.equal(pkg.packed_attention(q, k, v, far), want)
    with pytest.raises(ValueError, match="ascend"):
        pkg.packed_attention(q, k, v, far, check=True)
    with pytest.raises(ValueError, match="ascend"):
        pkg.packed_attention(q, k, v, torch.tensor([0, 60, 50], dtype=torch.int32, device=DEV), check=True)


def test_refusals(pkg):
    t = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, device=DEV, dtype=dtype)  # noqa: E731
    off = _offsets((4,))
    call = pkg.packed_attention
    for q, k, v, o, ko, kw in [
            (t(4, 2, 64, dtype=torch.float32), t(4, 2, 64), t(4, 2, 64), off, None, {}),
            (t(4, 2, 64), t(4, 2, 64, dtype=torch.float16), t(4, 2, 64), off, None, {}),
            (t(4, 128), t(4, 2, 64), t(4, 2, 64), off, None, {}),
            (t(4, 3, 64), t(4, 2, 64), t(4, 2, 64), off, None, {}),
            (t(4, 2, 64), t(4, 2, 32), t(4, 2, 64), off, None, {}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 1, 64), off, None, {}),
            (t(4, 2, 64), t(5, 2, 64), t(4, 2, 64), off, off, {}),
            (t(4, 2, 64), t(5, 2, 64), t(5, 2, 64), off, None, {}),
            (t(4, 2, 60), t(4, 2, 60), t(4, 2, 60), off, None, {}),
            (t(4, 2, 136), t(4, 2, 136), t(4, 2, 136), off, None, {}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), off.float(), None, {}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), off[None], None, {}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), off, _offsets((2, 2)), {}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), off, None, {"scale": 0.0}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), off, None, {"scale": -1.0}),
            (t(4, 2, 64), t(4, 2, 64), t(4, 2, 64), off, None, {"scale": float("nan")}),
            (t(4, 2, 64), t(4, 2, 64).cpu(), t(4, 2, 64), off, None, {})]:
        with pytest.raises(ValueError):
            call(q, k, v, o, ko, **kw)


@pytest.mark.parametrize("knob", ["1,1", "1,3", "1,64", "2", "3,1", "3,3", "3,64"])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_every_forward_kernel(pkg, tuning, knob, dim):
    """The kernels, whole and with their keys split over blocks (more blocks than key tiles among them)
    or taken in turn by a block's halves, whatever the sizes would choose."""
    tuning("RFDETR_ATTN_FWD", knob)
    _check(pkg, (1, 300, 0, 517, 64), heads=6, kv=2, dim=dim, causal=True, seed=dim)
    _check(pkg, (3, 130, 40, 7), (900, 0, 17, 129), heads=4, kv=1, dim=dim, seed=dim)
    _check(pkg, (130, 5), (30, 1000), heads=2, kv=2, dim=dim, causal=True, seed=dim)


@pytest.mark.parametrize("knob", ["1,1", "2,4", "4,2"])
@pytest.mark.parametrize("dim", [32, 64, 80, 128])
def test_every_backward_split(pkg, tuning, knob, dim):
    """Tiles shared by a cluster of blocks, some of them left without a step."""
    tuning("RFDETR_ATTN_BWD", knob)
    _check(pkg, (1, 300, 0, 517, 64), heads=6, kv=2, dim=dim, causal=True, seed=dim)
    _check(pkg, (3, 130, 40, 7), (900, 0, 17, 129), heads=4, kv=1, dim=dim, seed=dim)
    _check(pkg, (130, 5), (30, 1000), heads=2, kv=2, dim=dim, causal=True, seed=dim, with_lse_grad=True)


@pytest.mark.parametrize("dim", [32, 128])
def test_blocks_that_stay(pkg, tuning, dim):
    """More row tiles than the short kernel's resident blocks, with empty ones, tiles without keys and
    ragged ends between them, taken in turn."""
    tuning("RFDETR_ATTN_FWD", "2")
    rng = np.random.default_rng(21)
    lengths = [int(n) for n in rng.integers(0, 200, 150)]
    keys = [int(n) if rng.random() > 0.2 else 0 for n in rng.integers(0, 300, 150)]
    _check(pkg, lengths, keys, heads=8, kv=8, dim=dim, causal=True)
    _check(pkg, keys, heads=12, kv=4, dim=dim)


def test_one_token_over_long_keys(pkg):
    """The form for single tokens: the keys are split over blocks."""
    N = pkg._native
    assert N.lib().rfdetr_packed_attention_workspace_bytes(3, 3, 9000, 8, 2, 128) > 0
    _check(pkg, (1, 1, 1), (5000, 1, 3999), heads=8, kv=2, dim=128, causal=True, grad=False)
    _check(pkg, (1,), (7000,), heads=4, kv=4, dim=64)
    _check(pkg, (2, 0, 1), (3000, 3000, 3000), heads=7, kv=1, dim=80, causal=True)


@pytest.mark.parametrize("dim", [32, 64, 80, 128])
@pytest.mark.parametrize("heads,kv", [(16, 4), (6, 6), (12, 1)])
def test_keys_shared_out(pkg, heads, kv, dim):
    """Few rows over keys of very different lengths, none and one among them: how many blocks a slot gets
    depends on all of them."""
    keys = (5000, 0, 129, 3001, 1, 9000, 128, 40)
    size = pkg._native.lib().rfdetr_packed_attention_workspace_bytes
    assert size(8, 8, sum(keys), heads, kv, dim) > 0
    _check(pkg, (1,) * 8, keys, heads, kv, dim, causal=True, grad=False)
    _check(pkg, (3, 2, 0, 1, 5, 7, 1, 2), keys, heads, kv, dim, causal=True)
    _check(pkg, (1, 5, 0), (20000, 7, 300), heads, kv, dim)


def test_keys_shared_out_over_many_slots(pkg, tuning):
    """More slots than a warp has lanes, and more than the blocks look through (then none are shared out)."""
    rng = np.random.default_rng(3)
    for n, knob in ((40, "3,2"), (150, "3,3"), (400, "3,3")):
        tuning("RFDETR_ATTN_FWD", knob)
        lengths = [int(x) for x in rng.integers(0, 3, n)]
        keys = [int(x) if rng.random() > 0.3 else 0 for x in rng.integers(0, 2500 if n < 100 else 600, n)]
        _check(pkg, lengths, keys, heads=4, kv=2, dim=64, causal=True)


def test_offsets_that_do_not_ascend(pkg, tuning):
    """Unchecked: the results are then of no use, but every kernel stays within the tensors."""
    rng = np.random.default_rng(4)
    q, k, v = _bf16(rng, 300, 4, 64), _bf16(rng, 2000, 2, 64), _bf16(rng, 2000, 2, 64)
    off = torch.tensor([-5, 200, 100, 250, 7000, 20, 300], dtype=torch.int32, device=DEV)
    koff = torch.tensor([1500, 300, 2500, -1, 900, 100, 2000], dtype=torch.int32, device=DEV)
    for knob in ("1", "2", "3", "3,4"):
        tuning("RFDETR_ATTN_FWD", knob)
        pkg.packed_attention(q, k, v, off, koff, causal=True, return_lse=True)
        _fault_free(pkg)


def test_captured_in_a_graph(pkg):
    """Forward alone, with keys shared out and joined, replayed on other inputs and other lengths."""
    rng = np.random.default_rng(5)
    q, k, v = _bf16(rng, 8, 16, 128), _bf16(rng, 20000, 4, 128), _bf16(rng, 20000, 4, 128)
    off, koff = _offsets((1,) * 8), _offsets((9000, 1, 3000, 0, 500, 64, 7000, 435))
    call = lambda: pkg.packed_attention(q, k, v, off, koff, causal=True, return_lse=True)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (6, 7):
        rng = np.random.default_rng(seed)
        for x in (q, k, v):
            x.copy_(_bf16(rng, *x.shape))
        cuts = np.sort(rng.integers(0, 20001, 7))
        koff.copy_(torch.tensor([0, *cuts.tolist(), 20000], dtype=torch.int32))
        graph.replay()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets(pkg):
    """Keys, values and cotangents whose rows lie further apart than 2^31 elements (a wide cache)."""
    rng = np.random.default_rng(31)
    wide = torch.empty((1400, 1_600_000), device=DEV, dtype=torch.bfloat16)  # 4.5 GB
    rows = _bf16(rng, 1400, 8, 64)
    wide[:, :512] = rows.view(1400, 512)
    k, v, q, g = (wide[:, i * 128:(i + 1) * 128].view(1400, 2, 64) for i in range(4))
    off = _offsets((100, 1300))
    a = [x.detach().requires_grad_(True) for x in (q, k, v)]
    b = [x.detach().contiguous().requires_grad_(True) for x in (q, k, v)]
    x, y = pkg.packed_attention(*a, off, causal=True), pkg.packed_attention(*b, off, causal=True)
    assert torch.equal(x, y)
    for d, e in zip(torch.autograd.grad(x, a, g), torch.autograd.grad(y, b, g.contiguous())):
        assert torch.equal(d, e)
    pos, freq = torch.rand((1400, 1), device=DEV), torch.rand(32, device=DEV)
    for d, e in zip(pkg.axial_rotary(q, k, pos, freq, (32,)),
                    pkg.axial_rotary(q.contiguous(), k.contiguous(), pos, freq, (32,))):
        assert torch.equal(d, e)
