"""Calls from threads of their own while a graph is captured."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_a_new_thread_during_a_capture(pkg):
    """A thread without a current context gets the device's by a call that a capture (of the strictest mode, which looks
    at every thread) allows."""
    rng = np.random.default_rng(0)
    q, k, v = (torch.tensor(rng.standard_normal((40, 2, 64)).astype(np.float32), device=DEV).to(torch.bfloat16)
               for _ in range(3))
    off = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    want = pkg.packed_attention(q, k, v, off)
    out, status = torch.zeros_like(q), []
    lib = pkg._native.lib()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="global"):
        args = [torch.cuda.current_stream().cuda_stream]
        for x in (q, k, v):
            args += [x.data_ptr(), *x.stride()[:2]]
        args += [off.data_ptr(), None, out.data_ptr(), None, None, None, 0, 1, 40, 40, 2, 2, 64, 0, 0.125]
        thread = threading.Thread(target=lambda: status.append(lib.rfdetr_packed_attention(*args)))
        thread.start()
        thread.join()
    assert status == [pkg._native.OK]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def _bf16(rng, *shape):
    return torch.tensor(rng.standard_normal(shape).astype(np.float32), device=DEV).to(torch.bfloat16)


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_both_passes_in_a_graph(pkg, dim):
    """Replayed on other inputs and other lengths, with the same bits as calls outside; the second backward kernel, which
    starts before the first has ended, among them."""
    rng = np.random.default_rng(dim)
    q, k, v = (_bf16(rng, 1500, h, dim).requires_grad_(True) for h in (4, 2, 2))
    g = _bf16(rng, 1500, 4, dim)
    off = torch.tensor([0, 700, 701, 1500], dtype=torch.int32, device=DEV)

    def call():
        out = pkg.packed_attention(q, k, v, off, causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for cuts in ((10, 900), (0, 0), (333, 1400)):
        with torch.no_grad():
            for x in (q, k, v, g):
                x.copy_(_bf16(rng, *x.shape))
        off.copy_(torch.tensor([0, *cuts, 1500], dtype=torch.int32))
        graph.replay()
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


def test_streams_side_by_side(pkg):
    """Both passes of every width at once on streams of their own, short and long, alone on few SMs or in clusters: the
    bits are those of one after the other."""
    rng = np.random.default_rng(9)
    jobs = []
    for dim in (32, 64, 128):
        for lengths in ((300,) * 4, (1700, 45, 900), (2500,)):
            n = sum(lengths)
            x = [_bf16(rng, n, h, dim).requires_grad_(True) for h in (6, 2, 2)]
            off = torch.tensor(np.cumsum([0, *lengths]), dtype=torch.int32, device=DEV)
            jobs.append((x, off, _bf16(rng, n, 6, dim)))

    def call(job):
        x, off, g = job
        out = pkg.packed_attention(*x, off, causal=True)
        return (out, *torch.autograd.grad(out, x, g))

    want = [call(job) for job in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for job, stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                got.append(call(job))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    pkg.check_device_faults()
