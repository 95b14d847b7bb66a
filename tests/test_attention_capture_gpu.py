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
