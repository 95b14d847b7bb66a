"""The current stream's handle, with and without torch's shorter way to it."""

from __future__ import annotations

import types

import pytest
import torch


def test_without_the_short_way(pkg, monkeypatch):
    """A torch that has no ``_cuda_getCurrentRawStream`` gives the same handle through its public function."""
    N = pkg._native
    asked = []

    def current_stream(device):
        asked.append(device)
        return types.SimpleNamespace(cuda_stream=77)

    monkeypatch.setattr(N, "_raw_stream", None)
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    tensor = types.SimpleNamespace(device=torch.device("cuda", 3))
    assert N.stream_of(tensor) == 77 and asked == [torch.device("cuda", 3)]


@pytest.mark.gpu
def test_both_ways_agree(pkg, monkeypatch):
    N = pkg._native
    x = torch.zeros(1, device="cuda:0")
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            short = N.stream_of(x)
            with monkeypatch.context() as m:
                m.setattr(N, "_raw_stream", None)
                assert N.stream_of(x) == short == stream.cuda_stream
