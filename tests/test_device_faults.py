"""A wait that gave up on the device becomes an exception for who asks."""

from __future__ import annotations

import contextlib
import types

import pytest
import torch


@pytest.mark.parametrize("status,error", [("OK", None), ("ERR_LIMIT", "gave up"), ("ERR_CUDA", "device_fault")])
def test_statuses(pkg, monkeypatch, status, error):
    N = pkg._native
    text = N.lib().rfdetr_status_string
    asked = []

    def take(stream):
        asked.append(stream)
        return getattr(N, status)

    monkeypatch.setattr(N, "lib", lambda: types.SimpleNamespace(rfdetr_take_device_fault=take,
                                                                rfdetr_status_string=text))
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream=5))
    if error is None:
        pkg.check_device_faults()
    else:
        with pytest.raises(RuntimeError, match=error):
            pkg.check_device_faults()
    assert asked == [5]


@pytest.mark.gpu
def test_a_wait_that_runs_out(pkg):
    """The library's self-test makes one give up; the next call finds the word clear."""
    N = pkg._native
    pkg.check_device_faults("cuda:0")
    result = torch.full((1,), -1, dtype=torch.int32, device="cuda:0")
    N.check(N.lib().rfdetr_selftest_bounded_wait(N.stream_of(result), 2000, result.data_ptr()), "selftest")
    with pytest.raises(RuntimeError, match="gave up"):
        pkg.check_device_faults()
    pkg.check_device_faults(0)
