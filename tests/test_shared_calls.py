"""
What attend_shared hands to which kernels, without a GPU.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_amd import backend

from ._host import host_backend, sharing_batch


@pytest.mark.parametrize("scale, shared", [
    (0.125, True), (1e-38, True), (1e-50, False), (0.0, False), (-1e-50, False),
    (float("nan"), False)])
def test_a_scale_that_is_not_positive_in_32_bits_runs_as_attend(scale, shared, monkeypatch):
    monkeypatch.setattr(backend, "SHARED_PART_BYTES", 0)
    monkeypatch.setattr(backend, "SHARED_LEAST_BYTES", 0)
    bk = host_backend(monkeypatch)
    a = sharing_batch(bk)
    bk.attend_shared(torch.zeros((3, 32, 64), dtype=torch.float16), 0, scale, a)
    assert bk._lib.calls[-1][0] == ("pkv_attend_shared_batch" if shared else "pkv_attend_batch")


@pytest.mark.parametrize("scale", [0.125, -0.125])
def test_launches_go_to_the_backends_device(scale, monkeypatch):
    """Another device is current: both ways a batch may run make theirs current
    for their launch."""
    import contextlib

    monkeypatch.setattr(backend, "SHARED_PART_BYTES", 0)
    monkeypatch.setattr(backend, "SHARED_LEAST_BYTES", 0)
    bk, entered = host_backend(monkeypatch), []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        yield
        entered.append(len(bk._lib.calls))

    monkeypatch.setattr(backend, "_current_device", lambda: 5)
    monkeypatch.setattr(torch.cuda, "device", device)
    a = sharing_batch(bk)
    bk.attend_shared(torch.zeros((3, 32, 64), dtype=torch.float16), 0, scale, a)
    assert entered == [bk.device, 1]
