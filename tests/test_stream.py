"""The stream helper: whatever names a device gets that device's current stream (CPU, with a stand-in for torch's)."""
import types

import pytest
import torch

from fastmd_b200 import _lib


@pytest.fixture
def two_devices(monkeypatch):
    """Two devices whose current streams have the handles 100 and 101; device 0 is the current one."""

    def index(device):
        return 0 if device is None else device if isinstance(device, int) else torch.device(device).index or 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=100 + index(device)))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(_lib, "_raw_stream", lambda i: 100 + i, raising=False)


@pytest.mark.parametrize("device,handle", [(None, 100), (0, 100), (1, 101), ("cuda", 100), ("cuda:1", 101),
                                           (torch.device("cuda"), 100), (torch.device("cuda:1"), 101)])
def test_the_named_device_counts(two_devices, device, handle):
    assert _lib.stream(device) == handle


@pytest.mark.gpu
def test_the_current_stream_is_the_one(cuda):
    side = torch.cuda.Stream()
    for want in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(want):
            for device in (None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda:0")):
                assert _lib.stream(device) == want.cuda_stream
