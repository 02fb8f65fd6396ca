"""The cache's Python calls beside several devices, with a stand-in for the library and for tensors: no GPU."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from h3vae_b200 import kernels as K


class Tensor:
    """What the calls ask of a CUDA tensor."""

    def __init__(self, shape, dtype, device):
        self.shape, self.dtype, self.device, self.ndim = torch.Size(shape), dtype, device, len(shape)

    def stride(self):
        return tuple(torch.Size(self.shape[i + 1:]).numel() for i in range(self.ndim))

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 64

    def new_empty(self, shape):
        return Tensor(shape if isinstance(shape, tuple) else (shape,), self.dtype, self.device)


class Library:
    """Records the current device at every call; workspaces depend on it."""

    def __init__(self, current):
        self.current, self.launched, self.workspaces = current, [], []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_workspace_size"):
                return 1000 * (1 + self.current[0])
            self.launched.append((name, self.current[0]))
            if "attention" in name or "select" in name:
                self.workspaces.append(args[-2])
            return 0
        return call


@pytest.fixture
def two_devices(monkeypatch):
    current = [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        try:
            yield
        finally:
            current[0] = before

    lib = Library(current)
    monkeypatch.setattr(K._lib, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(K, "_device_index", lambda: current[0], raising=False)
    monkeypatch.setattr(K, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch, "empty", lambda shape, device, dtype: Tensor(shape, dtype, device))
    monkeypatch.setattr(torch, "empty_like", lambda t: t)
    K._kv_workspace_bytes.cache_clear()
    yield lib
    K._kv_workspace_bytes.cache_clear()


def _calls(index):
    dev = torch.device("cuda", index)
    cache = SimpleNamespace(device=dev, struct=0, kv_heads=2, page_size=16, head_dim=64, num_pages=4,
                            k=Tensor((4, 2, 16, 64), torch.int8, dev))
    table, lens = Tensor((1, 2), torch.int32, dev), Tensor((1,), torch.int32, dev)
    k = Tensor((1, 2, 3, 64), torch.float16, dev)
    K.kv_write_i8(cache, table, lens, k, k)
    K.kv_read_i8(cache, table, lens, 3)
    K.attention_kv_i8(k, cache, table, lens, 1.0, out=k)
    K.kv_select_i8(k, cache, table, lens, 1)


def test_workspaces_are_those_of_the_device(two_devices):
    """The plan behind a workspace goes by the device's SMs: what was asked on one device is not used on another."""
    for index in (0, 1, 0):
        two_devices.current[0] = index
        _calls(index)
    assert two_devices.workspaces == [1000] * 2 + [2000] * 2 + [1000] * 2


def test_calls_launch_on_the_device_of_the_cache(two_devices):
    """With another device current, every call runs on the cache's and leaves the current one as it was."""
    for current, index in ((0, 1), (1, 0), (1, 1)):
        two_devices.current[0] = current
        two_devices.launched.clear()
        _calls(index)
        assert [d for _, d in two_devices.launched] == [index] * 4 and two_devices.current[0] == current
    assert two_devices.workspaces == [2000] * 2 + [1000] * 2 + [2000] * 2
