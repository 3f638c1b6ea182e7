"""The paged cache's and the sampler's launches go to their tensors' device, whichever is current (no GPU: the
runtime's current device and streams are stand-ins)."""
import contextlib
import types

import pytest
import torch

from fp4_attn_b200 import _lib, paged_cache, sampling


@pytest.fixture
def runtime(monkeypatch):
    """.current: the current device; .calls: (entry, arguments, device that was current)."""
    r = types.SimpleNamespace(current=0, calls=[], fail=False)

    @contextlib.contextmanager
    def device(index):
        was, r.current = r.current, index
        try:
            yield
        finally:
            r.current = was

    class Library:
        def __getattr__(self, name):
            def call(*args):
                r.calls.append((name, args, r.current))
                return 1 if r.fail else 0
            return call

        def fp4attn_last_error(self):
            return b"refused"

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: r.current)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "load", Library)
    return r


class Tensor:
    """As much of a CUDA tensor as the host side of a call looks at."""

    is_cuda = True

    def __init__(self, shape, dtype, index):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device("cuda", index)

    def dim(self):
        return len(self.shape)

    def stride(self):
        return (self.shape[-1], 1)

    def is_contiguous(self):
        return True

    def contiguous(self):
        return self

    def data_ptr(self):
        return 256


@pytest.mark.parametrize("current,index", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_calls_run_with_their_device_current(runtime, monkeypatch, current, index):
    runtime.current = current
    c = object.__new__(paged_cache.PagedNVFP4Cache)
    c._index, c._ref, c.max_seqs = index, 4096, 2
    c.release()
    monkeypatch.setattr(torch, "empty", lambda *shape, dtype, device: Tensor(
        shape if isinstance(shape[0], int) else shape[0], dtype, device.index))
    sampling.sample(Tensor((2, 5), torch.float32, index), Tensor((2,), torch.float32, index))
    t = Tensor((2, 3), torch.int64, index)
    sampling.accept_tree(Tensor((2, 3), torch.int32, index), t, t)
    assert [n for n, _, _ in runtime.calls] == ["fp4paged_truncate", "fp4_sample", "fp4_accept_tree"]
    for _, args, was in runtime.calls:
        assert was == index and args[-1] == 1000 + index
    assert runtime.current == current


def test_the_current_device_comes_back_after_an_error(runtime):
    runtime.fail = True
    with pytest.raises(RuntimeError, match="entry failed .1.: refused"):
        _lib.call_on(1, "entry")
    assert runtime.current == 0 and runtime.calls == [("entry", (1001,), 1)]


def test_a_workspaces_size_is_that_of_the_caches_device(runtime, monkeypatch):
    seen = []
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(
        fp4paged_attention_workspace_size=lambda B, Hq, Hkv, N: seen.append(runtime.current) or 64))
    c = object.__new__(paged_cache.PagedNVFP4Cache)
    c._index, c.device, c.num_kv_heads, c._work_bytes, c._spaces = 1, torch.device("cpu"), 2, {}, []
    assert c._workspace(1, 4, 1).numel() == 64 and c._workspace(1, 4, 1).numel() == 64
    assert seen == [1] and runtime.current == 0
