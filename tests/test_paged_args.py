"""The Python layer's checks of what the paged operators would read or write out of
range, on the CPU: the library is a recorder and the current device is the CPU's."""
import pytest
import torch

import ternative_b200.backend as backend
from ternative_b200 import CUDABackend, DeviceWeight, LoraTable, PagedBatch, PagedCache, RopeConfig


class Recorder:
    """Stands in for the library: takes every call."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


@pytest.fixture
def be(monkeypatch):
    monkeypatch.setattr(backend, "_tensor", lambda x, name, dtype, ndim: x)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)   # what get_device() says of CPU tensors
    b = CUDABackend.__new__(CUDABackend)
    b.lib, b.ctx = Recorder(), None
    return b


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def cache(pages=8, page=16):
    k = torch.zeros(pages, page, 2, 64)
    return PagedCache(k, torch.zeros_like(k))


def both(be, c, b, **kw):
    """Each of the two calls over a cache."""
    q, k = torch.zeros(b.n_tokens, 4, 64), torch.zeros(b.n_tokens, 2, 64)
    yield lambda: be.attention_paged_d(torch.zeros_like(q), q, c, b, 4, 2, 64, 0.125, **kw)
    yield lambda: be.rope_append_paged_d(torch.zeros_like(q), q, k, k, c, b, RopeConfig(64), 4, 2, 64, **kw)


def table(ranks, K=64, N=32, values=None):
    return LoraTable([torch.zeros(r, K) for r in ranks], [torch.zeros(N, r) for r in ranks],
                     ints(*(ranks if values is None else values)), torch.ones(len(ranks)), 8)


def project(be, t, K=64, N=32, adapter=ints(0, 0), **kw):
    be.matmul_lora_d(torch.zeros(2, N), torch.zeros(2, K), 2, K, DeviceWeight(4096), N, t, adapter, **kw)


def test_a_table_that_is_a_slice(be):
    """Rows of a wider table are far enough apart for max_kv, but the slice has not the pages for it: the last row would
    be read behind its end."""
    wide = torch.zeros(2, 8, dtype=torch.int32)
    for pages, max_kv, ok in ((4, 64, True), (4, 65, False), (8, 128, True), (1, 17, False), (1, 16, True)):
        b = PagedBatch(ints(0, 1, 2), ints(max_kv, max_kv), wide[:, 8 - pages:], 2, 1, max_kv)
        for call in both(be, cache(), b):
            if ok:
                call()
            else:
                with pytest.raises(ValueError, match="block_table"):
                    call()
    assert len(be.lib.calls) == 6


def test_descriptors_of_another_device(be, monkeypatch):
    """A cache, a batch or adapters made on another device than the current one."""
    b = PagedBatch(ints(0, 1), ints(5), torch.zeros(1, 1, dtype=torch.int32), 1, 1, 5)
    c, t = cache(), table([4])
    for call in both(be, c, b):
        call()
    project(be, t)
    done = len(be.lib.calls)
    for d in (c, b, t):
        d.device = 3
        calls = [lambda: project(be, t)] if d is t else list(both(be, c, b))
        for call in calls:
            with pytest.raises(ValueError, match="device"):
                call()
        d.device = -1
    assert len(be.lib.calls) == done


@pytest.mark.parametrize("word", [torch.zeros(8, dtype=torch.uint8)[1:], torch.zeros(1, dtype=torch.int16),
                                  torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int32).numpy(), "status"],
                         ids=lambda w: str(getattr(w, "dtype", w)))
def test_status_words_that_are_none(be, word):
    """The kernels write 32 bits of device memory."""
    b = PagedBatch(ints(0, 1), ints(5), torch.zeros(1, 1, dtype=torch.int32), 1, 1, 5)
    calls = list(both(be, cache(), b, status=word)) + [lambda: project(be, table([4]), status=word)]
    for call in calls:
        with pytest.raises((ValueError, TypeError), match="status"):
            call()
    assert not be.lib.calls
    for ok in (None, 4096, ints(0), ints(0, 0)[1:]):
        for call in list(both(be, cache(), b, status=ok)) + [lambda: project(be, table([4]), status=ok)]:
            call()


def test_ranks_that_contradict_the_factors(be):
    """The kernels read rank[i] rows of A[i] and rows of B[i] rank[i] apart."""
    project(be, table([4, 8]))
    project(be, table([4, 8], values=[0, 8]))   # an adapter that is switched off
    for values in ([4, 7], [8, 8], [4, -8], [5, 8]):
        with pytest.raises(ValueError, match="rank"):
            table([4, 8], values=values)


def test_no_adapters_need_no_ids(be):
    project(be, table([]), adapter=None)
    with pytest.raises(ValueError, match="adapter"):
        project(be, table([4]), adapter=None)
