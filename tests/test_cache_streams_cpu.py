"""Streams of the paged KV cache's calls without a GPU: stand-ins for torch's streams record what would be done."""
import sys
import types
import weakref

import pytest
import torch

from lestramanika_b200.pages import KVPages, PageBatch


class FakeStream:
    done = False                                       # whether events have come to pass

    def __init__(self, handle, kind="stream"):
        self.cuda_stream, self.kind, self.waits = handle, kind, 0

    def record_event(self):
        return types.SimpleNamespace(query=lambda: FakeStream.done)

    def synchronize(self):
        self.waits += 1


class FakeTorch:
    """What KVPages asks of torch, on the CPU. ExternalStream of handle 0 is a stream of its own, as torch's is."""

    def __init__(self):
        self.default, self.now, self.scratch = FakeStream(0), FakeStream(11), []
        self.uint8, self.int32, self.float32, self.bfloat16 = torch.uint8, torch.int32, torch.float32, torch.bfloat16
        self.device = lambda *a: torch.device("cpu")
        self._C = types.SimpleNamespace(_cuda_getCurrentRawStream=lambda d: self.now.cuda_stream)
        self.cuda = types.SimpleNamespace(
            current_stream=lambda d=None: self.now, default_stream=lambda d=None: self.default,
            ExternalStream=lambda h, device=None: FakeStream(h or 99, "external"), Stream=FakeStream, stream=self._on,
            is_current_stream_capturing=lambda: False)

    class _On:
        def __init__(self, t, s):
            self.t, self.s = t, s

        def __enter__(self):
            self.was, self.t.now = self.t.now, self.s

        def __exit__(self, *a):
            self.t.now = self.was

    def _on(self, s):
        return self._On(self, s)

    def empty(self, n, **kw):
        self.scratch.append(self.now.cuda_stream)
        return torch.empty(n, dtype=torch.uint8)

    def zeros(self, *n, **kw):
        kw.pop("device")
        self.filled = self.now.waits
        return torch.zeros(*n, **kw)


@pytest.fixture
def fake():
    return FakeTorch()


def _cache(fake, monkeypatch):
    with monkeypatch.context() as m:
        m.setitem(sys.modules, "torch", fake)          # what the constructor imports and keeps
        return KVPages(1, 4, 16, 2, 64)


@pytest.mark.parametrize("given,handle", [(None, 11), (0, 0), (7, 7), (FakeStream(5), 5)])
def test_scratch_belongs_to_the_call_s_stream(fake, monkeypatch, given, handle):
    cache = _cache(fake, monkeypatch)
    cache._scratch(64, given)
    assert fake.scratch == [handle]


def test_sync_waits_for_the_stream_of_handle_0(fake, monkeypatch):
    cache = _cache(fake, monkeypatch)
    cache.sync(0)
    assert fake.default.waits == 1


@pytest.mark.parametrize("given,handle", [(None, 11), (0, 0), (FakeStream(5), 5)])
@pytest.mark.parametrize("starts", [False, True])
def test_a_batch_outlives_the_streams_that_read_it(fake, monkeypatch, given, handle, starts):
    seen = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: seen.append((t.data_ptr(), s.cuda_stream)))
    kv, table, start = (torch.tensor(x, dtype=torch.int32) for x in ([3, 5], [[0, 1], [2, 3]], [0, 1, 2]))
    batch = PageBatch(kv, table, q_start=start if starts else None)
    cache = _cache(fake, monkeypatch)
    for _ in range(2):
        assert cache._call(batch, 0, given) == handle
        assert cache._call(batch, 0, FakeStream(23)) == 23
    want = [kv, table] + [start] * starts
    own = {t.data_ptr() for t in cache.pools + [cache.err]}
    for h in (handle, 23):
        assert sorted(p for p, s in seen if s == h and p not in own) == sorted(t.data_ptr() for t in want)


def test_a_cache_outlives_the_streams_that_use_it(fake, monkeypatch):
    seen = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: seen.append((t.data_ptr(), s.cuda_stream)))
    rope = torch.zeros(2, 40, 32)
    with monkeypatch.context() as m:
        m.setitem(sys.modules, "torch", fake)
        cache = KVPages(1, 4, 16, 2, 64, n_layers=2, rope=(rope[0], rope[1]))
    own = sorted(t.data_ptr() for t in (*cache.pools, cache.err, rope[0], rope[1]))
    batch = PageBatch(torch.tensor([3], dtype=torch.int32), torch.tensor([[0]], dtype=torch.int32))
    batch._streams.update((11, 5))                     # used with another cache before
    cache._call(batch, 0, None)
    cache._call(batch, 1, FakeStream(5))
    for h in (11, 5):
        assert sorted(p for p, s in seen if s == h and p in own) == own
    # once: a new batch costs its own arrays, whatever the number of layers
    before = len(seen)
    cache._call(PageBatch(torch.tensor([3], dtype=torch.int32), torch.tensor([[0]], dtype=torch.int32)), 0, None)
    assert len(seen) == before + 2


def test_a_new_cache_is_filled_before_any_stream_can_use_it(fake, monkeypatch):
    _cache(fake, monkeypatch)
    assert fake.now.waits == fake.filled + 1


def test_what_the_stream_of_a_handle_reads_is_held(fake, monkeypatch):
    """No stream that may be gone is asked: batches are held until an event behind their last call has come to pass."""
    monkeypatch.setattr(torch.Tensor, "record_stream", None)
    monkeypatch.setattr(FakeStream, "done", False)
    cache, alive = _cache(fake, monkeypatch), []

    def call(n, also=None):
        for _ in range(n):
            batch = PageBatch(torch.tensor([3], dtype=torch.int32), torch.tensor([[0]], dtype=torch.int32))
            alive.append(weakref.ref(batch.kv_len))
            for layer in range(2):
                assert cache._call(batch, 0, 7) == 7
            if also is not None:
                cache._call(also, 0, 7)

    kept = PageBatch(torch.tensor([4], dtype=torch.int32), torch.tensor([[0]], dtype=torch.int32))
    mine = weakref.ref(kept.kv_len)
    call(200, kept)
    assert all(x() is not None for x in alive)
    FakeStream.done = True
    call(130, kept)
    del kept                                           # its last call is not behind an event yet
    assert mine() is not None
    assert sum(x() is not None for x in alive) <= 3 * 64 and all(x() is not None for x in alive[-64:])
    call(200)
    assert mine() is None
    cache.sync(7)
    assert all(x() is None for x in alive)
