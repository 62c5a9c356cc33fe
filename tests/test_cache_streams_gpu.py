"""Streams of the paged KV cache's calls: whose memory is whose, and who waits for whom."""
import gc
import weakref

import pytest
import torch

import pages_ref as R
from lestramanika_b200 import PickleError
from lestramanika_b200.pages import KVPages, PageBatch, PageSlots

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_the_default_stream_as_a_handle():
    """Handle 0, given while another stream is the current one: scratch, and the wait for what was recorded there."""
    B = R.Batch("i8", 1, 128, 16, [5000], [1], 3)
    kv, table, _ = B.tensors()
    cache, batch = KVPages(1, B.n_pages, 16, 1, 128, pools=[B.pool]), PageBatch(kv, table)
    q = B.randn(1, 4, 128)
    want, out = torch.empty_like(q), torch.empty_like(q)
    assert cache.attn_workspace(batch, 4, 0) > 0
    cache.attn_dev(0, batch, q, want)
    short = PageBatch(kv, table, max_kv=4999)                 # a length above the bound: recorded
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(20_000_000)                         # on the other stream
        cache.attn_dev(0, batch, q, out, stream=0)
        cache.sync(0)
        assert torch.equal(out, want)
        with torch.cuda.stream(torch.cuda.default_stream()):
            torch.cuda._sleep(20_000_000)
        cache.attn_dev(0, short, q, out, stream=0)
        with pytest.raises(PickleError):
            cache.sync(0)


@pytest.mark.parametrize("handle", ["stream", "raw", "current"])
@pytest.mark.parametrize("prompt", [1, 20])
def test_batches_dropped_while_a_side_stream_is_behind(handle, prompt):
    """A serving loop on a stream that runs late: every step's batch is dropped at once, and the memory of the current stream
    is written over meanwhile. The same as the loop without haste."""
    HK, H, D, steps = 2, 8, 64, 24
    g = torch.Generator().manual_seed(4)
    rows = [[torch.randn((2 * prompt, n, D), generator=g).to(DEV) for n in (H, HK, HK)] for _ in range(steps)]

    def loop(stream, late):
        cache = KVPages(1, 80, 16, HK, D, rope_len=600)
        slots = PageSlots(cache)
        slots.admit("a")
        slots.admit("b")
        outs = []
        torch.cuda.synchronize()
        if late:
            with torch.cuda.stream(stream):
                torch.cuda._sleep(400_000_000)
        for q, k, v in rows:
            q, out = q.clone(), torch.empty_like(q)
            torch.cuda.current_stream().synchronize()
            batch = slots.batch(["a", "b"], [prompt, prompt])
            if handle == "current":
                with torch.cuda.stream(stream):
                    slots.step(0, batch, q, k, v, out)
            else:
                slots.step(0, batch, q, k, v, out, stream=stream if handle == "stream" else stream.cuda_stream)
            slots.advance(batch)
            outs.append((q, out))
            del batch
            junk = [torch.full((n,), 3, dtype=torch.int32, device=DEV) for n in (2, 2, 3, 4, 8, 16, 32, 64)]
            del junk
        torch.cuda.synchronize()
        cache.sync(stream)
        return [o for _, o in outs], cache.pools[0].clone()

    side = torch.cuda.Stream()
    want, got = loop(side, False), loop(side, True)
    assert torch.equal(want[1], got[1])
    for a, b in zip(want[0], got[0]):
        assert torch.equal(a, b)


def test_a_new_cache_on_a_stream_that_is_behind():
    """The constructor's fill is over before a call on another stream writes rows."""
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn((40, 2, 64), generator=g).to(DEV) for _ in "kv")
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    cache = KVPages(0, 2000, 16, 2, 64)
    kv, table = torch.tensor([40], dtype=torch.int32), torch.tensor([[5, 1900, 7]], dtype=torch.int32)
    start = torch.tensor([0, 40], dtype=torch.int32)
    with torch.cuda.stream(side):
        batch = PageBatch(kv.to(DEV), table.to(DEV), q_start=start.to(DEV))
    cache.append_dev(0, batch, k, v, stream=side)
    torch.cuda.synchronize()
    cache.read_dev(0, batch, ko, vo, stream=side)
    cache.sync(side)
    assert torch.equal(ko, k.bfloat16().float()) and torch.equal(vo, v.bfloat16().float())


def test_a_kept_batch_keeps_no_cache():
    B = R.Batch("i8", 1, 128, 16, [4000], [1], 7)
    kv, table, _ = B.tensors()
    batch, q = PageBatch(kv, table), B.randn(1, 4, 128)
    out, other = torch.empty_like(q), torch.empty_like(q)
    cache = KVPages(1, B.n_pages, 16, 1, 128, pools=[B.pool])
    cache.attn_dev(0, batch, q, out)
    gone = weakref.ref(cache)
    cache.sync()
    del cache
    gc.collect()
    assert gone() is None
    # another cache of the same sizes, and one of another type, whose call takes other pieces
    KVPages(1, B.n_pages, 16, 1, 128, pools=[B.pool]).attn_dev(0, batch, q, other)
    wide = R.Batch("bf16", 1, 128, 16, [4000], [1], 7)
    assert torch.equal(wide.tensors()[1], table)
    KVPages(0, wide.n_pages, 16, 1, 128, pools=[wide.pool]).attn_dev(0, batch, q, torch.empty_like(q))
    torch.cuda.synchronize()
    assert torch.equal(out, other)
