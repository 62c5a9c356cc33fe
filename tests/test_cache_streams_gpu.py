"""Streams of the paged KV cache's calls: whose memory is whose, and who waits for whom."""
import pytest
import torch

import pages_ref as R
from lestramanika_b200 import PickleError
from lestramanika_b200.pages import KVPages, PageBatch

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
