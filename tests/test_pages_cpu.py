"""The paged KV cache without a GPU: sizes, refusals (decided before anything touches a device) and page bookkeeping."""
import ctypes

import pytest
import torch

import pages_ref as R
from lestramanika_b200 import PickleError, lib
from lestramanika_b200.pages import BatchParams, PageBatch, PagesParams, PageSlots, pages_bytes
from lestramanika_b200.slots import SlotError

ARG, RANGE = -6, -7
A = 1 << 20          # a 16-byte aligned address that no refused call may touch


def _pages(**kw):
    d = dict(pool=A, kv_type=1, n_pages=4, page_size=16, n_kv_heads=2, head_dim=128, err=None)
    d.update(kw)
    return PagesParams(**d)


def _batch(**kw):
    d = dict(n_seqs=2, n_tok=2, max_q=1, max_kv=32, q_start=None, kv_len=A, table=A, table_stride=2)
    d.update(kw)
    return BatchParams(**d)


def _append(p=None, b=None, **kw):
    a = dict(H=8, rt=0, q=A, qs=0, k=A, ks=0, v=A, vs=0, sin=A, cos=A, half=64, rl=64, ot=0, qo=A, os=0)
    a.update(kw)
    p, b = p or _pages(), b or _batch()
    return lib().pickle_cuda_pages_append_dev(ctypes.byref(p), ctypes.byref(b), *a.values(), None)


def _read(p=None, b=None, **kw):
    a = dict(rt=0, k=A, ks=0, v=A, vs=0)
    a.update(kw)
    p, b = p or _pages(), b or _batch()
    return lib().pickle_cuda_pages_read_dev(ctypes.byref(p), ctypes.byref(b), *a.values(), None)


def _attn(p=None, b=None, **kw):
    a = dict(H=8, rt=0, q=A, qs=0, out=A, os=0, window=0, sinks=0, ws=A, wb=1 << 40)
    a.update(kw)
    p, b = p or _pages(), b or _batch()
    return lib().pickle_cuda_pages_attn_dev(ctypes.byref(p), ctypes.byref(b), *a.values(), None)


@pytest.mark.parametrize("kv,D", [("bf16", 64), ("i8", 128), ("e4m3", 64)])
def test_pool_bytes(kv, D):
    assert pages_bytes(R.KV[kv], 5, 48, 3, D) == 5 * 3 * 3 * R.cell_bytes(kv, D)
    assert pages_bytes(R.KV[kv], 1 << 24, 128, 8, D) == (1 << 24) * 8 * 8 * R.cell_bytes(kv, D)     # above 2^32


@pytest.mark.parametrize("bad", [dict(kv_type=3), dict(kv_type=-1), dict(n_pages=0), dict(page_size=0),
                                 dict(page_size=24), dict(page_size=-16), dict(n_kv_heads=0), dict(head_dim=96),
                                 dict(head_dim=0), dict(pool=None), dict(pool=A + 8)])
def test_refused_pages(bad):
    for call in (_append, _read, _attn):
        assert call(p=_pages(**bad)) == ARG
    if "pool" not in bad:
        d = dict(kv_type=1, n_pages=4, page_size=16, n_kv_heads=2, head_dim=128)
        d.update(bad)
        assert pages_bytes(*d.values()) == 0


@pytest.mark.parametrize("bad,code", [(dict(n_seqs=0), ARG), (dict(n_tok=-1), ARG), (dict(max_q=0), ARG),
                                      (dict(max_kv=-1), ARG), (dict(kv_len=None), ARG), (dict(table=None), ARG),
                                      (dict(table_stride=0), ARG), (dict(max_kv=33), RANGE),
                                      (dict(n_tok=3), ARG), (dict(max_q=2), ARG)])
def test_refused_batches(bad, code):
    for call in (_append, _read, _attn):
        assert call(b=_batch(**bad)) == code


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(q=None), dict(qo=None), dict(k=A + 4), dict(v=A + 8),
                                 dict(q=A + 2), dict(rt=2), dict(ot=-1), dict(ks=255), dict(ks=258), dict(vs=2),
                                 dict(qs=1020), dict(rt=1, ks=260), dict(H=0), dict(half=4), dict(half=72),
                                 dict(half=-8), dict(sin=None), dict(cos=None), dict(sin=A + 4), dict(rl=-1)])
def test_refused_append(bad):
    assert _append(**bad) == ARG


def test_append_past_the_rope_table_is_refused():
    assert _append(rl=31) == RANGE


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(rt=2), dict(k=A + 8), dict(ks=100), dict(vs=257)])
def test_refused_read(bad):
    assert _read(**bad) == ARG


@pytest.mark.parametrize("bad", [dict(H=0), dict(H=7), dict(H=18), dict(q=None), dict(out=None), dict(q=A + 8),
                                 dict(out=A + 4), dict(rt=2), dict(qs=1000), dict(os=1026), dict(window=-1),
                                 dict(sinks=-1)])
def test_refused_attn(bad):
    assert _attn(**bad) == ARG


def test_calls_without_rows_do_nothing():
    b = _batch(n_tok=0, q_start=A)
    assert _append(b=b) == 0 and _read(b=b) == 0 and _attn(b=b) == 0


def test_null_structures_are_refused():
    L = lib()
    assert L.pickle_cuda_pages_attn_dev(None, None, 8, 0, A, 0, A, 0, 0, 0, None, 0, None) == ARG
    assert L.pickle_cuda_pages_workspace(None, None, 8, 0, 0, 0) == 0


def test_batch_checks_its_tensors():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for args in ((i(2).long(), i(2, 3)), (i(2), i(3, 3)), (i(2), i(2)), (i(2), i(2, 3), i(2)),
                 (i(2), i(2, 6)[:, ::2])):
        with pytest.raises(PickleError) as e:
            PageBatch(*args)
        assert e.value.code == ARG
    b = PageBatch(torch.tensor([3, 5], dtype=torch.int32), i(2, 3), torch.tensor([0, 2, 7], dtype=torch.int32))
    assert (b.n_tok, b.max_q, b.max_kv) == (7, 5, 5)


class _FakeCache:
    n_pages, page_size, _dev = 6, 16, torch.device("cpu")


def test_slots_hand_out_and_take_back_pages():
    s = PageSlots(_FakeCache())
    s.admit("a")
    s.admit("b")
    b = s.batch(["a", "b"], [17, 1])
    assert b.kv_len.tolist() == [17, 1] and b.q_start.tolist() == [0, 17, 18] and b.max_q == 17
    assert len(s.free) == 3 and b.table.shape == (2, 2) and b.table[1, 1] == -1
    assert s.batch(["a", "b"], [17, 1]).table.tolist() == b.table.tolist()      # asked again before it ran
    s.advance(b)
    one = s.batch(["b", "a"])
    assert one.q_start is None and one.kv_len.tolist() == [2, 18] and one.max_q == 1
    with pytest.raises(SlotError):
        s.batch(["a", "b"], [60, 20])
    assert len(s.free) == 3                                                     # nothing was taken
    with pytest.raises(SlotError):
        s.batch(["a", "a"])
    with pytest.raises(SlotError):
        s.admit("a")
    s.release("a")
    assert len(s.free) == 5 and s.position("b") == 1
    s.admit("a")
    assert s.position("a") == 0


def test_trim_keeps_sinks_and_the_window():
    s = PageSlots(_FakeCache())
    s.admit("a")
    s.advance(s.batch(["a"], [90]))
    s.trim("a", 0)
    assert len(s.free) == 0
    s.trim("a", 30, 4)              # the next row (position 90) sees 61..90 and 0..3: pages 0 and 3..5 stay
    assert [p >= 0 for p in s.pages["a"]] == [True, False, False, True, True, True]
    t = s.batch(["a"], [6]).table.tolist()[0]
    assert t[1] == t[2] == -1 and len(s.free) == 2
    s.release("a")
    assert sorted(s.free) == list(range(6))


def test_reference_blocks():
    """The 64-bit restatement itself: exact round trips and the borders of a scale."""
    x = torch.zeros(1, 32)
    x[0, 0] = 127.0
    assert R.quantise(x, "i8")[2].item() == 127
    x[0, 0] = 127.5
    assert R.quantise(x, "i8")[2].item() == 128
    x[0, 0] = 464.0
    v, _, s = R.quantise(x, "e4m3")
    assert s.item() == 127 and v[0, 0] == 448
    x[0, 1] = float("inf")
    assert torch.isnan(R.quantise(x, "e4m3")[0]).all()
