"""The paged KV cache on the GPU: writer, reader and attention against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import pages_ref as R
from lestramanika_b200 import PickleError
from lestramanika_b200.pages import KVPages, PageBatch, PageSlots

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _cache(B, rope=None):
    return KVPages(R.KV[B.kv], B.n_pages, B.page, B.HK, B.D, pools=[B.pool], rope=rope)


def _batch(B, **kw):
    kv, table, start = B.tensors()
    return PageBatch(kv, table, q_start=start, **kw)


def _tables(n, half, seed=5):
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand((n, half), generator=g, dtype=torch.float64) * 6.283185307179586
    return ang.sin().float().to(DEV), ang.cos().float().to(DEV)


def _check_attn(B, G, rows, window=0, sinks=0, q=None, out=None, batch=None, cache=None):
    q = B.randn(B.n_tok, G * B.HK, B.D).to(R.ROWS[rows]) if q is None else q
    out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format) if out is None else out
    cache = cache or _cache(B)
    batch = batch or _batch(B)
    cache.attn_dev(0, batch, q, out, window=window, sinks=sinks)
    cache.sync()
    for b, (n, m) in enumerate(zip(B.q_len, B.kv_len)):
        if not n:
            continue
        t = B.start[b]
        ref, mass, size = R.attend(q[t:t + n], B.k[b], B.v[b], B.positions(b), window, sinks)
        tol = R.attn_bound(mass, size, ref, rows, m, rows == "bf16")
        err = (out[t:t + n].double() - ref).abs()
        assert torch.isfinite(out[t:t + n]).all(), f"sequence {b}"
        assert (err <= tol).all(), f"sequence {b}: {float((err / tol).max()):.2f} of the bound"
    return out


# ---- append and read --------------------------------------------------------------

@pytest.mark.parametrize("kv", ["bf16", "i8", "e4m3"])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("D,half,HK,H,page", [(128, 64, 8, 32, 16), (64, 32, 3, 9, 48), (128, 16, 1, 1, 32),
                                              (64, 0, 2, 10, 128)])
def test_append_writes_the_defined_codes(kv, rows, D, half, HK, H, page):
    kv_len, q_len = [1, 40, 0, 129, 33], [1, 17, 0, 129, 2]
    B = R.Batch(kv, HK, D, page, kv_len, q_len, 11)
    before = B.pool.clone()
    rope = _tables(256, half) if half else None
    q, k, v = (B.randn(B.n_tok, n, D).to(R.ROWS[rows]) for n in (H, HK, HK))
    for q_type in ("f32", "bf16"):
        B.pool.copy_(before)
        cache, batch = _cache(B, rope), _batch(B)
        q_out = torch.empty((B.n_tok, H, D), dtype=R.ROWS[q_type], device=DEV)
        cache.append_dev(0, batch, k, v, q=q, q_out=q_out)
        cache.sync()
        written = torch.zeros_like(B.pool, dtype=torch.bool)
        for b, n in enumerate(q_len):
            if not n:
                continue
            t, pos = B.start[b], B.positions(b)
            if half:
                sin, cos = rope[0][pos], rope[1][pos]
                kr, qr = (R.rotate(x[t:t + n], sin, cos, half) for x in (k, q))
                size = R.rotate(q[t:t + n].abs(), -sin.abs(), cos.abs(), half).abs() + R.rotate(
                    q[t:t + n].abs(), sin.abs(), cos.abs(), half).abs()
            else:
                kr, qr = k[t:t + n].double(), q[t:t + n].double()
                size = qr.abs()
            # two products and a sum, each off by half a step of at most |c x| + |s y|
            tol = 2 * 2.0 ** -24 * size + (2.0 ** -8 * qr.abs() if q_type == "bf16" else 0) + 1e-37
            assert ((q_out[t:t + n].double() - qr).abs() <= tol).all()
            for which, x in ((0, kr.float()), (1, v[t:t + n].float())):
                val, codes, scale = R.quantise(x, kv)
                for i, j in enumerate(pos):
                    raw, s = B.stored(None, b, j, which)
                    if kv == "bf16":
                        assert torch.equal(raw.contiguous().view(torch.bfloat16).double(), val[i])
                    else:
                        assert torch.equal(s.long(), scale[i].long())
                        typ = torch.int8 if kv == "i8" else torch.float8_e4m3fn
                        assert torch.equal(raw.contiguous().view(typ).double(), codes[i])
        # nothing but the rows of the call was written
        n_rows = sum(q_len) * HK * 2
        per_row = D * 2 if kv == "bf16" else D + D // 32
        changed = int((B.pool != before).sum())
        assert changed <= n_rows * per_row
        for b, m in enumerate(kv_len):
            for j in range(m - q_len[b]):
                for which in (0, 1):
                    raw, s = B.stored(None, b, j, which)
                    keep = B.k[b][:, j] if which == 0 else B.v[b][:, j]
                    typ = {"bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}[kv]
                    x = raw.contiguous().view(typ).double()
                    if s is not None:
                        x = x * R.pow2(s.long() - 127).repeat_interleave(32, -1)
                    assert torch.equal(x, keep)
        # q may be rotated in place, and be left out
        if q_type == rows:
            q2 = q.clone()
            cache.append_dev(0, batch, k, v, q=q2, q_out=q2)
            assert torch.equal(q2, q_out)
        cache.append_dev(0, batch, k, v)
        # and the rows read back are what the codes stand for
        for r_type in ("f32", "bf16"):
            ko, vo = (torch.full((B.n_tok, HK, D), 9.0, dtype=R.ROWS[r_type], device=DEV) for _ in "kv")
            cache.read_dev(0, batch, ko, vo)
            cache.sync()
            for b, n in enumerate(q_len):
                if n:
                    t, pos = B.start[b], B.positions(b)
                    kr = R.rotate(k[t:t + n], rope[0][pos], rope[1][pos], half) if half else k[t:t + n].double()
                    assert torch.equal(ko[t:t + n], R.quantise(kr.float(), kv)[0].to(R.ROWS[r_type]))
                    assert torch.equal(vo[t:t + n], R.quantise(v[t:t + n].float(), kv)[0].to(R.ROWS[r_type]))


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_append_of_extreme_blocks(kv):
    """Ties, borders of a scale, the smallest and largest numbers, zeros, infinities and NaN."""
    top = 127.5 if kv == "i8" else 464.0
    rows = []
    for amp in (1.0, 2.0 ** -20, 2.0 ** 90, 2.0 ** -111, 2.0 ** -118, 1e-40, 1.5 * 2.0 ** 127 / top, 2.0 ** 119):
        for a in (top, np.nextafter(np.float32(top), np.float32(0)), np.nextafter(np.float32(top), np.float32(1e9)),
                  top / 2, 1.0):
            x = np.linspace(-1, 1, 32) * a * 0.99
            x[5] = a
            x[6:14] = np.array([0.5, 1.5, 2.5, -0.5, -1.5, 17.0, 0.0, -0.0]) * a / top
            rows.append(np.float64(x) * amp)
    for bad in (np.inf, -np.inf, np.nan):
        x = np.ones(32)
        x[31] = bad
        rows.append(x)
    rows.append(np.zeros(32))
    rows += [np.ones(32)] * (-len(rows) % 4)
    x = torch.tensor(np.array(rows), dtype=torch.float64).clamp(-3.4028234e38, 3.4028234e38).where(
        torch.isfinite(torch.tensor(np.array(rows))), torch.tensor(np.array(rows))).float().view(-1, 1, 128)
    n = x.shape[0]
    B = R.Batch(kv, 1, 128, 16, [n], [n], 3, fill=False)
    cache, batch = _cache(B), _batch(B)
    x = x.to(DEV).contiguous()
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    cache.append_dev(0, batch, x, x.flip(0).contiguous())
    cache.read_dev(0, batch, ko, vo)
    cache.sync()
    ref = R.quantise(x, kv)[0]
    for got, want in ((ko, ref), (vo, ref.flip(0))):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.double()), torch.nan_to_num(want))


@pytest.mark.parametrize("op", ["append", "read", "attn"])
def test_padded_entries_and_rows_behind_the_last_sequence(op):
    B = R.Batch("i8", 2, 64, 16, [5, 0, 20], [1, 1, 1], 4)
    rope = _tables(32, 32)
    cache = _cache(B, rope)
    kv, table, start = B.tensors()
    batch = PageBatch(kv, table, q_start=start, n_tok=5, max_q=1, max_kv=20)      # 3 rows used, 2 behind
    x = B.randn(5, 2, 64)
    q = B.randn(5, 6, 64)
    before = B.pool.clone()
    a, c = torch.full_like(x, 3.0), torch.full_like(x, 3.0)
    qo = torch.full_like(q, 3.0)
    if op == "append":
        cache.append_dev(0, batch, x, x, q=q, q_out=qo)
        assert (qo[1] == 0).all() and (qo[3:] == 3).all() and (qo[0] != 3).any()
        # one row of each live sequence, and nothing else
        assert int((B.pool != before).any(-1).sum()) <= 2 * B.HK
    elif op == "read":
        cache.read_dev(0, batch, a, c)
        assert (a[1] == 0).all() and (c[1] == 0).all() and (a[3:] == 3).all() and (c[3:] == 3).all()
        assert torch.equal(a[2].double(), B.k[2][:, 19])
    else:
        cache.attn_dev(0, batch, q, qo)
        assert (qo[1] == 0).all() and (qo[3:] == 3).all()
    cache.sync()


def test_more_rows_than_positions_gives_zero_rows():
    """A sequence with more rows than its length: the first ones lie before position 0."""
    B = R.Batch("bf16", 1, 64, 16, [3], [3], 6)
    kv, table, _ = B.tensors()
    batch = PageBatch(kv, table, q_start=torch.tensor([0, 40], dtype=torch.int32, device=DEV))
    q = B.randn(40, 4, 64)
    out = torch.full_like(q, 5.0)
    cache = _cache(B)
    cache.attn_dev(0, batch, q, out)
    cache.sync()
    assert (out[:37] == 0).all()
    ref, mass, size = R.attend(q[37:], B.k[0], B.v[0], [0, 1, 2], 0, 0)
    assert ((out[37:].double() - ref).abs() <= R.attn_bound(mass, size, ref, "f32", 3, False)).all()


# ---- attention ------------------------------------------------------------------------

LENS = [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("kv", ["bf16", "i8", "e4m3"])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,HK,page", [(1, 3, 16), (4, 2, 48), (8, 1, 32), (5, 2, 128)])
def test_single_tokens(kv, rows, D, G, HK, page):
    B = R.Batch(kv, HK, D, page, LENS + [0], [1] * (len(LENS) + 1), 21)
    _check_attn(B, G, rows)
    # without q_start: one row each
    q = B.randn(B.n_tok, G * HK, D).to(R.ROWS[rows])
    o1, o2 = torch.empty_like(q), torch.empty_like(q)
    c = _cache(B)
    kvl, table, start = B.tensors()
    c.attn_dev(0, PageBatch(kvl, table), q, o1)
    c.attn_dev(0, PageBatch(kvl, table, q_start=start), q, o2)
    assert torch.equal(o1, o2)


@pytest.mark.parametrize("kv", ["bf16", "i8", "e4m3"])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,HK,page", [(1, 2, 16), (3, 1, 48), (4, 2, 128), (8, 1, 32)])
def test_chunks(kv, rows, D, G, HK, page):
    kv_len = [1, 40, 0, 129, 300, 511, 64]
    q_len = [1, 3, 0, 129, 60, 257, 2]
    _check_attn(R.Batch(kv, HK, D, page, kv_len, q_len, 22), G, rows)


@pytest.mark.parametrize("kv,D", [("bf16", 64), ("bf16", 128), ("i8", 64), ("i8", 128), ("e4m3", 128)])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("G,n", [(1, 300), (2, 256), (8, 20), (3, 40)])
def test_tiles_of_rows_that_end_apart(kv, rows, D, G, n):
    """Both tiles of rows over long contexts: with few heads a group the first one's keys end tiles before the other's."""
    _check_attn(R.Batch(kv, 1, D, 32, [1500, 1100], [n, 1], 41), G, rows)


@pytest.mark.parametrize("kv,rows,D", [("i8", "f32", 128), ("e4m3", "bf16", 128), ("bf16", "bf16", 64),
                                       ("bf16", "f32", 128), ("i8", "bf16", 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 16), (100, 0), (100, 300), (128, 33),
                                          (1000, 5), (2147483647, 0)])
@pytest.mark.parametrize("one", [True, False])
def test_window_and_sinks(kv, rows, D, window, sinks, one):
    kv_len = [1, 20, 129, 300, 777]
    q_len = [1] * 5 if one else [1, 20, 100, 3, 400]
    _check_attn(R.Batch(kv, 2, D, 16, kv_len, q_len, 23), 4, rows, window, sinks)


@pytest.mark.parametrize("one", [True, False])
def test_pages_out_of_the_window_are_never_touched(one):
    """Stale table entries and NaN rows where no row of the call can see."""
    m, W, S = 700, 100, 20
    B = R.Batch("i8", 2, 128, 16, [m], [1 if one else 50], 24)
    first = m - B.q_len[0] - W + 1
    for i in range(-(-S // 16), first // 16):
        B.pool[B.table_host[0][i]] = 255
        B.table_host[0][i] = -1 if i % 2 else 10 ** 9
    _check_attn(B, 4, "bf16", W, S)


@pytest.mark.parametrize("kv", ["bf16", "i8"])
def test_long_contexts_split_and_join(kv):
    B = R.Batch(kv, 1, 128, 64, [9001], [1], 25)
    _check_attn(B, 8, "f32")
    B = R.Batch(kv, 1, 64, 64, [9001, 5], [40, 2], 26)
    _check_attn(B, 4, "bf16")
    B = R.Batch(kv, 1, 64, 64, [9001, 5], [40, 2], 26)
    _check_attn(B, 4, "f32", 8000, 3)


@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
def test_large_scores_stay_finite(one, rows):
    """Scores of several thousands: the softmax is one-hot."""
    B = R.Batch("e4m3", 1, 128, 16, [400], [1 if one else 64], 27)
    q = (B.randn(B.n_tok, 4, 128) * 1000).to(R.ROWS[rows])
    out = torch.empty_like(q)
    c = _cache(B)
    c.attn_dev(0, _batch(B), q, out)
    c.sync()
    ref, mass, size = R.attend(q, B.k[0], B.v[0], B.positions(0), 0, 0)
    # the scores' own rounding decides between near ties: the output stays inside the values' range
    assert torch.isfinite(out).all()
    assert (out.double().abs() <= B.v[0].abs().max() * (1 + 2.0 ** -7)).all()
    sure = (R.attend(q * 1.001, B.k[0], B.v[0], B.positions(0), 0, 0)[0] - ref).abs().amax(-1) < 1e-6
    assert ((out.double() - ref).abs() <= 2.0 ** -7 * mass + 1e-5)[sure].all() and sure.any()


@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
def test_strided_rows(one, rows):
    """q as a slice of a fused projection's rows, out as a slice of a wider buffer."""
    B = R.Batch("i8", 2, 64, 16, [50, 33], [1, 1] if one else [40, 33], 28)
    H = 8
    fused = B.randn(B.n_tok, H + 4, 64).to(R.ROWS[rows])
    wide = torch.full((B.n_tok, H + 3, 64), 4.0, dtype=R.ROWS[rows], device=DEV)
    _check_attn(B, 4, rows, q=fused[:, :H], out=wide[:, 2:2 + H])
    assert (wide[:, :2] == 4).all() and (wide[:, 2 + H:] == 4).all()
    rope = _tables(64, 32)
    c, batch = _cache(B, rope), _batch(B)
    q1, k1, v1 = (x.contiguous() for x in (fused[:, :H], fused[:, H:H + 2], fused[:, H + 2:]))
    o1, o2 = torch.empty_like(q1), torch.empty_like(wide)
    c.append_dev(0, batch, k1, v1, q=q1, q_out=o1)
    p1 = B.pool.clone()
    c.append_dev(0, batch, fused[:, H:H + 2], fused[:, H + 2:], q=fused[:, :H], q_out=o2[:, 1:1 + H])
    assert torch.equal(o1, o2[:, 1:1 + H]) and torch.equal(p1, B.pool)
    c.sync()


@pytest.mark.parametrize("one", [True, False])
def test_pool_beyond_4_gib(one):
    """Pages at the end of a pool whose byte offsets pass 2^32."""
    n_pages = (5 << 30) // (33 * 128)
    small = R.Batch("i8", 1, 128, 16, [100], [1 if one else 70], 29)
    pool = torch.empty(n_pages * 33 * 128, dtype=torch.uint8, device=DEV)
    at = n_pages - small.n_pages
    pool.view(n_pages, -1)[at:] = small.pool.view(small.n_pages, -1)
    small.table_host = [[p + at for p in small.table_host[0]]]
    cache = KVPages(1, n_pages, 16, 1, 128, pools=[pool])
    _check_attn(small, 4, "bf16", cache=cache)


@pytest.mark.parametrize("one", [True, False])
def test_device_side_errors_are_reported_and_contained(one):
    n = 1 if one else 20
    B = R.Batch("i8", 2, 64, 16, [40, 50, 60], [n] * 3, 30)
    q = B.randn(B.n_tok, 8, 64)
    good = torch.empty_like(q)
    cache = _cache(B)
    cache.attn_dev(0, _batch(B), q, good)
    cache.sync()
    kv, table, start = B.tensors()

    def same_but(batch, bad):
        out = torch.full_like(q, 2.0)
        cache.attn_dev(0, batch, q, out)
        with pytest.raises(PickleError) as e:
            cache.sync()
        assert e.value.code == -9
        keep = [b for b in range(3) if b != bad]
        for b in keep:
            assert torch.equal(out[b * n:(b + 1) * n], good[b * n:(b + 1) * n])
        assert torch.isfinite(out).all()

    t = table.clone()
    t[1, 1] = B.n_pages                                                   # a page id outside the pool
    same_but(PageBatch(kv, t, q_start=start), 1)
    t[1, 1] = -1
    same_but(PageBatch(kv, t, q_start=start), 1)
    same_but(PageBatch(kv, table, q_start=start, n_tok=3 * n, max_q=n, max_kv=55), 2)      # a length above max_kv
    k = B.randn(B.n_tok, 2, 64)
    before = B.pool.clone()
    t = table.clone()
    t[1, 3] = -1                                                          # the page of sequence 1's last positions
    cache.append_dev(0, PageBatch(kv, t, q_start=start, n_tok=3 * n, max_q=n, max_kv=60), k, k)
    with pytest.raises(PickleError):
        cache.sync()
    written = [B.table_host[b][j // 16] for b in range(3) for j in B.positions(b) if (b, j // 16) != (1, 3)]
    others = [p for p in range(B.n_pages) if p not in written]
    assert torch.equal(B.pool[others], before[others]) and not torch.equal(B.pool, before)
    cache.attn_dev(0, _batch(B), q, good)
    cache.sync()


# ---- streams, graphs, sessions ------------------------------------------------------------

@pytest.mark.parametrize("one", [True, False])
def test_graph_follows_lengths_and_two_graphs_run_at_once(one):
    n = 1 if one else 33
    B = R.Batch("i8", 2, 128, 16, [600, 300], [n, n], 31)
    cache = _cache(B)
    kv, table, start = B.tensors()
    batch = PageBatch(kv, table, q_start=start, n_tok=2 * n, max_q=n, max_kv=600)
    q = [B.randn(B.n_tok, 8, 128) for _ in range(2)]
    out = [torch.zeros_like(x) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    cache.attn_dev(0, batch, q[0], out[0])
    graphs = []
    for s, x, o in zip(streams, q, out):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cache.attn_dev(0, batch, x, o)
        graphs.append(g)
    for lens in ([600, 300], [n, 299], [37, n]):
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        B.kv_len = lens
        torch.cuda.synchronize()
        for _ in range(5):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, o in zip(q, out):
            for b in range(2):
                ref, mass, size = R.attend(x[b * n:(b + 1) * n], B.k[b][:, :lens[b]], B.v[b][:, :lens[b]],
                                           B.positions(b), 0, 0)
                assert ((o[b * n:(b + 1) * n].double() - ref).abs() <=
                        R.attn_bound(mass, size, ref, "f32", 600, False)).all()
    cache.sync()


def test_other_streams_and_explicit_workspace():
    B = R.Batch("e4m3", 2, 128, 16, [5000, 10], [1, 1], 32)
    cache, batch = _cache(B), _batch(B)
    q = B.randn(2, 8, 128).bfloat16()
    want = _check_attn(B, 4, "bf16", q=q, cache=cache, batch=batch)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        out = torch.empty_like(q)
        torch.cuda.synchronize()
        cache.attn_dev(0, batch, q, out, stream=stream)
        cache.sync(stream)
        assert torch.equal(out, want)
    need = cache.attn_workspace(batch, 8, 1)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(q)
    cache.attn_dev(0, batch, q, out, workspace=ws)
    assert torch.equal(out, want)
    if need:
        with pytest.raises(PickleError) as e:
            cache.attn_dev(0, batch, q, out, workspace=ws[:need - 16])
        assert e.value.code == -6
    cache.sync()


@pytest.mark.parametrize("kv,rows,window,sinks", [("i8", "f32", 0, 0), ("e4m3", "bf16", 40, 5), ("bf16", "f32", 40, 0)])
def test_session_of_requests(kv, rows, window, sinks):
    """Prompts, mixed steps, window eviction, release and reuse through PageSlots; every row against the whole history."""
    HK, G, D, page = 2, 4, 64, 16
    cache = KVPages(R.KV[kv], 24, page, HK, D, n_layers=2, rope_len=400, rope_theta=500.0)
    slots = PageSlots(cache)
    g = torch.Generator().manual_seed(8)
    hist = {}

    def call(counts):
        reqs = list(counts)
        batch = slots.batch(reqs, [counts[r] for r in reqs])
        T = sum(counts.values())
        for layer in range(2):
            q, k, v = (torch.randn((T, n, D), generator=g).to(DEV).to(R.ROWS[rows]) for n in (G * HK, HK, HK))
            raw = q.clone()
            out = torch.empty_like(q)
            slots.step(layer, batch, q, k, v, out, window=window, sinks=sinks)
            cache.sync()
            t = 0
            for r in reqs:
                n, p0 = counts[r], slots.position(r)
                pos = list(range(p0, p0 + n))
                sin, cos = cache.rope[0][pos], cache.rope[1][pos]
                kk = R.quantise(R.rotate(k[t:t + n], sin, cos, D // 2).float(), kv)[0].transpose(0, 1)
                vv = R.quantise(v[t:t + n].float(), kv)[0].transpose(0, 1)
                old = hist.setdefault((r, layer), (kk[:, :0], vv[:, :0]))
                hist[r, layer] = kk, vv = torch.cat([old[0], kk], 1), torch.cat([old[1], vv], 1)
                qr = R.rotate(raw[t:t + n], sin, cos, D // 2)
                assert ((q[t:t + n].double() - qr).abs() <= 2.0 ** (-8 if rows == "bf16" else -22) * (qr.abs() + 6)).all()
                ref, mass, size = R.attend(q[t:t + n], kk, vv, pos, window, sinks)
                tol = R.attn_bound(mass, size, ref, rows, kk.shape[1], rows == "bf16")
                assert ((out[t:t + n].double() - ref).abs() <= tol).all(), r
                t += n
        slots.advance(batch)
        for r in reqs:
            slots.trim(r, window, sinks)

    slots.admit("a")
    slots.admit("b")
    call({"a": 70, "b": 9})
    for _ in range(3):
        call({"b": 1, "a": 1})
    slots.admit("c")
    call({"c": 50, "a": 1, "b": 17})
    slots.release("b")
    del hist["b", 0], hist["b", 1]
    slots.admit("b")
    call({"b": 33, "c": 1, "a": 2})
    for _ in range(20):
        call({"a": 1, "b": 1, "c": 1})
    if window:
        assert len(slots.free) + sum(p >= 0 for o in slots.pages.values() for p in o) == 24
        assert any(p < 0 for p in slots.pages["a"])


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[9000] + [1] * 40, [1] * 300, [5000, 0, 4999, 0, 0, 3], [513] * 97, list(range(1, 700, 2))])
def test_ragged_decodes(rows, lens):
    """Long sequences next to short ones and unused entries, more sequences than a CTA has threads: the pieces that the
    longest one is cut into leave the others with empty ones."""
    B = R.Batch("e4m3", 2, 64, 16, lens, [1] * len(lens), 43)
    q = B.randn(B.n_tok, 6, 64).to(R.ROWS[rows])
    first = _check_attn(B, 3, rows, q=q)
    assert torch.equal(first, _check_attn(B, 3, rows, q=q))             # the same bits again
    _check_attn(B, 3, rows, 300, 20, q=q)


def test_starts_that_do_not_ascend_touch_nothing_else():
    """q_start [0, 5, 3, 4]: the second sequence has -2 rows, row 4 lies in no sequence, and row 3 is the third's. What has
    rows is written and attended to, and the error word says the rest."""
    B = R.Batch("i8", 2, 128, 16, [40, 32, 48], [5, 0, 1], 51)
    cache, H = _cache(B), 6
    kv, table, _ = B.tensors()
    start = torch.tensor([0, 5, 3, 4], dtype=torch.int32, device=DEV)
    batch = PageBatch(kv, table, q_start=start, n_tok=6, max_q=5, max_kv=48)
    q = torch.randn((6, H, 128), generator=torch.Generator().manual_seed(1)).to(DEV)
    out = torch.full_like(q, 7.0)
    for window in (0, 20):
        cache.attn_dev(0, batch, q, out, window=window)
        with pytest.raises(PickleError):
            cache.sync()
    pool = B.pool.clone()
    k = torch.randn((6, 2, 128), generator=torch.Generator().manual_seed(2)).to(DEV)
    cache.append_dev(0, batch, k, k)
    with pytest.raises(PickleError):
        cache.sync()
    k_out, v_out = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    cache.read_dev(0, batch, k_out, v_out)
    with pytest.raises(PickleError):
        cache.sync()
    assert torch.equal(out[5], torch.full_like(out[5], 7.0)) and torch.equal(k_out[4:], torch.full_like(k_out[4:], 7.0))
    changed = (pool != B.pool).view(B.n_pages, -1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {p for row in B.tensors()[1].tolist() for p in row if p >= 0}


@pytest.mark.parametrize("rows", ["f32", "bf16"])
def test_calls_without_rows(rows):
    B = R.Batch("i8", 2, 64, 16, [20, 0], [0, 0], 52)
    cache = _cache(B)
    kv, table, start = B.tensors()
    batch = PageBatch(kv, table, q_start=start)
    before = B.pool.clone()
    k, q = (torch.empty((0, h, 64), dtype=R.ROWS[rows], device=DEV) for h in (2, 4))
    cache.append_dev(0, batch, k, k, q=q, q_out=q)
    cache.read_dev(0, batch, k, k)
    cache.attn_dev(0, batch, q, q)
    cache.sync()
    assert torch.equal(before, B.pool)


def test_refused_workspaces():
    B = R.Batch("i8", 1, 128, 16, [4000], [1], 53)
    cache, batch = _cache(B), _batch(B)
    q = B.randn(1, 4, 128)
    need = cache.attn_workspace(batch, 4, 0)
    assert need > 0
    for ws in (torch.empty(need - 1, dtype=torch.uint8, device=DEV), torch.empty(need, dtype=torch.uint8),
               torch.empty(2 * need, dtype=torch.uint8, device=DEV)[::2], torch.empty(need + 8, dtype=torch.uint8, device=DEV)[8:]):
        with pytest.raises(PickleError):
            cache.attn_dev(0, batch, q, torch.empty_like(q), workspace=ws)


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("lens,most", [([4000, 30, 1, 700, 0, 2000], 4000), ([600, 590], 16000), ([3000], 3000),
                                       ([2500] + [17] * 60, 2500), ([500] * 128, 2000), ([500] * 129, 2000)])
def test_chunks_of_ragged_contexts(rows, lens, most):
    """Pieces are cut to what the sequences' lengths say, not to the longest that the host allows for."""
    new = [min(9, m) for m in lens]
    B = R.Batch("i8", 1, 128, 32, lens, new, 61)
    kv, table, start = B.tensors()
    wide = torch.full((len(lens), -(-most // 32)), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    batch = PageBatch(kv, wide, q_start=start, n_tok=B.n_tok, max_q=9, max_kv=most)
    q = B.randn(B.n_tok, 4, 128).to(R.ROWS[rows])
    first = _check_attn(B, 4, rows, q=q, batch=batch)
    assert torch.equal(first, _check_attn(B, 4, rows, q=q, batch=batch))
    _check_attn(B, 4, rows, 300, 20, q=q, batch=batch)


@pytest.mark.parametrize("kv", ["bf16", "i8", "e4m3"])
@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,n", [(1, 5), (2, 4), (4, 40), (8, 60), (1, 200)])
@pytest.mark.parametrize("which,window", [("k", 0), ("v", 0), ("k", 3), ("v", 3)])
def test_rows_that_do_not_see_a_number_that_is_not_finite(kv, rows, D, G, n, which, window):
    """A NaN or an infinity in k or v at a position that some rows of the call see and others do not: those that do not
    get their numbers, those that do get none. Without a window it is the last row but two of the call, with one the row
    before the call."""
    _check_unseen(kv, rows, D, G, n, which, window, 300)


@pytest.mark.parametrize("kv,rows", [("bf16", "f32"), ("bf16", "bf16"), ("i8", "bf16"), ("e4m3", "f32")])
@pytest.mark.parametrize("G,n", [(2, 3), (4, 20)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_numbers_that_are_not_finite_in_split_contexts(kv, rows, G, n, which):
    """The same where the keys are cut into pieces that are joined."""
    _check_unseen(kv, rows, 128, G, n, which, 0, 9000)


def _check_unseen(kv, rows, D, G, n, which, window, length):
    B = R.Batch(kv, 2, D, 16, [length, 77], [n, 3], 71)
    cache, batch = _cache(B), _batch(B)
    assert length < 9000 or cache.attn_workspace(batch, 2 * G, 0 if rows == "f32" else 1, window) > 0
    at = length - (2 if n < 5 else 3) if not window else length - n - 1
    k, v = torch.zeros((1, 2, D), device=DEV), torch.zeros((1, 2, D), device=DEV)
    k[0, 0], v[0, 0] = B.k[0][0, at].float(), B.v[0][0, at].float()
    k[0, 1], v[0, 1] = B.k[0][1, at].float(), B.v[0][1, at].float()
    (k if which == "k" else v)[0, 1, D - 7] = float("inf") if which == "v" and not window else float("nan")
    one = PageBatch(torch.tensor([at + 1], dtype=torch.int32, device=DEV), B.tensors()[1][:1].contiguous())
    cache.append_dev(0, one, k, v)
    q = B.randn(B.n_tok, 2 * G, D).to(R.ROWS[rows])
    out = torch.full_like(q, 7.0)
    cache.attn_dev(0, batch, q, out, window=window)
    cache.sync()
    for b, t in ((0, 0), (1, n)):
        m = B.q_len[b]
        ref, mass, size = R.attend(q[t:t + m], B.k[b], B.v[b], B.positions(b), window, 0)
        tol = R.attn_bound(mass, size, ref, rows, B.kv_len[b], rows == "bf16")
        sees = torch.tensor([b == 0 and at <= p and (not window or at > p - window) for p in B.positions(b)], device=DEV)
        good = torch.ones_like(ref, dtype=torch.bool)
        good[sees, G:] = False                                       # KV head 1's query heads
        err = (out[t:t + m].double() - ref).abs()
        assert torch.isfinite(out[t:t + m][good]).all()
        assert (err[good] <= tol[good]).all(), f"{float((err / tol)[good].max()):.2f} of the bound"
        if b == 0:
            assert 0 < int(sees.sum()) < m
            bad = out[:m][sees, G:]
            assert (~torch.isfinite(bad)).any(-1).all()
            if which == "k":
                assert torch.isnan(bad).all()
