"""Attention over pages whose rows differ in magnitude: along the sequence, between blocks of 32, and far apart."""
import pytest
import torch

import pages_ref as R
from lestramanika_b200.pages import KVPages, PageBatch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)

# Rows of two sequences and query heads of a KV head: the kernel for few rows with one token and with several; the one
# for many with both its tiles on the same rows, and with two blocks of rows.
CALLS = {"one": (4, [1, 1]), "few": (2, [4, 3]), "twin": (2, [40, 5]), "many": (4, [70, 5])}
FORMS = [(kv, rows, D, call) for kv in ("i8", "e4m3", "bf16") for rows in ("f32", "bf16") for D in (64, 128) for call in CALLS]


@pytest.fixture(params=["1", "2", "0"], ids=["whole", "halves", "planned"])
def pieces(request, monkeypatch):
    """How many pieces a sequence's keys are cut into: a piece finds its own magnitudes, and the planned ones are short."""
    monkeypatch.setenv("PICKLE_CUDA_PAGES_SPLITS", request.param)


def _amp(pattern, f, D):
    """2^0 to 2^f over positions or blocks, as a function for R.Batch."""
    def of(b, which, m):
        j = torch.arange(m, dtype=torch.float32)
        one, top = torch.ones(m), torch.full((m,), 2.0 ** f)
        col = {"rise": torch.where(j < m // 2, one, top), "fall": torch.where(j < m // 2, top, one),
               "drift up": 2.0 ** (f * j / max(1, m - 1)), "drift down": 2.0 ** (f * (1 - j / max(1, m - 1))),
               "first": torch.where(j < 4, one, top), "block": one}[pattern]
        x = col[:, None].expand(m, D).clone()
        if pattern == "block":
            x[:, D - 32:] *= 2.0 ** f
        return x
    return of


def _check(B, G, rows, q, extra=None, window=0, sinks=0):
    """attn_dev of q against 64 bits, with R.attn_bound, the held weights of 8-bit pages and `extra`."""
    kv, table, start = B.tensors()
    cache = KVPages(R.KV[B.kv], B.n_pages, B.page, B.HK, B.D, pools=[B.pool])
    out = torch.full_like(q, 7.0)
    cache.attn_dev(0, PageBatch(kv, table, q_start=start), q, out, window=window, sinks=sinks)
    cache.sync()
    assert torch.isfinite(out).all()
    for b, (n, m) in enumerate(zip(B.q_len, B.kv_len)):
        t = B.start[b]
        ref, mass, size = R.attend(q[t:t + n], B.k[b], B.v[b], B.positions(b), window, sinks)
        tol = R.attn_bound(mass, size, ref, rows, m, rows == "bf16")
        if B.kv != "bf16":
            held = [R.held_weights(B.k[b][h], B.v[b][h], B.positions(b), window, sinks) for h in range(B.HK)]
            tol = tol + torch.cat([x.expand(-1, G, -1) for x in held], 1)
        if extra is not None:
            tol = tol + extra(b, mass)
        err = (out[t:t + n].double() - ref).abs()
        assert (err <= tol).all(), f"sequence {b}: {float((err / tol).max()):.2f} of the bound"


@pytest.mark.parametrize("kv,rows,D,call", FORMS)
@pytest.mark.parametrize("pattern", ["rise", "fall", "drift up", "drift down", "first", "block"])
def test_magnitudes_that_differ(pattern, kv, rows, D, call, monkeypatch):
    """Steps of every power of two up to 2^12, over which every code of both 8-bit types is exact in the products. One
    piece: what follows a step is taken with what came before it."""
    monkeypatch.setenv("PICKLE_CUDA_PAGES_SPLITS", "1")
    G, q_len = CALLS[call]
    for f in range(13) if pattern in ("rise", "fall") else (5, 6, 7, 12):
        B = R.Batch(kv, 1, D, 16, [260, 37], q_len, 81 + f, amp=_amp(pattern, f, D))
        _check(B, G, rows, (B.randn(B.n_tok, G, D) * 2.0 ** -f).to(R.ROWS[rows]))


@pytest.mark.parametrize("kv,rows,D", [("i8", "f32", 128), ("i8", "bf16", 64), ("e4m3", "f32", 64), ("e4m3", "bf16", 128),
                                       ("bf16", "f32", 128)])
@pytest.mark.parametrize("call", ["one", "twin"])
@pytest.mark.parametrize("pattern", ["rise", "fall", "drift up"])
def test_magnitudes_that_differ_between_pieces(pattern, call, kv, rows, D, pieces):
    """Long contexts, whole and cut into pieces that find different magnitudes and are joined."""
    G, q_len = CALLS[call]
    for f in (6, 12):
        B = R.Batch(kv, 1, D, 64, [2501, 5], q_len, 91 + f, amp=_amp(pattern, f, D))
        _check(B, G, rows, (B.randn(B.n_tok, G, D) * 2.0 ** -f).to(R.ROWS[rows]))


@pytest.mark.parametrize("kv,rows,D,call", [x for x in FORMS if x[0] != "bf16"])
@pytest.mark.parametrize("which", ["k", "v", "v first"])
def test_a_key_far_larger_than_what_is_attended_to(which, kv, rows, D, call, monkeypatch):
    """k: a block of one key is 2^f larger than all others, and q is next to 0 there. v: the same key's v is, and no row
    gives it weight. The others lose 2^-24 of it at most, and nothing while they lie within 2^15 of it."""
    monkeypatch.setenv("PICKLE_CUDA_PAGES_SPLITS", "1")
    G, q_len = CALLS[call]
    for f in (9, 13, 15, 17, 20, 23, 25, 30):
        at = 0 if which == "v first" else 133

        def amp(b, w, m):
            x = torch.ones(m, D)
            if m > at:
                if which == "k" and w == 0:
                    x[at, :32] = 2.0 ** f
                elif which != "k" and w == 1:
                    x[at] = 2.0 ** f
                elif which != "k":
                    x[at] = 0.0
            return x

        B = R.Batch(kv, 1, D, 16, [260, 37], q_len, 101 + f, amp=amp)
        q = B.randn(B.n_tok, G, D)
        if which == "k":
            q[..., :32] *= 2.0 ** (-f - 12)
        else:
            # Every other key has a score near 40 or more: its weight is e^-40 of theirs.
            kv_len, table, start = B.tensors()
            cache = KVPages(R.KV[kv], B.n_pages, 16, 1, D, pools=[B.pool])
            for b, m in enumerate(B.kv_len):
                every = [j for j in range(m) if j != at]
                B.k[b][:, every, 0] = 64.0
            k = torch.cat([x[0] for x in B.k]).float().unsqueeze(1).contiguous()
            v = torch.cat([x[0] for x in B.v]).float().unsqueeze(1).contiguous()
            whole = torch.tensor([0] + [sum(B.kv_len[:i + 1]) for i in range(2)], dtype=torch.int32, device=DEV)
            cache.append_dev(0, PageBatch(kv_len, table, q_start=whole), k, v)
            ko, vo = torch.empty_like(k), torch.empty_like(v)
            cache.read_dev(0, PageBatch(kv_len, table, q_start=whole), ko, vo)
            cache.sync()
            for b in range(2):
                B.k[b] = ko[whole[b]:whole[b + 1], 0].double().unsqueeze(0)
                B.v[b] = vo[whole[b]:whole[b + 1], 0].double().unsqueeze(0)
            q[..., 0] = 40.0 * D ** 0.5 / 64.0
        q = q.to(R.ROWS[rows])

        def extra(b, mass):
            if f <= 9:
                return 0.0
            t = B.start[b]
            return R.shared_exponents(q[t:t + B.q_len[b]], B.k[b], B.v[b], mass)

        _check(B, G, rows, q, extra)


@pytest.mark.parametrize("kv,rows,D", [("i8", "f32", 128), ("i8", "bf16", 64), ("e4m3", "f32", 64), ("e4m3", "bf16", 128),
                                       ("bf16", "f32", 128), ("bf16", "bf16", 64)])
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("k,v", [(60, 80), (-60, -80), (-60, 80), (0, 88)])
def test_magnitudes_far_from_1(k, v, kv, rows, D, call):
    G, q_len = CALLS[call]
    B = R.Batch(kv, 1, D, 16, [260, 37], q_len, 111, amp=lambda b, which, m: 2.0 ** (v if which else k))
    _check(B, G, rows, (B.randn(B.n_tok, G, D) * 2.0 ** -k).to(R.ROWS[rows]))


@pytest.mark.parametrize("kv", ["i8", "e4m3"])
@pytest.mark.parametrize("call", CALLS)
def test_a_key_that_is_not_finite_among_the_largest(kv, call, pieces):
    """Scales at the top of their range, and one of 255 behind them, which all rows see."""
    G, q_len = CALLS[call]
    B = R.Batch(kv, 1, 128, 16, [260, 37], q_len, 99, amp=lambda b, which, m: 1.0 if which else 2.0 ** 124)
    cache = KVPages(R.KV[kv], B.n_pages, 16, 1, 128, pools=[B.pool])
    kv_len, table, start = B.tensors()
    k, v = torch.full((1, 1, 128), 2.0 ** 127, device=DEV), torch.ones((1, 1, 128), device=DEV)
    for at in (48, 49, 179):                        # cells 3 and 11: the same warp's first and last, where four share them
        if at == 179:
            k[0, 0, 70] = float("nan")
        one = PageBatch(torch.tensor([at + 1], dtype=torch.int32, device=DEV), table[:1].contiguous())
        cache.append_dev(0, one, k, v)
    q = B.randn(B.n_tok, G, 128) * 2.0 ** -120
    out = torch.empty_like(q)
    cache.attn_dev(0, PageBatch(kv_len, table, q_start=start), q, out)
    cache.sync()
    assert torch.isnan(out[:q_len[0]]).all()


@pytest.mark.parametrize("rows", ["f32", "bf16"])
@pytest.mark.parametrize("D,half,H,HK", [(128, 64, 32, 8), (64, 32, 9, 3), (128, 16, 5, 1)])
def test_rotated_q_is_rounded_once(rows, D, half, H, HK):
    """To F32: half a step, 2^-24 of the value, and 2^-46 of the products' size for the errors' own sum. To BF16: half of
    its step, 2^-8, from a sum whose two roundings are half an F32 step of the size each."""
    B = R.Batch("i8", HK, D, 16, [400], [400], 61, fill=False)
    kv, table, start = B.tensors()
    ang = torch.rand((400, half), generator=torch.Generator().manual_seed(5), dtype=torch.float64) * 6.283185307179586
    rope = ang.sin().float().to(DEV), ang.cos().float().to(DEV)
    cache = KVPages(1, B.n_pages, 16, HK, D, pools=[B.pool], rope=rope)
    batch = PageBatch(kv, table, q_start=start)
    q, k = B.randn(400, H, D).to(R.ROWS[rows]), B.randn(400, HK, D).to(R.ROWS[rows])
    wide, narrow = torch.empty((400, H, D), device=DEV), torch.empty((400, H, D), dtype=torch.bfloat16, device=DEV)
    cache.append_dev(0, batch, k, k, q=q, q_out=wide)
    cache.append_dev(0, batch, k, k, q=q, q_out=narrow)
    cache.sync()
    ref = R.rotate(q, *rope, half)
    lo, hi = q[..., :half].double().abs(), q[..., half:2 * half].double().abs()
    s, c = (x.double().abs()[:, None] for x in rope)
    size = torch.cat([c * lo + s * hi, s * lo + c * hi, 0 * q[..., 2 * half:].double()], -1)
    assert ((wide.double() - ref).abs() <= 2.0 ** -24 * ref.abs() + 2.0 ** -46 * size).all()
    off = 2 * 2.0 ** -24 * size
    assert ((narrow.double() - ref).abs() <= off + 2.0 ** -8 * (ref.abs() + off)).all()
    if half < D // 2:                                  # and what is not rotated stays
        assert torch.equal(wide[..., 2 * half:], q[..., 2 * half:].float())
