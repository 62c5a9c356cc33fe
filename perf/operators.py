"""Measured cases of the paged KV cache: its writer, its reader and the attention that reads it.

A page pool is one uint8 tensor [n_pages][n_kv_heads][page_size / 16][cell]. A cell holds 16 positions of one
KV head: K rows, V rows, then (8-bit types) K scales and V scales, with one scale byte for 32 elements:

  bf16   a row is D BF16 numbers, there are no scales
  i8     a row is D int8 codes c, element = c * 2^(scale - 127)
  e4m3   a row is D E4M3 codes c, element = c * 2^(scale - 127)

The scale of a block is the smallest power of two that keeps every code in range (2^-111 at least); a block with a
value that is not finite gets scale 255 and reads back as NaN. Position p of sequence b lies in page
table[b][p / page_size]. Sequence b's rows of a call are its last positions: row i of n is position kv_len[b] - n + i.

  append  rotates q and k by the position's sin / cos row (NeoX halves, rounded once to F32), writes k and v
          into their pages, gives the rotated q; the rows are then read back
  read    gives rows of the cache as F32 or BF16 numbers
  attn    softmax(q k^T / sqrt(D)) v over the keys at or before each query's position and, with a window, the last
          `window` of them and the first `sinks` of the sequence
"""
import math

import torch

own = False

_KV = {"bf16": 0, "i8": 1, "e4m3": 2}
_ROWS = {"f32": torch.float32, "bf16": torch.bfloat16}


def _case(name, op, kv, rows, B, H, HK, D, page, ctx, qlen, ragged, window=0, sinks=0):
    c = {"op": op, "kv": kv, "rows": rows, "B": B, "H": H, "HK": HK, "D": D, "page": page, "ctx": ctx, "qlen": qlen,
         "ragged": ragged, "window": window, "sinks": sinks}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decode step of 64 requests, 8B-shaped heads: the projections' F32 rows go into the cache.
        _case("append-step-b64", "append", "i8", "f32", 64, 32, 8, 128, 16, 4096, 1, True),
        # Four prompts of up to 2048 tokens, 7B-shaped heads, BF16 activations.
        _case("append-prompts-4x2048", "append", "e4m3", "bf16", 4, 32, 32, 128, 64, 2048, 2048, True),
        # The last rows of a few short sequences, as a check or a copy to another cache takes them.
        _case("read-tails", "read", "e4m3", "f32", 3, 12, 4, 64, 32, 777, 101, True),
        # Eight whole sequences out of the pages, for another device or another cache.
        _case("read-8x4096", "read", "i8", "bf16", 8, 32, 8, 128, 16, 4096, 4096, False),
        # One conversation, 8B-shaped: latency counts.
        _case("decode-b1-4096", "attn", "i8", "bf16", 1, 32, 8, 128, 16, 4096, 1, False),
        # A server's decode step: 64 requests of different lengths, F32 activations.
        _case("decode-b64-ragged", "attn", "e4m3", "f32", 64, 32, 8, 128, 32, 4096, 1, True),
        # 70B-shaped heads, 16 long contexts.
        _case("decode-70b-b16-32768", "attn", "i8", "bf16", 16, 64, 8, 128, 16, 32768, 1, False),
        # The same heads with a sliding window and visible first tokens over unquantised pages.
        _case("decode-window-b16", "attn", "bf16", "f32", 16, 64, 8, 128, 64, 32768, 1, True, 4096, 64),
        # Sixteen new tokens each (a short question, or drafted tokens to check) over existing contexts.
        _case("chunk-8x16-4096", "attn", "i8", "bf16", 8, 32, 8, 128, 16, 4096, 16, True),
        # A long prompt taken in pieces: 2048 tokens after 8192 cached ones.
        _case("chunk-2048-on-8192", "attn", "e4m3", "bf16", 1, 32, 8, 128, 32, 10240, 2048, False),
        # Whole prompts, 7B-shaped heads, unquantised pages.
        _case("prompts-4x2048", "attn", "bf16", "bf16", 4, 32, 32, 128, 128, 2048, 2048, False),
        # Ragged prompts with a window and sinks, F32 activations, head_dim 64.
        _case("prompts-window-f32", "attn", "i8", "f32", 2, 16, 2, 64, 16, 4001, 4001, True, 1000, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["append", "read", "attn", "attn", "attn"])
        HK = rng.choice([1, 2, 4, 8, 8, 32])
        G = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        c = _case(None, op, rng.choice(list(_KV)), rng.choice(list(_ROWS)), _log(rng, 1, 64), HK * G, HK,
                  rng.choice([64, 128, 128]), rng.choice([16, 32, 48, 64, 128]), _log(rng, 1, 32768), 1,
                  rng.random() < 0.7)
        if op != "attn" or rng.random() < 0.5:
            c["qlen"] = min(c["ctx"], _log(rng, 1, 4096))
        if op == "attn" and rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 1, 8192), rng.choice([0, 1, 4, 64, 100])
        rows = c["B"] * c["ctx"] * HK * c["D"]
        if rows > 16 * 32768 * 8 * 128 // 2 or c["B"] * c["qlen"] * c["H"] * c["D"] > 4 * 2048 * 32 * 128:
            continue
        if op == "attn" and (c["B"] * c["H"] * c["qlen"] * c["ctx"] > 6e8 or work(c)["flops"] > 1.3e11):
            continue
        return c


def _lengths(c):
    """(rows of the call, length) of each sequence; a ragged decode batch of 8 or more has an unused last entry."""
    B, n, ctx = c["B"], c["qlen"], c["ctx"]
    q, kv = [n] * B, [ctx] * B
    if c["ragged"]:
        for b in range(1, B):
            kv[b] = 1 + int((ctx - 1) * (b * 0.6180339887 % 1.0))
            q[b] = min(kv[b], 1 + int((n - 1) * (b * 0.7548776662 % 1.0)))
        if n == 1 and B >= 8:
            kv[B - 1] = 0
    return q, kv


def _elem_bytes(c):
    return 2.0 if c["kv"] == "bf16" else 1.0 + 1.0 / 32


def work(c):
    q, kv = _lengths(c)
    H, HK, D = c["H"], c["HK"], c["D"]
    io = 4 if c["rows"] == "f32" else 2
    tok = sum(n for n, m in zip(q, kv) if m)
    new = 2.0 * tok * HK * D
    if c["op"] == "append":   # q, k, v in; q and the cache rows out; the rows in again and out as numbers
        return {"bytes": tok * H * D * io * 2 + new * io * 2 + new * _elem_bytes(c) * 2, "flops": 0}
    if c["op"] == "read":
        return {"bytes": new * (io + _elem_bytes(c)), "flops": 0}
    W, S, rows, pairs = c["window"], c["sinks"], 0, 0
    for n, m in zip(q, kv):
        if not m:
            continue
        first = m - n
        if not W:
            rows += m
            pairs += n * (2 * m - n + 1) // 2
        else:
            lo = max(0, first - W + 1)
            rows += m - lo + min(S, lo)
            # position p sees min(p + 1, W) recent keys and the sinks before them
            full = max(0, min(n, W - 1 - first + 1))          # queries at p < W see p + 1 keys
            pairs += full * (2 * first + full + 1) // 2
            for_rest = n - full
            p0 = first + full
            sunk = max(0, min(for_rest, S + W - 1 - p0))      # queries whose sinks are partly in the window
            pairs += for_rest * W + sunk * (2 * (p0 + 1 - W) + sunk - 1) // 2 + (for_rest - sunk) * S
    return {"bytes": rows * 2.0 * HK * D * _elem_bytes(c) + tok * H * D * io * 2, "flops": 4.0 * D * H * pairs}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _quantise(x, kv):
    """Codes (uint8 [..., D * bytes]) and scales (uint8 [..., D / 32], or None) of F32 rows [..., D]."""
    if kv == "bf16":
        return x.to(torch.bfloat16).view(torch.uint8), None
    blocks = x.unflatten(-1, (-1, 32))
    amax = blocks.abs().amax(-1)
    finite = torch.isfinite(blocks).all(-1)
    # the power of two from the bits of the largest value: one more where it would round past the largest code
    bump, shift = (0x10000, 6) if kv == "i8" else (0x17FFFF, 8)
    scale = (((amax.view(torch.int32) + bump) >> 23) - shift).clamp_(min=16)
    scale = torch.where(finite, scale, 255)
    factor = torch.where(finite, (254 - scale) << 23, 0).to(torch.int32).view(torch.float32)     # 2^(127 - scale)
    scaled = torch.where(finite[..., None], blocks, 0.0).double() * factor[..., None]
    if kv == "i8":
        codes = torch.round(scaled).to(torch.int8).view(torch.uint8)
    else:
        codes = scaled.float().to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.flatten(-2), scale.to(torch.uint8)


def _numbers(codes, scales, kv):
    """F32 numbers [..., D] that codes (and scales) stand for."""
    if kv == "bf16":
        return codes.view(torch.bfloat16).float()
    x = (codes.view(torch.int8) if kv == "i8" else codes.view(torch.float8_e4m3fn)).float().unflatten(-1, (-1, 32))
    s = scales.to(torch.int32)
    f = torch.where(s == 255, float("nan"), (s << 23).view(torch.float32))
    return (x * f[..., None]).flatten(-2)


def _fields(pool, c):
    """Views of a pool (or of gathered pages [..., HK, cells, bytes]): K codes, V codes, K scales, V scales."""
    D, n = c["D"], c["D"] * (2 if c["kv"] == "bf16" else 1)
    k = pool[..., :16 * n].unflatten(-1, (16, n))
    v = pool[..., 16 * n:32 * n].unflatten(-1, (16, n))
    if c["kv"] == "bf16":
        return k, v, None, None
    s = pool[..., 32 * n:].unflatten(-1, (2, 16, D // 32))
    return k, v, s[..., 0, :, :], s[..., 1, :, :]


def prepare(case, seed):
    c = case
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    B, H, HK, D, ps = c["B"], c["H"], c["HK"], c["D"], c["page"]
    q_len, kv_len = _lengths(c)
    per = -(-c["ctx"] // ps)
    n_pages = B * per + 3
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    lens = torch.tensor(kv_len, device=dev)
    table = order[:B * per].view(B, per).contiguous()
    used = torch.arange(per, device=dev)[None, :] * ps < lens[:, None]
    # pages are not shared; entries past a sequence's end name no page
    table = torch.where(used, table, -1)
    n = D * (2 if c["kv"] == "bf16" else 1)
    cell = 32 * n + (0 if c["kv"] == "bf16" else D)
    # Rows that no sequence owns hold what is never to be read: NaN codes and scales.
    pool = torch.full((n_pages, HK, ps // 16, cell), 255, dtype=torch.uint8, device=dev)
    if c["op"] != "append":
        row_of = torch.arange(per * ps, device=dev)[None, :] < lens[:, None]
        filled = torch.zeros((n_pages, ps), dtype=torch.bool, device=dev)
        pages = table[used].long()
        filled[pages] = row_of.view(B, per, ps)[used]
        keep = filled.view(n_pages, 1, ps // 16, 16, 1)
        kc, vc, ks, vs = _fields(pool, c)
        for code, scale in ((kc, ks), (vc, vs)):
            for p0 in range(0, n_pages, 2048):
                p1 = min(n_pages, p0 + 2048)
                x = torch.randn((p1 - p0, HK, ps // 16, 16, D), generator=g, device=dev)
                a, s = _quantise(x, c["kv"])
                code[p0:p1] = torch.where(keep[p0:p1], a, code[p0:p1])
                if s is not None:
                    scale[p0:p1] = torch.where(keep[p0:p1], s, scale[p0:p1])
    rows = _ROWS[c["rows"]]
    T = sum(q_len)
    st = {"case": c, "pool": pool, "table": table, "kv_len": lens.to(torch.int32),
          "q_start": torch.tensor([0] + q_len, device=dev).cumsum(0).to(torch.int32),
          "n_tok": T, "max_q": max(q_len), "max_kv": max(kv_len)}
    if c["op"] == "attn":
        st["q"] = torch.randn((T, H, D), generator=g, device=dev).to(rows)
        st["out"] = torch.empty((T, H, D), dtype=rows, device=dev)
        return st
    st["k_out"] = torch.zeros((T, HK, D), dtype=rows, device=dev)
    st["v_out"] = torch.zeros((T, HK, D), dtype=rows, device=dev)
    if c["op"] == "append":
        st["q"] = torch.randn((T, H, D), generator=g, device=dev).to(rows)
        st["k"] = torch.randn((T, HK, D), generator=g, device=dev).to(rows)
        st["v"] = torch.randn((T, HK, D), generator=g, device=dev).to(rows)
        st["q_out"] = torch.zeros((T, H, D), dtype=rows, device=dev)
        inv = 1.0 / 500000.0 ** (torch.arange(D // 2, device=dev, dtype=torch.float64) * 2 / D)
        ang = torch.arange(c["ctx"], device=dev, dtype=torch.float64)[:, None] * inv
        st["sin"], st["cos"] = ang.sin().float(), ang.cos().float()
    return st


# ---- one pass --------------------------------------------------------------------------------------------------

def _places(st):
    """Sequence, position and (for rows of unused entries) validity of every row of a call."""
    start, lens = st["q_start"].long(), st["kv_len"].long()
    t = torch.arange(st["n_tok"], device=lens.device)
    b = torch.searchsorted(start[1:], t, right=True)
    pos = lens[b] - (start[b + 1] - t)
    return b, pos, pos >= 0


def _row_index(st, b, pos):
    """Page, cell and row in the cell of each (sequence, position)."""
    ps = st["case"]["page"]
    page = st["table"][b, pos // ps].long()
    return page, pos % ps // 16, pos % 16


def _gather(st):
    """(k, v) numbers of every row of the call, F32 [rows][HK][D], zero for unused entries."""
    c = st["case"]
    b, pos, ok = _places(st)
    page, cell, r = _row_index(st, b, pos.clamp(min=0))
    kc, vc, ks, vs = _fields(st["pool"], c)
    out = []
    for code, scale in ((kc, ks), (vc, vs)):
        x = _numbers(code[page, :, cell, r], None if scale is None else scale[page, :, cell, r], c["kv"])
        out.append(torch.where(ok[:, None, None], x, 0.0))
    return out


def _rotate(x, sin, cos):
    a, b = x.double().chunk(2, -1)
    s, c = sin.double()[:, None], cos.double()[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1).float()


def _plain_append(st):
    c = st["case"]
    rows = _ROWS[c["rows"]]
    b, pos, ok = _places(st)
    at = pos.clamp(min=0)
    sin, cos = st["sin"][at], st["cos"][at]
    q = torch.where(ok[:, None, None], _rotate(st["q"], sin, cos), 0.0).to(rows)
    page, cell, r = _row_index(st, b[ok], pos[ok])
    kc, vc, ks, vs = _fields(st["pool"], c)
    for code, scale, x in ((kc, ks, _rotate(st["k"], sin, cos)), (vc, vs, st["v"].float())):
        a, s = _quantise(x[ok], c["kv"])
        code[page, :, cell, r] = a
        if s is not None:
            scale[page, :, cell, r] = s
    k, v = _gather(st)
    return {"q": q, "k": k.to(rows), "v": v.to(rows)}


def _plain_attn(st):
    c = st["case"]
    HK, D, ps = c["HK"], c["D"], c["page"]
    G, W, S = c["H"] // HK, c["window"], c["sinks"]
    lens = st["kv_len"].long()
    B, n = lens.numel(), st["max_q"]
    b, pos, _ = _places(st)
    i = torch.arange(st["n_tok"], device=lens.device) - st["q_start"].long()[b]
    q = torch.zeros((B, n, HK, G, D), device=lens.device)
    q[b, i] = st["q"].float().view(-1, HK, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(B, HK, G * n, D)
    qpos = torch.full((B, n), -1, device=lens.device)
    qpos[b, i] = pos
    pages = st["pool"][st["table"].clamp(min=0).long()]              # [B][P][HK][cells][bytes]
    kc, vc, ks, vs = _fields(pages, c)
    j = torch.arange(kc.shape[1] * ps, device=lens.device)
    inside = j[None, :] < lens[:, None]                               # [B][keys]

    def rows(code, scale):
        x = _numbers(code, scale, c["kv"]).permute(0, 2, 1, 3, 4, 5).flatten(2, 4)
        return torch.where(inside[:, None, :, None], x, 0.0)

    s = (q @ rows(kc, ks).mT) * (1.0 / math.sqrt(D))                  # [B][HK][G * n][keys]
    seen = (j <= qpos[..., None]) & inside[:, None, :]
    if W:
        seen &= (j > qpos[..., None] - W) | (j < S)
    s = s.view(B, HK, G, n, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == float("-inf"), 0.0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ rows(vc, vs)).view(B, HK, G, n, D) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, c["H"], D).to(_ROWS[c["rows"]])


def _own_cache(st):
    """The cache over the state's pool and the batch of its sequences, made once as a server keeps them."""
    if "cache" not in st:
        from lestramanika_b200.pages import KVPages, PageBatch
        c = st["case"]
        st["cache"] = KVPages(_KV[c["kv"]], st["pool"].shape[0], c["page"], c["HK"], c["D"], pools=[st["pool"]],
                              rope=(st["sin"], st["cos"]) if "sin" in st else None)
        st["batch"] = PageBatch(st["kv_len"], st["table"], q_start=st["q_start"], n_tok=st["n_tok"],
                                max_q=st["max_q"], max_kv=st["max_kv"])
    return st["cache"], st["batch"]


def run(state):
    st, op = state, state["case"]["op"]
    if own:
        cache, batch = _own_cache(st)
        if op == "attn":
            cache.attn_dev(0, batch, st["q"], st["out"], window=st["case"]["window"], sinks=st["case"]["sinks"])
            return st["out"]
        if op == "append":
            cache.append_dev(0, batch, st["k"], st["v"], q=st["q"], q_out=st["q_out"])
        cache.read_dev(0, batch, st["k_out"], st["v_out"])
        out = {"k": st["k_out"], "v": st["v_out"]}
        return dict(out, q=st["q_out"]) if op == "append" else out
    if op == "attn":
        return _plain_attn(st)
    if op == "append":
        return _plain_append(st)
    k, v = _gather(st)
    rows = _ROWS[st["case"]["rows"]]
    return {"k": k.to(rows), "v": v.to(rows)}


# ---- the definition in 64 bits, sequence by sequence --------------------------------------------------------------

def _pow2(e):
    """2^e in F64, from the bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _block_value(x, kv):
    """What F64 blocks [..., 32] of F32 values read back as."""
    if kv == "bf16":
        return x.float().to(torch.bfloat16).double()
    amax = x.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(torch.clamp(amax, min=2.0 ** -140))[1].double() - 1       # floor(log2(amax))
    top, reach, digits = (127.5, 6, None) if kv == "i8" else (464.0, 8, 3)
    e = exponent - reach
    past = amax >= top * _pow2(e) if kv == "i8" else amax > top * _pow2(e)
    e = torch.clamp(e + past.double(), min=-111.0)
    y = x * _pow2(-e)
    if kv == "i8":
        return torch.round(y) * _pow2(e)
    mag = torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -12))), min=-6.0)
    step = _pow2(mag - digits)
    return torch.clamp(torch.round(y / step) * step, -448.0, 448.0) * _pow2(e)


def _sequence_rows(st, b, first, last):
    """K and V of positions [first, last) of sequence b, F64 [HK][rows][D]."""
    c, dev = st["case"], st["pool"].device
    D, ps = c["D"], c["page"]
    p = torch.arange(first, last, device=dev)
    cell = st["pool"][st["table"][b].long()[p // ps], :, (p % ps) // 16]       # [rows][HK][bytes]
    at = (p % 16)[:, None, None]
    wide = 2 if c["kv"] == "bf16" else 1
    found = []
    for which in (0, 1):
        i = which * 16 * D * wide + at * D * wide + torch.arange(D * wide, device=dev)
        raw = torch.gather(cell, 2, i.expand(-1, c["HK"], -1)).contiguous()
        if wide == 2:
            x = raw.view(torch.bfloat16).double()
        else:
            i = 32 * D + which * D // 2 + at * (D // 32) + torch.arange(D, device=dev) // 32
            e = torch.gather(cell, 2, i.expand(-1, c["HK"], -1)).double() - 127
            x = raw.view(torch.int8 if c["kv"] == "i8" else torch.float8_e4m3fn).double() * _pow2(e)
        found.append(x.transpose(0, 1))
    return found


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    q_len, kv_len = _lengths(c)
    H, HK, D, W, S = c["H"], c["HK"], c["D"], c["window"], c["sinks"]
    G, dev, t = H // HK, st["pool"].device, 0
    if c["op"] == "attn":
        out = torch.zeros((st["n_tok"], H, D), dtype=torch.float64, device=dev)
        for b, (n, m) in enumerate(zip(q_len, kv_len)):
            if m:
                k, v = _sequence_rows(st, b, 0, m)
                at = torch.arange(m - n, m, device=dev)[:, None]
                key = torch.arange(m, device=dev)
                hidden = key > at
                if W:
                    hidden |= (key <= at - W) & (key >= S)
                for h in range(H):
                    s = st["q"][t:t + n, h].double() @ k[h // G].T / math.sqrt(D)
                    out[t:t + n, h] = torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ v[h // G]
            t += n
        return out
    out = {x: torch.zeros((st["n_tok"], HK, D), dtype=torch.float64, device=dev) for x in "kv"}
    if c["op"] == "append":
        out["q"] = torch.zeros((st["n_tok"], H, D), dtype=torch.float64, device=dev)
    for n, m, b in zip(q_len, kv_len, range(c["B"])):
        if m and c["op"] == "read":
            k, v = _sequence_rows(st, b, m - n, m)
            out["k"][t:t + n], out["v"][t:t + n] = k.transpose(0, 1), v.transpose(0, 1)
        elif m:
            sin, cos = (st[x][m - n:m].double()[:, None] for x in ("sin", "cos"))

            def turn(x):
                lo, hi = x[..., :D // 2].double(), x[..., D // 2:].double()
                return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)

            out["q"][t:t + n] = turn(st["q"][t:t + n])
            k = turn(st["k"][t:t + n]).float().double()
            out["k"][t:t + n] = _block_value(k.unflatten(-1, (-1, 32)), c["kv"]).flatten(-2)
            out["v"][t:t + n] = _block_value(st["v"][t:t + n].double().unflatten(-1, (-1, 32)), c["kv"]).flatten(-2)
        t += n
    return out
