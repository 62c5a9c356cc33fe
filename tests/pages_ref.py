"""The paged KV cache restated in 64 bits, one sequence and one block at a time, and random batches for it."""
import math

import numpy as np
import torch

KV = {"bf16": 0, "i8": 1, "e4m3": 2}
ROWS = {"f32": torch.float32, "bf16": torch.bfloat16}


def cell_bytes(kv, D):
    return 64 * D if kv == "bf16" else 33 * D


def pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x, kv):
    """F32 rows [..., D] -> (values F64 [..., D], codes F64 [..., D], scale bytes [..., D/32]); BF16: values only.

    The scale: the smallest power of two >= 2^-111 for which the largest element's code, rounded to nearest even,
    is at most 127 (i8), or is at most 448 (E4M3, whose next number would be 480: halfway is 464, which goes to 448)."""
    if kv == "bf16":
        return x.float().to(torch.bfloat16).double(), None, None
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    ok = torch.isfinite(b).all(-1)
    amax = torch.where(ok, amax, 1.0)
    e = torch.full(amax.shape, -111, dtype=torch.long, device=x.device)
    fits = (lambda y: y < 127.5) if kv == "i8" else (lambda y: y <= 464.0)
    for _ in range(260):
        e = torch.where(fits(amax * pow2(-e)), e, e + 1)
    y = torch.where(ok[..., None], b, 0.0) * pow2(-e)[..., None]
    if kv == "i8":
        codes = torch.round(y)
    else:
        mag = y.abs()
        step = torch.full_like(y, 2.0 ** -9)
        for k in range(-5, 9):
            step = torch.where(mag >= 2.0 ** k, 2.0 ** (k - 3), step)
        codes = torch.round(y / step) * step
        codes = torch.where(codes.abs() > 448, torch.sign(codes) * 448.0, codes)
    v = torch.where(ok[..., None], codes * pow2(e)[..., None], float("nan"))
    return v.flatten(-2), codes.flatten(-2), torch.where(ok, e + 127, 255)


def rotate(x, sin, cos, half):
    """F64 NeoX rotation of [T][heads][D] rows by table rows sin, cos [T][half]."""
    x, s, c = x.double(), sin.double()[:, None], cos.double()[:, None]
    lo, hi, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([c * lo - s * hi, s * lo + c * hi, rest], -1)


def visible(pos, n_keys, window, sinks, device):
    """[len(pos)][n_keys] truth values: key j is seen from position pos."""
    p = torch.as_tensor(pos, device=device)[:, None]
    j = torch.arange(n_keys, device=device)
    see = j <= p
    if window:
        see &= (j > p - window) | (j < sinks)
    return see


def attend(q, k, v, pos, window, sinks):
    """F64 attention of q [n][H][D] at positions pos over k, v [HK][m][D]; also sum_j p_j |v_j| [n][H][D] and
    max_j sum_d |q_d k_jd| / sqrt(D) [n][H][1], which scale the error bounds."""
    n, H, D = q.shape
    G = H // k.shape[0]
    see = visible(pos, k.shape[1], window, sinks, q.device)
    out, mass, size = [], [], []
    for h in range(H):
        kk, vv, qq = k[h // G], v[h // G], q[:, h].double()
        s = (qq @ kk.T) / math.sqrt(D)
        s = s.masked_fill(~see, -math.inf)
        p = torch.softmax(s, -1) if k.shape[1] else s
        p = torch.where(see.any(-1, keepdim=True), p, 0.0) if k.shape[1] else s
        vz = torch.where(see.any(0)[:, None], vv, 0.0)
        kz = torch.where(see.any(0)[:, None], kk, 0.0)
        out.append(p @ vz)
        mass.append(p @ vz.abs())
        size.append((torch.where(see, qq.abs() @ kz.abs().T, 0.0).amax(-1, keepdim=True) if k.shape[1]
                     else torch.zeros(n, 1, device=q.device, dtype=torch.float64)) / math.sqrt(D))
    return (torch.stack(out, 1), torch.stack(mass, 1), torch.stack(size, 1))


def attn_bound(mass, size, out, rows, n_keys, rounded_p):
    """How far a kernel's output may be from F64, element by element.

    A score is a sum of D exact products in F32: at most 32 roundings on any path (16 in a tensor-core step's tree, D / 16
    steps, the parts of a split q), each 2^-24 of a partial sum that is at most size. A weight exp2(x) is off by 2 ln 2
    times nothing more than the score's error plus the argument's own rounding (2^-24 of |x| <= 2 size * 1.45) and
    2^-22 of the exponential; numerator and denominator both carry it, hence the factor 2. The sums over the keys add at
    most (n_keys / 16 + 16) 2^-24, and the final division 2^-23. Weights rounded to BF16: half a step, 2^-8.
    BF16 output: half a step, 2^-8 of the value."""
    u = 2.0 ** -24
    rel = 2 * (32 * u * size + 3 * u * size + 4 * u) + (n_keys / 16 + 20) * u
    if rounded_p:
        rel = rel + 2.0 ** -8
    tol = rel * mass + 1e-30
    if rows == "bf16":
        tol = tol + 2.0 ** -8 * (out.abs() + tol)
    return tol


def held_weights(k, v, pos, window, sinks):
    """What the 8-bit pages' weights held as F16 add to the bound, [n][1][D] over a KV head's rows of k, v [m][D]: a
    weight is held as 2^7 or more times itself over the row's largest, so the rounding to F16's smallest step, 2^-24,
    moves it by at most 2^-25 / 2^7, whatever is far below the row's largest weight included."""
    see = visible(pos, k.shape[0], window, sinks, v.device).double()
    return (2.0 ** -32 * (see @ v.abs()))[:, None]


def shared_exponents(q, k, v, mass):
    """What blocks far below the largest ones add to the bound on 8-bit pages, [n][H][D] for q [n][H][D] over k, v
    [HK][m][D], all of whose rows some row of the call sees.

    A code is held as an F16 number under the exponent E of the largest scales: off by 2^-25 where the product is rounded to F16's
    smallest step, by 448 2^-25 (E4M3) or 127 2^-25 (int8) where 2^(e - E) itself rounds to 0, in units in which the
    largest magnitude is 232 or 63.75 at least (a scale is the smallest that holds it): 2^-24 of that magnitude. Of v it is the
    largest of the same 32 elements of all rows; of k, of all rows, and a score is then off by the sum of |q_d|
    times it over sqrt(D), which numerator and denominator both carry."""
    n, H, D = q.shape
    G = H // k.shape[0]
    top_v = v.abs().unflatten(-1, (-1, 32)).amax((1, 3)).repeat_interleave(32, -1).repeat_interleave(G, 0)      # [H][D]
    top_k = k.abs().amax((1, 2)).repeat_interleave(G, 0)                                                        # [H]
    off = 2.0 ** -24 * q.double().abs().sum(-1) * top_k / math.sqrt(D)
    return 2.0 ** -24 * top_v + 2 * off[..., None] * mass


class Batch:
    """A random pool and ragged batch. Rows that no sequence owns are 255 bytes: NaN codes and NaN scales.

    amp: what the N(0, 1) rows are multiplied by, a number or a function of (sequence, which, length) that gives a
    tensor for [HK][length][D], which being 0 for K and 1 for V."""

    def __init__(self, kv, HK, D, page, kv_len, q_len, seed, device="cuda:0", spare=3, fill=True, amp=1.0):
        self.kv, self.HK, self.D, self.page = kv, HK, D, page
        self.kv_len, self.q_len, self.dev = list(kv_len), list(q_len), torch.device(device)
        g = self.g = torch.Generator(device="cpu").manual_seed(seed)
        n = len(kv_len)
        per = max(1, max(-(-m // page) for m in kv_len))
        self.n_pages = sum(-(-m // page) for m in kv_len) + spare
        order = torch.randperm(self.n_pages, generator=g).tolist()
        table = [[-1] * per for _ in range(n)]
        for b, m in enumerate(kv_len):
            for i in range(-(-m // page)):
                table[b][i] = order.pop()
        self.table_host = table
        cells = page // 16
        pool = np.full((self.n_pages, HK, cells, cell_bytes(kv, D)), 255, np.uint8)
        self.k, self.v = [], []                      # F64 [HK][m][D] per sequence: what the cache stands for
        for b, m in enumerate(kv_len):
            pair = []
            for which in (0, 1):
                x = torch.randn((HK, m, D), generator=g) * (amp(b, which, m) if callable(amp) else amp)
                val, codes, scale = quantise(x, kv)
                pair.append(val.to(self.dev))
                if fill and m:
                    if kv == "bf16":
                        raw = val.to(torch.bfloat16).view(torch.uint8).numpy()
                    elif kv == "i8":
                        raw = codes.to(torch.int8).view(torch.uint8).numpy()
                    else:
                        raw = codes.float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
                    w = raw.shape[-1]
                    for j in range(m):
                        c = pool[table[b][j // page], :, j % page // 16]
                        r = j % 16
                        c[:, (which * 16 + r) * w:(which * 16 + r + 1) * w] = raw[:, j]
                        if scale is not None:
                            o = 32 * D + (which * 16 + r) * (D // 32)
                            c[:, o:o + D // 32] = scale[:, j].numpy().astype(np.uint8)
            self.k.append(pair[0])
            self.v.append(pair[1])
        self.pool = torch.from_numpy(pool).to(self.dev)
        self.start = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
        self.n_tok = int(self.start[-1])

    def tensors(self):
        i32 = dict(dtype=torch.int32, device=self.dev)
        return (torch.tensor(self.kv_len, **i32), torch.tensor(self.table_host, **i32),
                torch.tensor(self.start, **i32))

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dev)

    def positions(self, b):
        return list(range(self.kv_len[b] - self.q_len[b], self.kv_len[b]))

    def stored(self, kv_row, b, j, which):
        """Bytes (codes, scales) of row j of sequence b in the pool: [HK][...]."""
        w = self.D * (2 if self.kv == "bf16" else 1)
        c = self.pool[self.table_host[b][j // self.page], :, j % self.page // 16]
        r = which * 16 + j % 16
        s = None if self.kv == "bf16" else c[:, 32 * self.D + r * (self.D // 32):32 * self.D + (r + 1) * (self.D // 32)]
        return c[:, r * w:(r + 1) * w], s
