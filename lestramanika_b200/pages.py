"""Paged KV cache with BF16 or 8-bit rows, and the bookkeeping of its pages.

The reference keeps one F32 cache of max_seq positions per conversation
(src/pickle_fast.c:1793-1811), as PickleCuda does per slot. KVPages keeps
pages of page_size positions that any sequence can own, with rows in BF16 or
in 8-bit blocks of 32 (int8 or E4M3 codes under a power-of-two scale), and
the calls of include/pickle_cuda.h on them:

  * append_dev rotates a call's q and k, and writes k and v to their pages;
  * read_dev gives rows back as F32 or BF16 numbers;
  * attn_dev is causal attention of the call's rows over the pages, from one
    token per sequence to whole prompts, with an optional sliding window and
    first positions that stay visible.

PageBatch names the sequences of a call. PageSlots hands out the pages:

  slots = PageSlots(cache)
  slots.admit("a")
  batch = slots.batch(["a"], [len(prompt)])        # pages for the new tokens
  for layer in range(cache.n_layers):
      slots.step(layer, batch, q, k, v, out)       # append, then attend
  slots.advance(batch)

Calls run on torch's current stream unless `stream` (a torch.cuda.Stream or
a handle) says otherwise, and are asynchronous; sync() reports device-side
errors. A batch may be dropped at any time after the call, and a cache too,
unless a stream was given as a handle: then after sync(handle). What the
arrays hold is the caller's to keep until the call has run, and so are q, k, v
and the outputs.
"""
import ctypes
import itertools

import numpy as np

from .api import PICKLE_OK, PickleError, lib
from .slots import SlotError

KV_BF16, KV_I8, KV_E4M3 = 0, 1, 2
ROW_F32, ROW_BF16 = 0, 1
ERR_ARG, ERR_RANGE, ERR_DEVICE = -6, -7, -9


class PagesParams(ctypes.Structure):
    """pickle_cuda_pages_t."""
    _fields_ = [("pool", ctypes.c_void_p), ("kv_type", ctypes.c_int), ("n_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("err", ctypes.c_void_p)]


class BatchParams(ctypes.Structure):
    """pickle_cuda_batch_t."""
    _fields_ = [("n_seqs", ctypes.c_int), ("n_tok", ctypes.c_int), ("max_q", ctypes.c_int), ("max_kv", ctypes.c_int),
                ("q_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("table_stride", ctypes.c_int)]


def pages_bytes(kv_type, n_pages, page_size, n_kv_heads, head_dim):
    """pickle_cuda_pages_bytes: bytes of one layer's pool (0: sizes the pages do not take)."""
    return lib().pickle_cuda_pages_bytes(kv_type, n_pages, page_size, n_kv_heads, head_dim)


def _ints(t, what):
    import torch
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise PickleError(ERR_ARG, "PageBatch", f"{what} must be a contiguous int32 tensor")
    return t


_serials = itertools.count()


class PageBatch:
    """The sequences of one call (pickle_cuda_batch_t).

    kv_len [n], table [n][pages] and q_start [n + 1] are int32 device tensors,
    read when the kernels run (a captured graph follows them); sequence b's
    rows are [q_start[b], q_start[b + 1]) of the call's tensors and its last
    positions, kv_len[b] counting them. q_start None: one row per sequence.
    n_tok, max_q and max_kv are host bounds; left out, they are read from the
    tensors (a host sync).
    """

    def __init__(self, kv_len, table, q_start=None, n_tok=None, max_q=None, max_kv=None):
        self.kv_len, self.table = _ints(kv_len, "kv_len"), _ints(table, "table")
        self.q_start = None if q_start is None else _ints(q_start, "q_start")
        n = kv_len.numel()
        if table.dim() != 2 or table.shape[0] != n or (q_start is not None and q_start.numel() != n + 1):
            raise PickleError(ERR_ARG, "PageBatch", "table is [n][pages], q_start [n + 1]")
        tensors = [kv_len, table] + ([] if q_start is None else [q_start])
        if len({t.device for t in tensors}) != 1:
            raise PickleError(ERR_ARG, "PageBatch", "tensors on different devices")
        self.device = kv_len.device
        if q_start is None:
            n_tok, max_q = n, 1
        else:
            n_tok = int(q_start[-1].item()) if n_tok is None else n_tok
            max_q = max(1, int((q_start[1:] - q_start[:-1]).max().item())) if max_q is None else max_q
        max_kv = int(kv_len.max().item()) if max_kv is None else max_kv
        self.n_seqs, self.n_tok, self.max_q, self.max_kv = n, n_tok, max_q, max_kv
        self._c = BatchParams(n, n_tok, max_q, max_kv, None if q_start is None else q_start.data_ptr(),
                              kv_len.data_ptr(), table.data_ptr(), table.shape[1])
        self._ref = ctypes.byref(self._c)
        self._ws = {}
        self._tensors, self._streams, self._serial = tensors, set(), next(_serials)


class _Held:
    """Arrays of the batches that the stream of a handle reads: `old` ones until the event, `young` ones after it."""

    def __init__(self):
        self.young, self.old, self.event = {}, {}, None


class KVPages:
    """Pools of n_pages pages for n_layers layers, and the calls on them.

    kv_type: KV_BF16, KV_I8 or KV_E4M3. pools: uint8 device tensors of
    pages_bytes(...) bytes to use in place of new ones. rope: the (sin, cos)
    F32 device tables [rope_len][half] that append_dev rotates with; with
    rope_len > 0 they are made from rope_theta (or rope_inv_freq) as
    PickleCuda makes its own; neither: rows are taken as rotated already.
    """

    def __init__(self, kv_type, n_pages, page_size, n_kv_heads, head_dim, *, n_layers=1, pools=None, rope=None,
                 rope_len=0, rope_theta=10000.0, rope_inv_freq=None, device=0):
        import torch
        self._torch = torch
        self.kv_type, self.n_pages, self.page_size = kv_type, n_pages, page_size
        self.HK, self.D, self.n_layers, self.device = n_kv_heads, head_dim, n_layers, device
        self._sizes = (kv_type, n_pages, page_size, n_kv_heads, head_dim, device)
        nbytes = pages_bytes(*self._sizes[:5])
        if nbytes == 0 or n_layers < 1:
            raise PickleError(ERR_ARG, "KVPages", "page_size is a multiple of 16, head_dim 64 or 128")
        dev = torch.device("cuda", device)
        if pools is None:
            pools = [torch.zeros(nbytes, dtype=torch.uint8, device=dev) for _ in range(n_layers)]
        for p in pools:
            if (p.numel() * p.element_size() != nbytes or not p.is_contiguous() or p.device != dev or
                    p.data_ptr() % 16):
                raise PickleError(ERR_ARG, "KVPages", f"a pool is {nbytes} contiguous bytes on {dev}")
        if len(pools) != n_layers:
            raise PickleError(ERR_ARG, "KVPages", "one pool per layer")
        if rope is None and rope_len > 0:
            rope = self._tables(rope_len, rope_theta, rope_inv_freq, dev)
        self.rope, self.half, self.rope_len = rope, 0, 0
        if rope is not None:
            s, c = rope
            if s.shape != c.shape or s.dim() != 2 or any(
                    t.dtype != torch.float32 or not t.is_contiguous() or t.device != dev for t in rope):
                raise PickleError(ERR_ARG, "KVPages", "rope is two contiguous F32 tables [rope_len][half]")
            self.rope_len, self.half = s.shape
        self._rope_args = (None, None) if rope is None else (rope[0].data_ptr(), rope[1].data_ptr())
        self.pools = list(pools)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self._dev = dev
        # The first call may be on another stream: what this one fills has to be there.
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(dev).synchronize()
        self._c = [PagesParams(p.data_ptr(), kv_type, n_pages, page_size, n_kv_heads, head_dim, self.err.data_ptr())
                   for p in self.pools]
        self._refs = [ctypes.byref(c) for c in self._c]
        self._row_types = {torch.float32: ROW_F32, torch.bfloat16: ROW_BF16}
        self._lib = lib()
        self._layouts = {}
        self._held, self._streams = {}, set()
        self._own = self.pools + [self.err] + list(rope or ())

    def _tables(self, rope_len, theta, inv_freq, dev):
        # src/pickle_fast.c:1638-1640, 1772-1788: half = min(D/2, 64), inv_freq and angles in F32.
        half = min(self.D // 2, 64)
        i = np.arange(half, dtype=np.float32)
        inv = (np.float32(1.0) / np.power(np.float64(np.float32(theta)), np.float64(2 * i / np.float32(self.D)))
               .astype(np.float32)) if inv_freq is None else np.asarray(inv_freq, np.float32)[:half]
        ang = np.outer(np.arange(rope_len, dtype=np.float32), inv.astype(np.float32)).astype(np.float64)
        return tuple(self._torch.from_numpy(f(ang).astype(np.float32)).to(dev) for f in (np.sin, np.cos))

    # -- argument checks -------------------------------------------------
    def _rows(self, t, heads, n_tok, what):
        """(address, element type, elements between tokens) of rows [n_tok][heads][D]."""
        shape = t.shape
        key = (t.dtype, shape, t.stride(), heads)
        known = self._layouts.get(key)
        if known is None:
            known = self._layout(t, heads, what)
            if len(self._layouts) >= 1024:
                self._layouts.clear()
            self._layouts[key] = known
        if shape[0] < n_tok or t.get_device() != self.device:
            raise PickleError(ERR_ARG, "KVPages", f"{what}: fewer rows than the batch's {n_tok}, or not on {self._dev}")
        return t.data_ptr(), known[0], known[1]

    def _layout(self, t, heads, what):
        """(element type, elements between tokens) of a tensor's shape and strides, or an error."""
        rt = self._row_types.get(t.dtype)
        shape, st = t.shape, t.stride()
        if rt is None or len(shape) != 3 or shape[2] != self.D or (heads and shape[1] != heads) or (
                st[2] != 1 or (st[1] != self.D and shape[1] > 1)):
            raise PickleError(ERR_ARG, "KVPages", f"{what}: F32 or BF16 rows [n_tok][heads][{self.D}], heads and "
                              "elements dense")
        if shape[0] <= 1:
            return rt, 0
        if st[0] < shape[1] * self.D:
            raise PickleError(ERR_ARG, "KVPages", f"{what}: rows overlap")
        return rt, st[0]

    def _call(self, batch, layer, stream):
        if not 0 <= layer < self.n_layers or batch.device != self._dev:
            raise PickleError(ERR_ARG, "KVPages", "layer out of range, or a batch on another device")
        if stream is None:
            st = self._torch._C._cuda_getCurrentRawStream(self.device)
        else:
            st = stream if isinstance(stream, int) else stream.cuda_stream
        # A batch is often dropped while its kernels still wait for their turn: its memory is not handed out before the
        # streams that read it are through. The allocator asks a stream that is marked when the memory is dropped, and
        # the stream of a handle may be gone by then: what those read is held here.
        if isinstance(stream, int) and stream:
            self._hold(batch, stream)
            return st
        for tensors, known in ((batch._tensors, batch._streams), (self._own, self._streams)):
            if st not in known:
                s = self._stream(stream)
                for t in tensors:
                    t.record_stream(s)
                known.add(st)
        return st

    def _hold(self, batch, handle):
        held = self._held.get(handle)
        if held is None:
            held = self._held[handle] = _Held()
        if len(held.young) >= 64 and batch._serial not in held.young:
            cuda, s = self._torch.cuda, self._stream(handle)
            captured = cuda.is_current_stream_capturing()
            with cuda.stream(s):
                captured = captured or cuda.is_current_stream_capturing()
            if not captured and (held.event is None or held.event.query()):
                held.old, held.young, held.event = held.young, {}, s.record_event()
        held.young[batch._serial] = batch._tensors

    def _run(self, fn, what, *args):
        if self._torch._C._cuda_getDevice() == self.device:
            rc = fn(*args)
        else:
            with self._torch.cuda.device(self.device):
                rc = fn(*args)
        if rc != PICKLE_OK:
            raise PickleError(rc, what)

    # -- calls -----------------------------------------------------------
    def append_dev(self, layer, batch, k, v, q=None, q_out=None, stream=None):
        """pickle_cuda_pages_append_dev: k, v [n_tok][HK][D] rotated (k) and written to their pages; q
        [n_tok][H][D] (k's type) rotated into q_out (F32 or BF16; q itself where the types agree)."""
        st = self._call(batch, layer, stream)
        kp, rt, ks = self._rows(k, self.HK, batch.n_tok, "k")
        vp, vt, vs = self._rows(v, self.HK, batch.n_tok, "v")
        qp = qs = op = ot = os_ = H = 0
        if q is not None or q_out is not None:
            if q is None or q_out is None:
                raise PickleError(ERR_ARG, "KVPages", "q and q_out go together")
            H = q.shape[1]
            qp, qt, qs = self._rows(q, H, batch.n_tok, "q")
            op, ot, os_ = self._rows(q_out, H, batch.n_tok, "q_out")
            if qt != rt:
                raise PickleError(ERR_ARG, "KVPages", "q, k and v have one element type")
        if vt != rt:
            raise PickleError(ERR_ARG, "KVPages", "q, k and v have one element type")
        if batch.n_tok == 0:                 # tensors without rows have no address
            return
        self._run(self._lib.pickle_cuda_pages_append_dev, "pickle_cuda_pages_append_dev", self._refs[layer],
                  batch._ref, H, rt, qp or None, qs, kp, ks, vp, vs, *self._rope_args, self.half, self.rope_len, ot,
                  op or None, os_, st)

    def read_dev(self, layer, batch, k_out, v_out, stream=None):
        """pickle_cuda_pages_read_dev: the call's rows of the cache into k_out, v_out [n_tok][HK][D]."""
        st = self._call(batch, layer, stream)
        kp, rt, ks = self._rows(k_out, self.HK, batch.n_tok, "k_out")
        vp, vt, vs = self._rows(v_out, self.HK, batch.n_tok, "v_out")
        if rt != vt:
            raise PickleError(ERR_ARG, "KVPages", "k_out and v_out have one element type")
        if batch.n_tok == 0:
            return
        self._run(self._lib.pickle_cuda_pages_read_dev, "pickle_cuda_pages_read_dev", self._refs[layer], batch._ref,
                  rt, kp, ks, vp, vs, st)

    def attn_dev(self, layer, batch, q, out, window=0, sinks=0, stream=None, workspace=None):
        """pickle_cuda_pages_attn_dev: attention of the rotated rows q [n_tok][H][D] over the pages into out (q's
        type). window > 0: the last `window` positions of each row and the sequence's first `sinks` only.
        workspace: a device tensor for the split partials; by default one is taken from torch's allocator for the
        call, so calls on several streams and captured graphs do not share one."""
        st = self._call(batch, layer, stream)
        H = q.shape[1] if q.dim() == 3 else 0
        qp, rt, qs = self._rows(q, H, batch.n_tok, "q")
        op, ot, os_ = self._rows(out, H, batch.n_tok, "out")
        if rt != ot:
            raise PickleError(ERR_ARG, "KVPages", "q and out have one element type")
        if window < 0 or sinks < 0:
            raise PickleError(ERR_ARG, "KVPages", "window and sinks are not negative")
        if batch.n_tok == 0:
            return
        key = (self._sizes, H, rt, window, sinks)           # not the cache, which a kept batch would keep
        need = batch._ws.get(key)
        if need is None:
            need = batch._ws[key] = self.attn_workspace(batch, H, rt, window, sinks)
        wp = 0
        if workspace is not None:
            if not workspace.is_contiguous() or workspace.get_device() != self.device:
                raise PickleError(ERR_ARG, "KVPages", f"workspace is contiguous and on {self._dev}")
            wp, need = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        elif need:
            workspace = self._scratch(need, stream)
            wp = workspace.data_ptr()
        self._run(self._lib.pickle_cuda_pages_attn_dev, "pickle_cuda_pages_attn_dev", self._refs[layer], batch._ref,
                  H, rt, qp, qs, op, os_, window, sinks, wp or None, need, st)

    def attn_workspace(self, batch, n_heads, row_type, window=0, sinks=0):
        """pickle_cuda_pages_workspace: device bytes attn_dev's split partials take for such a call."""
        if self._torch._C._cuda_getDevice() == self.device:
            return self._lib.pickle_cuda_pages_workspace(self._refs[0], batch._ref, n_heads, row_type, window, sinks)
        with self._torch.cuda.device(self.device):
            return self._lib.pickle_cuda_pages_workspace(self._refs[0], batch._ref, n_heads, row_type, window, sinks)

    def _stream(self, stream):
        """The torch stream that a call's `stream` stands for. (ExternalStream makes a new stream of handle 0.)"""
        cuda = self._torch.cuda
        if stream is None:
            return cuda.current_stream(self._dev)
        if not isinstance(stream, int):
            return stream
        return cuda.ExternalStream(stream, device=self._dev) if stream else cuda.default_stream(self._dev)

    def _scratch(self, nbytes, stream):
        """Bytes from torch's allocator, tied to the stream that uses them."""
        torch = self._torch
        if stream is None:
            return torch.empty(nbytes, dtype=torch.uint8, device=self._dev)
        with torch.cuda.stream(self._stream(stream)):
            return torch.empty(nbytes, dtype=torch.uint8, device=self._dev)

    def sync(self, stream=None):
        """Wait for the stream's work and raise PICKLE_ERR_DEVICE for a device-side error recorded since the last."""
        torch = self._torch
        self._stream(stream).synchronize()
        if isinstance(stream, int):
            self._held.pop(stream, None)
        code = int(self.err.item())
        if code:
            self.err.zero_()
            torch.cuda.current_stream(self._dev).synchronize()
            raise PickleError(ERR_DEVICE, "KVPages.sync", f"device error {code}")


class PageSlots:
    """Which pages each request owns: admission, growth, release, and the batches of a call.

    No counterpart in the reference (one cache per conversation); KVSlots is
    the same bookkeeping over fixed slots. Every page has one owner.
    """

    def __init__(self, cache):
        self.cache = cache
        self.free = list(range(cache.n_pages - 1, -1, -1))
        self.pages = {}
        self.pos = {}

    def admit(self, req):
        if req in self.pages:
            raise SlotError(f"request {req!r} is already admitted")
        self.pages[req] = []
        self.pos[req] = 0

    def release(self, req):
        self.free.extend(p for p in reversed(self.pages.pop(req)) if p >= 0)
        del self.pos[req]

    def position(self, req):
        return self.pos[req]

    def reserve(self, reqs, counts):
        """Pages for counts[i] more positions of reqs[i]; all of them or, with SlotError, none."""
        if len(set(reqs)) != len(reqs) or len(reqs) != len(counts):
            raise SlotError("requests of a call are distinct, with a count each")
        ps = self.cache.page_size
        need = [-(-(self.pos[r] + n) // ps) - len(self.pages[r]) for r, n in zip(reqs, counts)]
        if sum(max(0, x) for x in need) > len(self.free):
            raise SlotError("no free KV pages")
        for r, x in zip(reqs, need):
            for _ in range(max(0, x)):
                self.pages[r].append(self.free.pop())

    def trim(self, req, window, sinks=0):
        """Release the pages of `req` that no later row with this window and these sinks can see."""
        if window <= 0:
            return
        ps, owned = self.cache.page_size, self.pages[req]
        first = self.pos[req] - window + 1              # the next row's oldest position in the window
        for i in range(-(-sinks // ps), min(len(owned), max(0, first) // ps)):
            if owned[i] >= 0:
                self.free.append(owned[i])
                owned[i] = -1

    def batch(self, reqs, counts=None):
        """A PageBatch of counts[i] new tokens (1 each by default) for reqs[i], on reserved pages."""
        import torch
        counts = [1] * len(reqs) if counts is None else list(counts)
        if not reqs or min(counts) < 0:
            raise SlotError("a batch has requests, and no negative counts")
        self.reserve(reqs, counts)
        width = max(1, max(len(self.pages[r]) for r in reqs))
        table = torch.tensor([self.pages[r] + [-1] * (width - len(self.pages[r])) for r in reqs], dtype=torch.int32)
        kv = [self.pos[r] + n for r, n in zip(reqs, counts)]
        start = None
        if any(n != 1 for n in counts):
            start = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).to(self.cache._dev)
        b = PageBatch(torch.tensor(kv, dtype=torch.int32).to(self.cache._dev), table.to(self.cache._dev),
                      q_start=start, n_tok=sum(counts), max_q=max(1, max(counts)), max_kv=max(kv))
        b.reqs, b.counts = list(reqs), counts
        return b

    def step(self, layer, batch, q, k, v, out, window=0, sinks=0, q_rot=None, stream=None):
        """One layer of a call: rotate q (into q_rot, or in place) and k, append, attend into out."""
        q_rot = q if q_rot is None else q_rot
        self.cache.append_dev(layer, batch, k, v, q=q, q_out=q_rot, stream=stream)
        self.cache.attn_dev(layer, batch, q_rot, out, window=window, sinks=sinks, stream=stream)

    def advance(self, batch):
        """The batch's tokens are in the cache of every layer."""
        for r, n in zip(batch.reqs, batch.counts):
            self.pos[r] += n
