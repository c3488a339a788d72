"""g9kv -- the paged key-value cache of libgen9blas.so (include/gen9blas_kv.h) over torch tensors.

    kv = g9kv.PagedKV(K, V, table, bounds=bounds)           # pool tensors and the page table of a batch of streams
    kv.append(k, v, length)                                 # the new tokens' keys and values enter the pages
    out = kv.attend(q, length + k.shape[1])                 # attention of the new tokens over the pages
    sel = kv.select(q, visible, 64)                         # or: the 64 pages of each head that may matter most,
    out = kv.attend(q, visible, sel=sel)                    #     and attention over those alone
    out = kv.attend(q, visible, acc=acc)                    # also adds up the attention each slot receives
    length = kv.evict(length, 4096, acc, pos, recent=64)    # keeps the 4096 slots of each head that received most

K and V: float16 [pages, kv heads, page size, head size], unit stride in the last dimension, any others a multiple of 8
elements (so both [page][head][slot] and [page][slot][head] pools serve, the latter as a permuted view). table: int32
[streams, pages per stream], -1 where a stream has no page. q, k, v: float32 [streams, tokens, heads, head size], unit
stride in the last dimension. Everything lies on one GPU; calls run on torch's current stream and do not wait. They are for
serving: results carry no gradient, and a tensor that requires one is refused unless gradients are off (torch.no_grad()). Shape and
type errors raise ValueError, library errors RuntimeError with gen9blas_error().

One cache object is used by one thread at a time, as the library is. A captured call (torch.cuda.graph) needs a workspace
of its own: pass `workspace=g9kv.Workspace()` to the constructor and make one call of each shape before the capture. The
tensors and the workspace of a captured call have to live as long as its graph is replayed.
"""
import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.realpath(__file__))
_I, _P, _L, _F = ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_float


class _Cache(ctypes.Structure):   # gen9blas_kv_cache
    _fields_ = [("D", _I), ("HKV", _I), ("page", _I), ("n_pages", _I),
                ("K", _P), ("kp", _L), ("kk", _L), ("kh", _L), ("k_bytes", ctypes.c_size_t),
                ("V", _P), ("vp", _L), ("vk", _L), ("vh", _L), ("v_bytes", ctypes.c_size_t),
                ("bounds", _P), ("table", _P), ("ts", _L), ("mp", _I), ("ns", _I), ("stream", _P)]


_C = ctypes.POINTER(_Cache)
_SIGNATURES = {
    "init": ([], _I), "error": ([], ctypes.c_char_p), "set_device": ([_I], _I),
    "kv_supported": ([_I, _I, _I], _I), "kv_ws_create": ([], _P), "kv_ws_free": ([_P], None),
    "kv_append": ([_C, _I, _P, _L, _L, _L, _P, _L, _L, _L, _P, _P, _P, _P, _L, _L, _P, _I, _P], _I),
    "attn_paged": ([_C, _I, _I, _P, _L, _L, _L, _P, _I, _I, _P, _I, _F, _P, _P, _P, _L, _L, _P, _I], _I),
    "kv_select": ([_C, _I, _I, _P, _L, _L, _L, _P, _I, _I, _I, _I, _P, _P, _I], _I),
    "kv_evict": ([_C, _P, _I, _I, _I, _P, _P, _L, _L, _P, _P, _I], _I),
}
_lib = ctypes.CDLL(os.environ.get("GEN9BLAS_LIB") or os.path.join(_HERE, "libgen9blas.so"))
_fn = {}
for _name, (_args, _res) in _SIGNATURES.items():
    _f = getattr(_lib, "gen9blas_" + _name)
    _f.argtypes, _f.restype = _args, _res
    _fn[_name] = _f
_append, _attend, _select, _evict = (_fn[n] for n in ("kv_append", "attn_paged", "kv_select", "kv_evict"))
_LEGACY = 1   # cudaStreamLegacy: torch's default stream (a null stream would mean the library's own)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # torch's accessor without the Stream object, 1.2 us less
if _raw_stream is None:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream
_capturing = torch.cuda.is_current_stream_capturing
_grad_enabled = torch.is_grad_enabled
_f32, _i32 = torch.float32, torch.int32
_END = 2 ** 31   # of the library's counts; ctypes would cut larger ones short without a word


def _check(status, what):
    if status == 1:
        raise ValueError(f"{what}: shape outside gen9blas_kv_supported (head size a multiple of 8 up to 256)")
    if status:
        raise RuntimeError(_fn["error"]().decode(errors="replace"))


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def set_device(index):
    """The device of later calls of the library (gen9blas_set_device): that of the caches. Default: the one that was current
    when the library was first used."""
    _check(_fn["set_device"](index), "set_device")


_dead = []   # workspaces whose last reference went during a capture


class Workspace:
    """Device memory for attend, select and evict of calls that run one after the other (see gen9blas_kv_ws_create). One that
    a captured call has used keeps its memory until `free`, whether or not anything still refers to it: its graph may. `free`
    waits for the device, so not during a capture; a workspace that is collected during one is freed behind it."""

    def __init__(self):
        self.captured = False
        if _dead and not _capturing():
            while _dead:
                _fn["kv_ws_free"](_dead.pop())
        self.handle = _fn["kv_ws_create"]()
        if not self.handle:
            raise RuntimeError(_fn["error"]().decode(errors="replace"))

    def free(self):
        if self.handle:
            _fn["kv_ws_free"](self.handle)
            self.handle = None

    def __del__(self):
        if getattr(self, "handle", None) and _fn and not self.captured:
            if _capturing():
                _dead.append(self.handle)
            else:
                self.free()


class PagedKV:
    """A batch's view of one layer's cache: the pool, the page table and, on request, the bounds of the pages."""

    def __init__(self, K, V, table, bounds=None, workspace=None):
        for name, x in (("K", K), ("V", V)):
            _need(x.dtype == torch.float16 and x.dim() == 4 and x.is_cuda,
                  f"{name}: float16 [pages, kv heads, page size, head size] on a GPU")
            _need(x.stride(3) == 1 or x.shape[3] == 1, f"{name}: the last dimension has stride {x.stride(3)}")
        _need(K.shape == V.shape and K.device == V.device, "K and V differ in shape or device")
        _need(table.dtype == torch.int32 and table.dim() == 2 and table.device == K.device, "table: int32 [streams, pages]")
        _need(table.stride(1) == 1 or table.shape[1] <= 1, "table: the last dimension is not contiguous")
        pages, heads, page, dim = K.shape
        if bounds is not None:
            _need(bounds.dtype == torch.float16 and tuple(bounds.shape) == (pages, heads, 2, dim) and
                  bounds.is_contiguous() and bounds.device == K.device,
                  "bounds: contiguous float16 [pages, kv heads, 2, head size] beside K")
        self.K, self.V, self.table, self.bounds, self.workspace = K, V, table, bounds, workspace
        self.device, self.streams, self.slots = K.device, table.shape[0], table.shape[1] * page
        self.heads, self.page, self.dim = heads, page, dim
        self._index = K.device.index
        self._leaf = K.requires_grad or V.requires_grad
        self._per_stream = torch.Size([self.streams])
        self._logs = torch.empty(0, device=K.device)

        def span(x):
            return 2 * (sum((n - 1) * s for n, s in zip(x.shape, x.stride())) + 1) if x.numel() else 0
        ks, vs = K.stride(), V.stride()
        self._c = _Cache(dim, heads, page, pages, K.data_ptr(), ks[0], ks[2], ks[1], span(K), V.data_ptr(), vs[0], vs[2],
                         vs[1], span(V), bounds.data_ptr() if bounds is not None else None, table.data_ptr(),
                         table.stride(0), table.shape[1], table.shape[0])
        self._ref = ctypes.byref(self._c)
        if _fn["init"]():
            raise RuntimeError(_fn["error"]().decode(errors="replace"))

    def _run(self, what, fn, *args):
        """One library call on torch's current stream of this cache's device."""
        if self._leaf and _grad_enabled():
            raise ValueError("K or V requires a gradient, which the paged cache does not give: call it under torch.no_grad()")
        self._c.stream = _raw_stream(self._index) or _LEGACY
        status = fn(self._ref, *args)
        if status:
            _check(status, what)

    def _space(self):
        """The workspace's handle as it is now: a freed one must not reach the library."""
        w = self.workspace
        if w is None:
            return None
        if not w.handle:
            raise ValueError("the cache's workspace has been freed")
        if not w.captured and _capturing():
            w.captured = True
        return w.handle

    # The checks run in every call, so their messages are put together only when one fails.
    def _rows(self, name, x, heads):
        n, st = x.shape, x.stride()
        if not (x.dtype is _f32 and len(n) == 4 and x.get_device() == self._index and n[0] == self.streams and n[3] == self.dim
                and (heads is None or n[2] == heads) and st[3] == 1):
            raise ValueError(f"{name}: float32 [{self.streams}, tokens, {heads or 'heads'}, {self.dim}] on {self.device}, unit "
                             f"stride last; got {x.dtype} {list(n)} on {x.device}")
        if x.requires_grad and _grad_enabled():
            raise ValueError(f"{name} requires a gradient, which the paged cache does not give: call it under torch.no_grad()")
        return n, st

    def _ints(self, name, x):
        if not (x.dtype is _i32 and x.shape == self._per_stream and x.get_device() == self._index and x.is_contiguous()):
            raise ValueError(f"{name}: contiguous int32 [{self.streams}] on {self.device}; got {x.dtype} {list(x.shape)} on "
                             f"{x.device}")
        return x.data_ptr()

    def _mark(self, name, x, dtype):
        n, st = x.shape, x.stride()
        if not (x.dtype is dtype and len(n) == 3 and n[0] == self.streams and n[1] == self.heads and n[2] >= self.slots and
                x.get_device() == self._index and (st[2] == 1 or n[2] <= 1)):
            raise ValueError(f"{name}: {dtype} [{self.streams}, {self.heads}, at least {self.slots}] on {self.device}, unit "
                             f"stride last; got {x.dtype} {list(n)} on {x.device}")
        return st

    def _marks(self, acc, pos):
        """Pointers of acc and pos, and the strides (stream, head) that they share."""
        st = (0, 0)
        if acc is not None:
            st = self._mark("acc", acc, _f32)
        if pos is not None:
            other = self._mark("pos", pos, _i32)
            if acc is not None and other != st:
                raise ValueError("acc and pos differ in their strides")
            st = other
        return None if acc is None else acc.data_ptr(), None if pos is None else pos.data_ptr(), st[0], st[1]

    def _like(self, q, n):
        """A contiguous float32 tensor of q's shape."""
        return torch.empty_like(q) if q.is_contiguous() else q.new_empty(n)

    def _given(self, x, shape, dtype):
        if not (x.dtype is dtype and tuple(x.shape) == shape and x.is_contiguous() and x.get_device() == self._index):
            raise ValueError(f"out: contiguous {dtype} {list(shape)} on {self.device}; got {x.dtype} {list(x.shape)} on {x.device}")

    def append(self, k, v, length, count=None, acc=None, pos=None, pos0=None, wait=False):
        """Writes the tokens k, v [streams, tokens, kv heads, dim] behind each stream's `length` slots, of stream s the
        first count[s] (all without count); bounds follow. acc and pos [streams, kv heads, slots]: set to 0 and
        pos0[s] + t (the slot's number without pos0). With wait, returns whether every token found a page."""
        n, ks = self._rows("k", k, self.heads)
        m, vs = self._rows("v", v, self.heads)
        if n != m:
            raise ValueError(f"k {list(n)} and v {list(m)} differ in shape")
        a, p, ms, mh = self._marks(acc, pos) if acc is not None or pos is not None else (None, None, 0, 0)
        bad = _I(0) if wait else None
        self._run("append", _append, n[1], k.data_ptr(), ks[1], ks[2], ks[0], v.data_ptr(), vs[1], vs[2], vs[0],
                  self._ints("length", length), None if count is None else self._ints("count", count), a, p, ms, mh,
                  None if pos0 is None else self._ints("pos0", pos0), 1 if wait else 0, ctypes.addressof(bad) if wait else None)
        return not bad.value if wait else None

    def attend(self, q, visible, step=1, scale=None, window=0, sel=None, acc=None, out=None, lse=False):
        """Attention of the tokens q [streams, tokens, heads, dim]: token t of stream s sees visible[s] + step·t slots
        (the last `window` of them, if given; those of the pages sel[s, t, g], if given). acc gains the weights each slot
        received. Returns out (float32, as q), and with lse=True also the logarithms of the softmax sums
        [streams, tokens, heads]."""
        n, qs = self._rows("q", q, None)
        ns, nq, h, d = n
        see = self._ints("visible", visible)
        a, _, ms, mh = self._marks(acc, None) if acc is not None else (None, None, 0, 0)
        if not (-_END <= step < _END and -_END <= window < _END):
            raise ValueError(f"step = {step}, window = {window}")
        nsel = 0
        sp = None
        if sel is not None:
            if not (sel.dtype is _i32 and sel.dim() == 4 and sel.shape[:3] == (ns, nq, self.heads) and sel.is_contiguous() and
                    sel.get_device() == self._index):
                raise ValueError(f"sel: contiguous int32 [{ns}, {nq}, {self.heads}, pages] on {self.device}; got {sel.dtype} "
                                 f"{list(sel.shape)} on {sel.device}")
            nsel, sp = sel.shape[3], sel.data_ptr() or see   # no pages at all: the list is there, and nothing is read
        if out is None:
            out = self._like(q, n)
        else:
            self._given(out, tuple(n), _f32)
        logs = None
        if lse:
            shape = n[:3]
            if self._logs.shape != shape:
                self._logs = q.new_empty(shape)        # only its shape is used: empty_like costs 0.5 us less than new_empty
            logs = torch.empty_like(self._logs)
        self._run("attend", _attend, h, nq, q.data_ptr(), qs[1], qs[2], qs[0], see, step, window, sp, nsel,
                  d ** -0.5 if scale is None else scale, out.data_ptr(), logs.data_ptr() if lse else None, a, ms, mh, self._space(), 0)
        return (out, logs) if lse else out

    def select(self, q, visible, pages, step=1, first=1, last=1, out=None):
        """The `pages` pages that each token and kv head attends to: the first and the last ones it sees, then those whose
        bounds allow the largest q·k. int32 [streams, tokens, kv heads, pages], ascending, -1 behind."""
        n, qs = self._rows("q", q, None)
        if not (max(step, first, last, pages) < _END and 0 <= min(step, first, last, pages)):
            raise ValueError(f"step = {step}, first = {first}, last = {last}, pages = {pages}")
        if out is None:
            out = q.new_empty((n[0], n[1], self.heads, pages), dtype=_i32)
        else:
            self._given(out, (n[0], n[1], self.heads, pages), _i32)
        self._run("select", _select, n[2], n[1], q.data_ptr(), qs[1], qs[2], qs[0], self._ints("visible", visible), step, first,
                  last, pages, out.data_ptr(), self._space(), 0)
        return out

    def evict(self, length, keep, acc, pos=None, first=0, recent=0, out=None):
        """Thins every stream and head to `keep` slots: those whose position is below `first` or among the `recent` newest,
        then those with the largest acc; the slots that stay from behind `keep` fill the free ones, in K, V, acc and pos.
        Returns the new lengths."""
        a, p, ms, mh = self._marks(acc, pos)
        n = self._ints("length", length)
        if not (max(keep, first, recent) < _END and 0 <= min(keep, first, recent)):
            raise ValueError(f"keep = {keep}, first = {first}, recent = {recent}")
        if out is None:
            out = torch.empty_like(length)
        else:
            self._ints("out", out)
        self._run("evict", _evict, n, keep, first, recent, a, p, ms, mh, out.data_ptr(), self._space(), 0)
        return out
