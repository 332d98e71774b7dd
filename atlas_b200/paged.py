"""A packed serving step over the C ABI: block tables and slots from request lengths (page_plan), the four-bit paged KV cache
(PagedKvCache) and the causal attention of whole packed prompts (prompt_attention).

The calls take device arrays: a DeviceArray of this module, or anything with data_ptr(), shape, stride(),
is_contiguous(), dtype and get_device() as a PyTorch tensor has them (PyTorch itself is not imported).  They run on the context's stream and return at once; arrays that another
stream fills have to be ordered before them (`Context.stream`), and arrays must live until the stream has passed the call.
"""
import ctypes as C
import math

import numpy as np

from . import _ffi
from ._ffi import AtlasError, BF16, F16, F32, check
from .tensor import Context

I32 = "int32"
_NAMES = {"torch.float32": F32, "torch.bfloat16": BF16, "torch.float16": F16, "torch.int32": I32}
_NUMPY = {F32: np.float32, BF16: np.uint16, F16: np.float16, I32: np.int32}     # bf16 as its bit patterns
_SHOWN = {F32: "f32", BF16: "bf16", F16: "f16", I32: "int32"}


class DeviceArray:
    """A typed array in HBM; strides in elements (None: contiguous).  dtype F32, BF16 (uint16 bit patterns on the host), F16 or I32."""

    def __init__(self, ctx, ptr, shape, dtype, strides=None, owner=False, base=None):
        self.ctx, self.ptr, self.shape, self.dtype = ctx, int(ptr), tuple(int(n) for n in shape), dtype
        if strides is None:
            strides, n = [], 1
            for m in reversed(self.shape):
                strides.insert(0, n)
                n *= m
        self.strides, self._owner, self._base = tuple(int(n) for n in strides), owner, base

    @classmethod
    def empty(cls, shape, dtype, ctx=None):
        ctx = ctx or Context.default()
        n = int(np.prod(shape, dtype=np.int64)) * np.dtype(_NUMPY[dtype]).itemsize
        return cls(ctx, ctx.malloc(max(n, 16)), shape, dtype, owner=True)

    @classmethod
    def from_host(cls, data, dtype, ctx=None):
        a = np.ascontiguousarray(data, dtype=_NUMPY[dtype])
        out = cls.empty(a.shape, dtype, ctx)
        if a.size:
            out.ctx.upload(out.ptr, a)
        return out

    def is_contiguous(self):
        n = 1
        for m, s in zip(reversed(self.shape), reversed(self.strides)):
            if m > 1 and s != n:
                return False
            n *= m
        return True

    def download(self):
        """The values of a contiguous array."""
        if not self.is_contiguous():
            raise AtlasError("download needs a contiguous array")
        return self.ctx.download(self.ptr, self.shape, _NUMPY[self.dtype])

    def columns(self, first, shape, strides):
        """A view that starts `first` elements in, with a shape and strides of its own; all of it lies within this array."""
        def reach(shape, strides):
            if 0 in shape:
                return 0, -1
            ends = [(int(n) - 1) * int(s) for n, s in zip(shape, strides)]
            return sum(e for e in ends if e < 0), sum(e for e in ends if e > 0)
        if len(shape) != len(strides) or any(n < 0 for n in shape):
            raise AtlasError("a view needs sizes of zero or more and a stride for each")
        (lo, hi), (first_here, last_here) = reach(shape, strides), reach(self.shape, self.strides)
        if hi >= lo and (first + lo < first_here or first + hi > last_here):
            raise AtlasError(f"a view of elements {first + lo}..{first + hi} leaves an array of elements {first_here}..{last_here}")
        return DeviceArray(self.ctx, self.ptr + first * np.dtype(_NUMPY[self.dtype]).itemsize, shape, self.dtype, strides, base=self)

    def __del__(self):
        try:
            if self._owner and self.ptr and self.ctx.handle:
                self.ctx.free(self.ptr)
        except Exception:
            pass
        self.ptr = 0


_CODES = {}      # dtype objects of other libraries seen so far → codes


def _code(dtype):
    c = _CODES.get(dtype)
    if c is None:
        c = _NAMES.get(str(dtype), -1)
        _CODES[dtype] = c
    return c


def _refuse(x, name, dtypes, ndim, device):
    """Says what is wrong with an array that did not pass."""
    if type(x) is DeviceArray:
        shape, dtype, at = x.shape, x.dtype, x.ctx.device
    else:
        try:
            shape, dtype, at = x.shape, _code(x.dtype), x.get_device()
            x.data_ptr, x.stride
        except AttributeError:
            raise AtlasError("%s is not a device array" % name) from None
    if dtype not in dtypes:
        raise AtlasError("%s must be %s" % (name, " or ".join(_SHOWN[d] for d in dtypes)))
    if len(shape) != ndim:
        raise AtlasError("%s must have %d dimensions, not %d" % (name, ndim, len(shape)))
    if at != device:
        raise AtlasError("%s is not on device %d" % (name, device))


def _ints(x, name, n, device):
    """Pointer of a contiguous int32 array of n numbers (None: any)."""
    try:
        if type(x) is DeviceArray:
            fine, ptr = x.dtype is I32 and x.ctx.device == device and len(x.shape) == 1 and x.is_contiguous() and (n is None or x.shape[0] == n), x.ptr
        else:
            fine = _CODES.get(x.dtype) is I32 and x.get_device() == device and x.ndim == 1 and x.is_contiguous() and (n is None or x.numel() == n)
            ptr = x.data_ptr()
    except AttributeError:
        fine = False
    if not fine:
        ptr = _ints_slowly(x, name, (n,), device)
    return ptr


def _ints_slowly(x, name, shape, device):
    """The same for any number of dimensions (None in `shape` stands for any extent); says what is wrong."""
    _refuse(x, name, (I32,), len(shape), device)
    for m, n in zip(shape, x.shape):
        if m is not None and m != n:
            raise AtlasError("%s must have shape %s, not %s" % (name, tuple(shape), tuple(x.shape)))
    if not x.is_contiguous():
        raise AtlasError("%s must be contiguous" % name)
    return x.ptr if type(x) is DeviceArray else x.data_ptr()


def _length(x):
    return x.shape[0] if type(x) is DeviceArray else x.numel()


def _rows(x, name, dtypes, device, heads=None, head_dim=None):
    """(ptr, rows, token stride, head stride, dtype, heads, head_dim) of [rows, heads, head_dim] with unit stride along a row."""
    try:
        if type(x) is DeviceArray:
            ptr, shape, strides, dtype, at = x.ptr, x.shape, x.strides, x.dtype, x.ctx.device
        else:
            ptr, shape, strides, dtype, at = x.data_ptr(), x.shape, x.stride(), _code(x.dtype), x.get_device()
        fine = dtype in dtypes and len(shape) == 3 and at == device
    except AttributeError:
        fine = False
    if not fine:
        _refuse(x, name, dtypes, 3, device)
    n, h, d = shape
    if (heads is not None and h != heads) or (head_dim is not None and d != head_dim):
        raise AtlasError("%s must be [rows, %s, %s], not %s" % (name, heads, head_dim, tuple(shape)))
    if d > 1 and strides[2] != 1:
        raise AtlasError("%s must have unit stride along head_dim" % name)
    return ptr, n, strides[0], strides[1], dtype, h, d


def _contiguous(view, name):
    _, rows, tok, head, _, heads, hd = view
    if (heads > 1 and head != hd) or (rows > 1 and tok != heads * hd):
        raise AtlasError("%s must be contiguous" % name)
    return view


def _device(ctx):
    """Device of the call: the context's, or that of the default context (device 0), which may not exist yet."""
    ctx = ctx or Context._default
    return ctx.device if ctx is not None else 0


def _whole(x, name, limit=0x7FFFFFFF):
    """An int argument that a C int can hold."""
    if not -limit - 1 <= x <= limit:
        raise AtlasError("%s is out of range" % name)
    return x


def page_plan(cached, fresh, free_pages, table, cu, lens, slots, pos, status, page_size, n_pages, ctx=None):
    """Block tables, slots and positions of a step from request lengths: see atlasx_page_plan.  int32 device arrays: cached, fresh,
    lens [batch]; free_pages [any]; table [batch, width], extended in place; cu [batch + 1]; slots, pos [rows]; status [3]."""
    dev = _device(ctx)
    p_cached = _ints(cached, "cached", None, dev)
    b = _length(cached)
    p_slots = _ints(slots, "slots", None, dev)
    rows = _length(slots)
    args = _ffi.PAGE_PLAN.pack(
        p_cached, _ints(fresh, "fresh", b, dev), _ints(free_pages, "free_pages", None, dev), _ints_slowly(table, "table", (b, None), dev),
        _ints(cu, "cu", b + 1, dev), _ints(lens, "lens", b, dev), p_slots, _ints(pos, "pos", rows, dev),
        _ints(status, "status", 3, dev), b, _length(free_pages), _whole(page_size, "page_size"), _whole(n_pages, "n_pages"), table.shape[1], rows)
    check(_ffi.lib().atlasx_page_plan((ctx or Context.default()).handle, args))


class PagedKvCache:
    """Keys and values of many requests in pages of four-bit numbers with a bf16 scale per `group` of them (GpuKvCache with pages
    and the Int4Tensor number format): 4.25 or 4.5 bits per number instead of 16 or 32."""

    def __init__(self, n_pages, page_size, n_kv_heads, head_dim, group=32, ctx=None):
        self.ctx = ctx or Context.default()
        self._h = None
        h = C.c_void_p()
        for n, name in ((n_pages, "n_pages"), (page_size, "page_size"), (n_kv_heads, "n_kv_heads"), (head_dim, "head_dim"), (group, "group")):
            _whole(n, name)
        check(_ffi.lib().atlasx_pagedkv_create(self.ctx.handle, n_pages, page_size, n_kv_heads, head_dim, group, C.byref(h)))
        self._h = h
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim, self.group = n_pages, page_size, n_kv_heads, head_dim, group
        pool, n, w = C.c_void_p(), C.c_size_t(), C.c_size_t()
        check(_ffi.lib().atlasx_pagedkv_ptrs(h, C.byref(pool), C.byref(n), C.byref(w)))
        self.bytes, self.workspace_bytes = n.value, w.value

    def workspace(self):
        """A zeroed workspace for decode_attention calls that may run beside others of this cache."""
        p = DeviceArray.empty((self.workspace_bytes + 3) // 4 * np.ones(1, np.int64), I32, self.ctx)
        check(_ffi.lib().atlasx_memset(self.ctx.handle, C.c_void_p(p.ptr), 0, self.workspace_bytes))
        return p

    def append(self, k, v, slots):
        """Rows of k and v [rows, n_kv_heads, head_dim] (f32, bf16 or f16, any strides of whole 16 bytes) into their slots;
        a negative slot marks a row that is not there."""
        dev, types = self.ctx.device, (F32, BF16, F16)
        kp, n, kt, kh, dt, _, _ = _rows(k, "k", types, dev, self.n_kv_heads, self.head_dim)
        vp, m, vt, vh, dv, _, _ = _rows(v, "v", types, dev, self.n_kv_heads, self.head_dim)
        if n != m or dt != dv:
            raise AtlasError("k and v must have the same rows and type")
        check(_ffi.lib().atlasx_pagedkv_append(self.ctx.handle, self._h,
                                               _ffi.PAGED_ROWS.pack(kp, vp, _ints(slots, "slots", n, dev), kt, kh, vt, vh, dt, n)))

    def read(self, slots, k_out, v_out):
        """The values that the slots hold into contiguous [rows, n_kv_heads, head_dim] arrays (f32, bf16 or f16)."""
        dev, types = self.ctx.device, (F32, BF16, F16)
        kp, n, _, _, dt, _, _ = _contiguous(_rows(k_out, "k_out", types, dev, self.n_kv_heads, self.head_dim), "k_out")
        vp, m, _, _, dv, _, _ = _contiguous(_rows(v_out, "v_out", types, dev, self.n_kv_heads, self.head_dim), "v_out")
        if n != m or dt != dv:
            raise AtlasError("k_out and v_out must have the same rows and type")
        check(_ffi.lib().atlasx_pagedkv_read(self.ctx.handle, self._h, _ints(slots, "slots", n, dev), n, dt, kp, vp))

    def decode_attention(self, q, out, table, lens, scale, window_size=0, workspace=None):
        """Attention of one token per request: q, out [batch, n_heads, head_dim] f32, table [batch, width] page numbers, lens [batch]
        cached rows (the new token's own among them)."""
        dev = self.ctx.device
        qp, b, _, _, _, nh, _ = _contiguous(_rows(q, "q", (F32,), dev, None, self.head_dim), "q")
        op = _contiguous(_rows(out, "out", (F32,), dev, nh, self.head_dim), "out")
        if op[1] != b:
            raise AtlasError("out must have the rows of q")
        wp, wn = (0, 0) if workspace is None else (_ints(workspace, "workspace", None, dev), 4 * _length(workspace))
        p_table = _ints_slowly(table, "table", (b, None), dev)
        check(_ffi.lib().atlasx_pagedkv_decode_attention(
            self.ctx.handle, self._h, _ffi.PAGED_ATTN.pack(qp, op[0], p_table, _ints(lens, "lens", b, dev), wp, wn, nh, table.shape[1], b,
                                                           _whole(window_size, "window_size"), scale)))

    def __del__(self):
        try:
            if self._h and self.ctx.handle:
                _ffi.lib().atlasx_pagedkv_free(self._h)
        except Exception:
            pass
        self._h = None


def prompt_attention(q, k, v, out, cu_q, cu_k, scale=None, window_size=0, ctx=None):
    """Causal attention of packed prompts: q, out [rows, n_heads, head_dim], k, v [key rows, n_kv_heads, head_dim], bf16 or f16; sequence
    b owns rows cu_q[b]..cu_q[b + 1] of q and cu_k[b]..cu_k[b + 1] of k and v, its last query at its last key.  scale None: 1/√head_dim."""
    dev, types = _device(ctx), (BF16, F16)
    qp, n, qt, qh, dt, nh, hd = _rows(q, "q", types, dev)
    kp, m, kt, kh, dk, nk, _ = _rows(k, "k", types, dev, None, hd)
    vp, mv, vt, vh, dv, _, _ = _rows(v, "v", types, dev, nk, hd)
    op, on, ot, oh, do, _, _ = _rows(out, "out", types, dev, nh, hd)
    if m != mv or on != n:
        raise AtlasError("k and v, and q and out, must have the same rows")
    if not dt == dk == dv == do:
        raise AtlasError("q, k, v and out must have the same type")
    p_cu_q = _ints(cu_q, "cu_q", None, dev)
    b = _length(cu_q) - 1
    args = _ffi.PROMPT.pack(qp, kp, vp, op, qt, qh, kt, kh, vt, vh, ot, oh, p_cu_q, _ints(cu_k, "cu_k", b + 1, dev), dt, b, n, m, nh, nk, hd,
                            _whole(window_size, "window_size"), 1.0 / math.sqrt(hd) if scale is None else scale)
    check(_ffi.lib().atlasx_prompt_attention((ctx or Context.default()).handle, args))
