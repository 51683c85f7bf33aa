"""Several sequences at once: attention of packed prompts, and a paged KV cache held in 4 bits.

``attn_varlen`` is the prompt attention of a packed batch; ``PagedKV4`` holds the K and V rows of
n_slots sequences in pages of 4-bit values (4.5 bits with their scales, a quarter of an fp16 cache), which
``append`` writes, ``attend`` reads for the new tokens of every slot and ``reserve``, ``fork``, ``free`` and
``compact`` manage.  The kernels and the format are those of include/sx8_paged.h; lengths, tables and
counts live on the device and no call waits for it, so a step of all of them can be captured in a
graph.  The reference serves one sequence with the Hugging Face cache (scripts/infer_sx8.py:109-173).
"""
from __future__ import annotations

import ctypes
import math

import torch

import _sx8lib as _L

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_STATUS = {1: "bad slot or count", 2: "no free pages", 3: "the slot's table row is full",
           4: "the target slot is in use, named twice or a source"}


def _dtype(name, t):
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be float16 or bfloat16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _rows(name, t, heads, hd, device, dtype=None, min_ts=0):
    """A (rows, heads, hd) tensor that the kernels can read in place, or a contiguous copy of it."""
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != hd:
        raise RuntimeError(f"{name} must be (rows, {heads}, {hd}), got {tuple(t.shape)}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    _dtype(name, t)
    t = t.resolve_neg()                                             # (a view that negates on reading)
    return t if _in_place(t, min_ts) else t.clone(memory_format=torch.contiguous_format)


def _in_place(t, min_ts=0):
    ts, hs, es = t.stride()
    return es == 1 and ts % 8 == 0 and hs % 8 == 0 and t.data_ptr() % 16 == 0 and min_ts <= ts <= 1 << 23 and hs >= 0


def _out(name, out, like, heads, hd):
    """The output to write: `out` checked, or a new one."""
    if out is None:
        return torch.empty(like.shape[0], heads, hd, dtype=like.dtype, device=like.device)
    if out.shape != (like.shape[0], heads, hd) or out.dtype != like.dtype or out.device != like.device:
        raise RuntimeError(f"{name} must be {(like.shape[0], heads, hd)} {like.dtype} on {like.device}")
    if out.is_neg():
        raise RuntimeError(f"{name} may not be a view that negates on reading")
    # no two rows of the output may share memory
    ts, hs = out.stride()[:2]
    apart = hs >= hd and ts >= (heads - 1) * hs + hd or ts >= hd and hs >= (out.shape[0] - 1) * ts + hd
    if out.shape[0] and not (_in_place(out) and apart):
        raise RuntimeError(f"{name} needs contiguous head rows that begin on 16 bytes and do not overlap")
    return out


def _ints(name, t, n, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device or t.dim() != 1 \
            or (n is not None and t.numel() != n) or not t.is_contiguous() or t.is_neg():
        raise RuntimeError(f"{name} must be a contiguous int32 vector{'' if n is None else f' of {n}'} on {device}")
    return t


def _scale(scale, hd):
    s = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not (s > 0.0 and s < math.inf):
        raise RuntimeError(f"scale must be positive and finite, got {s}")
    return s


def attn_varlen(q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None):
    """softmax(scale * q k^T) v of packed sequences: q (Tq, heads, hd), k and v (Tk, kv heads, hd) fp16 or
    bf16, sequence b the query rows cu_q[b] .. cu_q[b + 1] - 1 and the keys cu_k[b] .. cu_k[b + 1] - 1 (int32 on
    the device; cu_k = None: cu_q, keys and queries of the same tokens).  causal: the last query of a
    sequence attends all of its keys, the one before it one key less, and so on; a query with no key gives
    zeros.  Rows of no sequence are left as they are (in a new `out`: unset); out shares no memory with k and v.  hd 64, 128 or 256; scale
    1 / sqrt(hd) unless given.  Sums are held in float32, the weights of the values rounded to the inputs' type (fp16 outputs
    are then 2.1 to 2.5e-4 off in the 2-norm where their own rounding is 1.8 to 2.0e-4, bf16 2.1e-3 where it is 1.6e-3).  Forward
    only: outputs have no gradient of either mode.  Returns out (Tq, heads, hd)."""
    if out is None and q.dim() == 3:
        got = _L.py().varlen(q, k, v, cu_q, cu_k, _scale(scale, q.shape[2]), causal)
        if got is not None:
            return got
    if q.dim() != 3 or k.dim() != 3 or q.device.type != "cuda":
        raise RuntimeError("q, k and v must be (rows, heads, hd) tensors on the GPU")
    nh, hd, nk = q.shape[1], q.shape[2], k.shape[1]
    if k.shape[0] != v.shape[0]:
        raise RuntimeError(f"k and v have {k.shape[0]} and {v.shape[0]} rows")
    if cu_k is None:
        cu_k = cu_q
    with torch.cuda.device(q.device):
        q = _rows("q", q, nh, hd, q.device)
        k = _rows("k", k, nk, hd, q.device, q.dtype, hd)
        v = _rows("v", v, nk, hd, q.device, q.dtype, hd)
        out = _out("out", out, q, nh, hd)
        if out.data_ptr() and out.data_ptr() in (k.data_ptr(), v.data_ptr()):
            raise RuntimeError("out may not be k or v")
        _ints("cu_q", cu_q, None, q.device)
        _ints("cu_k", cu_k, cu_q.numel(), q.device)
        nb = int(_L.lib().sx8_attn_varlen_workspace_bytes(cu_q.numel() - 1, q.shape[0], k.shape[0], nh, hd))
        ws = torch.empty(nb, dtype=torch.uint8, device=q.device) if nb > 0 else None
        _L.call("sx8_attn_varlen", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(),
                cu_q.numel() - 1, q.shape[0], k.shape[0], nh, nk, hd, q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                v.stride(0), v.stride(1), out.stride(0), out.stride(1), _scale(scale, hd), int(bool(causal)),
                _DTYPES[q.dtype], None if ws is None else ws.data_ptr(), max(nb, 0), _L.stream(q.device))
    return out


class PagedKV4:
    """The 4-bit KV cache of n_slots sequences and n_layers layers.

    pages  (n_layers, n_pages, page bytes) uint8     table  (n_slots, max_pages) int32, -1: no page
    lens   (n_slots,) int32, tokens of a slot        refs   (n_pages,) int32, slots that hold a page
    status (2,) int32: 0, or the first page operation's error (``check`` raises it)

    A step of new tokens is: ``reserve`` (lens grows, pages are taken), then for each layer ``append`` of the new K and V
    rows and ``attend`` of the new query rows.  Rows are packed by slot: slot s has the rows cu[s] .. cu[s + 1] - 1,
    or row s alone without cu; they are the last tokens of the slot.  Every call runs on the current stream of
    the cache's device; calls on one cache from several streams need the caller's ordering, as any tensors do.
    The calls stand outside autograd: inputs that require a gradient or carry a tangent give outputs that do not.
    """

    def __init__(self, n_layers, n_kv, head_dim, n_pages, n_slots, max_pages, page_tokens=64, device=None):
        device = torch.device(device or "cuda")
        nb = self._page_bytes(n_kv, head_dim, page_tokens)
        i32 = dict(dtype=torch.int32, device=device)
        self._bind(torch.zeros(n_layers, n_pages, nb, dtype=torch.uint8, device=device),
                   torch.full((n_slots, max_pages), -1, **i32), torch.zeros(n_slots, **i32),
                   torch.zeros(n_pages, **i32), n_kv, head_dim, page_tokens)

    @classmethod
    def from_tensors(cls, pages, table, lens, refs, *, n_kv, head_dim, page_tokens):
        """A cache over tensors that exist already (they are used in place)."""
        self = cls.__new__(cls)
        self._bind(pages, table, lens, refs, n_kv, head_dim, page_tokens)
        return self

    @staticmethod
    def _page_bytes(n_kv, head_dim, page_tokens):
        nb = int(_L.lib().sx8_kv4_page_bytes(int(n_kv), int(head_dim), int(page_tokens)))
        if nb < 0:
            raise RuntimeError(f"no 4-bit page of {n_kv} heads of {head_dim} and {page_tokens} tokens "
                               "(1..256 heads of 64, 128 or 256; 32, 64, 128 or 256 tokens)")
        return nb

    def _bind(self, pages, table, lens, refs, n_kv, head_dim, page_tokens):
        nb = self._page_bytes(n_kv, head_dim, page_tokens)
        if pages.dtype != torch.uint8 or pages.dim() != 3 or pages.shape[2] != nb or not pages.is_contiguous() \
                or pages.numel() == 0 or pages.device.type != "cuda" or pages.is_neg():
            raise RuntimeError(f"pages must be a contiguous (layers, pages, {nb}) uint8 tensor on the GPU")
        if table.dim() != 2 or not table.is_contiguous():
            raise RuntimeError("table must be a contiguous (slots, pages) int32 tensor")
        self.device = pages.device
        self.n_layers, self.n_pages = pages.shape[:2]
        self.n_slots, self.max_pages = table.shape
        _ints("table", table.view(-1), None, self.device)
        _ints("lens", lens, self.n_slots, self.device)
        _ints("refs", refs, self.n_pages, self.device)
        self.n_kv, self.head_dim, self.page_tokens, self.page_bytes = int(n_kv), int(head_dim), int(page_tokens), nb
        status = torch.zeros(2, dtype=torch.int32, device=self.device)
        self._ws_pages = int(_L.lib().sx8_kv4_pages_workspace_bytes(self.n_slots, self.n_pages))
        if self._ws_pages < 0 or self.max_pages * self.page_tokens > 1 << 22:
            raise RuntimeError("a cache has 1..4096 slots of up to 2^22 tokens and up to 2^28 pages")
        self._ws_attend = int(_L.lib().sx8_kv4_attend_workspace_bytes(self.head_dim))
        self._t = (pages, table, lens, refs, status, nb, self.n_kv, self.head_dim, self.page_tokens, self._ws_attend,
                   self._ws_pages)

    pages = property(lambda self: self._t[0])
    table = property(lambda self: self._t[1])
    lens = property(lambda self: self._t[2])
    refs = property(lambda self: self._t[3])
    status = property(lambda self: self._t[4])

    # ---------------------------------------------------------------- rows
    def _slots(self, layer, cu):
        if not 0 <= layer < self.n_layers:
            raise RuntimeError(f"layer {layer} of {self.n_layers}")
        if cu is not None:
            _ints("cu", cu, self.n_slots + 1, self.device)
        return (self.pages.data_ptr() + layer * self.n_pages * self.page_bytes, self.table.data_ptr(), self.lens.data_ptr(),
                None if cu is None else cu.data_ptr(), self.n_slots, self.max_pages, self.n_pages)

    def append(self, layer, k, v, cu=None):
        """Write the new tokens' k and v rows (rows, n_kv, head_dim), fp16 or bf16, into the slots' pages."""
        if _L.py().kv4_append(self._t, layer, k, v, cu):
            return
        with torch.cuda.device(self.device):
            k = _rows("k", k, self.n_kv, self.head_dim, self.device)
            v = _rows("v", v, self.n_kv, self.head_dim, self.device, k.dtype)
            if k.shape[0] != v.shape[0]:
                raise RuntimeError(f"k and v have {k.shape[0]} and {v.shape[0]} rows")
            _L.call("sx8_kv4_append", *self._slots(layer, cu), k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0),
                    k.stride(1), v.stride(0), v.stride(1), self.n_kv, self.head_dim, self.page_tokens, _DTYPES[k.dtype],
                    _L.stream(self.device))

    def read(self, layer, rows, cu=None, dtype=torch.float16, out=None):
        """The values of the slots' last tokens: k and v (rows, n_kv, head_dim), packed as `append` takes them (cu of
        all lengths reads whole slots).  out: (k, v) to write into.  Tokens without a page and rows without a token give zeros;
        rows of no slot are left as they are (in new tensors: unset)."""
        if dtype not in _DTYPES:
            raise RuntimeError(f"dtype must be float16 or bfloat16, got {dtype}")
        if out is None:
            got = _L.py().kv4_read(self._t, layer, rows, cu, dtype is torch.bfloat16)
            if got is not None:
                return got
        with torch.cuda.device(self.device):
            like = torch.empty(int(rows), 0, 0, dtype=dtype, device=self.device)
            if out is None:
                out = tuple(torch.empty(int(rows), self.n_kv, self.head_dim, dtype=dtype, device=self.device)
                            for _ in range(2))
            k, v = (_out(n, t, like, self.n_kv, self.head_dim) for n, t in zip(("k", "v"), out))
            if k.shape[0] and k.data_ptr() == v.data_ptr():
                raise RuntimeError("k and v may not share memory")
            _L.call("sx8_kv4_read", *self._slots(layer, cu), k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0), k.stride(1),
                    v.stride(0), v.stride(1), self.n_kv, self.head_dim, self.page_tokens, _DTYPES[dtype],
                    _L.stream(self.device))
        return k, v

    def attend(self, layer, q, cu=None, scale=None, out=None):
        """Attention of the new query rows q (rows, heads, head_dim), fp16 or bf16: row i of a slot's n new ones attends
        the slot's tokens 0 .. lens - n + i (zeros where that is none).  Returns out (rows, heads, head_dim)."""
        if out is None:
            got = _L.py().kv4_attend(self._t, layer, q, cu, _scale(scale, self.head_dim))
            if got is not None:
                return got
        with torch.cuda.device(self.device):
            nh = q.shape[1] if q.dim() == 3 else 0
            q = _rows("q", q, nh, self.head_dim, self.device)
            out = _out("out", out, q, nh, self.head_dim)
            ws = torch.empty(self._ws_attend, dtype=torch.uint8, device=self.device)
            _L.call("sx8_kv4_attend", *self._slots(layer, cu), q.data_ptr(), out.data_ptr(), q.shape[0], q.stride(0),
                    q.stride(1), out.stride(0), out.stride(1), nh, self.n_kv, self.head_dim, self.page_tokens,
                    _scale(scale, self.head_dim), _DTYPES[q.dtype], ws.data_ptr(), self._ws_attend,
                    _L.stream(self.device))
        return out

    # ---------------------------------------------------------------- pages
    def _ws(self):
        return torch.empty(self._ws_pages, dtype=torch.uint8, device=self.device)

    def reserve(self, add):
        """Slot s grows by add[s] tokens (int32 on the device): lens, and pages for them, lowest free page first."""
        if _L.py().kv4_pages(self._t, "reserve", add):
            return
        with torch.cuda.device(self.device):
            _ints("add", add, self.n_slots, self.device)
            ws = self._ws()
            _L.call("sx8_kv4_reserve", self.table.data_ptr(), self.lens.data_ptr(), self.refs.data_ptr(), add.data_ptr(),
                    self.n_slots, self.max_pages, self.n_pages, self.page_tokens, self.status.data_ptr(), ws.data_ptr(),
                    self._ws_pages, _L.stream(self.device))

    def fork(self, src, dst):
        """The empty slots dst[i] become copies of the slots src[i] (int32 on the device): full pages are shared, a last
        page that is partly filled is copied."""
        if _L.py().kv4_pages(self._t, "fork", src, dst):
            return
        with torch.cuda.device(self.device):
            _ints("src", src, None, self.device)
            _ints("dst", dst, src.numel(), self.device)
            ws = self._ws()
            _L.call("sx8_kv4_fork", self.pages.data_ptr(), self.n_layers, self.page_bytes, self.table.data_ptr(),
                    self.lens.data_ptr(), self.refs.data_ptr(), src.data_ptr(), dst.data_ptr(), src.numel(), self.n_slots,
                    self.max_pages, self.n_pages, self.page_tokens, self.status.data_ptr(), ws.data_ptr(),
                    self._ws_pages, _L.stream(self.device))

    def free(self, slots):
        """Empty the slots (int32 on the device); pages that no other slot holds are free."""
        if _L.py().kv4_pages(self._t, "free", slots):
            return
        with torch.cuda.device(self.device):
            _ints("slots", slots, None, self.device)
            _L.call("sx8_kv4_free", self.table.data_ptr(), self.lens.data_ptr(), self.refs.data_ptr(), slots.data_ptr(),
                    slots.numel(), self.n_slots, self.max_pages, self.n_pages, self.status.data_ptr(),
                    _L.stream(self.device))

    def compact(self):
        """Move the used pages to the front of the pool: pages 0 .. (number of used ones) - 1."""
        if _L.py().kv4_pages(self._t, "compact"):
            return
        with torch.cuda.device(self.device):
            ws = self._ws()
            _L.call("sx8_kv4_compact", self.pages.data_ptr(), self.n_layers, self.page_bytes, self.table.data_ptr(),
                    self.refs.data_ptr(), self.n_slots, self.max_pages, self.n_pages, ws.data_ptr(), self._ws_pages,
                    _L.stream(self.device))

    def check(self):
        """Wait for the device and raise the first error that reserve, fork or free met since the last check."""
        code, item = self.status.tolist()
        if code:
            self.status.zero_()
            raise RuntimeError(f"paged cache: {_STATUS.get(code, code)} (slot or entry {item})")
