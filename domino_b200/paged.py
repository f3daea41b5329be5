"""A paged key / value cache and the operators that fill, read and move it.

``PagedKVCache`` is the serving form of ``stack.RaggedKVCache``: keys and values live in pages of a few tokens, a table
says which pages a row of the batch holds, and rows may share pages.  Its operators are hand-written sm_100a kernels
behind ``dd_pages_*`` and ``dd_cache_*`` of include/domino_draft.h:

* ``write``    query / key norm, rotary positions and the store of a chunk's keys and values into their pages;
* ``attend``   attention of a chunk of new tokens (one or many) over the cache, causal or over the whole chunk, also
               with a sliding window and first tokens that stay visible;
* ``reserve``, ``crop``, ``fork``, ``compact``  pages for new tokens, back after a rejection, shared between rows,
               moved to the front.

Everything runs on the current stream of the cache's device without host synchronisation and can be captured in a CUDA
graph (lengths, positions and tables are read on the device).  Calls on one cache must be ordered: use one stream, or
make streams wait for one another.  There is no backward pass.  The reference keeps one contiguous cache per sequence
(code/dflash.py:359-360, 488).
"""
from __future__ import annotations

import copy
import ctypes
import math
from typing import Optional

import torch

from . import _lib

__all__ = ["PagedKVCache", "Rope", "rope_frequencies"]

_DTYPES = {torch.bfloat16: _lib.DD_BF16, torch.float16: _lib.DD_FP16, torch.float32: _lib.DD_F32}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class Rope:
    """Rotary positions of one kind of head.

    Pair i of the first ``rotary_dim`` values (default: all of the head) turns by ``position * inv_freq[i]``, and the
    turned values are scaled by ``factor``.  Pairs are ``(i, i + rotary_dim / 2)``, or ``(2 i, 2 i + 1)`` with
    ``interleaved``.  ``inv_freq`` [rotary_dim / 2] gives the frequencies; without it they are ``theta ** (-2 i /
    rotary_dim)``, changed for long contexts by ``scaling``, a dict as in a ``transformers`` config:

    * ``{"rope_type": "linear", "factor": f}``: every frequency divided by f;
    * ``{"rope_type": "yarn", "factor": f, "original_max_position_embeddings": n, ...}``: frequencies that turn more
      than ``beta_fast`` (32) times within n positions stay, those below ``beta_slow`` (1) turns are divided by f, a
      linear ramp over the pair index between; ``attention_factor`` (default 0.1 ln f + 1) becomes ``factor``;
    * ``{"rope_type": "llama3", "factor": f, "low_freq_factor": a, "high_freq_factor": b,
      "original_max_position_embeddings": n}``: by wavelength, above n / a divided by f, below n / b kept, blended between.
    """

    def __init__(self, head_dim: int, theta: float = 1e6, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[dict] = None, inv_freq: Optional[torch.Tensor] = None, factor: Optional[float] = None,
                 device=None):
        if inv_freq is not None:
            if rotary_dim is not None and rotary_dim != 2 * inv_freq.numel():
                raise ValueError(f"rotary_dim {rotary_dim} but {inv_freq.numel()} frequencies")
            if scaling:
                raise ValueError("scaling changes the default frequencies: give either it or inv_freq")
            if inv_freq.dim() != 1:
                raise ValueError("inv_freq must be [rotary_dim / 2]")
            rotary_dim = 2 * inv_freq.numel()
        elif rotary_dim is None:
            rotary_dim = head_dim
        if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} must be even and at most head_dim {head_dim}")
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), int(rotary_dim), bool(interleaved)
        scale = 1.0
        if inv_freq is None:
            inv_freq, scale = rope_frequencies(theta, rotary_dim, scaling)
        self.factor = float(scale if factor is None else factor)
        self.inv_freq = inv_freq.detach().to(device=device, dtype=torch.float32).contiguous()

    def to(self, device) -> "Rope":
        if self.inv_freq.device == torch.device(device):
            return self
        return Rope(self.head_dim, interleaved=self.interleaved, inv_freq=self.inv_freq, factor=self.factor, device=device)


def rope_frequencies(theta: float, dim: int, scaling: Optional[dict]):
    """(inv_freq fp32 [dim / 2], factor) of the default frequencies, scaled for long contexts."""
    inv = 1.0 / (theta ** (torch.arange(0, dim, 2, dtype=torch.int64).float() / max(dim, 1)))
    kind = (scaling or {}).get("rope_type", (scaling or {}).get("type", "default"))
    if kind == "default" or dim == 0:
        return inv, 1.0
    f = float(scaling["factor"])
    if kind == "linear":
        return inv / f, 1.0
    if kind == "yarn":
        n = float(scaling["original_max_position_embeddings"])
        fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)

        def index(turns):  # the (real) pair index that turns this often within n positions
            return dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = index(fast), index(slow)
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float32) - lo) / (hi - lo if hi > lo else 0.001)).clamp(0, 1)
        if scaling.get("mscale") and scaling.get("mscale_all_dim"):
            raise NotImplementedError("yarn with mscale and mscale_all_dim")
        factor = scaling.get("attention_factor")
        if factor is None:
            factor = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
        return inv / f * ramp + inv * (1 - ramp), float(factor)
    if kind == "llama3":
        n = float(scaling["original_max_position_embeddings"])
        a, b = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        wave = 2 * math.pi / inv
        blend = (n / wave - a) / (b - a)
        mid = (1 - blend) * inv / f + blend * inv
        return torch.where(wave > n / a, inv / f, torch.where(wave < n / b, inv, mid)), 1.0
    raise NotImplementedError(f"rope_type {kind!r}")


class PagedKVCache:
    """Keys and values of ``layers`` layers in ``pages`` pages of ``page_size`` tokens, for ``batch`` rows.

    State, all on the device (a captured call reads and writes it in place):

    * ``data``   [layers, 2, pages, kv_heads, page_size, head_dim]: keys (0) and values (1);
    * ``table``  int32 [batch, row_pages]: row b holds position p in page ``table[b, p // page_size]``, -1 is no page;
    * ``length`` int64 [batch]: tokens of each row (set by the caller after its writes, cut by ``crop``);
    * ``refs``   int32 [pages]: rows that hold a page; 0 is free.  Free pages are taken lowest number first.

    A call that cannot do a part of its work (no free page, a position without a page, a page shared with another row,
    a source row that does not exist) leaves that part out and sets a ``DD_STATUS_*`` bit, which ``status()`` reads.
    """

    def __init__(self, layers: int, batch: int, kv_heads: int, pages: int, head_dim: int, dtype, device,
                 page_size: int = 64, row_pages: Optional[int] = None):
        if dtype not in _DTYPES:
            raise NotImplementedError(f"the paged cache holds bf16, fp16 or fp32, got {dtype}")
        row_pages = pages if row_pages is None else row_pages
        self.layers, self.batch, self.kv_heads, self.pages = int(layers), int(batch), int(kv_heads), int(pages)
        self.head_dim, self.page_size, self.row_pages, self.dtype = int(head_dim), int(page_size), int(row_pages), dtype
        self._lib = _lib.load()
        self._c = _lib.DDPagedCache(layers=self.layers, batch=self.batch, kv_heads=self.kv_heads, pages=self.pages,
                                    page_size=self.page_size, head_dim=self.head_dim, row_pages=self.row_pages,
                                    dtype=_DTYPES[dtype])
        self._cp = ctypes.byref(self._c)
        need = ctypes.c_uint64()
        rc = self._lib.dd_cache_scratch(self._cp, ctypes.byref(need))
        if rc < 0:
            raise ValueError(self._lib.dd_last_error(None).decode(errors="replace"))
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("PagedKVCache runs on a CUDA device (sm_100a)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.capacity = self.row_pages * self.page_size
        self._whole = True  # all rows that hold pages of this pool
        self.data = torch.zeros(self.layers, 2, self.pages, self.kv_heads, self.page_size, self.head_dim, dtype=dtype,
                                device=device)
        self.table = torch.full((self.batch, self.row_pages), -1, dtype=torch.int32, device=device)
        self.length = torch.zeros(self.batch, dtype=torch.long, device=device)
        self.refs = torch.zeros(self.pages, dtype=torch.int32, device=device)
        self._status = torch.zeros(1, dtype=torch.int32, device=device)
        self._scratch = torch.zeros(need.value, dtype=torch.uint8, device=device)
        c = self._c
        c.data, c.table, c.length, c.refs = (x.data_ptr() for x in (self.data, self.table, self.length, self.refs))
        c.scratch, c.status, c.device = self._scratch.data_ptr(), self._status.data_ptr(), device.index

    def first_rows(self, n: int) -> "PagedKVCache":
        """The first ``n`` rows as a cache of their own, with the same pages and state: for a call on them alone.

        ``compact`` is not for such a part: it moves pages of all rows, whose tables the part does not know.
        """
        if not 1 <= n <= self.batch:
            raise ValueError(f"{n} rows of {self.batch}")
        part = copy.copy(self)
        part._whole = self._whole and n == self.batch
        part.batch, part.table, part.length = n, self.table[:n], self.length[:n]
        part._c = _lib.DDPagedCache.from_buffer_copy(self._c)
        part._c.batch = n
        part._cp = ctypes.byref(part._c)
        return part

    # ---------------------------------------------------------------- checks
    def _stream(self) -> int:
        """The current stream of the cache's device (the object that torch.cuda.current_stream makes costs 2 us)."""
        return _raw_stream(self.device.index)

    def _check(self, rc: int, what: str) -> None:
        if rc < 0:
            _lib.check(rc, None, what)

    def _rows(self, t: torch.Tensor, name: str) -> int:
        """An int64 [batch] tensor of the cache's device."""
        if not isinstance(t, torch.Tensor) or t.dtype != torch.long or t.shape != self.length.shape:
            raise ValueError(f"{name} must be an int64 tensor [{self.batch}]")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr()

    def _heads(self, x: torch.Tensor, name: str, tokens: Optional[int], heads: Optional[int]):
        """[batch, tokens, heads, head_dim] of the cache's type and device with a contiguous last dimension."""
        s = x.shape
        if (len(s) != 4 or s[0] != self.batch or s[3] != self.head_dim or s[1] < 1 or s[2] < 1
                or (tokens is not None and s[1] != tokens) or (heads is not None and s[2] != heads)):
            raise ValueError(f"{name} must be [{self.batch}, {tokens or 'tokens'}, {heads or 'heads'}, "
                             f"{self.head_dim}], got {list(s)}")
        if x.dtype != self.dtype:
            raise TypeError(f"{name} is {x.dtype}, the cache holds {self.dtype}")
        if x.device != self.device:
            raise ValueError(f"{name} is on {x.device}, the cache on {self.device}")
        return x if x.stride(3) == 1 else x.contiguous()

    def _norm(self, w: Optional[torch.Tensor], name: str):
        if w is None:
            return None
        if w.dtype != self.dtype or w.device != self.device or tuple(w.shape) != (self.head_dim,):
            raise ValueError(f"{name} must be [{self.head_dim}], {self.dtype}, on {self.device}")
        return w.contiguous()

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} outside [0, {self.layers})")
        return layer

    # ---------------------------------------------------------------- operators
    def write(self, layer: int, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, rope: Optional[Rope],
              start: torch.Tensor, lens: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
              k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Optional[torch.Tensor]:
        """Store a chunk's keys and values; returns the queries ready for ``attend``.

        q [batch, tokens, heads, head_dim] (or None), k and v [batch, tokens, kv_heads, head_dim]; any strides with a
        contiguous last dimension.  Token t of row b, t < ``lens[b]`` (all of them without ``lens``), has position
        ``start[b] + t``, whose page ``reserve`` has provided.  q and k are RMS-normalised per head with ``q_norm`` /
        ``k_norm`` [head_dim] where given, then turned by ``rope`` (None: not turned); the arithmetic is fp32 (angles
        fp64) with one rounding.  Rows of the result behind ``lens[b]`` are zero.  ``length`` does not change.
        """
        k = self._heads(k, "k", None, self.kv_heads)
        tokens = k.shape[1]
        v = self._heads(v, "v", tokens, self.kv_heads)
        a = _lib.DDCacheWriteArgs(layer=self._layer(layer), tokens=tokens, eps=eps)
        out = None
        if q is not None:
            q = self._heads(q, "q", tokens, None)
            out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
            a.heads, a.q, a.q_out = q.shape[2], q.data_ptr(), out.data_ptr()
            a.q_stride0, a.q_stride1, a.q_stride2, _ = q.stride()
        a.k, a.v = k.data_ptr(), v.data_ptr()
        a.k_stride0, a.k_stride1, a.k_stride2, _ = k.stride()
        a.v_stride0, a.v_stride1, a.v_stride2, _ = v.stride()
        a.start = self._rows(start, "start")
        if lens is not None:
            a.lens = self._rows(lens, "lens")
        if q_norm is not None:
            q_norm = self._norm(q_norm, "q_norm")
            a.q_norm = q_norm.data_ptr()
        if k_norm is not None:
            k_norm = self._norm(k_norm, "k_norm")
            a.k_norm = k_norm.data_ptr()
        if rope is not None:
            if rope.head_dim != self.head_dim or rope.inv_freq.device != self.device:
                raise ValueError(f"rope is for heads of {rope.head_dim} on {rope.inv_freq.device}, the cache has "
                                 f"{self.head_dim} on {self.device}")
            a.rotary, a.inv_freq, a.factor = rope.rotary_dim, rope.inv_freq.data_ptr(), rope.factor
            a.interleaved = rope.interleaved
        self._check(self._lib.dd_cache_write(self._cp, ctypes.byref(a), self._stream()), "dd_cache_write")
        return out

    def attend(self, layer: int, q: torch.Tensor, start: torch.Tensor, lens: Optional[torch.Tensor] = None,
               causal: bool = True, window: int = 0, sinks: int = 0, scale: Optional[float] = None) -> torch.Tensor:
        """Attention of a chunk of new tokens over one layer of the cache -> [batch, tokens, heads, head_dim].

        q [batch, tokens, heads, head_dim] (any strides with a contiguous last dimension; ``heads`` a multiple of
        ``kv_heads``).  Query t of row b, t < ``lens[b]``, has position p = ``start[b] + t`` and sees the keys j <
        ``start[b] + lens[b]`` that have a page: with ``causal`` those up to p, and with ``window`` > 0 of these only
        ``p - j < window`` or ``j < sinks``.  ``scale`` (positive) defaults to ``head_dim ** -0.5``.  A query that sees
        no key, or none with a score above -infinity, gives zeros, as do the rows behind ``lens[b]``.  What a query does
        not see has no effect on it; an infinite or NaN value that it sees makes that element infinite or NaN.
        """
        q = self._heads(q, "q", None, None)
        _, tokens, heads, _ = q.shape
        if heads % self.kv_heads:
            raise ValueError(f"{heads} query heads for {self.kv_heads} key heads")
        if window < 0 or sinks < 0 or (sinks and not window) or (window and not causal):
            raise ValueError("a window needs causal attention, sinks need a window")
        out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
        a = _lib.DDCacheAttendArgs(layer=self._layer(layer), tokens=tokens, heads=heads, causal=bool(causal),
                                   window=min(window, 1 << 30), sinks=min(sinks, 1 << 30), q=q.data_ptr(), out=out.data_ptr(),
                                   start=self._rows(start, "start"),
                                   scale=self.head_dim ** -0.5 if scale is None else scale)
        a.q_stride0, a.q_stride1, a.q_stride2, _ = q.stride()
        if lens is not None:
            a.lens = self._rows(lens, "lens")
        self._check(self._lib.dd_cache_attend(self._cp, ctypes.byref(a), self._stream()), "dd_cache_attend")
        return out

    def reserve(self, upto: torch.Tensor) -> None:
        """Make positions ``length[b] .. upto[b] - 1`` of every row writable (int64 [batch], device).

        Missing pages are taken from the free ones in row order.  A page that other rows hold too and that these
        positions reach is replaced by a copy; the first of the rows that need it keeps the original when no row
        outside this call's holds it.  Call it before ``write``.
        """
        self._check(self._lib.dd_pages_reserve(self._cp, self._rows(upto, "upto"), self._stream()), "dd_pages_reserve")

    def crop(self, length: torch.Tensor) -> None:
        """Cut every row to at most ``length[b]`` tokens (int64 [batch], device); pages wholly behind that go back."""
        self._check(self._lib.dd_pages_crop(self._cp, self._rows(length, "length"), self._stream()), "dd_pages_crop")

    def fork(self, src: torch.Tensor) -> None:
        """Row b continues from row ``src[b]`` as it was before the call (int64 [batch], device).

        It shares that row's pages and takes its length; ``src[b] = b`` leaves the row as it is, -1 empties it.
        """
        self._check(self._lib.dd_pages_fork(self._cp, self._rows(src, "src"), self._stream()), "dd_pages_fork")

    def compact(self) -> None:
        """Move the pages in use to the lowest numbers, so that all pages behind them are free."""
        if not self._whole:
            raise ValueError(f"compact needs all rows of the cache, this is its first {self.batch}")
        self._check(self._lib.dd_pages_compact(self._cp, self._stream()), "dd_pages_compact")

    def status(self) -> int:
        """Synchronise and return (and clear) the ``DD_STATUS_*`` bits that calls have set, on whatever stream they ran."""
        torch.cuda.synchronize(self.device)
        s = int(self._status.item())
        self._status.zero_()
        if s & _lib.DD_STATUS_TIMEOUT:  # an attention gave up half-way: its counters start anew
            self._scratch.zero_()
        return s
