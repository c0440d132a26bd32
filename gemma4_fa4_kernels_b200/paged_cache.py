"""8-bit paged KV cache: storage, attention over it, and its pages.

The static caches of ``decode_ops`` are BF16, contiguous and one sequence each.
This cache serves many sequences from one pool of pages and holds a key or value
element in one byte:

* a page holds ``page_size`` tokens of every layer; per layer it is ``[KV head]
  [token][head_dim]`` codes, ``torch.float8_e4m3fn`` or ``torch.int8``;
* a block (one page of one KV head) has one float32 scale, value = code * scale.
  :meth:`PagedKVCache8.append` chooses powers of two: the least one that holds
  the block's largest magnitude.  Codes are finite (infinities saturate, NaN
  becomes 0);
* ``tables`` (slots, pages per slot) lists each sequence's pages, -1 where there
  is none; ``lengths`` (slots) counts its tokens; ``refcounts`` (pages) says how
  many tables list a page.  All three live on the device and are only changed
  there, so a serving loop neither waits for the device nor re-captures its graphs.

A step of a batch::

    starts, ends = cache.extend(slots, counts)       # reserve pages, advance lengths
    for layer in range(layers):
        cache.append(layer, k, v, slots, starts, ends)
        out, lse = cache.attention(layer, q, slots, starts, ends, window=window)

``starts``/``ends`` (int32, one per row) are the positions of the row's tokens.
Operands are padded batches ``(rows, tokens, heads, head_dim)``: row b uses its
first ``ends[b] - starts[b]`` tokens, outputs of padding are zero (LSE -inf).  A
row whose slot or positions are out of range counts as empty; a row that
:meth:`extend`, :meth:`fork` or :meth:`copy_pages` cannot serve is left as it was.
Both raise a bit of ``status``, which :meth:`check` turns into an exception.
Slots of one call must be distinct.

Head dims 256 and 512 (local and global layers), any number of query heads per KV
head, softmax scale 1, the causal and sliding-window masks of the attention
operators without vision or document ids.  Inference only.  Calls run on the
current stream of the cache's device and never synchronise it (but ``check``).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from .errors import UnsupportedB200Path
from .ops import _raise_for, _stream, _workspace

PAGE_SIZES = (16, 32, 64, 128)
CODE_DTYPES = {torch.float8_e4m3fn: _lib.G4_KV8_E4M3, torch.int8: _lib.G4_KV8_INT8}
MAX_ROWS = 1024

# Up to this many (token, query head) columns per KV head and row the queries read
# the codes directly; longer chunks of prompts run the tensor-core forward over a
# BF16 copy of the keys they see.
DIRECT_COLUMNS = 128


def _ints(t, rows: int | None, name: str, device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1:
        raise ValueError(f"{name} must be a one-dimensional int32 tensor")
    if rows is not None and t.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} entries, found {t.shape[0]}")
    if t.device != device:
        raise ValueError(f"{name} must be on the cache's device ({device})")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _strides(t: torch.Tensor) -> list[int]:
    """(batch, token, head) strides; a dimension of size one has none that matter."""
    return [t.shape[-1] if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]


class PagedKVCache8:
    """An 8-bit paged KV cache of ``num_layers`` layers with one head layout."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, *,
                 max_slots: int, pages_per_slot: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        for name, n in (("num_layers", num_layers), ("num_pages", num_pages),
                        ("num_kv_heads", num_kv_heads), ("max_slots", max_slots),
                        ("pages_per_slot", pages_per_slot)):
            if int(n) < 1:
                raise ValueError(f"{name} must be positive")
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        _check_pool(shape, dtype)
        device = torch.device(device)
        self._bind(torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype),
                   torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype),
                   torch.ones(shape[:3], dtype=torch.float32, device=device),
                   torch.ones(shape[:3], dtype=torch.float32, device=device),
                   torch.full((max_slots, pages_per_slot), -1, dtype=torch.int32, device=device),
                   torch.zeros(max_slots, dtype=torch.int32, device=device),
                   torch.zeros(num_pages, dtype=torch.int32, device=device))

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale, tables, lengths, refcounts) -> "PagedKVCache8":
        """A cache over existing tensors (kept, not copied): codes ``k``, ``v``
        (layers, pages, KV heads, page_size, head_dim), scales ``k_scale``,
        ``v_scale`` (layers, pages, KV heads) float32, ``tables`` (slots,
        pages per slot), ``lengths`` (slots) and ``refcounts`` (pages) int32."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale, tables, lengths, refcounts)
        return self

    def _bind(self, k, v, k_scale, v_scale, tables, lengths, refcounts) -> None:
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("k and v must be code pools of one shape (layers, pages, KV heads, "
                             "page_size, head_dim)")
        _check_pool(tuple(k.shape), k.dtype)
        for name, t, shape, dtype in (
                ("k_scale", k_scale, k.shape[:3], torch.float32),
                ("v_scale", v_scale, k.shape[:3], torch.float32),
                ("lengths", lengths, tables.shape[:1], torch.int32),
                ("refcounts", refcounts, k.shape[1:2], torch.int32)):
            if t.shape != shape or t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}")
        if tables.dim() != 2 or tables.dtype != torch.int32 or not tables.numel():
            raise ValueError("tables must be int32 of shape (slots, pages per slot)")
        tensors = (k, v, k_scale, v_scale, tables, lengths, refcounts)
        if any(t.device != k.device for t in tensors):
            raise ValueError("the cache's tensors must share one device")
        if any(not t.is_contiguous() for t in tensors):
            raise ValueError("the cache's tensors must be contiguous")
        if len({t.data_ptr() for t in tensors}) != len(tensors):
            raise ValueError("the cache's tensors must be distinct")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.tables, self.lengths, self.refcounts = tables, lengths, refcounts
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self.device = k.device
        self.num_layers, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        self.max_slots, self.pages_per_slot = tables.shape
        self.capacity = self.pages_per_slot * self.page_size  # tokens a slot can hold
        self._blocks: dict = {}

    # ----------------------------------------------------------------------------
    # arguments
    # ----------------------------------------------------------------------------
    def _on_device(self) -> None:
        if self.device.type != "cuda":
            raise UnsupportedB200Path("the paged cache's operators require a CUDA device")

    def _launch(self, fn, *args) -> None:
        """``fn(*args, stream)`` on the cache's device; the status as an exception."""
        if torch.cuda.current_device() == self.device.index:
            rc = fn(*args, _stream(self.device))
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args, _stream(self.device))
        if rc:
            _raise_for(rc, fn.__name__)

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.num_layers:
            raise IndexError(f"layer {layer} of a cache of {self.num_layers}")
        return layer

    def _operand(self, t: torch.Tensor, heads: int | None, name: str) -> None:
        if t.dim() != 4 or t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be BF16 (rows, tokens, heads, head_dim)")
        if t.shape[3] != self.head_dim or (heads is not None and t.shape[2] != heads):
            raise ValueError(f"{name} of shape {tuple(t.shape)} does not fit the cache "
                             f"({self.num_kv_heads} KV heads, head_dim {self.head_dim})")
        if t.device != self.device:
            raise ValueError(f"{name} must be on the cache's device ({self.device})")
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"{name} must have unit stride along head_dim")
        if t.requires_grad and torch.is_grad_enabled():
            raise UnsupportedB200Path(f"the paged cache is inference only: {name} requires grad")

    def _rows(self, a, batch: int, slots, starts, ends) -> None:
        if slots is None:
            if batch > self.max_slots:
                raise ValueError("more rows than slots")
        else:
            a.slots = _ints(slots, batch, "slots", self.device).data_ptr()
        a.starts = _ints(starts, batch, "starts", self.device).data_ptr()
        a.ends = _ints(ends, batch, "ends", self.device).data_ptr()

    def _check_rows(self, batch: int, tokens: int) -> None:
        if batch > MAX_ROWS:
            raise UnsupportedB200Path(f"at most {MAX_ROWS} rows per call")

    def _kv8(self, key, layer: int, batch: int, tokens: int, fill) -> _lib.G4Kv8Args:
        """The argument block of a call signature (a copy of a cached one): all
        but the pointers of the call's own tensors."""
        key = (layer, batch, tokens, *key)
        block = self._blocks.get(key)
        if block is None:
            a = _lib.G4Kv8Args()
            a.k_pages, a.v_pages = self.k[layer].data_ptr(), self.v[layer].data_ptr()
            a.k_scale, a.v_scale = self.k_scale[layer].data_ptr(), self.v_scale[layer].data_ptr()
            a.tables, a.status = self.tables.data_ptr(), self.status.data_ptr()
            a.format = CODE_DTYPES[self.k.dtype]
            a.num_pages, a.page_size = self.num_pages, self.page_size
            a.num_kv_heads, a.head_dim = self.num_kv_heads, self.head_dim
            a.num_slots, a.pages_per_slot = self.max_slots, self.pages_per_slot
            a.batch, a.tokens = batch, tokens
            fill(a)
            if len(self._blocks) >= 512:
                self._blocks.clear()
            self._blocks[key] = block = bytes(a)
        return _lib.G4Kv8Args.from_buffer_copy(block)

    def _pages(self, batch: int, first=None, second=None, workspace=False):
        block = self._blocks.get("pages")
        if block is None:
            a = _lib.G4PagesArgs()
            a.tables, a.lengths = self.tables.data_ptr(), self.lengths.data_ptr()
            a.refcounts, a.status = self.refcounts.data_ptr(), self.status.data_ptr()
            a.k_pages, a.v_pages = self.k.data_ptr(), self.v.data_ptr()
            a.k_scale, a.v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()
            a.num_layers, a.num_pages, a.page_size = self.num_layers, self.num_pages, self.page_size
            a.num_kv_heads, a.head_dim = self.num_kv_heads, self.head_dim
            a.num_slots, a.pages_per_slot = self.max_slots, self.pages_per_slot
            self._blocks["pages"] = block = bytes(a)
        a = _lib.G4PagesArgs.from_buffer_copy(block)
        a.batch = batch
        if first is not None:
            a.first = first.data_ptr()
        if second is not None:
            a.second = second.data_ptr()
        ws = None
        if workspace:
            ws = _workspace(_lib.load().g4_pages_workspace_bytes(ctypes.byref(a)), self.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        return a, ws

    # ----------------------------------------------------------------------------
    # storage
    # ----------------------------------------------------------------------------
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots, starts, ends) -> None:
        """Quantise ``k`` and ``v`` (rows, tokens, KV heads, head_dim) BF16 and write
        each row's first ``ends - starts`` tokens at its positions, whose pages the
        tables must list (:meth:`extend`).  ``slots`` None: row b is slot b."""
        self._layer(layer)
        self._operand(k, self.num_kv_heads, "k")
        self._operand(v, self.num_kv_heads, "v")
        if v.shape != k.shape:
            raise ValueError("k and v must have one shape")
        batch, tokens = k.shape[:2]
        self._check_rows(batch, tokens)
        ks, vs = _strides(k), _strides(v)

        def fill(a):
            a.k_stride[:], a.v_stride[:] = ks, vs

        if batch == 0 or tokens == 0:
            return
        a = self._kv8(("append", *ks, *vs), layer, batch, tokens, fill)
        self._rows(a, batch, slots, starts, ends)
        self._on_device()
        a.k, a.v = k.data_ptr(), v.data_ptr()
        self._launch(_lib.load().g4_kv8_append, ctypes.byref(a))

    def read(self, layer: int, slots, starts, ends, max_tokens: int):
        """Values at positions ``starts .. ends - 1`` of each row: K and V, BF16
        (rows, max_tokens, KV heads, head_dim), zeros past a row's end and where it
        has no page.  Exact for what :meth:`append` wrote."""
        self._layer(layer)
        batch = _ints(starts, None, "starts", self.device).shape[0]
        if max_tokens < 0:
            raise ValueError("max_tokens must be >= 0")
        self._check_rows(batch, max_tokens)
        shape = (batch, max_tokens, self.num_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        if k.numel():
            self._read(layer, slots, starts, ends, k, v, _strides(k), batch, max_tokens, None)
        return k, v

    def _read(self, layer, slots, starts, ends, k, v, strides, batch, tokens, out_rows) -> None:
        def fill(a):
            a.k_stride[:] = a.v_stride[:] = strides

        a = self._kv8(("read", *strides), layer, batch, tokens, fill)
        self._rows(a, batch, slots, starts, ends)
        self._on_device()
        a.k, a.v = k.data_ptr(), v.data_ptr()
        if out_rows is not None:
            a.out_rows, a.out_total = out_rows.data_ptr(), k.shape[0]
        self._launch(_lib.load().g4_kv8_read, ctypes.byref(a))

    # ----------------------------------------------------------------------------
    # attention
    # ----------------------------------------------------------------------------
    def attention(self, layer: int, q: torch.Tensor, slots, starts, ends, *, window: int = 0,
                  max_seqlen_k: int | None = None):
        """Attention of ``q`` (rows, tokens, query heads, head_dim) BF16 at positions
        ``starts .. ends - 1`` over each row's own keys up to the query's position
        (``window`` W > 0: the last W of them).

        Returns ``(out, lse)``: BF16 of q's shape and float32 (rows, query heads,
        tokens); zeros and -inf for padding and for a query without a visible key.
        ``max_seqlen_k`` (default: a slot's capacity) bounds ``ends``; a tighter bound
        sizes the launch and its buffers better, and a row beyond it counts as empty.
        """
        self._layer(layer)
        self._operand(q, None, "q")
        batch, tokens, heads, d = q.shape
        if heads == 0 or heads % self.num_kv_heads:
            raise ValueError(f"{heads} query heads for {self.num_kv_heads} KV heads")
        if window < 0:
            raise ValueError("window must be >= 0")
        max_k = self.capacity if max_seqlen_k is None else int(max_seqlen_k)
        if not 1 <= max_k:
            raise ValueError("max_seqlen_k must be positive")
        max_k = min(max_k, self.capacity)
        self._check_rows(batch, tokens)
        if batch == 0 or tokens == 0:
            return (torch.empty_like(q, memory_format=torch.contiguous_format),
                    q.new_empty((batch, heads, tokens), dtype=torch.float32))
        if tokens * (heads // self.num_kv_heads) > DIRECT_COLUMNS:
            return self._chunk(layer, q, slots, starts, ends, int(window), max_k)
        qs = _strides(q)
        sizes = (heads * tokens * d, heads * d, d), (heads * tokens, tokens)

        def fill(a):
            a.q_stride[:], a.o_stride[:], a.lse_stride[:] = qs, sizes[0], sizes[1]
            a.num_q_heads, a.window, a.max_seqlen_k = heads, window, max_k
            a.workspace_bytes = self._kv8_workspace(a)

        a = self._kv8(("attn", heads, window, max_k, *qs), layer, batch, tokens, fill)
        self._rows(a, batch, slots, starts, ends)
        self._on_device()
        out = torch.empty((batch, tokens, heads, d), dtype=torch.bfloat16, device=self.device)
        lse = torch.empty((batch, heads, tokens), dtype=torch.float32, device=self.device)
        ws = _workspace(a.workspace_bytes, self.device)
        a.q, a.o, a.lse, a.workspace = q.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr()
        self._launch(_lib.load().g4_kv8_attn, ctypes.byref(a))
        return out, lse

    def _kv8_workspace(self, a) -> int:
        a.starts, a.ends = 16, 16  # the size does not depend on the call's pointers
        n = _lib.load().g4_kv8_attn_workspace_bytes(ctypes.byref(a))
        a.starts = a.ends = None
        return n

    def _chunk(self, layer, q, slots, starts, ends, window, max_k):
        batch, tokens, heads, d = q.shape
        keys = tokens + (min(max_k, window) if window else max_k) - 1  # most a row can see
        total = batch * tokens
        # checked before the first launch, like the direct path's operands
        if q.data_ptr() % 16 or any(s % 8 for s in _strides(q)):
            raise ValueError("q must be 16-byte aligned with strides that are multiples of 8")

        def fill(a):
            a.num_q_heads, a.window, a.max_seqlen_k = heads, window, max_k
            a.o_stride[:] = (heads * tokens * d, heads * d, d)
            a.lse_stride[:] = (tokens, total)

        a = self._kv8(("chunk", heads, window, max_k), layer, batch, tokens, fill)
        self._rows(a, batch, slots, starts, ends)
        self._on_device()
        lib = _lib.load()
        plan = torch.empty(4 * batch + 2, dtype=torch.int32, device=self.device)
        cu_q, cu_k = plan[:batch + 1], plan[batch + 1:2 * batch + 2]
        first, last = plan[2 * batch + 2:3 * batch + 2], plan[3 * batch + 2:]
        self._launch(lib.g4_kv8_chunk_plan, ctypes.byref(a), cu_q.data_ptr(), cu_k.data_ptr(),
                     first.data_ptr(), last.data_ptr())
        shape = (batch * keys, self.num_kv_heads, d)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        self._read(layer, slots, first, last, k, v, [8, self.num_kv_heads * d, d], batch, keys,
                   cu_k)
        out = torch.empty((batch, tokens, heads, d), dtype=torch.bfloat16, device=self.device)
        with torch.cuda.device(self.device):
            _, lse = ops.attn_fwd(q.reshape(total, heads, d), k, v, window=window,
                                  cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=tokens,
                                  max_seqlen_k=keys, out=out.view(total, heads, d))
        a.o, a.lse = out.data_ptr(), lse.data_ptr()
        self._launch(lib.g4_kv8_pad_rows, ctypes.byref(a))
        return out, lse.view(heads, batch, tokens).transpose(0, 1)

    # ----------------------------------------------------------------------------
    # pages
    # ----------------------------------------------------------------------------
    def extend(self, slots: torch.Tensor, counts):
        """Reserve pages for ``counts`` (int32 per row, or one int) more tokens of each
        slot and advance its length.  Returns ``(starts, ends)``, the new tokens'
        positions; a row that does not fit (its table is full, the pool is empty, its
        slot is bad or listed before) is left as it was with start = end."""
        batch = self._page_rows(slots, "slots")
        if isinstance(counts, int):
            counts = torch.full((batch,), counts, dtype=torch.int32, device=self.device)
        _ints(counts, batch, "counts", self.device)
        span = torch.empty((2, batch), dtype=torch.int32, device=self.device)
        starts, ends = span[0], span[1]
        if batch:
            self._on_device()
            a, _ = self._pages(batch, slots)
            a.counts, a.starts, a.ends = counts.data_ptr(), starts.data_ptr(), ends.data_ptr()
            self._launch(_lib.load().g4_pages_extend, ctypes.byref(a))
        return starts, ends

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Make each child (an empty slot) a copy of its parent: whole pages are
        shared, a partly filled last page is copied in every layer."""
        batch = self._page_rows(parents, "parents")
        _ints(children, batch, "children", self.device)
        if batch:
            self._on_device()
            a, _ws = self._pages(batch, parents, children, workspace=True)
            self._launch(_lib.load().g4_pages_fork, ctypes.byref(a))

    def free(self, slots: torch.Tensor) -> None:
        """Empty the slots; pages that no other slot lists become free."""
        self._free(slots, 0)

    def trim(self, slots: torch.Tensor, window: int) -> None:
        """Give back the leading pages that no token from a slot's length on sees
        through a sliding window of ``window``; lengths stay."""
        if window < 1:
            raise ValueError("window must be positive")
        self._free(slots, int(window))

    def _free(self, slots, window) -> None:
        batch = self._page_rows(slots, "slots")
        if batch:
            self._on_device()
            a, _ = self._pages(batch, slots)
            a.window = window
            self._launch(_lib.load().g4_pages_free, ctypes.byref(a))

    def compact(self) -> None:
        """Move the live pages to the lowest ids, so that the pool's end is free."""
        self._on_device()
        a, _ws = self._pages(0, workspace=True)
        self._launch(_lib.load().g4_pages_compact, ctypes.byref(a))

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copy page ``src[i]`` to page ``dst[i]`` in every layer, with its scales;
        tables and refcounts stay.  A pair with a bad id, with a destination that an
        earlier pair has too, or whose destination is any pair's source is left out."""
        batch = _ints(src, None, "src", self.device).shape[0]
        _ints(dst, batch, "dst", self.device)
        if batch:
            self._on_device()
            a, _ = self._pages(batch, src, dst)
            self._launch(_lib.load().g4_pages_copy, ctypes.byref(a))

    def _page_rows(self, t: torch.Tensor, name: str) -> int:
        batch = _ints(t, None, name, self.device).shape[0]
        if batch > MAX_ROWS:
            raise UnsupportedB200Path(f"at most {MAX_ROWS} rows per call")
        return batch

    def check(self) -> None:
        """Wait for the device, and raise if a call since the last check had a row
        that it could not serve."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [text for bit, text in (
                (_lib.G4_PAGES_EXHAUSTED, "no free page was left"),
                (_lib.G4_PAGES_ROW_FULL, "a slot's table was full"),
                (_lib.G4_PAGES_BAD_INDEX, "a slot, page or count was out of range or listed twice"),
            ) if bits & bit]
            raise RuntimeError("paged cache: " + "; ".join(what))


def _check_pool(shape, dtype) -> None:
    layers, pages, heads, page, d = shape
    if dtype not in CODE_DTYPES:
        raise ValueError("the codes must be torch.float8_e4m3fn or torch.int8")
    if page not in PAGE_SIZES:
        raise UnsupportedB200Path(f"page_size must be one of {PAGE_SIZES}")
    if d not in (256, 512):
        raise UnsupportedB200Path("head_dim must be 256 or 512")
    if not layers or not pages or not heads:
        raise ValueError("layers, pages and KV heads must be positive")
