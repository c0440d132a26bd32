"""8-bit paged KV cache: storage, attention over it, and its pages.

The static caches of ``decode_ops`` are BF16, contiguous and one sequence each.
This cache serves many sequences from one pool of pages and holds a key or value
element in one byte:

* a page holds ``page_size`` tokens of every layer; per layer it is ``[KV head]
  [token][head_dim]`` codes, ``torch.float8_e4m3fn`` or ``torch.int8``;
* a block (one page of one KV head) has one float32 scale, value = code * scale.
  :meth:`PagedKVCache8.append` chooses powers of two: the least one that holds
  the block's largest magnitude.  Values are finite (infinities saturate, NaN
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
row with ``ends[b] <= starts[b]`` asks for nothing, whatever its slot.  One that
asks for a slot or positions out of range counts as empty; a row that
:meth:`extend`, :meth:`fork` or :meth:`copy_pages` cannot serve is left as it was.
Both raise a bit of ``status``, which :meth:`check` turns into an exception.
Slots of one call must be distinct; :meth:`append` overlooks rows that ask for nothing.

Head dims 256 and 512 (local and global layers), any number of query heads per KV
head, softmax scale 1, the causal and sliding-window masks of the attention
operators without vision or document ids.  Inference only.  Calls run on the
current stream of the cache's device and do not wait for it, except ``check`` and,
for prompt chunks whose scratch exceeds the forward's budget, ``attention`` (as the
packed forward does; such a call cannot be captured).  The cache's tensors are its own
for its life: their contents may be changed from outside, they are not to be replaced.

Rejected drafts are taken back by lowering their slots' ``lengths`` on the device
(``cache.lengths[slots] = ends - rejected``): the pages behind a length stay the slot's,
:meth:`extend` fills them before it takes new ones and :meth:`free` gives them back.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, ops
from .errors import UnsupportedB200Path
from .ops import _raise_for, _stream

PAGE_SIZES = (16, 32, 64, 128)
CODE_DTYPES = {torch.float8_e4m3fn: _lib.G4_KV8_E4M3, torch.int8: _lib.G4_KV8_INT8}
MAX_ROWS = 1024

# Up to this many (token, query head) columns per KV head and row, by head dim, the
# queries read the codes directly; longer chunks of prompts run the tensor-core forward
# over a BF16 copy of the keys they see, whose softmax weights are BF16 (error against 64
# bits 0.0023 of the output's size, 0.0017 directly).  One bound for any number of rows:
# with one row the direct kernels stay faster beyond it, with four they do not.  Measured,
# us, direct against copy (1 and 4 rows):
#   d512, 1500 keys     256 columns  38 / 65,   71 / 81    512 columns   46 / 67,  116 / 85
#   d512, 17000 keys    256 columns 118 / 419, 374 / 587   512 columns  206 / 423, 712 / 595
#   d256, window 1024    64 columns  32 / 36,   48 / 52    128 columns   34 / 36,   75 / 52
DIRECT_COLUMNS = {512: 256, 256: 64}

# Most bytes of that BF16 copy at once.  It is sized by the bound on the rows' keys, which
# may be a whole slot, and the forward's own scratch grows with it: calls of more rows run
# by groups of rows, one copy after another.  64 rows of 40 tokens behind 3000 keys, d512,
# slots of 32768 tokens (us, GB at most): in one 1708, 41; with 9 GiB 1775, 21; 4 GiB 1902, 9.
CHUNK_COPY_BYTES = 9 << 30


def _layout(*shape) -> tuple:
    """(shape, strides) of a contiguous tensor."""
    strides, n = [], 1
    for x in reversed(shape):
        strides.append(n)
        n *= max(x, 1)
    return shape, tuple(strides[::-1])


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
        """A cache over existing tensors (kept, not copied): finite codes ``k``, ``v``
        (layers, pages, KV heads, page_size, head_dim), scales ``k_scale``,
        ``v_scale`` (layers, pages, KV heads) float32, positive and at most 2^121,
        ``tables`` (slots, pages per slot), ``lengths`` (slots) and ``refcounts``
        (pages) int32."""
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
        self._calls: dict = {}

    # ----------------------------------------------------------------------------
    # arguments
    # ----------------------------------------------------------------------------
    # What a call checks and lays out depends on its operands' shapes, strides and
    # types only.  It is done once per signature and kept as a finished argument
    # block; a call copies the block and writes its pointers (a decode step of a
    # small batch is otherwise bound by this host work).
    def _on_device(self) -> None:
        if self.device.type != "cuda":
            raise UnsupportedB200Path("the paged cache's operators require a CUDA device")

    def _launch(self, fn, *args) -> None:
        rc = fn(*args, _stream(self.device))
        if rc:
            _raise_for(rc, fn.__name__)

    def _operand(self, t: torch.Tensor, heads: int | None, name: str) -> None:
        if t.dim() != 4 or t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be BF16 (rows, tokens, heads, head_dim)")
        if t.shape[3] != self.head_dim or (heads is not None and t.shape[2] != heads):
            raise ValueError(f"{name} of shape {tuple(t.shape)} does not fit the cache "
                             f"({self.num_kv_heads} KV heads, head_dim {self.head_dim})")
        if t.device != self.device:
            raise ValueError(f"{name} must be on the cache's device ({self.device})")
        if t.stride(3) != 1:
            raise ValueError(f"{name} must have unit stride along head_dim")
        if t.shape[0] > MAX_ROWS:
            raise UnsupportedB200Path(f"at most {MAX_ROWS} rows per call")

    @staticmethod
    def _grad(*tensors) -> None:
        for t in tensors:
            if t.requires_grad and torch.is_grad_enabled():
                raise UnsupportedB200Path("the paged cache is inference only: an operand "
                                          "requires grad")

    # empty_strided takes half the host time of torch.empty
    def _new(self, layout, dtype) -> torch.Tensor:
        return torch.empty_strided(layout[0], layout[1], dtype=dtype, device=self.device)

    def _ints(self, t, rows: int | None, name: str) -> torch.Tensor:
        """``t``, a contiguous int32 vector of ``rows`` entries on the cache's device."""
        if (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.dim() == 1
                and t.device == self.device and t.is_contiguous()
                and (rows is None or len(t) == rows)):
            return t
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1:
            raise ValueError(f"{name} must be a one-dimensional int32 tensor")
        if t.device != self.device:
            raise ValueError(f"{name} must be on the cache's device ({self.device})")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        raise ValueError(f"{name} must have {rows} entries, found {t.shape[0]}")

    def _rows(self, a, batch: int, slots, starts, ends) -> None:
        if slots is not None:
            a.slots = self._ints(slots, batch, "slots").data_ptr()
        elif batch > self.max_slots:
            raise ValueError("more rows than slots")
        a.starts = self._ints(starts, batch, "starts").data_ptr()
        a.ends = self._ints(ends, batch, "ends").data_ptr()
        if self.device.type != "cuda":
            self._on_device()

    def _block(self, layer: int, batch: int, tokens: int) -> _lib.G4Kv8Args:
        """A new argument block of one layer's cache."""
        if not 0 <= layer < self.num_layers:
            raise IndexError(f"layer {layer} of a cache of {self.num_layers}")
        a = _lib.G4Kv8Args()
        a.k_pages, a.v_pages = self.k[layer].data_ptr(), self.v[layer].data_ptr()
        a.k_scale, a.v_scale = self.k_scale[layer].data_ptr(), self.v_scale[layer].data_ptr()
        a.tables, a.status = self.tables.data_ptr(), self.status.data_ptr()
        a.format = CODE_DTYPES[self.k.dtype]
        a.num_pages, a.page_size = self.num_pages, self.page_size
        a.num_kv_heads, a.head_dim = self.num_kv_heads, self.head_dim
        a.num_slots, a.pages_per_slot = self.max_slots, self.pages_per_slot
        a.batch, a.tokens = batch, tokens
        a.device = -1 if self.device.index is None else self.device.index
        return a

    def _keep(self, key, call):
        if len(self._calls) >= 512:
            self._calls.clear()
        self._calls[key] = call
        return call

    def _pages(self, batch: int, first=None, second=None, workspace=False):
        block = self._calls.get("pages")
        if block is None:
            self._on_device()
            a = _lib.G4PagesArgs()
            a.tables, a.lengths = self.tables.data_ptr(), self.lengths.data_ptr()
            a.refcounts, a.status = self.refcounts.data_ptr(), self.status.data_ptr()
            a.k_pages, a.v_pages = self.k.data_ptr(), self.v.data_ptr()
            a.k_scale, a.v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()
            a.num_layers, a.num_pages, a.page_size = self.num_layers, self.num_pages, self.page_size
            a.num_kv_heads, a.head_dim = self.num_kv_heads, self.head_dim
            a.num_slots, a.pages_per_slot = self.max_slots, self.pages_per_slot
            a.device = -1 if self.device.index is None else self.device.index
            block = self._keep("pages", bytes(a))
        a = _lib.G4PagesArgs.from_buffer_copy(block)
        a.batch = batch
        if first is not None:
            a.first = first.data_ptr()
        if second is not None:
            a.second = second.data_ptr()
        ws = None
        if workspace:
            need = self._calls.get(("workspace", batch))
            if need is None:
                need = self._keep(("workspace", batch),
                                  _lib.load().g4_pages_workspace_bytes(ctypes.byref(a)))
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        return a, ws

    # ----------------------------------------------------------------------------
    # storage
    # ----------------------------------------------------------------------------
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots, starts, ends) -> None:
        """Quantise ``k`` and ``v`` (rows, tokens, KV heads, head_dim) BF16 and write
        each row's first ``ends - starts`` tokens at its positions, whose pages the
        tables must list (:meth:`extend`).  ``slots`` None: row b is slot b."""
        key = ("append", layer, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(),
               v.dtype, v.device)
        call = self._calls.get(key) or self._append_call(key, layer, k, v)
        self._grad(k, v)
        batch, block = call
        if block is None:
            return
        a = _lib.G4Kv8Args.from_buffer_copy(block)
        self._rows(a, batch, slots, starts, ends)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        self._launch(_lib.load().g4_kv8_append, ctypes.byref(a))

    def _append_call(self, key, layer, k, v):
        self._operand(k, self.num_kv_heads, "k")
        self._operand(v, self.num_kv_heads, "v")
        if v.shape != k.shape:
            raise ValueError("k and v must have one shape")
        batch, tokens = k.shape[:2]
        a = self._block(layer, batch, tokens)
        a.k_stride[:], a.v_stride[:] = _strides(k), _strides(v)
        return self._keep(key, (batch, bytes(a) if batch and tokens else None))

    def read(self, layer: int, slots, starts, ends, max_tokens: int):
        """Values at positions ``starts .. ends - 1`` of each row: K and V, BF16
        (rows, max_tokens, KV heads, head_dim), zeros past a row's end and where it
        has no page.  Exact for what :meth:`append` wrote."""
        batch = self._ints(starts, None, "starts").shape[0]
        key = ("read", layer, batch, max_tokens)
        call = self._calls.get(key)
        if call is None:
            if batch > MAX_ROWS:
                raise UnsupportedB200Path(f"at most {MAX_ROWS} rows per call")
            if max_tokens < 0:
                raise ValueError("max_tokens must be >= 0")
            layout = _layout(batch, max_tokens, self.num_kv_heads, self.head_dim)
            call = self._keep(key, (layout, self._read_block(layer, batch, max_tokens)))
        layout, block = call
        k, v = self._new(layout, torch.bfloat16), self._new(layout, torch.bfloat16)
        if batch and max_tokens:
            self._read(block, batch, slots, starts, ends, k, v, None)
        return k, v

    def _read_block(self, layer, batch, tokens) -> bytes:
        a = self._block(layer, batch, tokens)
        row = self.num_kv_heads * self.head_dim
        a.k_stride[:] = a.v_stride[:] = (tokens * row, row, self.head_dim)
        return bytes(a)

    def _read(self, block, batch, slots, starts, ends, k, v, out_rows, holes=None) -> None:
        a = _lib.G4Kv8Args.from_buffer_copy(block)
        self._rows(a, batch, slots, starts, ends)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        if out_rows is not None:
            a.out_rows, a.out_total, a.holes = out_rows.data_ptr(), k.shape[0], holes
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
        sizes the launch and its buffers better; a row beyond it is out of range.
        """
        key = ("attention", layer, window, max_seqlen_k, q.shape, q.stride(), q.dtype, q.device)
        call = self._calls.get(key) or self._attention_call(key, layer, q, window, max_seqlen_k)
        self._grad(q)
        batch, block, out_layout, lse_layout, ws_bytes, chunk = call
        out = self._new(out_layout, torch.bfloat16)
        if block is None:
            return out, self._new(lse_layout, torch.float32)
        a = _lib.G4Kv8Args.from_buffer_copy(block)
        self._rows(a, batch, slots, starts, ends)
        a.o = out.data_ptr()
        if chunk:
            return out, self._chunk(a, layer, q, out, slots)
        lse = self._new(lse_layout, torch.float32)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=self.device)
        a.q, a.lse, a.workspace = q.data_ptr(), lse.data_ptr(), ws.data_ptr()
        self._launch(_lib.load().g4_kv8_attn, ctypes.byref(a))
        return out, lse

    def _attention_call(self, key, layer, q, window, max_seqlen_k):
        self._operand(q, None, "q")
        batch, tokens, heads, d = q.shape
        if heads == 0 or heads % self.num_kv_heads:
            raise ValueError(f"{heads} query heads for {self.num_kv_heads} KV heads")
        if window < 0:
            raise ValueError("window must be >= 0")
        max_k = self.capacity if max_seqlen_k is None else int(max_seqlen_k)
        if max_k < 1:
            raise ValueError("max_seqlen_k must be positive")
        a = self._block(layer, batch, tokens)
        # (no position reaches the capacity: a window beyond it is the same, and fits 31 bits)
        a.num_q_heads, a.window = heads, min(int(window), self.capacity)
        a.max_seqlen_k = min(max_k, self.capacity)
        a.q_stride[:] = _strides(q)
        a.o_stride[:] = (heads * tokens * d, heads * d, d)
        if any(s <= 0 or s % 8 for s in a.q_stride):
            raise ValueError("q strides must be positive multiples of 8 elements")
        layouts = _layout(batch, tokens, heads, d), _layout(batch, heads, tokens)
        if not batch or not tokens:
            return self._keep(key, (batch, None, *layouts, 0, False))
        chunk = tokens * (heads // self.num_kv_heads) > DIRECT_COLUMNS[d]
        if chunk:  # LSE as the packed forward writes it: (head, row, token)
            a.lse_stride[:] = (tokens, batch * tokens)
            ws_bytes = 0
        else:
            a.lse_stride[:] = (heads * tokens, tokens)
            a.starts = a.ends = 16  # the size does not depend on the call's pointers
            ws_bytes = _lib.load().g4_kv8_attn_workspace_bytes(ctypes.byref(a))
            a.workspace_bytes = ws_bytes
        return self._keep(key, (batch, bytes(a), *layouts, ws_bytes, chunk))

    def _chunk(self, a, layer, q, out, slots):
        batch, tokens, heads, d = q.shape
        if q.data_ptr() % 16:
            raise ValueError("q must be 16-byte aligned")
        window, max_k = a.window, a.max_seqlen_k
        keys = tokens + (min(max_k, window) if window else max_k) - 1  # most a row can see
        rows = max(1, CHUNK_COPY_BYTES // (4 * keys * self.num_kv_heads * d))
        if batch <= rows:
            return self._chunk_rows(a, layer, q, out, slots, keys)
        lse = self._new(_layout(batch, heads, tokens), torch.float32)
        if slots is None:
            slots = torch.arange(batch, dtype=torch.int32, device=self.device)
        starts, ends = a.starts, a.ends
        rows = -(-batch // -(-batch // rows))  # groups of about one size
        for lo in range(0, batch, rows):
            hi = min(lo + rows, batch)
            a.batch, a.o = hi - lo, out[lo:hi].data_ptr()
            a.slots = slots[lo:hi].data_ptr()
            a.starts, a.ends = starts + 4 * lo, ends + 4 * lo
            a.lse_stride[1] = (hi - lo) * tokens
            lse[lo:hi] = self._chunk_rows(a, layer, q[lo:hi], out[lo:hi], slots[lo:hi], keys)
        return lse

    def _chunk_rows(self, a, layer, q, out, slots, keys):
        batch, tokens, heads, d = q.shape
        total = batch * tokens
        lib = _lib.load()
        plan = torch.empty(5 * batch + 2, dtype=torch.int32, device=self.device)
        cu_q, cu_k = plan[:batch + 1], plan[batch + 1:2 * batch + 2]
        first, last = plan[2 * batch + 2:3 * batch + 2], plan[3 * batch + 2:4 * batch + 2]
        a.holes = plan[4 * batch + 2:].data_ptr()
        self._launch(lib.g4_kv8_chunk_plan, ctypes.byref(a), cu_q.data_ptr(), cu_k.data_ptr(),
                     first.data_ptr(), last.data_ptr())
        k = torch.empty((batch * keys, self.num_kv_heads, d), dtype=torch.bfloat16,
                        device=self.device)
        v = torch.empty_like(k)
        self._read(self._read_block(layer, batch, keys), batch, slots, first, last, k, v, cu_k,
                   a.holes)
        with torch.cuda.device(self.device):
            _, lse = ops.attn_fwd(q.reshape(total, heads, d), k, v, window=a.window,
                                  cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=tokens,
                                  max_seqlen_k=keys, out=out.view(total, heads, d))
        a.q, a.lse = q.data_ptr(), lse.data_ptr()
        self._launch(lib.g4_kv8_pad_rows, ctypes.byref(a))  # and rows with missing pages
        return lse.view(heads, batch, tokens).transpose(0, 1)

    # ----------------------------------------------------------------------------
    # pages
    # ----------------------------------------------------------------------------
    def extend(self, slots: torch.Tensor, counts):
        """Reserve pages for ``counts`` (int32 per row, or one int) more tokens of each
        slot and advance its length.  Returns ``(starts, ends)``, the new tokens'
        positions; a row that does not fit (its table is full, the pool has too few
        pages left by the rows before it, its slot is bad or listed before, or its new
        tokens would go into a page that it shares) is left as it was with start = end."""
        batch = self._page_rows(slots, "slots")
        if isinstance(counts, int):
            counts = torch.full((batch,), counts, dtype=torch.int32, device=self.device)
        self._ints(counts, batch, "counts")
        starts = torch.empty(batch, dtype=torch.int32, device=self.device)
        ends = torch.empty_like(starts)
        if batch:
            a, _ = self._pages(batch, slots)
            a.counts, a.starts, a.ends = counts.data_ptr(), starts.data_ptr(), ends.data_ptr()
            self._launch(_lib.load().g4_pages_extend, ctypes.byref(a))
        return starts, ends

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Make each child (an empty slot without pages) a copy of its parent: whole pages are
        shared, a partly filled last page is copied in every layer."""
        batch = self._page_rows(parents, "parents")
        self._ints(children, batch, "children")
        if batch:
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
        self._free(slots, min(int(window), self.capacity))

    def _free(self, slots, window) -> None:
        batch = self._page_rows(slots, "slots")
        if batch:
            a, _ = self._pages(batch, slots)
            a.window = window
            self._launch(_lib.load().g4_pages_free, ctypes.byref(a))

    def compact(self) -> None:
        """Move the live pages to the lowest ids, so that the pool's end is free."""
        a, _ws = self._pages(0, workspace=True)
        self._launch(_lib.load().g4_pages_compact, ctypes.byref(a))

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copy page ``src[i]`` to page ``dst[i]`` in every layer, with its scales;
        tables and refcounts stay.  A pair with a bad id, with a destination that an
        earlier pair has too, or whose destination is any pair's source is left out."""
        batch = self._ints(src, None, "src").shape[0]
        self._ints(dst, batch, "dst")
        if batch:
            a, _ = self._pages(batch, src, dst)
            self._launch(_lib.load().g4_pages_copy, ctypes.byref(a))

    def _page_rows(self, t: torch.Tensor, name: str) -> int:
        batch = self._ints(t, None, name).shape[0]
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
                (_lib.G4_PAGES_EXHAUSTED, "too few free pages were left"),
                (_lib.G4_PAGES_ROW_FULL, "a slot's table was full"),
                (_lib.G4_PAGES_BAD_INDEX, "a slot, page or count was out of range or listed twice"),
                (_lib.G4_KV8_DEVICE_WAIT, "a kernel's bounded wait expired (invalid results)"),
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
