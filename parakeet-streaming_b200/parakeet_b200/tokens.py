"""Paged K/V that grows with its requests, for a text decoder behind the
transcripts.

``PagedKVPool`` (ops.py) holds the encoder's bounded window; a decoder that
checks drafted tokens against a transcript (the greedy path and its
alternatives, a tree of them in one pass) needs every token of a request, and
drops the ones it rejects.  ``TokenKVPool`` is that cache: pages from one free
stack, lengths and page tables on the device, so that a whole step runs without
a host read and can be captured in a CUDA graph::

    step = pool.begin_step(slots, counts, rows, parents)   # pages, slot map, tree masks
    for layer in ...:
        pool.append(layer, k, v, step)
        out = pool.attention(layer, q, step)
    pool.end_step(step, last)                              # keep the path to node last[b]
    pool.truncate(slots, lengths)                          # cut back, or release (0)

Calls on one pool are ordered by the stream they are made on; only ``attention``
calls, and ``append`` and ``attention`` of different layers, may run side by side.
Two steps of the same request are not begun at once, and a step's tables hold until
its requests are truncated or the pool is reset.  A step's block belongs to the
stream that it was begun on, as any tensor does.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import lib
from .ops import DTYPES, _launch, _ptr, _stream


class TokenStep:
    """One step's tables, made by ``TokenKVPool.begin_step`` (device tensors,
    views of one block):

    row_start   int32 [B + 1]  first row of each request
    context     int32 [B]      tokens kept before the step; -1: refused
    row_request int32 [rows]   the row's request, -1 behind the last one
    positions   int32 [rows]   context + depth in the tree
    slot_map    int32 [rows]   page * page_size + row in the page, -1: none
    masks       int64 [rows]   bits of a node's ancestors and itself (trees; else None)
    """

    __slots__ = ("pool", "block", "batch", "rows", "trees", "open", "_at", "_workspace")

    def __init__(self, pool, block, batch, rows, trees, at, workspace):
        self.pool, self.block, self.batch, self.rows, self.trees = pool, block, batch, rows, trees
        self.open = True     # until end_step
        self._at, self._workspace = at, workspace

    def _view(self, which, n):
        return self.block.as_strided((n,), (1,), self._at[which])

    @property
    def row_start(self):
        return self._view(_lib.PK_TOK_ROW_START, self.batch + 1)

    @property
    def context(self):
        return self._view(_lib.PK_TOK_CONTEXT, self.batch)

    @property
    def row_request(self):
        return self._view(_lib.PK_TOK_REQUEST, self.rows)

    @property
    def positions(self):
        return self._view(_lib.PK_TOK_POSITION, self.rows)

    @property
    def slot_map(self):
        return self._view(_lib.PK_TOK_SLOT_MAP, self.rows)

    @property
    def masks(self):
        return self._view(_lib.PK_TOK_MASK, 2 * self.rows).view(torch.int64) if self.trees else None


class TokenKVPool:
    """Paged K/V of ``num_slots`` requests of up to ``max_tokens`` tokens.

    kv          [num_pages, L, 2, Hkv, page_size, dh] dtype (head-major pages)
    page_table  [num_slots, ceil(max_tokens / page_size)] int32, -1 = none
    free_pages  [num_pages]  int32 stack of free page ids, the top at free_count
    free_count  [1]          int32
    lengths     [num_slots]  int32 tokens kept
    held        [num_slots]  int32 pages held
    error       [1]          int32 PK_DEV_* bits

    Query heads are a multiple of the K/V heads; head_dim 64 or 128; bfloat16,
    or float32 (the parity mode)."""

    def __init__(self, num_layers, num_heads, num_kv_heads, head_dim, num_slots, max_tokens, *,
                 num_pages=None, page_size=16, dtype=torch.bfloat16, device="cuda",
                 page_order=None):
        if dtype not in DTYPES:
            raise TypeError(f"dtype {dtype} not handled (float32 or bfloat16)")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("TokenKVPool needs a CUDA device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index
        if max_tokens <= 0 or page_size <= 0 or num_slots <= 0:
            raise ValueError("max_tokens, page_size and num_slots must be positive")
        self.num_layers, self.num_heads, self.num_kv_heads = num_layers, num_heads, num_kv_heads
        self.head_dim, self.num_slots, self.page_size, self.dtype = head_dim, num_slots, page_size, dtype
        self.table_width = -(-max_tokens // page_size)
        self.num_pages = int(num_pages if num_pages is not None else num_slots * self.table_width)
        dev = self.device

        def i32(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device=dev)

        self.kv = torch.zeros((self.num_pages, num_layers, 2, num_kv_heads, page_size, head_dim),
                              dtype=dtype, device=dev)
        self.page_table = i32(num_slots, self.table_width, fill=-1)
        self.free_pages, self.free_count = i32(self.num_pages), i32(1)
        self.lengths, self.held, self.error = i32(num_slots), i32(num_slots), i32(1)
        self._scratch = i32(4 * num_slots + 16)
        d = _lib.TokenKVDesc(
            kv=self.kv.data_ptr(), page_table=self.page_table.data_ptr(),
            free_pages=self.free_pages.data_ptr(), free_count=self.free_count.data_ptr(),
            lengths=self.lengths.data_ptr(), held=self.held.data_ptr(),
            scratch=self._scratch.data_ptr(), error=self.error.data_ptr(),
            num_pages=self.num_pages, num_slots=num_slots, num_layers=num_layers,
            num_heads=num_heads, num_kv_heads=num_kv_heads, head_dim=head_dim,
            page_size=page_size, table_width=self.table_width, dtype=DTYPES[dtype])
        h = ctypes.c_void_p()
        self._lib = lib()
        _launch(dev, self._lib.pk_token_kv_create, ctypes.byref(d), ctypes.byref(h))
        self._h = h
        # (batch, rows, trees): a step block's words and offsets, attention's workspace
        self._sizes: dict = {}
        self.reset(page_order)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                lib().pk_token_kv_destroy(h)
            except Exception:
                pass
            self._h = None

    # ------------------------------------------------------------ checks
    def _i32(self, t, n, name):
        """The length of an int32 vector, which has to be ``n`` where given."""
        if t.dtype is not torch.int32 or t.get_device() != self._index:
            raise TypeError(f"{name}: expected int32 on {self.device}, got {t.dtype} on {t.device}")
        if t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name}: expected a contiguous [{'n' if n is None else n}] tensor, "
                             f"got {tuple(t.shape)}")
        return t.shape[0]

    def _step(self, step, ending=False):
        if step.pool is not self:
            raise ValueError("the step belongs to another pool")
        if not step.open:
            raise ValueError("the step has been ended")
        if ending:
            step.open = False

    def _rows(self, t, heads, rows, name):
        """Leading dimensions and strides of t, [..., rows, heads, head_dim] or
        [..., rows, heads * head_dim]: (leading, all strides, row stride, head stride)."""
        if t.dtype is not self.dtype or t.get_device() != self._index:
            raise TypeError(f"{name}: expected {self.dtype} on {self.device}, got {t.dtype} on {t.device}")
        shape, strides, dh = t.shape, t.stride(), self.head_dim
        n = len(shape)
        if n >= 3 and shape[-1] == dh and shape[-2] == heads and shape[-3] == rows:
            rs, hs, column = strides[-3:]
            n -= 3
        elif n >= 2 and shape[-1] == heads * dh and shape[-2] == rows:
            rs, column = strides[-2:]
            hs = dh
            n -= 2
        else:
            raise ValueError(f"{name}: expected [..., {rows}, {heads}, {dh}] or [..., {rows}, "
                             f"{heads * dh}], got {tuple(shape)}")
        if column != 1:
            raise ValueError(f"{name}: last dimension must be contiguous")
        return n, strides, rs, hs

    # ------------------------------------------------------------ allocator
    def reset(self, page_order=None):
        """Every request empty, every page free; pages are taken from the end of
        ``page_order`` (default 0 .. num_pages - 1), which lists every page once (looked
        at where it is on the host; a device tensor's values are taken as they are)."""
        order = None
        if page_order is not None:
            order = torch.as_tensor(page_order, dtype=torch.int32)
            if order.numel() != self.num_pages or not order.is_cuda and not torch.equal(
                    order.flatten().sort().values, torch.arange(self.num_pages, dtype=torch.int32)):
                raise ValueError("page_order must list every page once")
            order = order.to(self.device).contiguous()
        self._order = order
        _launch(self.device, self._lib.pk_token_reset, self._h, _ptr(order), _stream(self.device))

    def begin_step(self, slots: torch.Tensor, counts: torch.Tensor, rows: int,
                   parents: torch.Tensor | None = None) -> TokenStep:
        """Pages and tables for ``counts[b]`` new tokens of each request
        ``slots[b]`` (int32 [B], distinct), packed in this order into ``rows``
        rows (at least their sum; rows behind it belong to nobody).  ``parents``
        (int32 [rows]): each token's parent node inside its request, below its
        own index, -1 for the context - a tree of at most 64 tokens; without it
        each token follows the one before, any number of them.

        A request that cannot be served (a slot out of range or named twice, a
        count out of range, no room or no pages left) sets its bit of ``error``
        and is left out: context -1, its rows not appended nor attended.  Pages go out
        in batch order and nobody overtakes: behind a request that finds too few, the
        later ones that need any are left out too, even where enough for them are left
        (those that need none are served)."""
        B = self._i32(slots, None, "slots")
        self._i32(counts, B, "counts")
        trees = parents is not None
        if trees:
            self._i32(parents, rows, "parents")
        key = (B, rows, trees)
        size = self._sizes.get(key)
        if size is None:
            at = (ctypes.c_int64 * _lib.PK_TOK_OFFSETS)()
            words = self._lib.pk_token_step_words(self._h, B, rows, trees, at)
            if words < 0:
                raise ValueError(f"rows must not be negative, got {rows}")
            if len(self._sizes) >= 64:
                self._sizes.clear()
            size = self._sizes[key] = (words, tuple(at),
                                       self._lib.pk_token_attention_workspace(self._h, B, rows))
        dev = self.device
        block = slots.new_empty(size[0])
        _launch(dev, self._lib.pk_token_begin_step, self._h, slots.data_ptr(), counts.data_ptr(), B,
                parents.data_ptr() if trees else None, rows, block.data_ptr(), _stream(dev))
        step = TokenStep(self, block, B, rows, trees, size[1], size[2])
        if B == 0:   # nothing was launched
            block.zero_()
            step.row_request.fill_(-1)
            step.slot_map.fill_(-1)
        return step

    def end_step(self, step: TokenStep, last: torch.Tensor):
        """Keep of each request the path to its node ``last[b]`` (int32 [B]; -1:
        nothing; a chain's ``n - 1``: all): its K/V rows are moved behind the
        context in every layer and ``lengths`` grows by them.  Pages stay with
        the request.  A request that gave pages of the step back since it began
        (``truncate``, ``reset``) keeps nothing of it and sets PK_DEV_BAD_COUNT."""
        self._i32(last, step.batch, "last")
        self._step(step, ending=True)
        _launch(self.device, self._lib.pk_token_end_step, self._h, last.data_ptr(), step.batch,
                step.rows, step.trees, step.block.data_ptr(), _stream(self.device))

    def truncate(self, slots: torch.Tensor, lengths: torch.Tensor):
        """Cut requests to ``lengths[b]`` tokens (0 releases them); the pages
        past the end go back on the stack."""
        n = self._i32(slots, None, "slots")
        self._i32(lengths, n, "lengths")
        _launch(self.device, self._lib.pk_token_truncate, self._h, slots.data_ptr(),
                lengths.data_ptr(), n, _stream(self.device))

    def read_error(self) -> int:
        return int(self.error.item())

    # ------------------------------------------------------------ data path
    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, step: TokenStep):
        """key/value [rows, Hkv, dh] (or [rows, Hkv * dh]) of one layer, or
        [nl, rows, ...] of layers layer .. layer + nl - 1, with any row and head
        strides (slices of a fused projection)."""
        self._step(step)
        leading, strides, rs, hs = self._rows(key, self.num_kv_heads, step.rows, "key")
        if leading > 1 or self._rows(value, self.num_kv_heads, step.rows, "value")[1] != strides or \
                value.shape != key.shape:
            raise ValueError("key and value must have the same shape and strides")
        nl, ls = (key.shape[0], strides[0]) if leading else (1, 0)
        _launch(self.device, self._lib.pk_token_append, self._h, layer, nl, key.data_ptr(),
                value.data_ptr(), ls, rs, hs, step.batch, step.rows, step.trees,
                step.block.data_ptr(), _stream(self.device))

    def attention(self, layer: int, query: torch.Tensor, step: TokenStep,
                  scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the step's rows over their request's context and, of the
        step's own tokens, their ancestors and themselves (without ``parents``:
        the rows before and themselves).  query [rows, H, dh] (or [rows, H * dh]);
        ``scale`` defaults to dh ** -0.5; returns ``out`` in the query's shape (it may
        be the query itself).
        Rows of no request, and of refused ones, are left as they were.

        Sums are float32.  A bfloat16 pool's weights are rounded to bfloat16 for the
        product with the values, as the tensor cores take them: off by 2^-8 of each term
        at most, beside the result's own rounding.  A float32 pool rounds neither."""
        self._step(step)
        leading, _, qrs, qhs = self._rows(query, self.num_heads, step.rows, "query")
        if leading:
            raise ValueError(f"query: one layer's rows, got {tuple(query.shape)}")
        if out is None:
            out = query.new_empty(query.shape)
            ors, ohs = self.num_heads * self.head_dim, self.head_dim
        elif out.shape != query.shape:
            raise ValueError(f"out: expected {tuple(query.shape)}, got {tuple(out.shape)}")
        else:
            _, _, ors, ohs = self._rows(out, self.num_heads, step.rows, "out")
        # a buffer of this call's own (the step's layers may run side by side), held until
        # both of its launches are made: another thread's call may be between them
        dev, need = self.device, step._workspace
        ws = step.block.new_empty(need // 4) if need else None
        _launch(dev, self._lib.pk_token_attention, self._h, layer, query.data_ptr(), qrs, qhs,
                self.head_dim ** -0.5 if scale is None else scale, step.batch, step.rows, step.trees,
                step.block.data_ptr(), out.data_ptr(), ors, ohs, _ptr(ws), _stream(dev))
        return out


__all__ = ["TokenKVPool", "TokenStep"]
