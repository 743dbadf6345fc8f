"""A 4-bit paged KV cache for batched decode: the pages of every layer, and which row holds which.

`ops.kv4_*` are the operators; this keeps their buffers together for a server or a decoder:

    cache = Kv4Cache(n_layers, n_pages, n_kv_heads, head_dim, batch, max_pages)
    cache.reserve(prompt_lens)                       # pages for every row's next tokens
    for l in range(n_layers): cache.append(l, k, v, pos, cu=cu)       # prompts, ragged
    cache.advance(prompt_lens)
    ...
    cache.reserve(1)                                 # a decode step: one more token a row in use
    pos = cache.positions()                          # -1 for the others
    for l in ...: cache.append(l, k, v, pos); out = cache.decode(l, q, pos, n_q_heads=40)
    cache.advance(1)
    cache.reorder(parent)                            # beams, rows that ended (-1)
    cache.reserve(new)                               # a request into a row that ended: its prompt's
                                                     # length there, 0 for the others

A value takes 4.5 bits (codes of 4 bits, a bf16 step and least value per token, kv head and
64 dims) where the dense cache of `ops.gqa_decode` takes 16.  Rows share full pages; the table
and its counts live on the device and nothing here waits for it: `info` of the last reorder or
compact can be read when a host wants to know what is free.  A row that a reorder emptied, or
that a new cache's first reserve gave no page, is not in use until pages are reserved for it: it
takes no page and no token of reserve(1) and advance(1), and attends to nothing.  The buffers
stay where they are, so a captured step sees what later calls put into them.  No reference
counterpart (the reference keeps one sequence's K and V in bf16,
designs/granite_gemv/granite_attention.h:80-213)."""

from __future__ import annotations

import torch

from . import ops


class Kv4Cache:
    """Pages, page table, lengths and page counts; see the module's text for a run of calls."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, batch: int, max_pages: int,
                 page: int = 64, device=None, summaries: bool = False):
        """page: tokens of a page, a multiple of 16.  summaries: keep the least and the largest
        key of every page per dim (4 bytes a kv head and dim), for decode's n_sel."""
        if min(n_layers, n_pages, n_kv_heads, batch, max_pages) < 1:
            raise ValueError("every size of a cache is 1 or more")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.page, self.head_dim, self.n_kv_heads, self.batch, self.max_pages = (page, head_dim, n_kv_heads, batch,
                                                                                 max_pages)
        nbytes = ops.kv4_page_bytes(page, head_dim)
        self.pool = torch.zeros(n_layers, n_pages, n_kv_heads, nbytes, dtype=torch.uint8, device=dev)
        self.summary = (torch.zeros(n_layers, n_pages, n_kv_heads, 2, head_dim, dtype=torch.bfloat16, device=dev)
                        if summaries else None)
        i32 = dict(dtype=torch.int32, device=dev)
        # info, counts, lengths and table after one another, as a reorder writes them
        self._state = torch.zeros(4 + n_pages + batch + batch * max_pages, **i32)
        self.info, self.refs, self.lens, table = self._state.split((4, n_pages, batch, batch * max_pages))
        self.table = table.view(batch, max_pages).fill_(-1)
        # 1 for a row in use; one more entry, 0, for those that go on with no row.  All are until the
        # first pages are given out: by a tensor, to the rows that begin with them
        self._use = torch.ones(batch + 1, **i32)
        self._use[batch] = 0
        self.used = self._use[:batch]
        self._fresh = True
        self._same = torch.arange(batch, **i32)
        self._layers = list(self.pool.unbind(0))
        self._near = list(self.summary.unbind(0)) if summaries else [None] * n_layers

    def bytes_per_token(self) -> int:
        """Bytes of one token's K and V in one layer."""
        return self.n_kv_heads * self.head_dim * 9 // 8

    def reorder(self, parent: torch.Tensor, reserve: torch.Tensor | None = None) -> torch.Tensor:
        """Row b goes on with the tokens of row parent[b] (-1: with none), and has pages for
        reserve[b] more (ops.kv4_reorder).  The row is in use if row parent[b] was, or if
        reserve[b] is above 0.  Returns info: free pages left, pages copied, pages missing, 0."""
        self._rows(parent, reserve)
        self.used.copy_(self._use[parent.clamp(-1, self.batch)])  # -1 and batch: the entry that is 0
        if reserve is not None:
            self._begin(reserve)
        self._fresh = False
        return self.info

    def _begin(self, tokens: torch.Tensor) -> None:
        if self._fresh and not torch.cuda.is_current_stream_capturing():
            self.used.copy_(tokens > 0)
        else:
            self.used.logical_or_(tokens > 0)

    def _rows(self, parent: torch.Tensor, reserve: torch.Tensor | None) -> None:
        anew, at = ops._kv4_reorder(self.pool, self.table, self.lens, self.refs, parent, self.head_dim, reserve,
                                    self.summary)
        self._state.copy_(anew[at:])

    def reserve(self, tokens: int | torch.Tensor) -> torch.Tensor:
        """Pages for that many tokens behind those that a row has: int32 [batch] (a row with more
        than 0 is in use from then on; where this is a new cache's first call, the others are
        not), or one number for every row in use (of a new cache: every row)."""
        if isinstance(tokens, torch.Tensor):
            self._rows(self._same, tokens)
            self._begin(tokens)
        else:
            self._rows(self._same, self.used * int(tokens))
        self._fresh = False
        return self.info

    def positions(self) -> torch.Tensor:
        """Where every row's next token goes: int32 [batch], -1 for a row that is not in use."""
        return torch.addcmul(self.used - 1, self.lens, self.used)

    def compact(self) -> torch.Tensor:
        """Live pages to the lowest numbers (ops.kv4_compact).  Returns info: live pages, pages moved, 0, 0."""
        table, refs, info = ops.kv4_compact(self.pool, self.table, self.refs, summary=self.summary)
        self.table.copy_(table)
        self.refs.copy_(refs)
        self.info.copy_(info)
        return self.info

    def advance(self, tokens: int | torch.Tensor) -> None:
        """The rows have that many more tokens, what has been appended to every layer (int32
        [batch], or one number for every row in use)."""
        if isinstance(tokens, torch.Tensor):
            self.lens.add_(tokens)
        else:
            self.lens.add_(self.used, alpha=int(tokens))

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, *,
               cu: torch.Tensor | None = None, theta: float | None = 10000.0) -> None:
        """New rows of one layer at positions pos (ops.kv4_append)."""
        ops.kv4_append(k, v, self._layers[layer], self.table, pos, n_kv_heads=self.n_kv_heads,
                       head_dim=self.head_dim, cu=cu, theta=theta, summary=self._near[layer])

    def gather(self, layer: int, pos: torch.Tensor, rows: int, *, cu: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows of one layer read back (ops.kv4_gather)."""
        return ops.kv4_gather(self._layers[layer], self.table, pos, rows, n_kv_heads=self.n_kv_heads,
                              head_dim=self.head_dim, cu=cu, dtype=dtype)

    def decode(self, layer: int, q: torch.Tensor, pos: torch.Tensor, *, n_q_heads: int, theta: float | None = 10000.0,
               scale: float | None = None, n_sel: int | None = None, max_len: int | None = None,
               **kw) -> torch.Tensor:
        """Attention of one query per row over tokens 0..pos (ops.kv4_decode), or over the n_sel
        pages that ops.kv4_select picks for it (a cache with summaries).  max_len, out, out_f32
        and workspace as ops.kv4_decode takes them."""
        heads = dict(n_q_heads=n_q_heads, n_kv_heads=self.n_kv_heads, head_dim=self.head_dim, theta=theta)
        select = None
        if n_sel is not None:
            if self.summary is None:
                raise ValueError("n_sel needs a cache with summaries")
            select = ops.kv4_select(q, self._near[layer], self.table, pos, page=self.page,
                                    n_sel=min(n_sel, self.max_pages), max_len=max_len, **heads)
        return ops.kv4_decode(q, self._layers[layer], self.table, pos, scale=scale, select=select, max_len=max_len,
                              **heads, **kw)
