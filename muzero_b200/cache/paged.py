"""Paged quantized KV cache: sequences of unlike lengths in one cache, pages that sequences share, 4-bit codes.

``MuZeroPagedCache`` holds all layers of a model.  A sequence is a *row*; its newest ``residual_length`` to ``residual_length + 63`` tokens stand in
16 bits in the row's ring, its older ones in pages of 64 tokens, which a block table lists and which rows share by reference count.  Lengths,
table and counts live on the device, so a step needs no host round trip and can be captured in a CUDA graph:

    cache = MuZeroPagedCache.allocate(layers=36, kv_heads=8, head_dim=128, pages=4096, rows=64, max_length=32768)
    cache.extend(rows=rows, offsets=offsets)                    # once per step: pages for the new tokens
    cache.append(layer, key, value, rows=rows, offsets=offsets) # per layer: quantizes what leaves the 16-bit window
    out = cache.attend(layer, query, rows=rows)                 # per layer
    cache.fork(parents, children); cache.free(ended); cache.compact()
    cache.check()                                               # raises what only the device could see (synchronises)

The codes are those of the zero-anchored log compander with alpha 2, its levels rounded to 127ths of a row's range (``include/muzero_b200.h`` has the
page's layout).  The contiguous ``MuZeroCache`` keeps the reference's codes bit for bit; these are its paged counterpart's own, with an
error 1.3 % larger on normally distributed values, and their attention runs without a book of values per row.

The reference has no paged store (its layer cache is muzero/cache/layer.py:39-217, one length for all batch entries).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ..kernels._cabi import (MuZeroKernelError, PagedAttentionArgs, PagedCache, check, dtype_code, load_library, on_device, stream_ptr)

PAGE_TOKENS = 64
_STATUS = {1: "the pool has too few free pages", 2: "a sequence outgrew its row of the block table", 4: "a row or page index is outside the cache"}
_ERRORS = sum(_STATUS)                               # the fourth bit says that the newest extension was refused; the device sets and clears it


def page_bytes(head_dim: int) -> int:
    """Bytes of a page per kv head: codes of 64 tokens' keys and values, and a 32-bit word per row of 64 codes."""
    return 72 * head_dim


def packed_tokens(length: int, residual_length: int) -> int:
    """Tokens of a sequence of this length that stand in pages."""
    return max(0, (length - residual_length) // PAGE_TOKENS) * PAGE_TOKENS


def _index(t: Optional[torch.Tensor], what: str, device: torch.device, n: Optional[int] = None) -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.dim() != 1 or t.device != device or not t.is_contiguous():
        raise ValueError(f"`{what}` must be a contiguous int32 vector on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"`{what}` has {t.shape[0]} entries, expected {n}")
    return t.data_ptr()


class MuZeroPagedCache:
    """The tensors of a paged cache and the calls on them.

    store        uint8 [layers, pages, kv_heads, page_bytes]
    tail         bf16 or fp16 [layers, rows, 2, kv_heads, ring, head_dim]: the rows' rings, token t at place t % ring
    block_table  int32 [rows, width], lengths int32 [rows], page_refs int32 [pages], status int32 [1]

    ``allocate`` makes them; the constructor takes them as they are.  All calls run on the current stream of the cache's device.
    """

    def __init__(self, *, store: torch.Tensor, tail: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, page_refs: torch.Tensor,
                 status: torch.Tensor, residual_length: int = 128):
        if store.dim() != 4 or tail.dim() != 6 or block_table.dim() != 2:
            raise ValueError("`store` is [layers, pages, kv_heads, bytes], `tail` [layers, rows, 2, kv_heads, ring, head_dim], `block_table` [rows, width]")
        for t in (store, tail, block_table, lengths, page_refs, status):
            if not t.is_cuda or t.device != store.device:
                raise MuZeroKernelError("a paged cache lives on one CUDA device; this package has no CPU path")
        layers, pages, kv_heads, pb = store.shape
        _, rows, _, _, ring, head_dim = tail.shape
        problems = []
        if store.dtype != torch.uint8:
            problems.append(f"`store` must be uint8, got {store.dtype}")
        if tail.dtype not in (torch.bfloat16, torch.float16):
            problems.append(f"`tail` must be bfloat16 or float16, got {tail.dtype}")
        if head_dim not in (64, 128):
            problems.append(f"head_dim must be 64 or 128, got {head_dim}")
        if pb != page_bytes(head_dim):
            problems.append(f"a page of head_dim {head_dim} has {page_bytes(head_dim)} bytes per kv head, got {pb}")
        if tuple(tail.shape[:4]) != (layers, rows, 2, kv_heads):
            problems.append(f"`tail` {tuple(tail.shape)} does not fit `store` {tuple(store.shape)}")
        if residual_length < 0 or residual_length % PAGE_TOKENS:
            problems.append(f"`residual_length` must be a multiple of {PAGE_TOKENS}, got {residual_length}")
        if ring < residual_length + PAGE_TOKENS:
            problems.append(f"a ring needs at least residual_length + {PAGE_TOKENS} places, got {ring}")
        if block_table.shape[0] != rows:
            problems.append(f"`block_table` has {block_table.shape[0]} rows, `tail` {rows}")
        for name, t, n in (("lengths", lengths, rows), ("page_refs", page_refs, pages), ("status", status, 1)):
            if tuple(t.shape) != (n,):
                problems.append(f"`{name}` must have {n} entries, got {tuple(t.shape)}")
        for name, t in (("block_table", block_table), ("lengths", lengths), ("page_refs", page_refs), ("status", status)):
            if t.dtype != torch.int32 or not t.is_contiguous():
                problems.append(f"`{name}` must be contiguous int32")
        if store.stride(3) != 1 or store.stride(2) != pb or tail.stride()[2:] != (kv_heads * ring * head_dim, ring * head_dim, head_dim, 1):
            problems.append("a page and a row's ring must be contiguous")
        if (store.data_ptr() | store.stride(0) | store.stride(1)) & 31 or tail.data_ptr() & 15 or (tail.stride(0) | tail.stride(1)) & 7:
            problems.append("pages must begin on 32-byte boundaries, rings on 16-byte boundaries")
        if problems:
            raise ValueError("; ".join(problems))
        self.store, self.tail, self.block_table, self.lengths, self.page_refs, self.status = store, tail, block_table, lengths, page_refs, status
        self.residual_length = residual_length
        self.layers, self.pages, self.kv_heads, self.rows, self.head_dim, self.dtype = layers, pages, kv_heads, rows, head_dim, tail.dtype
        self.device = store.device
        self._lib = load_library()
        check(on_device(self.device, self._lib.mz_paged_prepare), "mz_paged_prepare")      # so that a first call may stand in a captured graph
        self._c = PagedCache(layers, rows, pages, block_table.shape[1], kv_heads, head_dim, residual_length, ring, dtype_code(tail.dtype),
                             store.data_ptr(), store.stride(0), store.stride(1), tail.data_ptr(), tail.stride(0), tail.stride(1),
                             block_table.data_ptr(), lengths.data_ptr(), page_refs.data_ptr(), status.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._workspaces: dict = {}
        self._needs: dict = {}

    @classmethod
    def allocate(cls, *, layers: int, kv_heads: int, head_dim: int, pages: int, rows: int, max_length: int, residual_length: int = 128,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "MuZeroPagedCache":
        """An empty cache: ``pages`` pages of 64 tokens for all layers, ``rows`` sequences of at most ``max_length`` tokens."""
        ring = residual_length + 2 * PAGE_TOKENS          # two pages of slack: a short block of new tokens never meets one still to be quantized
        width = max(1, -(-max(0, max_length - residual_length) // PAGE_TOKENS))
        return cls(store=torch.zeros((layers, pages, kv_heads, page_bytes(head_dim)), dtype=torch.uint8, device=device),
                   tail=torch.zeros((layers, rows, 2, kv_heads, ring, head_dim), dtype=dtype, device=device),
                   block_table=torch.full((rows, width), -1, dtype=torch.int32, device=device),
                   lengths=torch.zeros(rows, dtype=torch.int32, device=device), page_refs=torch.zeros(pages, dtype=torch.int32, device=device),
                   status=torch.zeros(1, dtype=torch.int32, device=device), residual_length=residual_length)

    # ---- a step's tokens
    def _entries(self, rows, offsets) -> int:
        if rows is not None:
            return rows.shape[0]
        return self.rows if offsets is None else offsets.shape[0] - 1

    def extend(self, *, rows: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None) -> None:
        """Announces new tokens: entry i brings ``offsets[i+1] - offsets[i]`` of them (one each without ``offsets``) for row ``rows[i]`` (row i without
        ``rows``).  Lengths grow and the pages that they need are taken, for all layers at once, or nothing changes and ``check`` raises.  After
        an extension that was refused ``append`` writes nothing, until another one succeeds.  The rows of a call are distinct."""
        n = self._entries(rows, offsets)
        r, o = _index(rows, "rows", self.device), _index(offsets, "offsets", self.device, n + 1)
        check(on_device(self.device, self._lib.mz_paged_extend, self._ref, r, o, n, stream_ptr(self.device)), "mz_paged_extend")

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, *, rows: Optional[torch.Tensor] = None,
               offsets: Optional[torch.Tensor] = None, max_new: Optional[int] = None) -> None:
        """Writes the announced tokens of one layer: ``key`` and ``value`` [tokens, kv_heads, head_dim], entry after entry.  ``max_new``: the most
        tokens that an entry brings, if the host knows it.  Without it all might be one entry's, and the grid grows with entries times tokens: 64 prompts of 1000 tokens take
        943 instead of 138 us, 16 of 1777 150 instead of 71, one of 4096 the same 28 (8 kv heads, head_dim 128)."""
        n = self._entries(rows, offsets)
        r, o = _index(rows, "rows", self.device), _index(offsets, "offsets", self.device, n + 1)
        shape = (key.shape[0], self.kv_heads, self.head_dim)
        tensors = []
        for name, t in (("key", key), ("value", value)):
            if t.dtype != self.dtype or t.device != self.device or tuple(t.shape) != shape:
                raise ValueError(f"`{name}` must be {self.dtype} {shape} on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
            # rows of whole 16-byte pieces; anything else is laid out once
            tensors.append(t if t.stride(2) == 1 and not (t.stride(0) | t.stride(1)) & 7 and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format))
        k, v = tensors
        if offsets is None and shape[0] != n:
            raise ValueError(f"{shape[0]} tokens for {n} rows: without `offsets` each row brings one")
        if max_new is None:
            max_new = 1 if offsets is None else shape[0]
        check(on_device(self.device, self._lib.mz_paged_append, self._ref, layer, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                        v.stride(1), r, o, n, shape[0], max_new, stream_ptr(self.device)), "mz_paged_append")

    def _workspace(self, nbytes: int, stream: int) -> tuple:
        # One per stream, grown by replacement.  An outgrown one is kept, as a captured graph may hold its address; one that has to grow at least
        # doubles, so that its predecessors are smaller than it all together
        held = self._workspaces.get(stream)
        if held is None or held[-1][1] < nbytes:
            size = max(nbytes, 1 << 20, 2 * held[-1][1] if held else 0)
            t = torch.empty(size, dtype=torch.uint8, device=self.device)
            held = self._workspaces.setdefault(stream, [])
            held.append((t.data_ptr(), size, t))
        return held[-1]

    def attend(self, layer: int, query: torch.Tensor, *, rows: Optional[torch.Tensor] = None, scaling: Optional[float] = None,
               out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Attention of the rows' newest tokens, already appended: ``query`` [batch, q_len, q_heads, head_dim] or [batch, q_heads, head_dim] (one
        token), query l of a row being its (length - q_len + l)-th token.  Each sees the tokens up to its own.  Returns the query's shape."""
        q = query if query.dim() == 4 else query.unsqueeze(1)
        if q.dim() != 4 or q.shape[3] != self.head_dim or q.dtype != self.dtype or q.device != self.device:
            raise ValueError(f"`query` must be {self.dtype} [batch, (q_len,) q_heads, {self.head_dim}] on {self.device}, got {query.dtype} "
                             f"{tuple(query.shape)} on {query.device}")
        # rows of whole 16-byte pieces; anything else is laid out once
        if q.stride(3) != 1 or (q.stride(0) | q.stride(1) | q.stride(2)) & 7 or q.data_ptr() & 15:
            q = q.clone(memory_format=torch.contiguous_format)
        b, lq, hq, _ = q.shape
        if out is None:
            out = query.new_empty(query.shape) if out_dtype is None else torch.empty(query.shape, dtype=out_dtype, device=self.device)
        elif out.shape != query.shape or not out.is_contiguous() or out.device != self.device or (out_dtype or out.dtype) != out.dtype:
            raise ValueError("`out` must be a contiguous tensor of the query's shape on the cache's device")
        st = stream_ptr(self.device)
        need = self._needs.get((b, lq, hq))
        if need is None:                                  # 0: a shape that the call below refuses with its reason
            need = self._needs[b, lq, hq] = on_device(self.device, self._lib.mz_paged_attention_workspace_bytes, self._ref, b, lq, hq)
        ws = self._workspace(need, st)
        # a block per call: another thread may attend another layer meanwhile
        a = PagedAttentionArgs(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), b, lq, hq, _index(rows, "rows", self.device, b),
                               self.head_dim ** -0.5 if scaling is None else scaling, out.data_ptr(), dtype_code(out.dtype), ws[0], ws[1])
        check(on_device(self.device, self._lib.mz_paged_attention, self._ref, layer, ctypes.byref(a), st), "mz_paged_attention")
        return out

    # ---- rows and pages
    def fork(self, source: torch.Tensor, target: torch.Tensor) -> None:
        """Row ``target[i]`` becomes a copy of row ``source[i]`` in all layers: pages are shared, the ring is copied, what the target held is released.
        Targets are distinct, and none is a source."""
        n = target.shape[0]
        check(on_device(self.device, self._lib.mz_paged_fork, self._ref, _index(source, "source", self.device, n),
                        _index(target, "target", self.device), n, stream_ptr(self.device)), "mz_paged_fork")

    def free(self, rows: torch.Tensor) -> None:
        """Empties rows; pages that no other row holds are free again."""
        check(on_device(self.device, self._lib.mz_paged_free, self._ref, _index(rows, "rows", self.device), rows.shape[0],
                        stream_ptr(self.device)), "mz_paged_free")

    def compact(self) -> None:
        """Moves the live pages into the lowest places of the pool, so that what lies above them is free in one piece."""
        st = stream_ptr(self.device)
        ws = self._workspace(self._lib.mz_paged_compact_workspace_bytes(self._ref), st)
        check(on_device(self.device, self._lib.mz_paged_compact, self._ref, ws[0], ws[1], st), "mz_paged_compact")

    def copy_pages(self, source: torch.Tensor, target: torch.Tensor) -> None:
        """Copies page ``source[i]`` onto page ``target[i]`` in all layers; tables and counts stay as they are."""
        n = target.shape[0]
        check(on_device(self.device, self._lib.mz_paged_copy_pages, self._ref, _index(source, "source", self.device, n),
                        _index(target, "target", self.device), n, stream_ptr(self.device)), "mz_paged_copy_pages")

    def check(self) -> None:
        """Raises what a call on this cache found wrong on the device since the last check, and forgets it.  Synchronises."""
        seen = int(self.status.item()) & _ERRORS
        if seen:
            self.status.bitwise_and_(~seen)
            raise MuZeroKernelError("paged cache: " + "; ".join(text for bit, text in _STATUS.items() if seen & bit))

    def free_pages(self) -> int:
        """Pages that no row holds.  Synchronises."""
        return int((self.page_refs == 0).sum())
