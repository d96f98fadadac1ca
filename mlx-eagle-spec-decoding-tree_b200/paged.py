"""A KV cache in pages, with a prefix that requests share: append and attention for a pass of several requests.

``BatchKVCache`` gives every request a slab as long as its longest possible text, and a system prompt is held and read once per request.  Here
a request's rows lie in pages taken from one pool as it grows, and the rows of a common prefix are held, and read in a pass, once for all.

A pass holds, for each of ``B`` requests, any number of new tokens behind one another: ``row_starts (B + 1,)`` int32 gives where each
request's begin (tokens from ``row_starts[B]`` on are padding and left alone).  ``lengths (B,)`` int32 counts the rows of each request's own pages,
the pass's own included; row ``r`` of request ``b`` is row ``r % page_size`` of page ``page_table[b, r // page_size]``.  Everything a step changes is
read on the device, so a pass can be captured once and replayed:

    cache = PagedKVCache(layers, pages, page_size, kv_heads, head_dim, device=device)
    for layer in range(layers):
        q, k, v = projections ...
        q = append(q, k, v, *cache.layer(layer), page_table, lengths, row_starts, inv_freqs, prefix_length=P)
        o = attention(q, *cache.layer(layer), page_table, lengths, row_starts, prefix_pages=prefix_pages, prefix_length=P)
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib, rope

_errors: dict = {}


class PagedKVCache:
    """Pages of every layer in one allocation ``[layers][2][pages][kv_heads][page_size][head_dim]``.  Which page belongs to whom is the
    caller's: pages come from ``take`` and go back with ``give`` (host lists; no page is cleared, rows behind a length are never read)."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.float16, device="cuda"):
        _check_page_size(page_size)
        if dtype not in (torch.float16, torch.bfloat16):
            raise _lib.B200Error("a paged cache holds float16 or bfloat16")
        self.pages, self.page_size = int(pages), int(page_size)
        self.data = torch.zeros(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self._free = list(range(self.pages - 1, -1, -1))
        self._out: set = set()

    def layer(self, i):
        return self.data[i, 0], self.data[i, 1]

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self, rows: int) -> list:
        """Pages for ``rows`` more rows."""
        need = (int(rows) + self.page_size - 1) // self.page_size
        if need > len(self._free):
            raise _lib.B200Error(f"{need} pages wanted, {len(self._free)} free")
        got = [self._free.pop() for _ in range(need)]
        self._out.update(got)
        return got

    def give(self, pages) -> None:
        pages = [int(p) for p in pages]
        if len(set(pages)) != len(pages) or not self._out.issuperset(pages):
            raise _lib.B200Error("only pages that were taken, each once, can be given back")
        self._out.difference_update(pages)
        self._free.extend(pages)


def _check_page_size(n: int) -> None:
    if not (n in (8, 16, 32, 64) or (n >= 128 and n % 128 == 0)):
        raise _lib.B200Error(f"a page must hold 8, 16, 32, 64 or a multiple of 128 rows, not {n}")


def _paged(q, k_pages, v_pages, page_table, lengths, row_starts) -> _lib.Paged:
    """The descriptor of a pass, its tensors looked over."""
    _lib.require_tensor("q", q, (torch.float16, torch.bfloat16), (None, None, None), packed=False)
    _lib.require_tensor("k_pages", k_pages, (q.dtype,), (None, None, None, q.shape[2]), q, packed=False)
    _lib.require_tensor("v_pages", v_pages, (q.dtype,), k_pages.shape, q, packed=False)
    _lib.require_tensor("lengths", lengths, (torch.int32,), (None,), q)
    _lib.require_tensor("row_starts", row_starts, (torch.int32,), (lengths.numel() + 1,), q)
    _lib.require_tensor("page_table", page_table, (torch.int32,), (lengths.numel(), None), q, packed=False)
    if k_pages.stride() != v_pages.stride():
        raise _lib.B200Error("k_pages and v_pages must have the same strides")
    _lib.require_writable("k_pages", k_pages)
    pages, kv_heads, page_size, _ = k_pages.shape
    if pages < 1 or kv_heads < 1 or q.shape[1] < 1 or q.shape[1] % kv_heads or q.shape[1] > 4096:
        raise _lib.B200Error(f"{q.shape[1]} query heads (at most 4096) must be a multiple of the {kv_heads} key heads of at least one page")
    _check_page_size(page_size)
    if max(*q.shape, *k_pages.shape, *page_table.shape) > 0x7fffffff:
        raise _lib.B200Error("sizes must fit 32 bits")
    return _lib.Paged(_lib.DTYPES[q.dtype], lengths.numel(), q.shape[0], q.shape[1], kv_heads, q.shape[2], pages, page_size, page_table.shape[1],
                      _lib.ptr(page_table), page_table.stride(0), _lib.ptr(lengths), _lib.ptr(row_starts), _lib.ptr(k_pages), _lib.ptr(v_pages),
                      *k_pages.stride()[:3])


def append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
           lengths: torch.Tensor, row_starts: torch.Tensor, inv_freqs: torch.Tensor, *, positions: Optional[torch.Tensor] = None,
           prefix_length: int = 0, scaling_factor: float = 1.0, magnitude: float = 1.0, interleaved: bool = False,
           q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keys, rotated, and values of a pass into the pages of their requests, and the rotated queries, in one launch.

    ``q (tokens, heads, dim)``, ``k`` and ``v (tokens, kv_heads, dim)``: float16 or bfloat16, tokens and heads may be strided (slices of a fused
    projection), ``k`` and ``v`` alike (where a norm has made new keys, values are made contiguous too); pages ``(pages, kv_heads, page_size, dim)`` in any
    order of strides.  A token's position is its row behind ``prefix_length`` rows, or ``positions (tokens,)`` says it (a tree of drafted tokens: rows
    side by side, positions by depth); the rotation is ``rope.rotate``'s.  ``q_out`` may be ``q``.  Rows whose page number lies outside the cache, or that
    the table is too short for, are dropped.
    Two requests that write one page's row in the same pass leave either's."""
    if q_out is None:
        y = _lib.ops().paged_append(q, k, v, k_pages, v_pages, page_table, lengths, row_starts, prefix_length, positions, inv_freqs, scaling_factor,
                                    magnitude, interleaved, False)
        if y is not None:
            return y
    c = _paged(q, k_pages, v_pages, page_table, lengths, row_starts)
    _lib.require_tensor("k", k, (q.dtype,), (c.tokens, c.kv_heads, c.head_dim), q, packed=False)
    _lib.require_tensor("v", v, (q.dtype,), k.shape, q, packed=False)
    if k.stride() != v.stride() and k.numel() > 0:
        raise _lib.B200Error("k and v must have the same strides")
    if c.head_dim > 2048 or not 0 <= prefix_length <= 0x7fffffff:
        raise _lib.B200Error("append takes heads of at most 2048 dims and a prefix of 0 to 2^31 - 1 rows")
    r = rope._rotary(positions, inv_freqs, c.head_dim, c.tokens, q, scaling_factor, magnitude, interleaved)
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _lib.require_tensor("q_out", q_out, (q.dtype,), q.shape, q, packed=False)
        _lib.require_writable("q_out", q_out)
    with _lib.on_device(q):
        rc = _lib.lib().b200_paged_append(ctypes.byref(c), ctypes.byref(r), _lib.ptr(q), q.stride(0), q.stride(1), _lib.ptr(k), _lib.ptr(v),
                                          k.stride(0), k.stride(1), _lib.ptr(q_out), q_out.stride(0), q_out.stride(1), int(prefix_length),
                                          _lib.stream_ptr(q.device))
    _lib.check(rc, "b200_paged_append")
    return q_out


def _error_word(device) -> torch.Tensor:
    """One word per device that a wait inside the attention sets when it runs out; never freed, captured passes hold its address."""
    word = _errors.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise _lib.B200Error("the first attention on a device must not be captured: its error word would belong to the graph")
        word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()                  # (other streams set it and read it)
        _errors[device.index] = word
    return word


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
              row_starts: torch.Tensor, *, prefix_pages: Optional[torch.Tensor] = None, prefix_length: int = 0,
              mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale * q K^T) V`` of a pass's tokens over the ``prefix_length`` rows of ``prefix_pages``, read once for all requests, and the rows
    of their own request: causal, or by ``mask (tokens,)`` int64, whose bit ``j`` says that the token sees its request's ``j``-th new row (the
    older rows are seen by all; new rows from the 64th on are hidden).

    ``q (tokens, heads, dim)``, positions already in it; heads of 64 or 128; float16 or bfloat16, scores, statistics and sums in fp32, probabilities
    rounded to the type for the second product; NaN and infinities reach the tokens that see them, and no other.  ``out`` may be ``q``.  ``scale``, 0 or more, is
    ``dim ** -0.5`` unless given.  A token that sees no row gets zeros; results of tokens outside ``row_starts`` are
    not written (``append`` likewise).  Rows behind a length may hold anything; a page number outside the cache stands for rows of zeros.  At most 1024 requests.
    Rows of ``q``, ``out`` and the pages start at 16 bytes (strides of multiples of 8).  A call takes a workspace of 12 bytes for each value of the result and 39 MB (heads of
    128; 20 MB of 64); the prefix is gone over for all ``tokens``, padding among them."""
    if out is None and isinstance(q, torch.Tensor):
        y = _lib.ops().paged_attention(q, k_pages, v_pages, page_table, lengths, row_starts, prefix_pages, prefix_length, mask, scale,
                                       _errors.get(q.device.index))
        if y is not None:
            return y
    c = _paged(q, k_pages, v_pages, page_table, lengths, row_starts)
    if c.head_dim not in (64, 128):
        raise _lib.B200Error(f"attention takes heads of 64 or 128 dims, not {c.head_dim}")
    if c.requests > 1024:
        raise _lib.B200Error(f"attention takes at most 1024 requests, not {c.requests}")
    if not 0 <= prefix_length <= 1 << 30 or prefix_length > 0 and prefix_pages is None:
        raise _lib.B200Error("prefix_length needs prefix_pages, and must be 0 to 2^30 rows")
    if prefix_pages is not None:
        _lib.require_tensor("prefix_pages", prefix_pages, (torch.int32,), (None,), q)
        if prefix_pages.numel() * c.page_size < prefix_length:
            raise _lib.B200Error(f"{prefix_pages.numel()} pages of {c.page_size} rows cannot hold a prefix of {prefix_length}")
    scale = c.head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 <= scale <= 3e38:
        raise _lib.B200Error(f"attention takes a finite scale of 0 or more, not {scale}")
    if mask is not None:
        _lib.require_tensor("mask", mask, (torch.int64,), (c.tokens,), q)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _lib.require_tensor("out", out, (q.dtype,), q.shape, q, packed=False)
        _lib.require_writable("out", out)
    _lib.require_writable("q", q)
    if any(s % 8 for t in (q, out, k_pages) for s in t.stride()[:-1]) or any(t.data_ptr() % 16 for t in (q, out, k_pages, v_pages)):
        raise _lib.B200Error("attention needs rows that start at 16 bytes: q, out and pages with strides of multiples of 8")
    L = _lib.lib()
    with _lib.on_device(q):
        ws = torch.empty(L.b200_paged_attention_workspace_bytes(ctypes.byref(c)), dtype=torch.uint8, device=q.device)
        rc = L.b200_paged_attention(ctypes.byref(c), _lib.ptr(q), q.stride(0), q.stride(1), _lib.ptr(out), out.stride(0), out.stride(1),
                                    _lib.ptr(prefix_pages), int(prefix_length), _lib.ptr(mask), scale,
                                    _lib.ptr(ws), ws.numel(), _lib.ptr(_error_word(q.device)), _lib.stream_ptr(q.device))
    _lib.check(rc, "b200_paged_attention")
    return out


def attention_error(device, clear: bool = False) -> int:
    """Non-zero if a bounded wait inside an attention on this device (without an index: the current one) ever ran out, or ran out since the word
    was cleared (reads the flag, in the order of the current stream)."""
    device = torch.device(device)
    word = _errors.get(torch.cuda.current_device() if device.index is None and _errors else device.index)
    found = 0 if word is None else int(word.item())
    if clear and found:
        word.zero_()
        if word.is_cuda:
            torch.cuda.current_stream(word.device).synchronize()
    return found
