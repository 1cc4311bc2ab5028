"""Key-value cache of several sequences in one pool of pages in HBM: append with the rotary embedding on the way, and
attention of one new token per sequence."""

from __future__ import annotations

import math
import operator
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native
from .rotary import Rotary

HEAD_DIMS = (64, 80, 96, 128, 256)


class PagedKVCache:
    """A pool of pages and the operators on it.

    `pages` is (n_kv_heads, n_pages, page_size, 2, head_dim): token-major inside a page, key then value, the page format of
    `LRUCache`.  Which pages belong to a sequence, and in which order, is the caller's: `page_table` (n_sequences, columns)
    int32 holds token t of sequence b in page page_table[b, t // page_size]; entries that no token needs are never read.
    `lengths` (n_sequences,) int32 is the number of tokens of every sequence, the new ones of the step among them; 0 marks a
    row of the batch that is not in use.  Both are read on the device, so a captured step follows them from replay to replay.
    Calls work on the current stream of the pool's device and share nothing but the pool: ordering calls that write and read
    the same pages on several streams is the caller's.

    Args:
        n_pages, page_size: pages in the pool, tokens per page.
        n_kv_heads, head_dim: KV head count and channel count (64, 80, 96, 128 or 256).
        device: CUDA device of the pool.
        dtype: element type (bfloat16, float16 or float32)."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device: str = "cuda",
                 dtype: torch.dtype = torch.bfloat16):
        _native.dtype_code(dtype)
        self._set_pages(torch.zeros(n_kv_heads, n_pages, page_size, 2, head_dim, dtype=dtype, device=device))

    @classmethod
    def over(cls, pages: torch.Tensor) -> "PagedKVCache":
        """The operators on a pool that exists already: (n_kv_heads, n_pages, page_size, 2, head_dim), pages of a head and
        heads at any distance (a multiple of 16 bytes), or the slot table of an LRU cache,
        `lru.hbm_kv_cache.view(lru.num_kv_heads, -1, lru.page_size, 2, lru.head_dim)`.  Derivatives do not reach it."""
        self = cls.__new__(cls)
        self._set_pages(pages)
        return self

    def _set_pages(self, pages: torch.Tensor) -> None:
        assert pages.dim() == 5 and pages.shape[3] == 2 and pages.numel() > 0, \
            f"pages must be (n_kv_heads, n_pages, page_size, 2, head_dim), got {tuple(pages.shape)}"
        _native.dtype_code(pages.dtype)
        d, page_size = pages.shape[4], pages.shape[2]
        assert d in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {d}"
        _native.require_cuda(pages, "pages")
        assert all(size == 1 or stride == want for size, stride, want in zip(pages.shape[2:], pages.stride()[2:], (2 * d, d, 1))), \
            "the tokens of a page must be contiguous"
        assert not pages.is_neg(), "pages must be plain memory, not the negative of another tensor's"
        piece = 16 // pages.element_size()
        assert pages.data_ptr() % 16 == 0 and all(s % piece == 0 for n, s in zip(pages.shape, pages.stride()[:2]) if n > 1), \
            "pages must start on 16-byte boundaries"
        _native.lib()
        self._pages = pages.detach()
        self.n_kv_heads, self.n_pages, self.page_size, _, self.head_dim = pages.shape
        # (the stride of a dimension of one entry is never followed)
        head, page = pages.stride()[:2]
        self._layout = (page if self.n_pages > 1 else 0, head if self.n_kv_heads > 1 else 0, self.page_size, self.n_pages)
        self._device, self._dtype, self._dtype_code, self._piece = pages.get_device(), pages.dtype, _native.dtype_code(pages.dtype), piece
        self._scratch = {}
        self.status = torch.zeros(1, dtype=torch.int32, device=pages.device)

    @property
    def pages(self) -> torch.Tensor:
        return self._pages

    def __getstate__(self):
        return {"pages": self._pages}     # (a copied or saved cache works on its own pages)

    def __setstate__(self, state) -> None:
        self._set_pages(state["pages"])

    # ---- checks shared by the calls --------------------------------------------------------
    def _check_heads(self, t: torch.Tensor, name: str, rows: Optional[int], heads: Optional[int]) -> torch.Tensor:
        shape = t.shape
        assert len(shape) == 3 and shape[2] == self.head_dim and (rows is None or shape[0] == rows) and \
            (heads is None or shape[1] == heads), \
            f"{name} must be ({'rows' if rows is None else rows}, {'heads' if heads is None else heads}, {self.head_dim}), got {tuple(shape)}"
        if t.get_device() != self._device:
            self._wrong_device(t, name)
        assert t.dtype is self._dtype, f"{name} must be {self._dtype} like the pages, got {t.dtype}"
        if t.requires_grad or forward_ad._current_level >= 0:
            assert not (t.requires_grad and torch.is_grad_enabled()), \
                f"{name} requires a gradient, which the paged cache does not pass on: detach it or call under torch.no_grad()"
            assert not _native.has_tangent(t), f"{name} has a tangent, which the paged cache does not pass on: detach it"
        return t if t.stride(2) == 1 and not t.is_neg() else t.resolve_neg().contiguous()

    def _wrong_device(self, t: torch.Tensor, name: str) -> None:
        _native.require_cuda(t, name)
        raise AssertionError(f"{name} must be on the device of the pages ({self._pages.device}), got {t.device}")

    def _check_table(self, page_table: torch.Tensor, lengths: torch.Tensor):
        """Sequences, columns and row stride of the table"""
        shape, strides = page_table.shape, page_table.stride()
        assert len(shape) == 2 and shape[1] > 0 and page_table.dtype is torch.int32, \
            f"page_table must be (n_sequences, columns) int32, got {tuple(shape)} {page_table.dtype}"
        n, columns = shape
        assert lengths.dtype is torch.int32 and lengths.shape == (n,), \
            f"lengths must be ({n},) int32, got {tuple(lengths.shape)} {lengths.dtype}"
        assert (strides[1] == 1 or columns == 1) and (n <= 1 or lengths.stride(0) == 1), \
            "the rows of page_table and lengths must be contiguous"
        if page_table.get_device() != self._device:
            self._wrong_device(page_table, "page_table")
        if lengths.get_device() != self._device:
            self._wrong_device(lengths, "lengths")
        return n, columns, strides[0]

    # ---- operators ----------------------------------------------------------------------------
    def append_(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
                starts: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                rotary: Optional[Rotary] = None) -> Optional[torch.Tensor]:
        """Write the keys and values of new tokens to their pages, the keys rotated by their position when `rotary` is given.

        k, v (rows, n_kv_heads, D): without `starts` one row per sequence; with `starts` (n_sequences + 1,) int32, rows
        starts[b] to starts[b + 1] are the new tokens of sequence b (starts does not decrease).  `lengths` counts them already:
        the last new token of sequence b is its token lengths[b] - 1.  Rows in front of and behind the sequences (a padded
        batch), and those of sequences of length 0, are left out.
        q (rows, Hq, D), only with `rotary`: returned rotated like the keys (a new tensor; rows left out are zero).
        No two new tokens may have the same place (two sequences that append to one page, a page listed twice), and k, v and q
        must not lie in the pool.  A position outside the table or a page outside the pool writes nothing and is reported by
        `check_status`."""
        n, columns, table_stride = self._check_table(page_table, lengths)
        k = self._check_heads(k, "k", None, self.n_kv_heads)
        rows = k.shape[0]
        v = self._check_heads(v, "v", rows, self.n_kv_heads)
        if starts is None:
            assert rows == n, f"one row per sequence expected ({n}), got {rows}; pass starts for a ragged batch"
            starts_ptr = 0
        else:
            assert starts.dtype is torch.int32 and starts.shape == (n + 1,) and (n == 0 or starts.stride(0) == 1), \
                f"starts must be ({n + 1},) int32, contiguous, got {tuple(starts.shape)} {starts.dtype}"
            if starts.get_device() != self._device:
                self._wrong_device(starts, "starts")
            starts_ptr = starts.data_ptr()
        out, qp, qo, qs, hq, turn = None, 0, 0, (0, 0), 0, (0, 0, 0, 1.0)
        if rotary is not None:
            assert rotary.rotary_dim <= self.head_dim, f"rotary_dim {rotary.rotary_dim} exceeds head_dim {self.head_dim}"
            inv_freq = rotary.inv_freq
            if inv_freq.get_device() != self._device:
                self._wrong_device(inv_freq, "inv_freq")
            turn = (inv_freq.data_ptr(), rotary.rotary_dim, rotary.interleaved, rotary.factor)
        if q is not None:
            assert rotary is not None, "q is only rotated: pass rotary with it"
            q = self._check_heads(q, "q", rows, None)
            hq = q.shape[1]
            assert hq > 0, "q has no heads"
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            qp, qo, qs = q.data_ptr(), out.data_ptr(), q.stride()[:2]
        if rows == 0:
            return out
        if n == 0:
            return None if out is None else out.zero_()
        _native.launch(_native.lib().da_append_pages, _native.PACK_APPEND(
            qp, k.data_ptr(), v.data_ptr(), qo, *qs, *k.stride()[:2], *v.stride()[:2], self._pages.data_ptr(), *self._layout, page_table.data_ptr(),
            table_stride, columns, lengths.data_ptr(), starts_ptr, n, rows, *turn, hq, self.n_kv_heads, self.head_dim,
            self._dtype_code, self.status.data_ptr(), _native.stream_of(self._device)), self._device, "da_append_pages")
        return out

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *, window: int = 0,
               scale: Optional[float] = None, return_lse: bool = False):
        """Attention of one token per sequence, q (n_sequences, Hq, D) with Hq a multiple of n_kv_heads (query head h reads
        KV head h // (Hq / n_kv_heads)), over the first lengths[b] tokens of its sequence, or the last `window` of them.
        Logits are scaled by `scale` (default 1 / sqrt(D)).  Returns (n_sequences, Hq, D); with `return_lse` also the float32
        log-sum-exp of the scaled logits (n_sequences, Hq).  A sequence of length 0 gives zeros and -inf.  What pages hold beyond
        the attended tokens does not matter, NaN and infinities included; attended keys and values are taken to be finite.
        Where there are tokens, a row of q with a NaN or an infinity gives NaN, and no other row does.  The same inputs give the same
        bits.  Tokens in pages outside the pool are left out and lengths outside the table are cut; `check_status` reports both."""
        n, columns, table_stride = self._check_table(page_table, lengths)
        q = self._check_heads(q, "q", n, None)
        hq = q.shape[1]
        rep = hq // self.n_kv_heads
        assert rep > 0 and hq == rep * self.n_kv_heads, f"{hq} query heads do not divide among {self.n_kv_heads} KV heads"
        window = operator.index(window)
        assert window >= 0, f"window must not be negative, got {window}"
        if window >= columns * self.page_size:
            window = 0
        strides = q.stride()
        if q.data_ptr() % 16 or strides[0] % self._piece or strides[1] % self._piece:
            q = q.clone(memory_format=torch.contiguous_format)
            strides = q.stride()
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty(n, hq, dtype=torch.float32, device=q.device) if return_lse else None
        if n:
            # scratch of this call alone: two captured steps, or two streams, never share it
            size, like = self._scratch.get((n, rep)) or self._scratch_like(n, rep)
            scratch = torch.empty_like(like)
            _native.launch(_native.lib().da_paged_attention, _native.PACK_ATTEND(
                q.data_ptr(), strides[0], strides[1], self._pages.data_ptr(), *self._layout, page_table.data_ptr(), table_stride, columns, lengths.data_ptr(),
                n, window, 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale), out.data_ptr(),
                0 if lse is None else lse.data_ptr(), scratch.data_ptr(), size, self.status.data_ptr(), self.n_kv_heads, rep,
                self.head_dim, self._dtype_code, _native.stream_of(self._device)), self._device, "da_paged_attention")
        return (out, lse) if return_lse else out

    def _scratch_like(self, n: int, rep: int):
        """Bytes of scratch for n sequences with `rep` query heads per KV head, and a tensor of that many elements (one byte of
        memory) to make it like"""
        size = _native.lib().da_paged_attention_workspace_bytes(n, self.n_kv_heads, rep, self.head_dim, self._dtype_code)
        if len(self._scratch) >= 256:
            self._scratch.clear()
        entry = self._scratch[n, rep] = (size, torch.empty(1, dtype=torch.uint8, device=self._pages.device).expand(max(size, 16)))
        return entry

    def check_status(self) -> None:
        """Waits for all streams of the device; raises if any call on this pool flagged a problem since the last check.  (Calls that
        other threads enqueue meanwhile may be reported here or be missed.)"""
        torch.cuda.synchronize(self._device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            torch.cuda.synchronize(self._device)   # (or a later call on another stream could flag a problem first)
            raise RuntimeError("dram_attention_b200 device status: " + "; ".join(t for b, t in _STATUS_TEXT.items() if bits & b))


_STATUS_TEXT = {
    _native.STATUS_BAD_PAGE_ID: "a page id in the page table was outside the pool",
    _native.STATUS_BAD_POSITION: "a length or a position was outside the page table",
    _native.STATUS_WAIT_TIMEOUT: "a bounded wait on an asynchronous copy ran out",
}
