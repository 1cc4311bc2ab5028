"""Key-value cache of several sequences in one pool of pages in HBM: append with the rotary embedding on the way, and
attention of one new token per sequence."""

from __future__ import annotations

import math
from typing import Optional

import torch

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
        `lru.hbm_kv_cache.view(lru.num_kv_heads, -1, lru.page_size, 2, lru.head_dim)`."""
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
        piece = 16 // pages.element_size()
        assert pages.data_ptr() % 16 == 0 and all(s % piece == 0 for n, s in zip(pages.shape, pages.stride()[:2]) if n > 1), \
            "pages must start on 16-byte boundaries"
        _native.lib()
        self.pages = pages.detach()
        self.n_kv_heads, self.n_pages, self.page_size, _, self.head_dim = pages.shape
        # (the stride of a dimension of one entry is never followed)
        head, page = pages.stride()[:2]
        self._strides = (page if self.n_pages > 1 else 0, head if self.n_kv_heads > 1 else 0)
        self.status = torch.zeros(1, dtype=torch.int32, device=pages.device)

    # ---- checks shared by the calls --------------------------------------------------------
    def _check_heads(self, t: torch.Tensor, name: str, rows: Optional[int], heads: Optional[int]) -> torch.Tensor:
        assert t.dim() == 3 and t.shape[2] == self.head_dim and (rows is None or t.shape[0] == rows) and \
            (heads is None or t.shape[1] == heads), \
            f"{name} must be ({'rows' if rows is None else rows}, {'heads' if heads is None else heads}, {self.head_dim}), got {tuple(t.shape)}"
        self._check_device(t, name)
        assert t.dtype == self.pages.dtype, f"{name} must be {self.pages.dtype} like the pages, got {t.dtype}"
        assert not (t.requires_grad and torch.is_grad_enabled()), \
            f"{name} requires a gradient, which the paged cache does not pass on: detach it or call under torch.no_grad()"
        return t if t.stride(2) == 1 else t.contiguous()

    def _check_device(self, t: torch.Tensor, name: str) -> None:
        _native.require_cuda(t, name)
        assert t.device == self.pages.device, f"{name} must be on the device of the pages ({self.pages.device}), got {t.device}"

    def _check_table(self, page_table: torch.Tensor, lengths: torch.Tensor) -> int:
        assert page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.shape[1] > 0, \
            f"page_table must be (n_sequences, columns) int32, got {tuple(page_table.shape)} {page_table.dtype}"
        n = page_table.shape[0]
        assert lengths.dtype == torch.int32 and lengths.shape == (n,), \
            f"lengths must be ({n},) int32, got {tuple(lengths.shape)} {lengths.dtype}"
        assert (page_table.shape[1] == 1 or page_table.stride(1) == 1) and (n <= 1 or lengths.stride(0) == 1), \
            "the rows of page_table and lengths must be contiguous"
        self._check_device(page_table, "page_table")
        self._check_device(lengths, "lengths")
        return n

    # ---- operators ----------------------------------------------------------------------------
    def append_(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *,
                starts: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                rotary: Optional[Rotary] = None) -> Optional[torch.Tensor]:
        """Write the keys and values of new tokens to their pages, the keys rotated by their position when `rotary` is given.

        k, v (rows, n_kv_heads, D): without `starts` one row per sequence; with `starts` (n_sequences + 1,) int32, rows
        starts[b] to starts[b + 1] are the new tokens of sequence b.  `lengths` counts them already: the last
        new token of sequence b is its token lengths[b] - 1.  Rows in front of and behind the sequences (a padded batch), and those
        of sequences of length 0, are left out.
        q (rows, Hq, D), only with `rotary`: returned rotated like the keys (a new tensor; rows left out are zero).
        Two sequences must not append to the same page.  A position outside the table or a page outside the pool writes
        nothing and is reported by `check_status`."""
        n = self._check_table(page_table, lengths)
        k = self._check_heads(k, "k", None, self.n_kv_heads)
        v = self._check_heads(v, "v", k.shape[0], self.n_kv_heads)
        rows = k.shape[0]
        if starts is None:
            assert rows == n, f"one row per sequence expected ({n}), got {rows}; pass starts for a ragged batch"
        else:
            assert starts.dtype == torch.int32 and starts.shape == (n + 1,) and (n == 0 or starts.stride(0) == 1), \
                f"starts must be ({n + 1},) int32, contiguous, got {tuple(starts.shape)} {starts.dtype}"
            self._check_device(starts, "starts")
        out = None
        if q is not None:
            assert rotary is not None, "q is only rotated: pass rotary with it"
            q = self._check_heads(q, "q", rows, None)
            assert q.shape[1] > 0, "q has no heads"
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        turn = (0, 0, 0, 1.0)
        if rotary is not None:
            assert rotary.rotary_dim <= self.head_dim, f"rotary_dim {rotary.rotary_dim} exceeds head_dim {self.head_dim}"
            self._check_device(rotary.inv_freq, "inv_freq")
            turn = (rotary.inv_freq.data_ptr(), rotary.rotary_dim, rotary.interleaved, rotary.factor)
        if rows == 0:
            return out
        if n == 0:
            return None if out is None else out.zero_()
        qs = (0, 0) if q is None else q.stride()[:2]
        with torch.cuda.device(k.device):
            _native.check(_native.lib().da_append_pages(_native.PACK_APPEND(
                0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if q is None else out.data_ptr(),
                *qs, *k.stride()[:2], *v.stride()[:2], self.pages.data_ptr(), *self._strides, self.page_size, self.n_pages,
                page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(),
                0 if starts is None else starts.data_ptr(), n, rows, *turn, 0 if q is None else q.shape[1], self.n_kv_heads,
                self.head_dim, _native.dtype_code(k.dtype), self.status.data_ptr(), _native.stream_ptr())), "da_append_pages")
        return out

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, *, window: int = 0,
               scale: Optional[float] = None, return_lse: bool = False):
        """Attention of one token per sequence, q (n_sequences, Hq, D) with Hq a multiple of n_kv_heads (query head h reads
        KV head h // (Hq / n_kv_heads)), over the first lengths[b] tokens of its sequence, or the last `window` of them.
        Logits are scaled by `scale` (default 1 / sqrt(D)).  Returns (n_sequences, Hq, D); with `return_lse` also the float32
        log-sum-exp of the scaled logits (n_sequences, Hq).  A sequence of length 0 gives zeros and -inf."""
        n = self._check_table(page_table, lengths)
        q = self._check_heads(q, "q", n, None)
        hq = q.shape[1]
        assert hq > 0 and hq % self.n_kv_heads == 0, f"{hq} query heads do not divide among {self.n_kv_heads} KV heads"
        rep = hq // self.n_kv_heads
        assert window >= 0, f"window must not be negative, got {window}"
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale)
        piece = 16 // q.element_size()
        if q.data_ptr() % 16 or any(s % piece for s in q.stride()[:2]):
            q = q.clone(memory_format=torch.contiguous_format)
        with torch.cuda.device(q.device):
            out = torch.empty(n, hq, self.head_dim, dtype=q.dtype, device=q.device)
            lse = torch.empty(n, hq, dtype=torch.float32, device=q.device) if return_lse else None
            if n:
                dtype = _native.dtype_code(q.dtype)
                lib = _native.lib()
                # scratch of this call alone: two captured steps, or two streams, never share it
                size = lib.da_paged_attention_workspace_bytes(rep, self.head_dim, dtype)
                workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=q.device)
                _native.check(lib.da_paged_attention(_native.PACK_ATTEND(
                    q.data_ptr(), *q.stride()[:2], self.pages.data_ptr(), *self._strides, self.page_size, self.n_pages,
                    page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(), n, window, scale,
                    out.data_ptr(), 0 if lse is None else lse.data_ptr(), workspace.data_ptr(), size, self.status.data_ptr(),
                    self.n_kv_heads, rep, self.head_dim, dtype, _native.stream_ptr())), "da_paged_attention")
        return (out, lse) if return_lse else out

    def check_status(self) -> None:
        """Synchronises; raises if any call on this pool flagged a problem."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise RuntimeError("dram_attention_b200 device status: " + _native.status_message(bits))
