"""GPU tests of attention over a paged cache: queries that are no numbers."""

import pytest
import torch

from tests.test_gpu_paged import DEV, TYPES, _pool, _randn, da  # noqa: F401

pytestmark = pytest.mark.gpu


# how the parts of an item meet: (lengths, KV heads, rows per KV head)
JOINS = {
    "in one warp": ([1, 16, 0, 9, 16], 2, 3),
    "few rows, many parts": ([9000, 0, 40], 1, 3),
    "a CTA of narrow columns per row": ([2100, 17, 0, 1050, 1, 700, 2100, 0, 17], 3, 5),
    "a CTA per row": ([900, 0, 17, 450, 1, 300] * 3, 4, 5),
    "a warp per row": ([500, 17, 0, 250, 1, 160] * 7, 4, 4),
    "a warp per row, one item by all warps": ([3] * 300 + [20000] + [(i * 13) % 40 for i in range(300)], 1, 4),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("how", JOINS)
def test_queries_that_are_no_numbers_give_none(da, dtype, d, how):
    """The logits of a query with a NaN are NaN, those with an infinity infinite or NaN (channel 0 of the keys is positive, so a
    query of -inf there has only logits of -inf): 0 / 0.  Every other row keeps its bits."""
    lengths, hk, rep = JOINS[how]
    pool, table, _, _ = _pool(61, lengths, hk, 16, d, dtype)
    pool[:, :, :, 0, 0] = pool[:, :, :, 0, 0].abs() + 0.5
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = _randn(62, len(lengths), hk * rep, d, dtype=dtype)
    want, want_lse = cache.attend(q, table, n, return_lse=True)
    marked = q.clone()
    rows = torch.arange(len(lengths) * hk * rep, device=DEV).view(len(lengths), hk * rep)
    kind = torch.where(rows % 5 < 3, rows % 5, 3)                 # 0: a NaN, 1: +inf, 2: -inf in channel 0, 3: as it was
    marked[..., d - 1][kind == 0] = float("nan")
    marked[..., 0][kind == 1] = float("inf")
    marked[..., 0][kind == 2] = -float("inf")
    out, lse = cache.attend(marked, table, n, return_lse=True)
    cache.check_status()
    some = (n > 0)[:, None]
    for i in range(3):
        assert bool(torch.isnan(out[(kind == i) & some]).all())
    assert bool(torch.isnan(lse[(kind == 0) & some]).all()) and not bool(torch.isfinite(lse[(kind < 3) & some]).any())
    assert bool((lse[(kind == 2) & some] == -float("inf")).all())
    assert torch.equal(out[kind == 3], want[kind == 3]) and torch.equal(lse[kind == 3], want_lse[kind == 3])
    assert bool((out[n == 0] == 0).all()) and bool((lse[n == 0] == -float("inf")).all())     # nothing attended: zeros, whatever the query


@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_whose_pages_are_all_bad_gives_zeros_for_any_query(da, dtype):
    pool, table, _, _ = _pool(63, [40, 3000], 2, 16, 64, dtype)
    cache = da.PagedKVCache.over(pool)
    out, lse = cache.attend(torch.full((2, 4, 64), float("nan"), dtype=dtype, device=DEV), torch.full_like(table, -1),
                            torch.tensor([40, 3000], dtype=torch.int32, device=DEV), return_lse=True)
    with pytest.raises(RuntimeError, match="page id"):
        cache.check_status()
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
