"""GPU tests of attention over a paged cache: queries that are no numbers, and how finely the weights are kept.

Tolerance, in the terms of test_gpu_paged.py (u half a step of the element type, e what the logits and sums are off by, A the
weighted mean of |v|).  In 16-bit types a weight takes part in the second product as the sum of two numbers of the type: the first
leaves at most u of it, the second u of that, so u^2 relative.  Float16 has no numbers between 0 and 2^-24: what lies there is off by
2^-25, and the weights are kept as multiples of 2^-15 of the largest, so a token by at most 2^-40 of the largest weight."""

import math

import pytest
import torch

from tests.test_gpu_paged import DEV, HALF_STEP, TYPES, _assert_attended, _attention, _pool, _randn, da  # noqa: F401

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rep", [4, 12])
@pytest.mark.parametrize("n,batch", [(16, 1), (1000, 1), (1000, 2500), (32768, 2500)])
def test_many_small_weights_beside_a_large_one(da, dtype, rep, n, batch):
    """One key 17.4 above the others, whose values are 1 and its own 0: the output is the others' share.  Many sequences share the
    pages, so that a warp has all of an item."""
    d, page = 64, 16
    pool = torch.zeros(1, -(-n // page), page, 2, d, dtype=dtype, device=DEV)
    pool[0, :, :, 1] = 1.0
    outlier = n // 2
    pool[0, outlier // page, outlier % page, 0, 0] = 139.0
    pool[0, outlier // page, outlier % page, 1] = 0.0
    cache = da.PagedKVCache.over(pool)
    q = torch.zeros(batch, rep, d, dtype=dtype, device=DEV)
    q[..., 0] = 1.0
    table = torch.arange(pool.shape[1], dtype=torch.int32, device=DEV).expand(batch, -1)
    out, lse = cache.attend(q, table, torch.full((batch,), n, dtype=torch.int32, device=DEV), return_lse=True)
    cache.check_status()
    small = (n - 1) * math.exp(-139.0 / 8)
    want = small / (1 + small)
    u = HALF_STEP[dtype]
    e = (d + 8) * 2.0 ** -23 * 139.0 / 8 + (n / 16 + 64) * 2.0 ** -23
    tol = want * (2 * (e + (u * u if dtype != torch.float32 else 0.0)) + u) * (1 + u)
    if dtype == torch.float16:
        tol += n * 2.0 ** -40 + 2.0 ** -25
    err = float((out.double() - want).abs().max())
    assert err <= tol, (err, tol, want)
    want_lse = 139.0 / 8 + math.log1p(small)
    assert float((lse.double() - want_lse).abs().max()) <= e + 2.0 ** -22 * (1 + want_lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rep", [(64, 3), (64, 16), (80, 5), (128, 4), (256, 12)])
def test_weights_are_kept_to_twice_the_bits_of_the_type(da, dtype, d, rep):
    """Few tokens, so that the values of a row cancel in many channels and their outputs show the weights' own errors: rounded once to
    bfloat16 or float16 they would leave the bound."""
    lengths = [2 + i % 19 for i in range(200)]
    pool, table, keys, values = _pool(64, lengths, 1, 16, d, dtype)
    q = _randn(65, len(lengths), rep, d, dtype=dtype)
    cache = da.PagedKVCache.over(pool)
    out = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=0.25 * d ** -0.5)
    want, _, tol, rounded_once = _fine_tolerance(q, keys, values, 0.25 * d ** -0.5)
    _assert_attended(out, want, tol)
    if dtype != torch.float32:       # (the bound tells the two apart: the definition with weights of one number is outside it)
        assert bool(((rounded_once - want).abs() > tol).any())


def _fine_tolerance(q, keys, values, scale):
    """(out, lse, tolerance of out, out with every weight rounded once) in 64 bits"""
    out, lse, _, _ = _attention(q, keys, values, 0, scale)
    u = HALF_STEP[q.dtype]
    u_w = 0.0 if q.dtype == torch.float32 else u * u
    tol, once = torch.zeros_like(out), torch.zeros_like(out)
    for b, (k, v) in enumerate(zip(keys, values)):
        hk, n, d = k.shape
        x = q[b].double().reshape(hk, -1, d)
        s = x @ k.transpose(1, 2) * scale
        size = (x.abs() @ k.abs().transpose(1, 2)).amax(-1) * abs(scale)
        w = torch.softmax(s, -1)
        mean = w @ v.abs()
        e = (d + 8) * 2.0 ** -23 * size + (n / 16 + 64) * 2.0 ** -23
        tol[b] = (mean * (u_w + 2 * e)[..., None] * (1 + u) + u * (w @ v).abs()).reshape(out[b].shape)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        once[b] = ((p.to(q.dtype).double() @ v) / p.sum(-1, keepdim=True)).to(q.dtype).double().reshape(out[b].shape)
    if q.dtype == torch.float16:
        tol += 2.0 ** -25 + 20 * 2.0 ** -40 * max(float(v.abs().max()) for v in values)
    return out, lse, tol, once


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rep,batch,n", [(64, 4, 1800, 1048576), (128, 12, 1200, 262144), (256, 2, 900, 196608), (96, 5, 1800, 196608)])
def test_sums_over_very_many_tokens_in_one_warp(da, dtype, d, rep, batch, n):
    """Equal weights over values near 1: the output is their mean.  The sequences share the pages, and there are as many as warps, so
    that a warp has (nearly) all tokens of one.  Tolerance: the products of a unit and the join 64 * 2^-23; one rounding to nearest
    per 16 tokens, 2^-24 of the sum each, which add up like independent ones, six deviations: 6 sqrt(n / 16) 2^-24; u of the output."""
    if dtype == torch.float32:
        batch, n = batch // 4, n // 4
    pool = torch.zeros(1, n // 16, 16, 2, d, dtype=dtype, device=DEV)
    pool[0, :, :, 1] = (1 + 0.25 * torch.rand(n // 16, 16, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(66))).to(dtype)
    table = torch.arange(n // 16, dtype=torch.int32, device=DEV).expand(batch, -1)
    cache = da.PagedKVCache.over(pool)
    out, lse = cache.attend(torch.zeros(batch, rep, d, dtype=dtype, device=DEV), table, torch.full((batch,), n, dtype=torch.int32, device=DEV),
                            return_lse=True)
    cache.check_status()
    want = pool[0, :, :, 1].double().mean((0, 1))
    tol = want * (64 * 2.0 ** -23 + 6 * math.sqrt(n / 16) * 2.0 ** -24 + HALF_STEP[dtype])
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), float((err / want).max())
    assert float((lse.double() - math.log(n)).abs().max()) <= 2.0 ** -20 * (1 + math.log(n))
