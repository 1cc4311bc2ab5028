"""GPU tests of the paged-cache operators at the sizes of real prompts and batches, where the kernels take other forms than for a few
hundred tokens: several heads per thread (as many as leave few places empty, the last group of a kind smaller), several tokens
of a thread under way or in turn, sums over more than 32 or 1024 sequences.  Tolerances as in test_gpu_paged.py."""

import pytest
import torch

from tests.test_gpu_paged import (DEV, TYPES, _assert_attended, _assert_turned, _assert_within, _attention, _frequencies, _pool,
                                  _randn, _turned, da)  # noqa: F401

pytestmark = pytest.mark.gpu


def _ragged(rows, n):
    """n numbers of new tokens that add up to `rows`, an empty sequence among them"""
    new = [rows // n + (i * 37) % 23 - 11 for i in range(n)]
    new[2] = 0
    new[-1] += rows - sum(new)
    return new


# query and KV heads (the values' count too): (32, 8) are four to a thread, (31, 7) four with smaller last groups, (9, 3) three, (6, 2) two,
# (5, 1) and (1, 1) one
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hq,hk,d,rot,rows,shift", [
    (32, 8, 64, 64, 11003, 0), (31, 7, 64, 64, 6007, 0), (9, 3, 96, 48, 4900, 0), (9, 3, 96, 96, 21001, 0), (6, 2, 64, 64, 20011, 0),
    (6, 2, 128, 128, 20011, 0), (5, 1, 128, 128, 20003, 0), (1, 1, 64, 64, 50021, 0), (4, 1, 80, 34, 30011, 0), (31, 2, 256, 100, 3001, 0),
    (9, 3, 96, 34, 15013, 0), (6, 2, 96, 34, 20011, 0), (14, 4, 64, 50, 8009, 1), (14, 4, 64, 50, 8009, 2), (3, 1, 64, 64, 30011, 1),
])
def test_append_of_long_prompts(da, dtype, interleaved, hq, hk, d, rot, rows, shift):
    """A ragged batch: rows in front of and behind the sequences, a sequence without new tokens, one of length 0 that has rows all the
    same, one with a page outside the pool, one whose last tokens pass the end of the table.  Sources `shift` elements behind a 16-byte
    boundary."""
    page, front, behind = 16, 5, 9
    new = _ragged(rows, 7)
    before = [0, 100, 33, 7, 0, 250, 3]
    after = [b + n for b, n in zip(before, new)]
    lengths = list(after)
    lengths[1] = 0
    columns = -(-max(after) // page)
    lengths[5] += columns * page - after[5] + 20                   # its last 20 tokens have no place
    n_pages = 7 * columns + 1
    table = torch.randperm(7 * columns, generator=torch.Generator().manual_seed(5)).view(7, columns).int().to(DEV)
    scrap = n_pages - 1                                            # in the reference the bad page
    kept = table.clone()
    bad = [(0, 2), (0, 3), (3, columns // 3), (6, after[6] // page // 2)]
    for b, c in bad:
        table[b, c], kept[b, c] = (-1, n_pages, 2 ** 31 - 1, -2 ** 31)[c % 4], scrap
    starts = torch.tensor([front + sum(new[:i]) for i in range(8)], device=DEV)
    total = int(starts[-1]) + behind
    fused = _randn(41, total * (hq + 2 * hk) * d + shift, dtype=dtype)[shift:].view(total, hq + 2 * hk, d)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
    f = _frequencies(rot)
    pool = _randn(42, hk, n_pages, page, 2, d, dtype=dtype)

    # row by row: its sequence, its position, whether it has a place
    row = torch.arange(total, device=DEV)
    seq = (torch.searchsorted(starts, row, right=True) - 1).clamp(0, 6)
    position = torch.tensor(lengths, device=DEV)[seq] - starts[seq + 1] + row
    used = (row >= starts[0]) & (row < starts[-1]) & (torch.tensor(lengths, device=DEV)[seq] > 0) & (position < columns * page)
    row, seq, position = row[used], seq[used], position[used]
    where = kept[seq, position // page].long()
    for rotary, queries in ((da.Rotary(f, factor=1.125, interleaved=interleaved), q), (None, None)):
        want, slack = pool.double(), torch.zeros(pool.shape, device=DEV)
        rk, sk = _turned(k[used], position, f, 1.125, interleaved) if rotary else (k[used].double(), torch.zeros(k[used].shape, device=DEV))
        want[:, where, position % page, 0], slack[:, where, position % page, 0] = rk.transpose(0, 1), sk.float().transpose(0, 1)
        want[:, where, position % page, 1] = v[used].double().transpose(0, 1)
        want[:, scrap], slack[:, scrap] = pool[:, scrap].double(), 0.0
        cache = da.PagedKVCache.over(pool.clone())
        out = cache.append_(k, v, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), starts=starts.int(), q=queries, rotary=rotary)
        with pytest.raises(RuntimeError, match="page id.*outside the page table"):
            cache.check_status()
        for h in range(hk):
            _assert_within(cache.pages[h], want[h], slack[h].double())
        if queries is not None:
            assert bool((out[~used] == 0).all())
            _assert_turned(out[used], q[used], position, f, 1.125, interleaved)
        del want, slack, rk, sk, cache, out


@pytest.mark.parametrize("interleaved", [True, False])
def test_append_of_one_token_to_many_sequences(da, interleaved):
    """A decode step of 5000 sequences, every third one not in use."""
    n, hq, hk, d, page = 5000, 8, 2, 64, 16
    lengths = torch.arange(n, device=DEV) % 70
    lengths[::3] = 0
    table = torch.randperm(n * 5, generator=torch.Generator().manual_seed(6)).view(n, 5).int().to(DEV)
    pool = torch.zeros(hk, n * 5, page, 2, d, dtype=torch.bfloat16, device=DEV)
    q, k, v = (_randn(43 + i, n, h, d, dtype=torch.bfloat16) for i, h in enumerate((hq, hk, hk)))
    f = _frequencies(d)
    cache = da.PagedKVCache.over(pool)
    out = cache.append_(k, v, table, lengths.int(), q=q, rotary=da.Rotary(f, interleaved=interleaved))
    cache.check_status()
    used = lengths > 0
    position = lengths[used] - 1
    where = table[used].long().gather(1, (position // page)[:, None])[:, 0]
    _assert_turned(out[used], q[used], position, f, 1.0, interleaved)
    _assert_turned(pool[:, where, position % page, 0].transpose(0, 1), k[used], position, f, 1.0, interleaved)
    assert torch.equal(pool[:, where, position % page, 1].transpose(0, 1), v[used])
    assert bool((out[~used] == 0).all())
    pool[:, where, position % page] = 0
    assert bool((pool == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hq,hk,d,rot,tokens", [
    (32, 8, 64, 64, 11003), (31, 7, 64, 64, 10007), (13, 2, 128, 32, 9001), (9, 3, 96, 48, 21001), (6, 2, 64, 64, 20011), (5, 1, 128, 128, 20003),
    (6, 2, 128, 128, 20011),
    (2, 2, 128, 128, 40013), (4, 1, 80, 34, 30011), (2, 1, 33, 12, 40009), (7, 3, 6, 4, 60013), (32, 8, 256, 256, 2503), (32, 8, 80, 34, 9001), (9, 3, 96, 34, 15013),
    (6, 2, 96, 34, 20011), (31, 9, 6, 4, 20011), (15, 4, 33, 12, 20011),
])
def test_rotation_of_long_sequences_and_its_gradient(da, dtype, interleaved, hq, hk, d, rot, tokens):
    f = _frequencies(rot)
    positions = torch.arange(tokens, device=DEV, dtype=torch.int32) + 1234
    q, k = (_randn(s, tokens, h, d, dtype=dtype).requires_grad_() for s, h in ((51, hq), (52, hk)))
    dq, dk = _randn(53, tokens, hq, d, dtype=dtype), _randn(54, tokens, hk, d, dtype=dtype)
    q2, k2 = da.Rotary(f, factor=1.25, interleaved=interleaved)(q, k, positions)
    gq, gk = torch.autograd.grad((q2, k2), (q, k), (dq, dk))
    for got, x, p in ((q2, q, positions), (k2, k, positions), (gq, dq, -positions), (gk, dk, -positions)):
        _assert_turned(got.detach(), x.detach(), p, f, 1.25, interleaved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("hq,hk,d", [(32, 8, 64), (9, 3, 96), (6, 2, 80)])
def test_rotation_of_long_batches_that_do_not_follow_one_another(da, dtype, interleaved, hq, hk, d):
    """Heads before tokens, positions of their own in every batch entry."""
    f = _frequencies(d)
    batch, tokens = 3, 7001
    q, k = _randn(55, batch, hq, tokens, d, dtype=dtype).transpose(1, 2), _randn(56, batch, tokens + 2, hk, d, dtype=dtype)[:, 1:-1]
    positions = torch.randint(0, 100000, (batch, tokens), device=DEV)
    q2, k2 = da.Rotary(f, interleaved=interleaved)(q, k, positions)
    _assert_turned(q2, q, positions, f, 1.0, interleaved)
    _assert_turned(k2, k, positions, f, 1.0, interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hk,rep,lengths", [
    (1, 4, [(i * 331) % 1700 for i in range(64)]),                # 256 rows
    (1, 1, [(i * 331) % 900 for i in range(37)]),                 # 37 rows: narrow columns
    (1, 2, [0] * 33 + [2500] + [0] * 30 + [700, 0, 1]),           # 134 rows, long runs of sequences not in use
    (1, 3, [5, 0, 1900] * 65),                                    # 585 rows
    (2, 2, [(i * 13) % 50 for i in range(1500)]),                 # sequences in runs of 47
    (1, 2, [0] * 1000 + [900] + [0] * 99 + [33] * 200 + [4000] + [0] * 300),
])
def test_attention_of_more_sequences_than_a_warp_has_lanes(da, dtype, hk, rep, lengths):
    pool, table, keys, values = _pool(71, lengths, hk, 16, 64, dtype)
    q = _randn(72, len(lengths), hk * rep, 64, dtype=dtype)
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, table, n, return_lse=True)
    cache.check_status()
    want, want_lse, tol, tol_lse = _attention(q, keys, values, 0, 0.125)
    _assert_attended(out, want, tol)
    some = n > 0
    assert bool((out[~some] == 0).all()) and bool((lse[~some] == -float("inf")).all())
    _assert_attended(lse[some], want_lse[some], tol_lse[some])
