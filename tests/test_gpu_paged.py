"""GPU tests of the paged-cache operators against their definitions in 64 bits.

Tolerances.  u = half a step of the element type (bf16 2^-8, fp16 2^-11, fp32 2^-24 relative).
Rotation: sine and cosine carry at most 3 * 2^-24 (argument rounded after the reduction: 0.8; the function itself: 2), the factor
and its product 2 * 2^-24, the two products and their sum 3 * 2^-24 of |a| + |b|: 8 * 2^-24 * factor * (|a| + |b|), then u of
the result for the rounding to the element type (float16 also loses 2^-25 in its subnormal range).
Attention: a logit of D fused 32-bit steps (the tensor cores' may truncate: 2^-23 each) is off by e = (D + 8) * 2^-23 * S with S the
largest sum of |scale q_i k_i|; a weight by e relative, its exponential by 2^-22 and, in 16-bit types, u for its
rounding in front of the second product; sums over n tokens by (n / 16 + 64) * 2^-23 (16 per warp step and lane, then the joins).
So |out - exact| <= A (u_w + 2 (e + (n / 16 + 64) 2^-23)) + u |out| with A the weighted mean of |v| and u_w = u for 16-bit
types, 0 for float32."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def da():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import dram_attention_b200 as pkg
    pkg._native.lib()
    return pkg


def _randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _frequencies(rot, base=10000.0):
    return (base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).float().to(DEV)


def _turned(x, positions, inv_freq, factor, interleaved):
    """x (..., heads, D), positions (...): the definition in 64 bits, and the bound on its 32-bit evaluation"""
    x = x.detach().double()
    half = inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    c, s = factor * angle.cos()[..., None, :], factor * angle.sin()[..., None, :]
    y, slack = x.clone(), torch.zeros_like(x)
    ia, ib = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    slack[..., ia] = slack[..., ib] = 8 * 2.0 ** -24 * abs(factor) * (a.abs() + b.abs())
    return y, slack


def _assert_turned(got, x, positions, inv_freq, factor, interleaved):
    want, slack = _turned(x, positions, inv_freq, factor, interleaved)
    u = HALF_STEP[got.dtype]
    tol = slack + u * (want.abs() + slack) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.detach().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    rot = 2 * inv_freq.numel()
    assert torch.equal(got[..., rot:], x[..., rot:])       # channels behind the rotated part are copied


# ---------------------------------------------------------------- rotation ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shape,hk,rot", [
    ((1, 8, 64), 2, 64),            # one token
    ((5, 4, 128), 4, 128), ((300, 32, 128), 8, 128),
    ((33, 3, 96), 1, 32),           # part of the head
    ((7, 5, 80), 5, 80), ((7, 5, 80), 1, 34), ((9, 2, 256), 2, 2), ((3, 4, 64), 1, 50),   # parts that end inside a piece
    ((2, 3, 6), 2, 4), ((4, 1, 510), 1, 510), ((3, 2, 512), 2, 512), ((11, 7, 33), 2, 12),   # heads that are no whole pieces
    ((2, 21, 4, 64), 2, 64), ((3, 1, 2, 128), 1, 96),                                        # batches
])
def test_rotation(da, dtype, interleaved, shape, hk, rot):
    q, k = _randn(1, *shape, dtype=dtype), _randn(2, *shape[:-2], hk, shape[-1], dtype=dtype)
    f = _frequencies(rot)
    positions = torch.randint(-5000, 2 ** 20, shape[:-2], device=DEV)
    for p in (positions, positions.int()):
        q2, k2 = da.Rotary(f, factor=1.25, interleaved=interleaved)(q, k, p)
        _assert_turned(q2, q, positions, f, 1.25, interleaved)
        _assert_turned(k2, k, positions, f, 1.25, interleaved)


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotation_at_far_positions(da, interleaved):
    f = _frequencies(64, 500000.0)
    positions = torch.tensor([0, 1, 2 ** 20 + 1, 2 ** 30 - 1, 2 ** 31 - 1, -2 ** 31 + 1, 123456789], device=DEV)
    q, k = _randn(3, 7, 4, 64), _randn(4, 7, 2, 64)
    q2, k2 = da.Rotary(f, interleaved=interleaved)(q, k, positions)
    _assert_turned(q2, q, positions, f, 1.0, interleaved)
    _assert_turned(k2, k, positions, f, 1.0, interleaved)


@pytest.mark.parametrize("d,tokens", [(8, 200003), (2, 100001), (64, 70001)])
def test_rotation_of_many_tokens_with_few_channels(da, d, tokens):
    f = _frequencies(d)
    positions = torch.arange(tokens, device=DEV, dtype=torch.int32)
    q, k = _randn(46, tokens, 1, d, dtype=torch.bfloat16), _randn(47, tokens, 1, d, dtype=torch.bfloat16)
    for interleaved in (True, False):
        q2, k2 = da.Rotary(f, interleaved=interleaved)(q, k, positions)
        _assert_turned(q2, q, positions, f, 1.0, interleaved)
        _assert_turned(k2, k, positions, f, 1.0, interleaved)


def test_rotation_equals_the_table_form(da):
    """The operator's own rotation (complex factors of the whole head) and this one agree to the bound."""
    f = _frequencies(128)
    positions = torch.arange(40, device=DEV) + 1000
    q, k = _randn(5, 40, 8, 128, dtype=torch.bfloat16), _randn(6, 40, 2, 128, dtype=torch.bfloat16)
    table = torch.polar(torch.ones(40, 64, device=DEV, dtype=torch.float64), positions.double()[:, None] * f.double()).to(torch.complex64)
    op = da.DRAMAttention(max_output_length=4, lru_hbm_cache_size=64, local_cache_size=32, page_size=16, top_k=32, n_kv_heads=2,
                          head_dim=128, device=DEV)
    a, b = op.rotate_(q[None], k[None], table)
    q2, k2 = da.Rotary(f)(q, k, positions)
    for x, y in ((a[0], q2), (b[0], k2)):
        assert float((x.double() - y.double()).abs().max()) <= 2.0 ** -7 * float(x.abs().max())
        assert float((x != y).float().mean()) < 0.01


@pytest.mark.parametrize("dtype", TYPES)
def test_rotation_of_strided_heads(da, dtype):
    f = _frequencies(64)
    positions = torch.arange(6, device=DEV)
    fused = _randn(7, 2, 6, 10, 64, dtype=dtype)
    q, k = fused[:, :, :6], fused[:, :, 6:8]
    r = da.Rotary(f, interleaved=False)
    q2, k2 = r(q, k, positions)                     # one row of positions for the batch
    _assert_turned(q2, q, positions.expand(2, 6), f, 1.0, False)
    _assert_turned(k2, k, positions.expand(2, 6), f, 1.0, False)
    heads_first = _randn(8, 2, 5, 6, 64, dtype=dtype).transpose(1, 2)
    channels_apart = _randn(9, 2, 6, 3, 128, dtype=dtype)[..., ::2]
    q2, k2 = r(heads_first, channels_apart, positions.flip(0).expand(2, 6))
    _assert_turned(q2, heads_first, positions.flip(0).expand(2, 6), f, 1.0, False)
    _assert_turned(k2, channels_apart, positions.flip(0).expand(2, 6), f, 1.0, False)
    # rows that start between 16-byte boundaries
    base = _randn(10, 6 * 4 * 64 + 1, dtype=dtype)
    q = base[1:].view(6, 4, 64)
    q2, k2 = r(q, q, positions)
    _assert_turned(q2, q, positions, f, 1.0, False)
    assert torch.equal(q2, k2)
    # positions with gaps between them, and the same one for every token
    far = torch.arange(60, device=DEV, dtype=torch.int32)[::10]
    _assert_turned(r(q, q, far)[0], q, far, f, 1.0, False)
    _assert_turned(r(q, q, far[3:4].expand(6))[1], q, far[3:4].expand(6), f, 1.0, False)


def test_rotation_without_tokens(da):
    r = da.Rotary(_frequencies(64))
    for lead in ((0,), (0, 4), (3, 0)):
        q, k = r(torch.zeros(*lead, 4, 64, device=DEV), torch.zeros(*lead, 2, 64, device=DEV), torch.zeros(lead, dtype=torch.int32, device=DEV))
        assert q.shape == lead + (4, 64) and k.shape == lead + (2, 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,rot", [(64, 64), (96, 32), (80, 34)])
def test_gradient_of_the_rotation_is_the_rotation_back(da, dtype, interleaved, d, rot):
    f = _frequencies(rot)
    positions = torch.arange(17, device=DEV) * 1001
    r = da.Rotary(f, factor=1.5, interleaved=interleaved)
    q, k = (_randn(s, 17, h, d, dtype=dtype).requires_grad_() for s, h in ((11, 4), (12, 2)))
    dq, dk = _randn(13, 17, 4, d, dtype=dtype), _randn(14, 17, 2, d, dtype=dtype)
    gq, gk = torch.autograd.grad(r(q, k, positions), (q, k), (dq, dk))
    _assert_turned(gq, dq, -positions, f, 1.5, interleaved)
    _assert_turned(gk, dk, -positions, f, 1.5, interleaved)
    # one side alone, a gradient that is one number for every element, and an input that needs none
    (only,) = torch.autograd.grad(r(q, k, positions)[0].sum(), (q,))
    _assert_turned(only, torch.ones_like(q), -positions, f, 1.5, interleaved)
    (only,) = torch.autograd.grad(r(q.detach(), k, positions)[1], (k,), dk)
    assert torch.equal(only, gk)
    assert not r(q.detach(), k.detach(), positions)[0].requires_grad
    with torch.no_grad():
        assert not r(q, k, positions)[0].requires_grad


def test_gradient_of_the_rotation_against_differences(da):
    """Linear in q and k, so a central difference of any step is exact up to the rounding of its float32 terms."""
    f = _frequencies(32)
    positions = torch.tensor([3, 70000, -9], device=DEV)
    r = da.Rotary(f, factor=0.75, interleaved=False)
    q, k = _randn(15, 3, 2, 64).requires_grad_(), _randn(16, 3, 1, 64).requires_grad_()
    wq, wk = _randn(17, 3, 2, 64).double(), _randn(18, 3, 1, 64).double()

    def loss(q, k):
        a, b = r(q, k, positions)
        return (a.double() * wq).sum() + (b.double() * wk).sum()

    gq, gk = torch.autograd.grad(loss(q, k), (q, k))
    with torch.no_grad():
        for x, g, dx in ((q, gq, _randn(19, 3, 2, 64)), (k, gk, _randn(20, 3, 1, 64))):
            plus, minus = ((x + dx), (x - dx))
            diff = (loss(plus, k) - loss(minus, k)) / 2 if x is q else (loss(q, plus) - loss(q, minus)) / 2
            slope = (g.double() * (plus.double() - minus.double()) / 2).sum()
            w = wq if x is q else wk
            # every output of the two evaluations and every gradient is off by at most 16 * 2^-24 of the values that make it
            bound = 16 * 2.0 ** -24 * float((w.abs().amax() * (x.abs() + dx.abs()).sum() * 4))
            assert abs(float(diff - slope)) <= bound


def test_second_derivatives_of_the_rotation(da):
    f = _frequencies(64)
    positions = torch.arange(4, device=DEV)
    r = da.Rotary(f)
    q, k = _randn(21, 4, 2, 64).requires_grad_(), _randn(22, 4, 1, 64).requires_grad_()
    dq = _randn(23, 4, 2, 64).requires_grad_()
    (g,) = torch.autograd.grad(r(q, k, positions)[0], (q,), dq, create_graph=True)
    z = _randn(24, 4, 2, 64)
    (back,) = torch.autograd.grad(g, (dq,), z)         # the gradient's gradient is the rotation itself
    _assert_turned(back, z, positions, f, 1.0, True)


def test_rotation_refuses(da):
    f = _frequencies(64)
    r = da.Rotary(f)
    q, k, p = _randn(1, 4, 2, 64), _randn(2, 4, 1, 64), torch.arange(4, device=DEV)
    for bad in (lambda: r(q, k[:3], p), lambda: r(q, k.half(), p), lambda: r(q[..., :32], k[..., :32], p), lambda: r(q, k, p[:3]),
                lambda: r(q, k, p.float()), lambda: r(q, k, p.cpu()), lambda: r(q[0], k[0], p[:1]),
                lambda: da.Rotary(f.double()), lambda: da.Rotary(f[None]), lambda: da.Rotary(f[:0])):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        r(q.double(), k.double(), p)
    with pytest.raises(RuntimeError, match="CUDA"):
        r(q.cpu(), k.cpu(), p)


# ------------------------------------------------------------------ pools -----

def _pool(seed, lengths, hk, page, d, dtype, layout="heads", poison=True, window=0, spare=3):
    """A pool with random tokens where sequences have them and NaN or infinities everywhere else, its table (entries that no
    token needs: -1 or far outside) and the sequences' keys and values (hk, n, d) in 64 bits"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pages_of = [-(-n // page) for n in lengths]
    total = sum(pages_of) + spare
    ids = torch.randperm(total, generator=g, device=DEV)
    fill = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV) if poison else torch.zeros(3, device=DEV)
    shape = (hk, total, page, 2, d)
    pool = fill[torch.randint(3, shape, generator=g, device=DEV)].to(dtype)
    if layout == "pages":        # every page holds all its heads
        pool = pool.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "gaps":       # pages and heads at a distance
        pool = torch.full((hk + 1, 2 * total, page, 2, d), float("nan"), dtype=dtype, device=DEV)[:hk, ::2].copy_(pool)
    table = torch.full((len(lengths), max(pages_of + [1]) + 2), -1, dtype=torch.int32, device=DEV)
    table[:, -1] = 2 ** 31 - 1
    keys, values, at = [], [], 0
    for b, n in enumerate(lengths):
        table[b, :pages_of[b]] = ids[at:at + pages_of[b]].int()
        at += pages_of[b]
        k = torch.randn(hk, n, d, generator=g, device=DEV).to(dtype)
        v = torch.randn(hk, n, d, generator=g, device=DEV).to(dtype)
        first = max(0, n - window) if window else 0
        t = torch.arange(first, n, device=DEV)
        place = table[b].long()[t // page] if n else t
        for h in range(hk):
            pool[h][place, t % page, 0] = k[h, first:]
            pool[h][place, t % page, 1] = v[h, first:]
        if window and first // page > 0:
            table[b, :first // page] = -7             # pages in front of the window may be gone
        keys.append(k.double())
        values.append(v.double())
    return pool, table, keys, values


def _attention(q, keys, values, window, scale):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits from the keys and values of every sequence"""
    n_seq, hq, d = q.shape
    u = HALF_STEP[q.dtype]
    u_w = 0.0 if q.dtype == torch.float32 else u
    out, lse = torch.zeros(n_seq, hq, d, dtype=torch.float64, device=DEV), torch.full((n_seq, hq), -float("inf"), dtype=torch.float64, device=DEV)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(n_seq):
        hk, n, _ = keys[b].shape
        if n == 0:
            continue
        first = max(0, n - window) if window else 0
        k, v = keys[b][:, first:], values[b][:, first:]
        x = q[b].double().reshape(hk, hq // hk, d)
        s = x @ k.transpose(1, 2) * scale
        size = (x.abs() @ k.abs().transpose(1, 2)).amax(-1) * abs(scale)       # (hk, rep)
        w = torch.softmax(s, -1)
        o = w @ v
        e = (d + 8) * 2.0 ** -23 * size + (n / 16 + 64) * 2.0 ** -23
        mean = w @ v.abs()
        out[b] = o.reshape(hq, d)
        lse[b] = torch.logsumexp(s, -1).reshape(hq)
        tol[b] = (mean * (u_w + 2 * e)[..., None] + u * (o.abs() + mean * 2 * (u_w + e)[..., None])).reshape(hq, d)
        tol_lse[b] = (e + 2.0 ** -22 * (1 + lse[b].reshape(hk, -1).abs())).reshape(hq)
    if q.dtype == torch.float16:
        tol += 2.0 ** -25
    return out, lse, tol, tol_lse


def _assert_attended(got, want, tol):
    assert bool(torch.isfinite(got).all())
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


# -------------------------------------------------------------- attention -----

RAGGED = [1, 0, 16, 17, 15, 700, 0, 33, 2, 129]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,hk,rep,page,lengths", [
    (128, 8, 4, 16, RAGGED), (64, 2, 1, 16, [1]), (64, 1, 8, 5, RAGGED), (80, 3, 7, 24, RAGGED), (96, 2, 12, 32, RAGGED),
    (256, 2, 2, 1, [40, 3, 0]), (256, 1, 16, 100, [1000, 99, 100, 101]), (128, 1, 32, 16, RAGGED), (64, 1, 71, 8, [300, 9]),
    (128, 2, 17, 64, [64, 65, 0, 1]), (128, 1, 4, 16, [20011]), (128, 8, 4, 16, [4096, 5000]), (96, 3, 5, 24, [6000, 0, 1]),
    (80, 1, 9, 7, [2, 9000]), (64, 4, 3, 128, list(range(0, 90))), (256, 3, 6, 16, [3333, 17]),
])
def test_attention(da, dtype, d, hk, rep, page, lengths):
    pool, table, keys, values = _pool(d + rep, lengths, hk, page, d, dtype)
    q = _randn(31, len(lengths), hk * rep, d, dtype=dtype)
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, table, n, return_lse=True)
    cache.check_status()
    want, want_lse, tol, tol_lse = _attention(q, keys, values, 0, d ** -0.5)
    _assert_attended(out, want, tol)
    empty = (n == 0)
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == -float("inf")).all())
    _assert_attended(lse[~empty], want_lse[~empty], tol_lse[~empty])
    assert torch.equal(cache.attend(q, table, n), out)         # the same bits, with and without the log-sum-exp


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("batch,hk,rep,long", [
    (1, 2, 3, 9000),      # few rows, each in hundreds of parts
    (9, 3, 5, 2100),      # 135 rows
    (16, 4, 5, 900),      # 320
    (40, 4, 4, 500),      # 640
    (5, 7, 17, 600),      # rows in several groups, 595 of them
])
def test_attention_with_few_rows_and_many(da, dtype, d, batch, hk, rep, long):
    """The number of rows decides how the parts of an item are joined; lengths from none to long, so that items have from one part to many."""
    lengths = [(long, 0, 17, long // 2, 1, long // 3)[i % 6] for i in range(batch)]
    pool, table, keys, values = _pool(91, lengths, hk, 16, d, dtype)
    q = _randn(92, batch, hk * rep, d, dtype=dtype)
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(q, table, n, return_lse=True)
    cache.check_status()
    want, want_lse, tol, tol_lse = _attention(q, keys, values, 0, d ** -0.5)
    _assert_attended(out, want, tol)
    empty = n == 0
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == -float("inf")).all())
    _assert_attended(lse[~empty], want_lse[~empty], tol_lse[~empty])
    again, lse_again = cache.attend(q, table, n, return_lse=True)
    assert torch.equal(again, out) and torch.equal(lse_again, lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 15, 16, 100, 513, 10 ** 6])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_in_a_window(da, dtype, window, page):
    lengths = [1, 16, 17, 0, 600, 513, 101, 2500]
    pool, table, keys, values = _pool(window, lengths, 2, page, 64, dtype, window=window)
    q = _randn(32, len(lengths), 6, 64, dtype=dtype)
    cache = da.PagedKVCache.over(pool)
    out = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window)
    cache.check_status()
    want, _, tol, _ = _attention(q, keys, values, window, 0.125)
    _assert_attended(out, want, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["pages", "gaps"])
def test_attention_over_other_pool_layouts(da, dtype, layout):
    lengths = [50, 301, 16]
    pool, table, keys, values = _pool(5, lengths, 3, 16, 64, dtype, layout=layout)
    wide = _randn(33, 3, 15, 64, dtype=dtype)
    q = wide[:, 2:14]                                            # heads of a fused projection
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out = cache.attend(q, table, n, scale=0.3)
    want, _, tol, _ = _attention(q, keys, values, 0, 0.3)
    _assert_attended(out, want, tol)
    odd = torch.empty(3 * 12 * 64 + 1, dtype=dtype, device=DEV)[1:].view(3, 12, 64).copy_(q)     # between 16-byte boundaries
    assert torch.equal(cache.attend(odd, table, n, scale=0.3), out)
    apart = torch.empty(3, 12, 128, dtype=dtype, device=DEV)[..., ::2].copy_(q)
    assert torch.equal(cache.attend(apart, table, n, scale=0.3), out)
    wider = torch.full((6, table.shape[1] + 5), 12345, dtype=torch.int32, device=DEV)
    wider[1:4, 2:-3] = table
    assert torch.equal(cache.attend(q, wider[1:4, 2:-3], n, scale=0.3), out)


def test_attention_where_sequences_share_pages(da):
    pool, table, keys, values = _pool(6, [64, 200], 2, 16, 128, torch.bfloat16)
    table[0, :4] = table[1, :4]                                  # a common prefix, read by both and twice by the third
    table = torch.cat([table, table[1:]])
    table[2, 4:8] = table[1, :4]
    keys = [keys[1][:, :64], keys[1], torch.cat([keys[1][:, :64], keys[1][:, :64]], 1)]
    values = [values[1][:, :64], values[1], torch.cat([values[1][:, :64], values[1][:, :64]], 1)]
    q = _randn(34, 3, 8, 128, dtype=torch.bfloat16)
    out = da.PagedKVCache.over(pool).attend(q, table, torch.tensor([64, 200, 128], dtype=torch.int32, device=DEV))
    want, _, tol, _ = _attention(q, keys, values, 0, 128 ** -0.5)
    _assert_attended(out, want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_with_large_logits(da, dtype):
    """Logits of some hundreds with one that stands out: the running maximum moves, most weights vanish."""
    lengths = [777, 40]
    pool, table, keys, values = _pool(7, lengths, 1, 16, 64, dtype)
    q = _randn(35, 2, 4, 64, dtype=dtype) * 4
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    for scale in (8.0, -8.0, 0.0):
        out = da.PagedKVCache.over(pool).attend(q, table, n, scale=scale)
        want, _, tol, _ = _attention(q, keys, values, 0, scale)
        _assert_attended(out, want, tol)


def test_bad_pages_and_lengths_are_left_out_and_reported(da):
    pool, table, keys, values = _pool(8, [100, 64, 30], 2, 16, 64, torch.bfloat16)
    cache = da.PagedKVCache.over(pool)
    q = _randn(36, 3, 4, 64, dtype=torch.bfloat16)
    n = torch.tensor([100, 64, 30], dtype=torch.int32, device=DEV)
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 1], bad[1, 2], bad[1, 3] = -5, pool.shape[1], 2 ** 31 - 1, -2 ** 31, -1
    out, lse = cache.attend(q, bad, n, return_lse=True)
    with pytest.raises(RuntimeError, match="page id"):
        cache.check_status()
    cache.check_status()                                          # reported once
    keep = [t for t in range(100) if t // 16 != 2]
    want, _, tol, _ = _attention(q[:1], [keys[0][:, keep]], [values[0][:, keep]], 0, 0.125)
    _assert_attended(out[:1], want, tol)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -float("inf")).all())     # a row whose tokens are all gone
    want, _, tol, _ = _attention(q[2:], keys[2:], values[2:], 0, 0.125)
    _assert_attended(out[2:], want, tol)

    capacity = 2 * 16
    out = cache.attend(q, table[:, :2].contiguous(), torch.tensor([-3, 64, 30], dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="outside the page table"):
        cache.check_status()
    assert bool((out[0] == 0).all())
    want, _, tol, _ = _attention(q[1:2], [keys[1][:, :capacity]], [values[1][:, :capacity]], 0, 0.125)
    _assert_attended(out[1:2], want, tol)


def test_attention_of_many_sequences_and_of_none(da):
    lengths = [(i * 37) % 70 for i in range(1000)]
    pool, table, keys, values = _pool(9, lengths, 1, 16, 64, torch.bfloat16)
    q = _randn(37, 1000, 4, 64, dtype=torch.bfloat16)
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out = cache.attend(q, table, n)
    want, _, tol, _ = _attention(q, keys, values, 0, 0.125)
    _assert_attended(out, want, tol)
    out, lse = cache.attend(q[:0], table[:0], n[:0], return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out = cache.attend(q, table, torch.zeros_like(n))
    assert bool((out == 0).all())
    cache.check_status()


@pytest.mark.parametrize("dtype", TYPES)
def test_one_long_sequence_among_many_short_ones(da, dtype):
    lengths = [3] * 300 + [20000] + [(i * 13) % 40 for i in range(400)]
    pool, table, keys, values = _pool(10, lengths, 2, 16, 64, dtype)
    q = _randn(44, len(lengths), 8, 64, dtype=dtype)
    cache = da.PagedKVCache.over(pool)
    out, lse = cache.attend(q, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), return_lse=True)
    cache.check_status()
    want, want_lse, tol, tol_lse = _attention(q, keys, values, 0, 0.125)
    _assert_attended(out, want, tol)
    some = torch.tensor(lengths, device=DEV) > 0
    _assert_attended(lse[some], want_lse[some], tol_lse[some])


def test_copied_and_saved_caches_work_on_their_own_pages(da):
    import copy
    import io
    cache = da.PagedKVCache(4, 16, 2, 64)
    table, one = torch.tensor([[2]], dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    k = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    cache.attend(k, table, one)
    twin = copy.deepcopy(cache)
    file = io.BytesIO()
    torch.save(cache, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=False)
    for other in (twin, loaded):
        other.append_(k, k, table, one)
        assert bool((other.attend(k, table, one) == 1).all()) and bool((other.pages[:, 2, 0] == 1).all())
    assert bool((cache.pages == 0).all()) and bool((cache.attend(k, table, one) == 0).all())
    with pytest.raises(AttributeError):
        cache.pages = twin.pages
    r = copy.deepcopy(da.Rotary(_frequencies(64)))
    assert r.rotary_dim == 64 and r(k[:, :, :], k, one)[0].shape == k.shape
    with pytest.raises(AttributeError):
        r.inv_freq = _frequencies(32)


def test_frequencies_changed_in_place_are_followed(da):
    f = _frequencies(64)
    r = da.Rotary(f)
    q, p = _randn(45, 5, 2, 64), torch.arange(5, device=DEV)
    r.inv_freq.mul_(0.5)
    _assert_turned(r(q, q, p)[0], q, p, _frequencies(64) * 0.5, 1.0, True)


def test_pool_of_more_than_2_to_31_elements(da):
    """Pages whose offset in elements passes 32 bits: appended to and attended to."""
    hk, page, d = 1, 16, 64
    n_pages = (2 ** 31 + 2 ** 28) // (page * 2 * d)
    cache = da.PagedKVCache.over(torch.empty(hk, n_pages, page, 2, d, dtype=torch.float16, device=DEV))
    table = torch.tensor([[n_pages - 1, 0, n_pages - 3], [n_pages - 2, 1, 2]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 40, 45], dtype=torch.int32, device=DEV)
    n = torch.tensor([40, 5], dtype=torch.int32, device=DEV)
    k, v = _randn(38, 45, hk, d, dtype=torch.float16), _randn(39, 45, hk, d, dtype=torch.float16)
    cache.append_(k, v, table, n, starts=starts)
    q = _randn(40, 2, 4, d, dtype=torch.float16)
    out = cache.attend(q, table, n)
    cache.check_status()
    part = lambda x: [x[:40].transpose(0, 1).double(), x[40:].transpose(0, 1).double()]
    want, _, tol, _ = _attention(q, part(k), part(v), 0, 0.125)
    _assert_attended(out, want, tol)


def test_page_of_more_than_a_million_tokens(da):
    """A contiguous cache per sequence is one page."""
    page, n = 1500001, 1499990
    pool = torch.empty(1, 2, page, 2, 256, dtype=torch.float16, device=DEV)
    k, v = _randn(48, 1, 300, 256, dtype=torch.float16), _randn(49, 1, 300, 256, dtype=torch.float16)
    pool[0, 1, n - 300:n, 0], pool[0, 1, n - 300:n, 1] = k[0], v[0]
    cache = da.PagedKVCache.over(pool)
    table, lengths = torch.tensor([[1]], dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    q = _randn(50, 1, 4, 256, dtype=torch.float16)
    out = cache.attend(q, table, lengths, window=300)
    cache.check_status()
    want, _, tol, _ = _attention(q, [k.double()], [v.double()], 0, 256 ** -0.5)
    _assert_attended(out, want, tol)
    cache.append_(k.transpose(0, 1), v.transpose(0, 1), table, lengths + 5, starts=torch.tensor([0, 300], dtype=torch.int32, device=DEV))
    assert torch.equal(pool[0, 1, n - 295:n + 5, 0], k[0])


# ----------------------------------------------------------------- append -----

def _append_reference(pool, table, lengths, starts, k, v, q, how):
    """What append_ leaves in the pool (64 bits, with slack) and returns"""
    page = pool.shape[2]
    want, slack = pool.double(), torch.zeros(pool.shape, dtype=torch.float64, device=DEV)
    q_want, q_slack = (None, None) if q is None else (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for b, n in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        if hi == lo or n == 0:
            continue
        position = torch.arange(n - (hi - lo), n, device=DEV)
        place, slot = table[b].long()[position // page], position % page
        rk, sk = (k[lo:hi].double(), torch.zeros_like(k[lo:hi], dtype=torch.float64)) if how is None else _turned(k[lo:hi], position, *how)
        for h in range(pool.shape[0]):
            want[h, place, slot, 0], slack[h, place, slot, 0] = rk[:, h], sk[:, h]
            want[h, place, slot, 1] = v[lo:hi, h].double()
        if q is not None:
            q_want[lo:hi], q_slack[lo:hi] = _turned(q[lo:hi], position, *how)
    return want, slack, q_want, q_slack


def _assert_within(got, want, slack):
    tol = slack + HALF_STEP[got.dtype] * (want.abs() + slack) * (slack > 0) + (2.0 ** -25 * (slack > 0) if got.dtype == torch.float16 else 0.0)
    err = (got.double() - want).abs()
    same = torch.isnan(want) & torch.isnan(got) | (got.double() == want)
    assert bool((same | (err <= tol)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,hq,hk,rot,page,before,new,layout", [
    (128, 32, 8, 128, 16, [0, 5, 16, 100], [1, 1, 1, 1], "heads"),
    (64, 4, 2, 64, 16, [0, 15, 16, 31, 0, 7], [17, 1, 0, 40, 0, 3], "heads"),
    (96, 6, 3, 32, 24, [3, 0, 50], [100, 1, 24], "pages"), (80, 5, 5, 34, 5, [2], [23], "heads"), (256, 2, 1, 256, 1, [0, 3], [2, 3], "gaps"),
    (128, 4, 4, 16, 64, [0], [1], "pages"),
])
def test_append(da, dtype, interleaved, d, hq, hk, rot, page, before, new, layout):
    after = [b + n for b, n in zip(before, new)]
    pool, table, _, _ = _pool(d, after, hk, page, d, dtype, layout=layout)
    starts = [4 + sum(new[:i]) for i in range(len(new) + 1)]      # four rows in front of the sequences, three behind
    rows = starts[-1] + 3
    fused = _randn(41, rows, hq + 2 * hk, d, dtype=dtype)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
    f = _frequencies(rot)
    n = torch.tensor(after, dtype=torch.int32, device=DEV)
    s = torch.tensor(starts, dtype=torch.int32, device=DEV)
    for rotary, queries in ((da.Rotary(f, factor=1.125, interleaved=interleaved), q), (None, None)):
        how = None if rotary is None else (f, 1.125, interleaved)
        want, slack, q_want, q_slack = _append_reference(pool, table, after, starts, k, v, queries, how)
        mine = pool.clone()
        if layout != "heads":
            mine = torch.empty_strided(pool.shape, pool.stride(), dtype=dtype, device=DEV).copy_(pool)
        cache = da.PagedKVCache.over(mine)
        out = cache.append_(k, v, table, n, starts=s, q=queries, rotary=rotary)
        cache.check_status()
        _assert_within(mine, want, slack)
        if queries is None:
            assert out is None
        else:
            _assert_within(out, q_want, q_slack)
            assert bool((out[:4] == 0).all()) and bool((out[-3:] == 0).all())
        if all(x == 1 for x in new):                              # the form without starts
            again = torch.empty_strided(pool.shape, pool.stride(), dtype=dtype, device=DEV).copy_(pool)
            cache = da.PagedKVCache.over(again)
            one = cache.append_(k[4:-3], v[4:-3], table, n, q=None if queries is None else queries[4:-3], rotary=rotary)
            assert torch.equal(again.view(torch.uint8), mine.view(torch.uint8)) if layout == "heads" else \
                torch.equal(again.nan_to_num(), mine.nan_to_num())
            assert one is None or torch.equal(one, out[4:-3])


def test_append_skips_what_is_not_in_use_and_reports_what_is_wrong(da):
    pool = _randn(42, 2, 6, 16, 2, 64, dtype=torch.bfloat16)
    table = torch.tensor([[0, 1], [2, 9], [-1, 3], [4, 5]], dtype=torch.int32, device=DEV)
    k, v, q = (_randn(43 + i, 4, h, 64, dtype=torch.bfloat16) for i, h in enumerate((2, 2, 4)))
    r = da.Rotary(_frequencies(64))
    cache = da.PagedKVCache.over(pool.clone())
    # rows not in use write nothing and are no mistake
    out = cache.append_(k, v, table, torch.tensor([0, 16, 20, 0], dtype=torch.int32, device=DEV), q=q, rotary=r)
    cache.check_status()
    assert bool((out[0] == 0).all()) and bool((out[3] == 0).all()) and bool((out[1] != 0).any())
    changed = (cache.pages != pool).flatten(3).any(-1).any(0)
    assert changed.nonzero().tolist() == [[2, 15], [3, 3]]
    # pages outside the pool: nothing is written for them, the queries are rotated all the same
    cache = da.PagedKVCache.over(pool.clone())
    good = da.PagedKVCache.over(pool.clone()).append_(k, v, torch.tensor([[0, 1]] * 4, dtype=torch.int32, device=DEV),
                                                      torch.tensor([1, 17, 1, 32], dtype=torch.int32, device=DEV), q=q, rotary=r)
    out = cache.append_(k, v, table, torch.tensor([1, 17, 1, 32], dtype=torch.int32, device=DEV), q=q, rotary=r)
    with pytest.raises(RuntimeError, match="page id"):
        cache.check_status()
    changed = (cache.pages != pool).flatten(3).any(-1).any(0)
    assert changed.nonzero().tolist() == [[0, 0], [5, 15]]
    assert torch.equal(out, good)
    # positions outside the table
    cache = da.PagedKVCache.over(pool.clone())
    out = cache.append_(k, v, table, torch.tensor([33, -1, 2 ** 31 - 1, 32], dtype=torch.int32, device=DEV), q=q, rotary=r)
    with pytest.raises(RuntimeError, match="outside the page table"):
        cache.check_status()
    assert bool((out[:3] == 0).all())
    changed = (cache.pages != pool).flatten(3).any(-1).any(0)
    assert changed.nonzero().tolist() == [[5, 15]]
    # more new tokens than the sequence has
    cache = da.PagedKVCache.over(pool.clone())
    cache.append_(k, v, table[:1], torch.tensor([2], dtype=torch.int32, device=DEV), starts=torch.tensor([0, 4], dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="outside the page table"):
        cache.check_status()
    changed = (cache.pages != pool).flatten(3).any(-1).any(0)
    assert changed.nonzero().tolist() == [[0, 0], [0, 1]]


def test_append_of_nothing(da):
    cache = da.PagedKVCache(4, 16, 2, 64)
    table, n = torch.zeros(0, 1, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    k, q = torch.ones(0, 2, 64, dtype=torch.bfloat16, device=DEV), torch.ones(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    r = da.Rotary(_frequencies(64))
    assert cache.append_(k, k, table, n, q=q, rotary=r).shape == (0, 4, 64)
    k, q = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=DEV), torch.ones(3, 4, 64, dtype=torch.bfloat16, device=DEV)
    out = cache.append_(k, k, table, n, starts=torch.zeros(1, dtype=torch.int32, device=DEV), q=q, rotary=r)
    assert bool((out == 0).all()) and bool((cache.pages == 0).all())


def test_paged_calls_refuse(da):
    cache = da.PagedKVCache(4, 16, 2, 64)
    table, n = torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    k, q = _randn(1, 3, 2, 64, dtype=torch.bfloat16), _randn(2, 3, 4, 64, dtype=torch.bfloat16)
    r = da.Rotary(_frequencies(64))
    wide = da.Rotary(_frequencies(128))
    s = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV)
    for bad in (lambda: cache.append_(k.float(), k, table, n), lambda: cache.append_(k, k[:2], table, n), lambda: cache.append_(k[:, :1], k, table, n),
                lambda: cache.append_(k[..., :32], k, table, n), lambda: cache.append_(k[:2], k[:2], table, n),
                lambda: cache.append_(k, k, table.long(), n), lambda: cache.append_(k, k, table, n.long()), lambda: cache.append_(k, k, table, n[:2]),
                lambda: cache.append_(k, k, table, n, starts=s[:3]), lambda: cache.append_(k, k, table, n, starts=s.long()),
                lambda: cache.append_(k, k, table, n, q=q), lambda: cache.append_(k, k, table, n, q=q[:2], rotary=r),
                lambda: cache.append_(k, k, table, n, rotary=wide), lambda: cache.append_(k, k, table.t(), n),
                lambda: cache.append_(k.clone().requires_grad_(), k, table, n),
                lambda: cache.attend(q[:2], table, n), lambda: cache.attend(q[:, :3], table, n), lambda: cache.attend(q.half(), table, n),
                lambda: cache.attend(q, table, n, window=-1), lambda: cache.attend(q.clone().requires_grad_(), table, n),
                lambda: cache.attend(q, table[:, :0], n), lambda: cache.attend(q[:, :0], table, n),
                lambda: da.PagedKVCache.over(torch.zeros(2, 4, 16, 2, 128, device=DEV)[..., :64]),
                lambda: da.PagedKVCache.over(torch.zeros(2 * 4 * 16 * 2 * 64 + 1, device=DEV)[1:].view(2, 4, 16, 2, 64)),
                lambda: da.PagedKVCache.over(torch.zeros(2, 0, 16, 2, 64, device=DEV))):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: cache.attend(q.cpu(), table, n), lambda: cache.attend(q, table.cpu(), n), lambda: cache.append_(k, k, table, n.cpu())):
        with pytest.raises(RuntimeError, match="CUDA"):
            bad()
    with pytest.raises(RuntimeError, match="outside"):
        cache.attend(_randn(3, 3, 2 * 300, 64, dtype=torch.bfloat16), table, n)      # more queries to a key than the kernels take
    with pytest.raises(TypeError):
        cache.attend(q, table, n, window=1.5)
    cache.attend(q, table, n, window=2 ** 62)
    with torch.no_grad():
        cache.attend(q.clone().requires_grad_(), table, n)
    cache.check_status()


# --------------------------------------------------------------- together -----

@pytest.mark.parametrize("dtype,d,rot,page,window", [(torch.bfloat16, 128, 128, 16, 0), (torch.float16, 96, 48, 24, 70), (torch.float32, 64, 64, 7, 0)])
def test_prompts_in_chunks_then_decode_steps(da, dtype, d, rot, page, window):
    """Three conversations: prompts arrive in two ragged calls, then tokens one by one, the third row joining late; every
    step's output is the attention over all keys rotated by their positions."""
    hq, hk, steps = 8, 2, 6
    chunks = [[30, 7, 0], [41, 0, 0]]
    f = _frequencies(rot)
    r = da.Rotary(f, factor=1.1, interleaved=False)
    cache = da.PagedKVCache(40, page, hk, d, dtype=dtype)
    table = torch.randperm(39, generator=torch.Generator().manual_seed(0))[:39].view(3, 13).int().to(DEV)
    lengths = torch.zeros(3, dtype=torch.int32, device=DEV)
    given = [([], []) for _ in range(3)]                # keys before their rotation, values

    def remember(b, k, v):
        given[b][0].append(k)
        given[b][1].append(v)

    def cached(b, n):
        """The sequence's rows in the pool, checked against what was given: (hk, n, d) keys and values"""
        t = torch.arange(n, device=DEV)
        rows = cache.pages[:, table[b].long()[t // page], t % page]
        if n:
            _assert_turned(rows[:, :, 0].transpose(0, 1), torch.cat(given[b][0]), t, f, 1.1, False)
            assert torch.equal(rows[:, :, 1].transpose(0, 1), torch.cat(given[b][1]))
        return rows[:, :, 0].double(), rows[:, :, 1].double()

    for i, new in enumerate(chunks):
        k, v = _randn(50 + i, sum(new), hk, d, dtype=dtype), _randn(60 + i, sum(new), hk, d, dtype=dtype)
        starts = [0, new[0], new[0] + new[1], sum(new)]
        for b in range(3):
            remember(b, k[starts[b]:starts[b + 1]], v[starts[b]:starts[b + 1]])
        lengths += torch.tensor(new, dtype=torch.int32, device=DEV)
        cache.append_(k, v, table, lengths, starts=torch.tensor(starts, dtype=torch.int32, device=DEV), rotary=r)
    for step in range(steps):
        joined = torch.tensor([1, 1, int(step >= 3)], dtype=torch.int32, device=DEV)
        lengths += joined
        k, v, q = (_randn(70 + 10 * i + step, 3, h, d, dtype=dtype) for i, h in enumerate((hk, hk, hq)))
        for b in range(3):
            if joined[b]:
                remember(b, k[b:b + 1], v[b:b + 1])
        q2 = cache.append_(k, v, table, lengths, q=q, rotary=r)
        out = cache.attend(q2, table, lengths, window=window)
        cache.check_status()
        rows = [cached(b, n) for b, n in enumerate(lengths.tolist())]
        want, _, tol, _ = _attention(q2, [x[0] for x in rows], [x[1] for x in rows], window, d ** -0.5)
        _assert_attended(out, want, tol)


def test_captured_step_follows_lengths_and_table(da):
    hq, hk, d, page = 8, 2, 128, 16
    r = da.Rotary(_frequencies(d))
    n_steps = 20
    q, k, v = (_randn(80 + i, n_steps, 4, h, d, dtype=torch.bfloat16) for i, h in enumerate((hq, hk, hk)))
    start = torch.tensor([300, 0, 15, 1000], dtype=torch.int32, device=DEV)
    table = torch.randperm(400, generator=torch.Generator().manual_seed(1))[:4 * 70].view(4, 70).int().to(DEV)
    prefix = _randn(90, hk, 400, page, 2, d, dtype=torch.bfloat16)

    def run(captured):
        cache = da.PagedKVCache.over(prefix.clone())
        lengths = start.clone()
        inputs = [x[0].clone() for x in (q, k, v)]

        def step():
            lengths.add_(1)
            q2 = cache.append_(inputs[1], inputs[2], table, lengths, q=inputs[0], rotary=r)
            return cache.attend(q2, table, lengths)

        outs = []
        if captured:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                step()
            torch.cuda.current_stream().wait_stream(stream)
            lengths.copy_(start)
            cache.pages.copy_(prefix)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        for i in range(n_steps):
            for x, y in zip(inputs, (q, k, v)):
                x.copy_(y[i])
            if captured:
                graph.replay()
                outs.append(out.clone())
            else:
                outs.append(step())
        cache.check_status()
        return torch.stack(outs), cache.pages

    eager, pages_eager = run(False)
    graph, pages_graph = run(True)
    assert torch.equal(eager, graph) and torch.equal(pages_eager, pages_graph)


def test_two_captured_graphs_run_side_by_side(da):
    lengths = [3000, 500, 0, 9000]
    pool, table, _, _ = _pool(91, lengths, 2, 16, 128, torch.bfloat16)
    cache = da.PagedKVCache.over(pool)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    qs = [_randn(92 + i, 4, 16, 128, dtype=torch.bfloat16) for i in range(2)]
    want = [cache.attend(q, table, n) for q in qs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in qs], [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.attend(q, table, n))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(50):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # and eagerly on two streams
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    results = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[i].append(cache.attend(qs[i], table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in results[i])


def test_captured_rotation_with_its_gradient(da):
    f = _frequencies(64)
    r = da.Rotary(f, interleaved=False)
    positions = torch.arange(9, device=DEV, dtype=torch.int32)
    q, k = _randn(95, 9, 4, 64).requires_grad_(), _randn(96, 9, 2, 64).requires_grad_()
    w = _randn(97, 9, 4, 64)

    def step():
        a, b = r(q, k, positions)
        return (a,) + torch.autograd.grad((a * w).sum() + b.sum(), (q, k))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        q.mul_(2.0)
        positions.add_(5)
    graph.replay()
    for a, b in zip(captured, step()):
        assert torch.equal(a, b)


def test_slot_table_of_the_lru_cache_is_a_pool(da):
    """What the LRU cache has resident, attended to by the paged call, is what its own views hold."""
    hk, d, page = 2, 64, 16
    k, v = _randn(98, hk, 1024, d, dtype=torch.bfloat16), _randn(99, hk, 1024, d, dtype=torch.bfloat16)
    lru = da.LRUCache(k_cache=k, v_cache=v, page_size=page, top_k=4, lru_hbm_cache_size=512)
    pool = lru.hbm_kv_cache.view(hk, -1, page, 2, d)
    cache = da.PagedKVCache.over(pool)
    table = torch.arange(32, dtype=torch.int32, device=DEV)[None]
    q = _randn(100, 1, 8, d, dtype=torch.bfloat16)
    out = cache.attend(q, table, torch.tensor([500], dtype=torch.int32, device=DEV))
    want, _, tol, _ = _attention(q, [pool[:, :, :, 0].reshape(hk, 512, d)[:, :500].double()], [pool[:, :, :, 1].reshape(hk, 512, d)[:, :500].double()], 0, 0.125)
    _assert_attended(out, want, tol)


def test_on_another_device_than_the_current_one(da):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    with torch.cuda.device(0):
        cache = da.PagedKVCache(4, 16, 2, 64, device="cuda:1")
        one = torch.ones(1, dtype=torch.int32, device="cuda:1")
        table = torch.zeros(1, 1, dtype=torch.int32, device="cuda:1")
        k = torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda:1")
        cache.append_(k, k, table, one)
        assert bool((cache.attend(k, table, one) == 1).all())
        with pytest.raises(AssertionError, match="device"):
            cache.append_(k.to("cuda:0"), k, table, one)
