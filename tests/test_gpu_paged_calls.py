"""GPU tests of how the paged-cache operators are called: derivatives in forward mode, inputs that need none, reports of calls on
other streams, the documented decode step."""

import pytest
import torch
from torch.autograd import forward_ad

from tests.test_gpu_paged import DEV, _frequencies, _randn, da  # noqa: F401

pytestmark = pytest.mark.gpu


def _rotation(da, **how):
    return da.Rotary(_frequencies(64), factor=1.25, **how), torch.arange(5, device=DEV) * 1001


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_forward_mode_derivatives_of_the_rotation(da, dtype, interleaved):
    """Linear in q and k: the tangents are rotated like the heads, bit by bit."""
    r, p = _rotation(da, interleaved=interleaved)
    q, k, tq, tk = (_randn(s, 5, h, 64, dtype=dtype) for s, h in ((1, 4), (2, 2), (3, 4), (4, 2)))
    want, want_t = r(q, k, p), r(tq, tk, p)
    apart = _randn(5, 5, 4, 128, dtype=dtype)[..., ::2]
    for grad in (False, True):
        with forward_ad.dual_level():
            a, b = (x.clone().requires_grad_(grad) for x in (q, k))
            both = r(forward_ad.make_dual(a, tq), forward_ad.make_dual(b, tk), p)
            for got, x, t in zip(both, want, want_t):
                primal, tangent = forward_ad.unpack_dual(got)
                assert torch.equal(primal, x) and torch.equal(tangent, t)
            # one side alone
            one = r(forward_ad.make_dual(a, tq), b, p)
            assert torch.equal(forward_ad.unpack_dual(one[0]).tangent, want_t[0])
            rest = forward_ad.unpack_dual(one[1]).tangent
            assert rest is None or bool((rest == 0).all())
            other = r(a, forward_ad.make_dual(b, tk), p)
            assert torch.equal(forward_ad.unpack_dual(other[1]).tangent, want_t[1]) and torch.equal(other[0].detach(), want[0])
            # tangents with gaps between their channels, and under no_grad
            with torch.no_grad():
                strided = r(forward_ad.make_dual(a.detach(), apart), b.detach(), p)[0]
            assert torch.equal(forward_ad.unpack_dual(strided).tangent, r(apart, k, p)[0])


def test_forward_mode_through_the_gradient_and_back(da):
    """Forward over reverse and reverse over forward: with y = R q and a loss of |y|^2 / 2 the gradient is f^2 q, its derivative
    along t is f^2 t; the sum of R t against w has R^T w as its gradient in t."""
    r, p = _rotation(da)
    q, k, t, w = _randn(1, 5, 4, 64), _randn(2, 5, 2, 64), _randn(3, 5, 4, 64), _randn(4, 5, 4, 64)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(q.clone().requires_grad_(), t)
        y, _ = r(x, k, p)
        (g,) = torch.autograd.grad((y * y).sum() / 2, x)
        got = forward_ad.unpack_dual(g).tangent
        # two rotations, each off by at most 8 * 2^-24 of the sum of the pair's magnitudes times the factor
        size = (t.unflatten(-1, (32, 2)).abs().sum(-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)).double()
        assert bool(((got.double() - 1.5625 * t.double()).abs() <= 2 * 16 * 2.0 ** -24 * 1.5625 * size).all())
    with forward_ad.dual_level():
        s = t.clone().requires_grad_()
        y, _ = r(forward_ad.make_dual(q, s), k, p)
        (g,) = torch.autograd.grad((forward_ad.unpack_dual(y).tangent * w).sum(), s)
    a = q.clone().requires_grad_()
    (want,) = torch.autograd.grad((r(a, k, p)[0] * w).sum(), a)
    assert torch.equal(g, want)


def test_function_transforms_are_refused(da):
    """What the rotation has no rule for ends in an error, never in a derivative of zero."""
    r, p = _rotation(da)
    q, k = _randn(1, 5, 4, 64), _randn(2, 5, 2, 64)
    for call in (lambda: torch.func.jvp(lambda x: r(x, k, p)[0], (q,), (q,)), lambda: torch.func.grad(lambda x: r(x, k, p)[0].sum())(q),
                 lambda: torch.func.vmap(lambda x: r(x, k, p)[0])(q[None])):
        with pytest.raises(Exception):
            call()


def test_tangents_are_refused_where_nothing_passes_them_on(da):
    cache = da.PagedKVCache(4, 16, 2, 64)
    table, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    k, q = _randn(1, 1, 2, 64, dtype=torch.bfloat16), _randn(2, 1, 4, 64, dtype=torch.bfloat16)
    r = da.Rotary(_frequencies(64))
    with forward_ad.dual_level():
        dk, dq = forward_ad.make_dual(k, k), forward_ad.make_dual(q, q)
        for bad in (lambda: cache.append_(dk, k, table, n), lambda: cache.append_(k, dk, table, n),
                    lambda: cache.append_(k, k, table, n, q=dq, rotary=r), lambda: cache.attend(dq, table, n)):
            with pytest.raises(AssertionError, match="tangent"):
                bad()
            with torch.no_grad(), pytest.raises(AssertionError, match="tangent"):
                bad()
        assert bool((cache.pages == 0).all())
        cache.append_(k, k, table, n)
        cache.attend(q, table, n)
    cache.check_status()


def test_an_input_that_needs_no_gradient_has_an_output_that_needs_none(da):
    """Frozen keys beside trained queries: their rotation can be appended to a cache like any other."""
    r, p = _rotation(da)
    q, k = _randn(1, 5, 4, 64).requires_grad_(), _randn(2, 5, 2, 64)
    q2, k2 = r(q, k, p)
    assert q2.requires_grad and not k2.requires_grad
    cache = da.PagedKVCache(1, 16, 2, 64, dtype=torch.float32)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    cache.append_(k2, k, torch.zeros(1, 1, dtype=torch.int32, device=DEV), starts[1:], starts=starts)
    assert torch.equal(cache.pages[:, 0, :5, 0].transpose(0, 1), r(q, k, p)[1])
    q2, k2 = r(q.detach(), k.requires_grad_(), p)
    assert k2.requires_grad and not q2.requires_grad


def test_status_of_calls_on_other_streams(da):
    cache = da.PagedKVCache(4, 16, 2, 64)
    bad, n = torch.full((1, 1), 9, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    q = torch.ones(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)            # (some 50 ms: the call has not run when its report is asked for)
            cache.attend(q, bad, n)
        with pytest.raises(RuntimeError, match="page id"):
            cache.check_status()
    cache.check_status()
    # asked for on a busy stream, reported on another: nothing that comes after the report is erased by it
    with torch.cuda.stream(side):
        cache.attend(q, bad, n)
    with pytest.raises(RuntimeError, match="page id"):
        cache.check_status()
    with torch.cuda.stream(side):
        cache.attend(q, bad, n)
    side.synchronize()
    with pytest.raises(RuntimeError, match="page id"):
        cache.check_status()
    cache.check_status()


def test_documented_decode_step_leaves_rows_alone_that_are_not_in_use(da):
    """lengths.add_(lengths.sign()): rows of length 0 stay so, whatever their table holds; one joins by its prompt."""
    cache = da.PagedKVCache(8, 16, 2, 64)
    r = da.Rotary(_frequencies(64))
    table = torch.tensor([[0, 1], [1, 0], [-1, -1], [2, 3]], dtype=torch.int32, device=DEV)     # rows 1 and 2 are free, 1 with an old entry
    lengths = torch.zeros(4, dtype=torch.int32, device=DEV)
    prompt = _randn(1, 25, 2, 64, dtype=torch.bfloat16)
    lengths[0], lengths[3] = 20, 5
    cache.append_(prompt, prompt, table, lengths, starts=torch.tensor([0, 20, 20, 20, 25], dtype=torch.int32, device=DEV), rotary=r)
    k, q = _randn(2, 4, 2, 64, dtype=torch.bfloat16), _randn(3, 4, 4, 64, dtype=torch.bfloat16)

    def step():
        lengths.add_(lengths.sign())
        return cache.attend(cache.append_(k, k, table, lengths, q=q, rotary=r), table, lengths)

    kept = cache.pages.clone()
    out = step()
    cache.check_status()
    assert lengths.tolist() == [21, 0, 0, 6] and bool((out[1:3] == 0).all()) and bool((out[0] != 0).any())
    assert (cache.pages != kept).flatten(3).any(-1).any(0).nonzero().tolist() == [[1, 4], [2, 5]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    table[1], lengths[1] = torch.tensor([4, 5], dtype=torch.int32, device=DEV), 3
    cache.append_(prompt[:3], prompt[:3], table[1:2], lengths[1:2], starts=torch.tensor([0, 3], dtype=torch.int32, device=DEV), rotary=r)
    graph.replay()
    cache.check_status()
    assert lengths.tolist() == [22, 4, 0, 7]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [5, 3000])
def test_queries_and_keys_that_are_both_copied_for_the_call(da, dtype, tokens):
    """Channels at a distance: the copies of q and k live side by side until the rotation is enqueued, forwards and backwards."""
    r, p = da.Rotary(_frequencies(64)), torch.arange(tokens, device=DEV)
    apart = lambda seed: _randn(seed, tokens, 4, 128, dtype=dtype)[..., ::2]
    q, k, dq, dk = (apart(s) for s in range(1, 5))
    dense = [x.contiguous() for x in (q, k, dq, dk)]
    want, want_g = r(dense[0], dense[1], p), r(dense[2], dense[3], -p)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(r(q, k, p), want))
        assert all(torch.equal(a, b) for a, b in zip(r(q, dense[1], p), want)) and all(torch.equal(a, b) for a, b in zip(r(dense[0], k, p), want))
    x, y = dense[0].clone().requires_grad_(), dense[1].clone().requires_grad_()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(r(x, y, p), (x, y), (dq, dk)), want_g))
    # gradients that are one number for every element
    ones = torch.autograd.grad(r(x, y, p), (x, y), (torch.ones((), dtype=dtype, device=DEV).expand(x.shape), torch.zeros((), dtype=dtype, device=DEV).expand(y.shape)))
    assert torch.equal(ones[0], r(torch.ones_like(x), y, -p)[0].detach()) and bool((ones[1] == 0).all())


def test_heads_and_gradients_that_are_negated_lazily(da):
    """Imaginary parts of conjugates share memory with what they are the negative of; gradients arrive in that form too."""
    r, p = _rotation(da)
    real = lambda seed, *shape: _randn(seed, *shape)
    zq, zk = torch.complex(real(1, 5, 4, 64), real(2, 5, 4, 64)), torch.complex(real(3, 5, 2, 64), real(4, 5, 2, 64))
    apart = lambda z: z.conj().imag                                       # every second word
    dense = lambda x: torch._neg_view(x)
    for q, k in ((apart(zq), apart(zk)), (dense(zq.imag.contiguous()), dense(zk.imag.contiguous()))):
        assert q.is_neg() and k.is_neg()
        for a, b in zip(r(q, k, p), r(-zq.imag, -zk.imag, p)):
            assert torch.equal(a, b)
    q, k = zq.real.contiguous().requires_grad_(), zk.real.contiguous().requires_grad_()
    dq, dk = dense(real(5, 5, 4, 64)), dense(real(6, 5, 2, 64))
    got = torch.autograd.grad(r(q, k, p), (q, k), (dq, dk))
    want = torch.autograd.grad(r(q, k, p), (q, k), (dq.resolve_neg(), dk.resolve_neg()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # as it comes about: the conjugate of what was rotated
    (got,) = torch.autograd.grad(torch.complex(r(q, k, p)[0], r(q, k, p)[0]).conj().imag.sum(), (q,))
    (want,) = torch.autograd.grad(-r(q, k, p)[0].sum(), (q,))
    assert torch.equal(got, want)
    with forward_ad.dual_level():
        out = r(forward_ad.make_dual(q.detach(), dq), forward_ad.make_dual(k.detach(), torch._efficientzerotensor(k.shape, device=DEV)), p)
        assert torch.equal(forward_ad.unpack_dual(out[0]).tangent, r(dq.resolve_neg(), k, p)[0])
        assert bool((forward_ad.unpack_dual(out[1]).tangent == 0).all())
    # and in the cache
    q, k = zq.imag.contiguous(), zk.imag.contiguous()
    starts = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    caches = [da.PagedKVCache(1, 16, 2, 64, dtype=torch.float32) for _ in range(2)]
    outs = []
    for cache, a, b in ((caches[0], dense(q), dense(k)), (caches[1], -q, -k)):
        outs.append((cache.append_(b, b, table, starts[1:], starts=starts, q=a, rotary=r), cache.attend(a[:1], table, starts[1:])))
    assert torch.equal(caches[0].pages, caches[1].pages) and all(torch.equal(a, b) for a, b in zip(*outs))
