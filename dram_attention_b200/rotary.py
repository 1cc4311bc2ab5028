"""Rotary positions by inverse frequencies: both pairings of the channels, all of the head or part of it, frequencies
stretched to long contexts, with gradients.  (`DRAMAttention.rotate_` is the reference caller's own form: the whole head
in adjacent pairs, from a table of complex factors.)"""

from __future__ import annotations

import math
from typing import Mapping, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[Mapping] = None,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """Inverse frequencies base^(-2i / rotary_dim), float32 (rotary_dim / 2,), and the amplitude that goes with them
    (1 unless the scaling changes it): the two arguments of `Rotary`.  Computed in 64 bits, rounded once.

    `scaling`, for contexts longer than the model was trained on (`factor` times as long):
        {"type": "linear", "factor": f}   every position divided by f
        {"type": "ntk", "factor": f}      the base raised so that the slowest pair turns f times slower and the fastest as before
        {"type": "llama3", "factor": f, "original_length": n, "low": 1.0, "high": 4.0}
            pairs that turn fewer than `low` times in n tokens are slowed by f, those that turn more than `high` times
            not at all, in between linearly in the number of turns
        {"type": "yarn", "factor": f, "original_length": n, "fast": 32.0, "slow": 1.0, "attention_factor": None}
            the same idea, linear in the index of the pair between the ones that turn `fast` and `slow` times; amplitude
            0.1 ln f + 1 unless `attention_factor` is given
    """
    assert rotary_dim >= 2 and rotary_dim % 2 == 0, f"rotary_dim must be even and at least 2, got {rotary_dim}"
    assert base > 1, f"base must be above 1, got {base}"
    scaling = dict(scaling or {"type": "none"})
    kind = scaling.pop("type")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    amplitude = 1.0
    if kind != "none":
        factor = float(scaling.pop("factor"))
        assert factor > 0, f"factor must be positive, got {factor}"
    if kind == "ntk":
        assert rotary_dim > 2, "ntk scaling needs more than one channel pair"
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-2.0 * i / rotary_dim)
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        n, low, high = float(scaling.pop("original_length")), float(scaling.pop("low", 1.0)), float(scaling.pop("high", 4.0))
        assert n > 0 and high > low, "llama3 scaling needs original_length > 0 and high > low"
        keep = ((n * inv / (2.0 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1.0 - keep)
    elif kind == "yarn":
        n, fast, slow = float(scaling.pop("original_length")), float(scaling.pop("fast", 32.0)), float(scaling.pop("slow", 1.0))
        assert n > 0 and fast > slow > 0, "yarn scaling needs original_length > 0 and fast > slow > 0"
        index = lambda turns: rotary_dim * math.log(n / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        first, last = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
        slowed = ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1.0 - slowed) + inv / factor * slowed
        given = scaling.pop("attention_factor", None)
        amplitude = (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0) if given is None else float(given)
    else:
        assert kind in ("none", "ntk"), f"unknown scaling type {kind!r}"
    assert not scaling, f"unknown entries of {kind} scaling: {sorted(scaling)}"
    return inv.to(torch.float32).to(device), amplitude


class Rotary:
    """Rotary positions with the given inverse frequencies.

    Args:
        inv_freq: float32 (rotary_dim / 2,) on a CUDA device; `rotary_frequencies` makes them.  Its values may be changed in
            place between calls, e.g. for frequencies that follow the length.
        factor: amplitude of the rotated channels.
        interleaved: channel pairs (2i, 2i + 1); otherwise (i, i + rotary_dim / 2).

    Angles are formed and reduced in 64 bits, so far positions keep the accuracy of near ones; the arithmetic is float32,
    rounded once to the type of the heads."""

    def __init__(self, inv_freq: torch.Tensor, factor: float = 1.0, interleaved: bool = True):
        _native.require_cuda(inv_freq, "inv_freq")
        assert inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.numel() > 0, \
            f"inv_freq must be a float32 vector, got {tuple(inv_freq.shape)} {inv_freq.dtype}"
        _native.lib()
        self._inv_freq = inv_freq.detach().resolve_neg().contiguous()
        self._rotary_dim = 2 * inv_freq.numel()
        self.factor = float(factor)
        self.interleaved = bool(interleaved)

    @property
    def inv_freq(self) -> torch.Tensor:
        return self._inv_freq

    @property
    def rotary_dim(self) -> int:
        return self._rotary_dim

    def __call__(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor):
        """q (s, Hq, D) or (b, s, Hq, D), k the same with its own number of heads; positions int32 or int64, (s,) or (b, s),
        magnitudes below 2^31.  Channels from rotary_dim on pass unchanged.  Returns the rotated pair (new tensors);
        differentiable in q and k, backwards and in forward mode; the output of one that needs no derivative needs none.  (As
        with every differentiable call: let go of results of eager calls on the same leaves before a call and its backward pass are
        captured into a graph, torch ties the leaves' gradients to the eager stream.)"""
        qs, ks, device = q.shape, k.shape, q.get_device()
        lead = len(qs) - 2
        assert 1 <= lead <= 2 and len(ks) == lead + 2 and ks[0] == qs[0] and ks[lead - 1] == qs[lead - 1] and ks[-1] == qs[-1], \
            f"q (..., heads, D) and k (..., heads, D) do not go together: {tuple(qs)}, {tuple(ks)}"
        if device < 0:
            _native.require_cuda(q, "q")
        assert k.dtype is q.dtype, "q and k must have the same dtype"
        assert self._rotary_dim <= qs[-1] <= 512, \
            f"head_dim must lie between rotary_dim ({self.rotary_dim}) and 512, got {qs[-1]}"
        assert positions.dtype in _POSITION_TYPES, f"positions must be int32 or int64, got {positions.dtype}"
        if positions.shape != qs[:lead]:
            assert positions.shape == qs[lead - 1:lead], \
                f"positions must be {tuple(qs[:lead])} or {tuple(qs[lead - 1:lead])}, got {tuple(positions.shape)}"
            positions = positions.expand(qs[:lead])
        inv_freq = self._inv_freq
        assert k.get_device() == positions.get_device() == inv_freq.get_device() == device, \
            f"k ({k.device}), positions ({positions.device}) and inv_freq ({inv_freq.device}) must be on the device of q ({q.device})"
        if q.requires_grad or k.requires_grad or forward_ad._current_level >= 0:
            by_q, by_k = _derives(q), _derives(k)
            if by_q or by_k:
                q2, k2 = _Rotate.apply(q, k, positions, inv_freq, self.factor, self.interleaved, False)
                # (the function gives both outputs a place in the graph)
                return q2 if by_q else q2.detach(), k2 if by_k else k2.detach()
        return _rotate(q, k, positions, inv_freq, self.factor, self.interleaved, False)


_POSITION_TYPES = (torch.int32, torch.int64)
_NOTHING = (0, 0, (0, 0, 0), 0)


def _derives(t: torch.Tensor) -> bool:
    """Whether something asks for the derivative by this tensor"""
    return (t.requires_grad and torch.is_grad_enabled()) or _native.has_tangent(t)


def _side(t: torch.Tensor):
    """The input (a copy where its channels lie apart or torch counts its memory as negated: the caller keeps it until the call is
    enqueued, or its memory is another's), the output, and what the call is told of the pair: addresses, strides (batch, token, head), heads"""
    strides = t.stride()
    if strides[-1] != 1 or t.is_neg():
        t = t.resolve_neg().contiguous()
        strides = t.stride()
    out = torch.empty_like(t, memory_format=torch.contiguous_format)
    # (a tensor without elements takes part in the call no more than None does: its address is null)
    return t, out, (t.data_ptr(), out.data_ptr(), strides[:3] if len(strides) == 4 else (0, strides[0], strides[1]), t.shape[-2])


def _rotate(q, k, positions, inv_freq, factor, interleaved, transposed):
    """Enqueue da_rotate; q or k may be None.  Returns new tensors."""
    x = k if q is None else q
    q, q2, (qp, qo, qs, hq) = (None, None, _NOTHING) if q is None else _side(q)
    k, k2, (kp, ko, ks, hk) = (None, None, _NOTHING) if k is None else _side(k)
    if not qo and not ko:
        return q2, k2
    shape, device, ps = x.shape, x.get_device(), positions.stride()
    batch, ps = (shape[0], ps) if len(shape) == 4 else (1, (0, ps[0]))
    _native.launch(_native.lib().da_rotate, _native.PACK_ROTATE(
        qp if qo else 0, kp if ko else 0, qo, ko, *qs, *ks, positions.data_ptr(), positions.dtype is torch.int64, *ps,
        inv_freq.data_ptr(), 2 * inv_freq.shape[0], interleaved, transposed, factor, batch, shape[-3], hq, hk, shape[-1],
        _native.dtype_code(x.dtype), _native.stream_of(device)), device, "da_rotate")
    return q2, k2


class _Rotate(torch.autograd.Function):
    """The rotation is linear in q and k: its gradient is the transposed rotation, which is one again, and in forward mode the
    tangents are rotated like the heads."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, factor, interleaved, transposed):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (factor, interleaved, transposed)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions, inv_freq)
            ctx.shapes = (q.shape, k.shape)
        ctx.set_materialize_grads(False)
        return _rotate(q, k, positions, inv_freq, factor, interleaved, transposed)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        factor, interleaved, transposed = ctx.how
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is None and dk is None:
            return (None,) * 7
        return _linear(dq, dk, positions, inv_freq, factor, interleaved, not transposed) + (None,) * 5

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        positions, inv_freq = ctx.saved_tensors
        # (torch has a kind of zeros without memory, and wants a tangent for each output)
        tq, tk = (t.clone() if t is not None and t._is_zerotensor() else t for t in (tq, tk))
        tangents = _linear(tq, tk, positions, inv_freq, *ctx.how)
        like = tq if tk is None else tk
        return tuple(like.new_zeros(shape) if t is None else t for t, shape in zip(tangents, ctx.shapes))


def _linear(x, y, *how):
    """The rotation of what belongs to q and to k, gradients or tangents, one of which may be missing; itself differentiable"""
    if (x is not None and _derives(x)) or (y is not None and _derives(y)):
        # (a second derivative: what is missing is passed on as a tensor without elements)
        none = lambda t, like: like.new_empty(like.shape[:-2] + (0, like.shape[-1])) if t is None else t
        a, b = _Rotate.apply(none(x, y), none(y, x), *how)
        return (None if x is None else a), (None if y is None else b)
    return _rotate(x, y, *how)
