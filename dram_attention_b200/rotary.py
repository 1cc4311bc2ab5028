"""Rotary positions by inverse frequencies: both pairings of the channels, all of the head or part of it, frequencies
stretched to long contexts, with gradients.  (`DRAMAttention.rotate_` is the reference caller's own form: the whole head
in adjacent pairs, from a table of complex factors.)"""

from __future__ import annotations

import math
from typing import Mapping, Optional, Tuple

import torch

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
        inv_freq: float32 (rotary_dim / 2,) on a CUDA device; `rotary_frequencies` makes them.
        factor: amplitude of the rotated channels.
        interleaved: channel pairs (2i, 2i + 1); otherwise (i, i + rotary_dim / 2).

    Angles are formed and reduced in 64 bits, so far positions keep the accuracy of near ones; the arithmetic is float32,
    rounded once to the type of the heads."""

    def __init__(self, inv_freq: torch.Tensor, factor: float = 1.0, interleaved: bool = True):
        _native.require_cuda(inv_freq, "inv_freq")
        assert inv_freq.dtype == torch.float32 and inv_freq.dim() == 1 and inv_freq.numel() > 0, \
            f"inv_freq must be a float32 vector, got {tuple(inv_freq.shape)} {inv_freq.dtype}"
        _native.lib()
        self.inv_freq = inv_freq.detach().contiguous()
        self.factor = float(factor)
        self.interleaved = bool(interleaved)

    @property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.numel()

    def __call__(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor):
        """q (s, Hq, D) or (b, s, Hq, D), k the same with its own number of heads; positions int32 or int64, (s,) or (b, s),
        magnitudes below 2^31.  Channels from rotary_dim on pass unchanged.  Returns the rotated pair (new tensors);
        differentiable in q and k."""
        assert q.dim() in (3, 4) and k.dim() == q.dim() and k.shape[:-2] == q.shape[:-2] and k.shape[-1] == q.shape[-1], \
            f"q (..., heads, D) and k (..., heads, D) do not go together: {tuple(q.shape)}, {tuple(k.shape)}"
        _native.require_cuda(q, "q")
        assert k.dtype == q.dtype, "q and k must have the same dtype"
        _native.dtype_code(q.dtype)
        assert self.rotary_dim <= q.shape[-1] <= 512, \
            f"head_dim must lie between rotary_dim ({self.rotary_dim}) and 512, got {q.shape[-1]}"
        assert positions.dtype in (torch.int32, torch.int64), f"positions must be int32 or int64, got {positions.dtype}"
        lead = q.shape[:-2]
        assert positions.shape == lead or positions.shape == lead[-1:], \
            f"positions must be {tuple(lead)} or {tuple(lead[-1:])}, got {tuple(positions.shape)}"
        for t, name in ((k, "k"), (positions, "positions"), (self.inv_freq, "inv_freq")):
            assert t.device == q.device, f"{name} must be on the device of q ({q.device}), got {t.device}"
        positions = positions.expand(lead)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
            return _Rotate.apply(q, k, positions, self.inv_freq, self.factor, self.interleaved, False)
        return _rotate(q, k, positions, self.inv_freq, self.factor, self.interleaved, False)


def _rotate(q, k, positions, inv_freq, factor, interleaved, transposed):
    """Enqueue da_rotate; q or k may be None.  Returns new tensors."""
    x = k if q is None else q
    lead, d = x.shape[:-2], x.shape[-1]
    out, fields = [], []
    for t in (q, k):
        if t is None:
            out.append(None)
            fields.append((0, 0, (0, 0, 0), 0))
            continue
        t = t if t.stride(-1) == 1 else t.contiguous()
        o = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        s = t.stride()
        # (a tensor without elements takes part in the call no more than None does)
        present = o.numel() > 0
        out.append(o)
        fields.append((t.data_ptr() if present else 0, o.data_ptr() if present else 0,
                       (s[0] if len(lead) == 2 else 0, s[-3], s[-2]), t.shape[-2]))
    (qp, qo, qs, hq), (kp, ko, ks, hk) = fields
    if not (qp or kp):
        return tuple(out)
    ps = positions.stride()
    with torch.cuda.device(x.device):
        _native.check(_native.lib().da_rotate(_native.PACK_ROTATE(
            qp, kp, qo, ko, *qs, *ks, positions.data_ptr(), positions.dtype == torch.int64, ps[0] if len(lead) == 2 else 0, ps[-1],
            inv_freq.data_ptr(), 2 * inv_freq.numel(), interleaved, transposed, factor,
            lead[0] if len(lead) == 2 else 1, lead[-1], hq, hk, d, _native.dtype_code(x.dtype), _native.stream_ptr())), "da_rotate")
    return tuple(out)


class _Rotate(torch.autograd.Function):
    """The rotation is linear in q and k: its gradient is the transposed rotation, which is one again."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, factor, interleaved, transposed):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (factor, interleaved, transposed)
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
        how = (positions, inv_freq, factor, interleaved, not transposed)
        if torch.is_grad_enabled() and any(g is not None and g.requires_grad for g in (dq, dk)):
            # (a second derivative: a missing gradient is passed on as one without elements)
            none = lambda g, like: like.new_empty(like.shape[:-2] + (0, like.shape[-1])) if g is None else g
            q, k = _Rotate.apply(none(dq, dk), none(dk, dq), *how)
            dq, dk = (None if dq is None else q), (None if dk is None else k)
        else:
            dq, dk = _rotate(dq, dk, *how)
        return dq, dk, None, None, None, None, None
