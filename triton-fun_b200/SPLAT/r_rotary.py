"""Rotary positions with one to four axes (text; rows and columns of an image; time, rows and columns of a video).

No counterpart in the reference, whose attention takes q and k as they come.  Pair i of a row turns by the angle
``positions[axis(i)] * inv_freq[i]``; the first ``sections[0]`` pairs go by axis 0, the next ``sections[1]`` by axis 1
and so on.  Pair i is elements i and i + len(inv_freq), or 2 i and 2 i + 1 with ``interleaved=True``; elements behind the
turned ones stay as they are.  float32, float16 and bfloat16; angles are formed in 64 bits, products in 32.
"""
from __future__ import annotations

import torch

import splat_native as _n


def rrotary_launcher(q: torch.Tensor, k, positions: torch.Tensor, inv_freq: torch.Tensor, sections=None, *,
                     interleaved: bool = False, inverse: bool = False, q_out=None, k_out=None):
    """q (B,H,L,d) and k (B,H',L,d) or None, any strides but a contiguous last dimension -> (q_out, k_out), new tensors
    where none are given; q_out may be q itself and k_out k.  positions: int32 or int64 (axes,B,L), (axes,L) or (L);
    inv_freq: float32, one for each turned pair, at most d / 2; sections may be left out for one axis.  inverse turns the
    other way.  No gradients: see ``rrotary``."""
    return _n.rotary(q, k, positions, inv_freq, sections, interleaved, inverse, q_out, k_out)


class _Rotary(torch.autograd.Function):
    """The gradient of a rotation is the rotation by the opposite angle."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, sections, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = sections, interleaved, inverse
        return _n.rotary(q, k, positions, inv_freq, sections, interleaved, inverse, None, None)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, inv_freq = ctx.saved_tensors
        sections, interleaved, inverse = ctx.how
        wanted = [g if need and g is not None else None for g, need in zip((dq, dk), ctx.needs_input_grad)]
        # (a gradient may come expanded, as that of a sum)
        rows = [g if g is None or g.stride(-1) == 1 else g.contiguous() for g in wanted]
        first, second = (rows[0], rows[1]) if rows[0] is not None else (rows[1], None)
        if first is None:
            return (None,) * 7
        a, b = _Rotary.apply(first, second, positions, inv_freq, sections, interleaved, not inverse)
        return (*((a, b) if rows[0] is not None else (None, a)), None, None, None, None, None)


def rrotary(q: torch.Tensor, k, positions: torch.Tensor, inv_freq: torch.Tensor, sections=None, *,
            interleaved: bool = False):
    """``rrotary_launcher`` into new tensors, differentiable in q and k (also twice): (q', k'), k' None without k."""
    if torch.is_grad_enabled():
        if inv_freq.requires_grad:
            raise ValueError("inv_freq must not require a gradient: there is none for the frequencies")
        if q.requires_grad or (k is not None and k.requires_grad):
            return _Rotary.apply(q, k, positions, inv_freq, sections, interleaved, False)
    return _n.rotary(q, k, positions, inv_freq, sections, interleaved, False, None, None)
