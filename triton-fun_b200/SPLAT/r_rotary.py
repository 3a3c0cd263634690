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


def rrotary(q: torch.Tensor, k, positions: torch.Tensor, inv_freq: torch.Tensor, sections=None, *,
            interleaved: bool = False):
    """``rrotary_launcher`` into new tensors, differentiable in q and k (also twice): (q', k'), k' None without k.  The
    gradient of a rotation is the rotation by the opposite angle, one launch for both; in forward mode the tangents are
    turned like the operands, by a launch of their own."""
    return _n.rotary_grad(q, k, positions, inv_freq, sections, interleaved)
