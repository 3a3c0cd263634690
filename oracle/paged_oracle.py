"""64-bit restatement of the paged cache's operators, of the rotary positions, and of the error that rounding allows.

An oracle, no part of the product.  Everything is written from the formulas, request by request and head by head, and runs on any device.
"""
from __future__ import annotations

import torch


def tables(ctx, new, table, ring, span, page, tokens):
    """Lists of ints (table: list of lists) -> dict of what rpaged_tables_launcher writes."""
    table = [list(row) for row in table]
    width = len(table[0]) if table else 0
    kv_lens, q_start, slots, positions, requests = [], [0], [], [], []
    head, tail, missing = span[0], span[1], 0
    avail = max(0, min(tail - head, len(ring)))
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        held, need = -(-c // page), -(-(c + n) // page)
        for i in range(held, need):
            if i >= width:
                missing += 1
            elif avail > 0:
                table[b][i] = ring[head % len(ring)]
                head, avail = head + 1, avail - 1
            else:
                table[b][i] = -1
                missing += 1
        for p in range(c, c + n):
            entry = table[b][p // page] if p // page < width else -1
            slots.append(entry * page + p % page if entry >= 0 else -1)
            positions.append(p)
            requests.append(b)
        kv_lens.append(c + n)
        q_start.append(q_start[-1] + n)
    pad = tokens - len(slots)
    return {"table": table, "kv_lens": kv_lens, "q_start": q_start, "slots": (slots + [-1] * pad)[:tokens],
            "positions": (positions + [0] * pad)[:tokens], "requests": (requests + [-1] * pad)[:tokens],
            "taken": [head, tail, missing]}


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    """x (B, H, L, d), positions (axes, B, L) -> float64."""
    half = inv_freq.numel()
    axis = sum(([a] * count for a, count in enumerate(sections)), [])
    out = x.double().clone()
    for i in range(half):
        w = positions[axis[i]].double() * inv_freq[i].double()              # (B, L)
        c, s = w.cos()[:, None], (-w.sin() if inverse else w.sin())[:, None]
        re, im = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., re].double(), x[..., im].double()
        out[..., re], out[..., im] = a * c - b * s, a * s + b * c
    return out


def attention(q, k_cache, v_cache, table, kv_lens, q_start, *, scale=1.0, taps=0, stride=1, softcap=0.0, slopes=None):
    """-> (out, lse, tolerance of out, tolerance of lse), float64; NaN in out's rows that belong to no request.

    The tolerance, with u = eps / 2 of the operands' type and w = 2^-23 (an fp32 operation, rounded in any direction):
      * a score is a sum of d products: off by (d + 8) w S at most, S = scale * max sum |q||k| + |bias|; probabilities
        are off by that, relatively, and so is their sum.  A cap's tanh does not enlarge what its argument is off by, and is off
        by 8 w of its own value at most, which is no more than the score's;
      * n terms are summed up, and rescaled: (n + 64) w, for the numerator and for the denominator;
      * a probability rounded to the operands' 16 bits before it is multiplied: u of sum p |v| / sum p;
      * the result is rounded once: u of itself, and half of the smallest number of its type.
    """
    T, H, d = q.shape
    pages, heads, page, _ = k_cache.shape
    g = H // heads
    type_info = torch.finfo(q.dtype)
    u, w = type_info.eps / 2, 2.0 ** -23
    out = torch.full((T, H, d), float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((T, H), float("nan"), dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    for b in range(len(kv_lens)):
        kv, t0, t1 = int(kv_lens[b]), int(q_start[b]), int(q_start[b + 1])
        n = t1 - t0
        for t in range(t0, t1):
            i = kv - n + (t - t0)
            js = [j for j in range(i, -1, -stride)][:taps or None]
            js = [j for j in js if j // page < table.shape[1] and 0 <= int(table[b, j // page]) < pages]
            if not js:
                out[t], lse[t] = 0.0, float("-inf")
                continue
            j = torch.tensor(js, device=q.device)
            where = table[b, j // page].long()
            k, v = k_cache[where, :, j % page].double(), v_cache[where, :, j % page].double()        # (n, heads, d)
            x = q[t].double().view(heads, g, d)
            s = torch.einsum("hgd,nhd->hgn", x, k) * scale
            mass = torch.einsum("hgd,nhd->hgn", x.abs(), k.abs()) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                bias = slopes.double().view(heads, g, 1) * (i - j)
                s, mass = s - bias, mass + bias.abs()
            total = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - total)
            o = torch.einsum("hgn,nhd->hgd", p, v)
            weight = torch.einsum("hgn,nhd->hgd", p, v.abs())
            # (keys that weigh nothing may be off by more)
            seen = mass.masked_fill(p < 2.0 ** -40, 0.0).amax(-1, keepdim=True)
            rel = 2 * ((d + 8) * w * seen + (len(js) + 64) * w)
            rounded = u if q.dtype != torch.float32 else 0.0
            out[t], lse[t] = o.view(H, d), total.view(H)
            tol[t] = ((rounded + rel) * weight + u * o.abs() + type_info.smallest_normal).view(H, d)
            lse_tol[t] = (rel / 2 + 4 * w * (1 + total.abs())).view(H)
    return out, lse, tol, lse_tol
