"""What serving and training with the paged cache and the rotary positions have this package do, as measurable cases.

Four kinds of call, all through the modules of the SPLAT directory:

  tables   rpaged_tables_launcher: block tables, slots and positions of a step, from the requests' lengths
  rotary   rrotary: rotary positions of several axes on queries and keys, and their gradients
  append   rpaged_append_launcher: a step's queries and keys turned to their positions, keys and values put into the
           paged cache
  attend   rpaged_attention_launcher: a step's queries (one token each, chunks of a prompt, or both) over the paged
           cache: full causal, a window, strided or dilated, scores capped by a tanh, or with a bias by distance

Where `own` is false every kind is computed from elementary torch operations instead, in 32 bits (angles in 64).
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


def _package():
    splat = os.path.join(os.getcwd(), "triton-fun_b200", "SPLAT")
    if splat not in sys.path:
        sys.path.insert(0, splat)
    import r_paged
    import r_rotary
    return r_paged, r_rotary


# ----------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------
def _tables(name, B, new, q_max, ctx_max, page, width):
    return {"name": name, "kind": "tables", "B": B, "new": new, "q_max": q_max, "ctx_max": ctx_max, "page": page,
            "width": width, "lens": 1}


def _rotary(name, dtype, B, Hq, Hkv, L, d, turned, axes, interleaved, backward):
    return {"name": name, "kind": "rotary", "dtype": dtype, "B": B, "Hq": Hq, "Hkv": Hkv, "L": L, "d": d,
            "turned": turned, "axes": axes, "interleaved": interleaved, "backward": backward}


def _append(name, dtype, T, Hq, Hkv, d, turned, axes, interleaved, page, rows_first=False):
    return {"name": name, "kind": "append", "dtype": dtype, "T": T, "Hq": Hq, "Hkv": Hkv, "d": d, "turned": turned,
            "axes": axes, "interleaved": interleaved, "page": page, "rows_first": rows_first}


def _attend(name, dtype, B, new, q_max, kv, kv_max, Hq, Hkv, d, page, taps=0, stride=1, cap=0.0, bias=False,
            rows_first=False, lens=1):
    return {"name": name, "kind": "attend", "dtype": dtype, "B": B, "new": new, "q_max": q_max, "kv": kv,
            "kv_max": kv_max, "Hq": Hq, "Hkv": Hkv, "d": d, "page": page, "taps": taps, "stride": stride, "cap": cap,
            "bias": bias, "rows_first": rows_first, "lens": lens}


def listed():
    return [
        # A decoding step's bookkeeping: one token for each of 128 requests.
        _tables("tables_decode", 128, "one", 1, 8191, 16, 1024),
        # Bookkeeping of a step that takes in prompts beside decoding requests, as long as the cache goes.
        _tables("tables_prompts", 500, "mixed", 2048, 30000, 32, 1024),
        # Queries and keys of a training batch of video (time, height, width), forward and backward.
        _rotary("rotary_bf16_video", "bf16", 2, 32, 32, 4096, 128, 128, 3, False, True),
        # Patches of images (height, width), pairs side by side, an odd number of them, in fp32.
        _rotary("rotary_fp32_image", "fp32", 3, 12, 4, 1369, 64, 32, 2, True, True),
        # A decoding step's queries, keys and values on their way into the cache: latency.
        _append("append_bf16_decode", "bf16", 64, 32, 8, 128, 128, 3, False, 16),
        # Chunks of prompts, an odd number of tokens.
        _append("append_fp16_chunk", "fp16", 8191, 16, 16, 64, 64, 1, False, 64, rows_first=True),
        # One request in a short conversation: nothing but latency.
        _attend("attend_bf16_single", "bf16", 1, "one", 1, "equal", 700, 16, 4, 64, 16),
        # A decoding batch of requests of all lengths, grouped heads: the cache has to be read once.
        _attend("attend_bf16_decode", "bf16", 64, "one", 1, "ragged", 16384, 32, 8, 128, 16),
        # Long contexts through the local window of the benchmark's largest configuration, scores capped.
        _attend("attend_fp16_window", "fp16", 96, "one", 1, "ragged", 32768, 16, 16, 128, 64, taps=1024, cap=50.0),
        # The checking type, with the bias by distance, drafted tokens beside the last one.
        _attend("attend_fp32_draft", "fp32", 9, "ragged", 5, "ragged", 4097, 16, 8, 64, 16, bias=True),
        # A long prompt's chunk beside decoding requests, dilated as in configuration 4 of the benchmark.
        _attend("attend_bf16_dilated", "bf16", 8, "mixed", 1024, "ragged", 8192, 32, 8, 128, 32, taps=512, stride=2,
                rows_first=True),
        # Chunks of two long prompts, full causal attention: the largest call.
        _attend("attend_bf16_prompt", "bf16", 2, "equal", 2048, "equal", 16384, 32, 8, 128, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["tables", "rotary", "append", "attend"], [15, 15, 15, 55])[0]
    dtype = rng.choices(["fp32", "fp16", "bf16"], [2, 3, 5])[0]
    if kind == "tables":
        new = rng.choice(["one", "mixed", "ragged"])
        page = rng.choice([1, 8, 16, 24, 32, 64, 128])
        q_max = 1 if new == "one" else _log(rng, 2, 2048)
        ctx = _log(rng, 16, 30000)
        case = _tables("", _log(rng, 1, 512 if q_max < 256 else 64), new, q_max, ctx, page,
                       -(-(ctx + q_max) // page) + rng.randrange(8))
        case["lens"] = rng.randrange(1 << 20)
    elif kind == "rotary":
        d = rng.choice([32, 64, 80, 96, 128])
        axes = rng.choice([1, 2, 3])
        Hkv = _log(rng, 1, 16)
        case = _rotary("", dtype, rng.choice([1, 2, 3]), Hkv * rng.choice([1, 2, 4]), Hkv, _log(rng, 17, 2048), d,
                       rng.choice([d, d // 2]), axes, rng.random() < 0.3, rng.random() < 0.7)
    elif kind == "append":
        d = rng.choice([64, 80, 128])
        Hkv = _log(rng, 1, 16)
        case = _append("", dtype, _log(rng, 1, 8191), Hkv * rng.choice([1, 2, 4]), Hkv, d, rng.choice([d, d // 2]),
                       rng.choice([1, 2, 3]), rng.random() < 0.3, rng.choice([8, 16, 24, 64]), rng.random() < 0.5)
    else:
        d = rng.choices([64, 80, 96, 128], [4, 1, 1, 6])[0]
        Hkv = rng.choice([1, 2, 4, 8, 16])
        Hq = Hkv * rng.choice([1, 2, 3, 4, 8])
        new = rng.choices(["one", "ragged", "mixed", "equal"], [5, 2, 2, 2])[0]
        q_max = 1 if new == "one" else _log(rng, 2, 8) if new == "ragged" else _log(rng, 16, 2048)
        if dtype == "fp32":           # what fp32 is used for: checks, not long prompts
            q_max = min(q_max, 256)
        kv_max = max(q_max, _log(rng, 64, 32768))
        shape = rng.choices(["full", "window", "strided", "dilated"], [5, 3, 1, 1])[0]
        taps, stride = 0, 1
        if shape == "window":
            taps = _log(rng, 64, 4096)
        elif shape == "strided":
            stride = rng.choice([4, 16, 64])
        elif shape == "dilated":
            taps, stride = _log(rng, 32, 1024), rng.choice([2, 3, 4])
        case = _attend("", dtype, 1, new, q_max, rng.choice(["ragged", "equal"]), kv_max, Hq, Hkv, d,
                       rng.choice([8, 16, 24, 32, 64, 128]), taps, stride, rng.choice([0.0, 0.0, 30.0]),
                       rng.random() < 0.2, rng.random() < 0.4, rng.randrange(1 << 20))
        # as many requests as the plain form's scores and the cache leave room for
        most = min(2.1e9 / (q_max * kv_max * Hq), 3.3e9 / (kv_max * Hkv * d * 2 * SIZE[dtype]))
        case["B"] = max(1, min(_log(rng, 1, 128), int(most)))
        while case["q_max"] > 1 and work(case)["flops"] > work(listed()[-1])["flops"]:
            case["q_max"] = max(1, case["q_max"] // 2)
    del case["name"]
    return case


def _spread(rng, how, n, most):
    """n lengths of up to `most`."""
    if how == "equal":
        return [most] * n
    if how == "one":
        return [1] * n
    if how == "mixed":                # most of the requests decode, some take in a chunk
        return [most if i == n // 2 else _log(rng, 1, most) if rng.random() < 0.25 else 1 for i in range(n)]
    return [most if i == n // 2 else _log(rng, 1, most) for i in range(n)]


def _lens(case):
    """(cached tokens, new tokens) of every request, the same for every seed."""
    rng = random.Random(case["lens"])
    new = _spread(rng, case["new"], case["B"], case["q_max"])
    if case["kind"] == "tables":
        return [rng.randrange(case["ctx_max"] + 1) for _ in new], new
    whole = _spread(rng, case["kv"], case["B"], case["kv_max"])
    return [max(0, w - n) for w, n in zip(whole, new)], new


# ----------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------
def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _normal(shape, dtype, g):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _turn(case):
    """Frequencies of the turned pairs, and how many of them go by each axis."""
    half, axes = case["turned"] // 2, case["axes"]
    inv_freq = torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda")
    first = half - (axes - 1) * (half * 3 // (4 * axes))
    return inv_freq, [first] + [half * 3 // (4 * axes)] * (axes - 1)


def _places(case, T, g):
    """(axes, T) positions: frames or text behind one another, rows and columns within them."""
    at = torch.arange(T, device="cuda") + torch.randint(0, 20000, (1,), device="cuda", generator=g)
    wide = max(1, math.isqrt(T // 4))
    return torch.stack([at, at // wide % wide, at % wide][: case["axes"]]).to(torch.int32)


def _cache(pages, Hkv, page, d, dtype, rows_first, g):
    """K and V of (pages, Hkv, page, d), in that order in memory or with a page's rows first."""
    shape = (pages, page, Hkv, d) if rows_first else (pages, Hkv, page, d)
    kv = [_normal(shape, dtype, g) for _ in range(2)]
    return [t.transpose(1, 2) for t in kv] if rows_first else kv


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = {"kind": kind, "case": case}
    if kind == "tables":
        ctx, new = _lens(case)
        page, width, B = case["page"], case["width"], case["B"]
        held = [-(-c // page) for c in ctx]
        free = sum(-(-(c + n) // page) for c, n in zip(ctx, new)) - sum(held)
        order = torch.randperm(sum(held) + free + 5, device="cuda", generator=g).to(torch.int32)
        column = torch.arange(width, device="cuda", dtype=torch.int32)
        h = _ints(held)
        before = h.cumsum(0) - h
        table = torch.where(column < h[:, None], order[(before[:, None] + column).clamp(max=len(order) - 1).long()], -1)
        T = sum(new)
        s.update(ctx=_ints(ctx), new=_ints(new), table=table.to(torch.int32).contiguous(),
                 ring=order[sum(held):].contiguous(), span=_ints([3, 3 + free + 5], torch.int64), page=page,
                 kv_lens=_ints([0] * B), q_start=_ints([0] * (B + 1)), slots=_ints([0] * T, torch.int64),
                 positions=_ints([0] * T), requests=_ints([0] * T), taken=_ints([0, 0, 0], torch.int64))
        return s
    dtype = DTYPES[case["dtype"]]
    Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
    if kind == "rotary":
        B, L = case["B"], case["L"]
        s["inv_freq"], s["sections"] = _turn(case)
        s["positions"] = torch.stack([_places(case, L, g) for _ in range(B)], dim=1)       # (axes, B, L)
        # as a projection leaves them: (B, L, H, d) in memory
        s["q"], s["k"] = (_normal((B, L, H, d), dtype, g).transpose(1, 2) for H in (Hq, Hkv))
        if case["backward"]:
            s["dq"], s["dk"] = (_normal((B, H, L, d), dtype, g) for H in (Hq, Hkv))
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
        return s
    page = case["page"]
    if kind == "append":
        T = case["T"]
        pages = -(-T // page) + 3
        s["inv_freq"], s["sections"] = _turn(case)
        s["positions"] = _places(case, T, g)
        # rows of one fused projection
        qkv = _normal((T, Hq + 2 * Hkv, d), dtype, g)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        s["k_cache"], s["v_cache"] = _cache(pages, Hkv, page, d, dtype, case["rows_first"], g)
        at = torch.arange(T, device="cuda")
        s["slots"] = torch.randperm(pages, device="cuda", generator=g)[at // page] * page + at % page
        s["q_out"] = torch.zeros((T, Hq, d), dtype=dtype, device="cuda")
        return s
    ctx, new = _lens(case)
    whole = [c + n for c, n in zip(ctx, new)]
    held = [-(-w // page) for w in whole]
    pages = sum(held) + 2
    s["k_cache"], s["v_cache"] = _cache(pages, Hkv, page, d, dtype, case["rows_first"], g)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    h = _ints(held)
    column = torch.arange(max(held), device="cuda", dtype=torch.int32)
    before = h.cumsum(0) - h
    table = torch.where(column < h[:, None], order[(before[:, None] + column).clamp(max=pages - 1).long()], -1)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    s.update(table=table.to(torch.int32).contiguous(), kv_lens=_ints(whole), q_start=_ints(start),
             q=_normal((start[-1], Hq, d), dtype, g), out=torch.zeros((start[-1], Hq, d), dtype=dtype, device="cuda"),
             lse=torch.zeros((start[-1], Hq), dtype=torch.float32, device="cuda"), slopes=None,
             q_max=max(new), kv_max=max(whole), scale=d ** -0.5)
    if case["bias"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device="cuda")
    return s


# ----------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------
def _tables_plain(s):
    page, table, ring = s["page"], s["table"], s["ring"]
    B, width = table.shape
    T = s["slots"].shape[0]
    ctx, new = s["ctx"].long(), s["new"].long()
    kv = ctx + new
    s["kv_lens"].copy_(kv)
    ends = new.cumsum(0)
    s["q_start"][0] = 0
    s["q_start"][1:] = ends
    held, need = (ctx + page - 1) // page, (kv + page - 1) // page
    before = (need - held).cumsum(0) - (need - held)
    column = torch.arange(width, device="cuda")
    fresh = (column >= held[:, None]) & (column < need[:, None])
    index = (s["span"][0] + before[:, None] + column - held[:, None]) % ring.shape[0]
    table.copy_(torch.where(fresh, ring[index.clamp(min=0)], table))
    total = (need - held).sum()
    s["taken"][0] = s["span"][0] + total
    s["taken"][1] = s["span"][1]
    s["taken"][2] = 0
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(ends, t, right=True)
    pos = ctx[r] + t - (ends - new)[r]
    s["slots"].copy_(table[r, pos // page].long() * page + pos % page)
    s["positions"].copy_(pos)
    s["requests"].copy_(r)


def _angles(positions, inv_freq, sections):
    """(axes, ...) positions -> cosines and sines (..., pairs)."""
    axis = torch.arange(len(sections), device="cuda").repeat_interleave(_ints(sections, torch.int64), output_size=len(inv_freq))
    angle = positions.double()[axis].movedim(0, -1) * inv_freq.double()
    return angle.cos().float(), angle.sin().float()


def _turned(x, cos, sin, interleaved):
    half = cos.shape[-1]
    x32 = x.float()
    a, b = (x32[..., 0:2 * half:2], x32[..., 1:2 * half:2]) if interleaved else (x32[..., :half], x32[..., half:2 * half])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x32[..., 2 * half:]), -1).to(x.dtype)


def _attend_plain(s):
    case = s["case"]
    kc, vc, table, q = s["k_cache"], s["v_cache"], s["table"].long(), s["q"]
    page, Hq, Hkv, d, stride = case["page"], case["Hq"], case["Hkv"], case["d"], case["stride"]
    B, g, T, n_q, n_kv = table.shape[0], Hq // Hkv, q.shape[0], s["q_max"], s["kv_max"]
    start, kv = s["q_start"].long(), s["kv_lens"].long()
    i, j = torch.arange(n_q, device="cuda"), torch.arange(n_kv, device="cuda")
    at = (start[:-1, None] + i).clamp(max=T - 1)
    pos = (kv - (start[1:] - start[:-1]))[:, None] + i                               # (B, n_q)
    where = table[:, j // page].clamp(min=0)                                         # (B, n_kv)
    k = kc[where, :, j % page].float().permute(0, 2, 3, 1)                           # (B, Hkv, d, n_kv)
    v = vc[where, :, j % page].float().transpose(1, 2)                               # (B, Hkv, n_kv, d)
    x = q[at].float().reshape(B, n_q, Hkv, g, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * n_q, d)
    scores = (x @ k).mul_(s["scale"])
    if case["cap"]:
        scores = scores.div_(case["cap"]).tanh_().mul_(case["cap"])
    scores = scores.view(B, Hkv, g, n_q, n_kv)
    away = pos[..., None] - j                                                        # (B, n_q, n_kv)
    if s["slopes"] is not None:
        scores -= s["slopes"].view(Hkv, g, 1, 1) * away[:, None, None]
    seen = (away >= 0) & (away % stride == 0) & (j < kv[:, None, None])
    if case["taps"]:
        seen &= away < case["taps"] * stride
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = (scores - top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, g * n_q, n_kv) @ v).view(B, Hkv, g, n_q, d) / torch.where(total > 0, total, 1.0)
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(start[1:], t, right=True)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[r, t - start[r]].reshape(T, Hq, d))
    s["lse"].copy_((top + total.log()).squeeze(-1).permute(0, 3, 1, 2)[r, t - start[r]].reshape(T, Hq))


# ----------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------
def run(state):
    s = state
    kind, case = s["kind"], s["case"]
    r_paged, r_rotary = _package() if own else (None, None)
    if kind == "tables":
        if own:
            r_paged.rpaged_tables_launcher(s["ctx"], s["new"], s["table"], s["ring"], s["span"], s["page"], s["kv_lens"],
                                           s["q_start"], s["slots"], s["positions"], s["requests"], s["taken"])
        else:
            _tables_plain(s)
        return {k: s[k] for k in ("table", "kv_lens", "q_start", "slots", "positions", "requests", "taken")}
    if kind == "rotary":
        if own:
            q, k = r_rotary.rrotary(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"],
                                    interleaved=case["interleaved"])
        else:
            cos, sin = (x[:, None] for x in _angles(s["positions"], s["inv_freq"], s["sections"]))    # (B, 1, L, pairs)
            q, k = (_turned(x, cos, sin, case["interleaved"]) for x in (s["q"], s["k"]))
        if not case["backward"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if kind == "append":
        if own:
            r_paged.rpaged_append_launcher(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["q_out"],
                                           positions=s["positions"], inv_freq=s["inv_freq"], sections=s["sections"],
                                           interleaved=case["interleaved"])
        else:
            cos, sin = (x[:, None] for x in _angles(s["positions"], s["inv_freq"], s["sections"]))    # (T, 1, pairs)
            page = case["page"]
            s["q_out"].copy_(_turned(s["q"], cos, sin, case["interleaved"]))
            s["k_cache"][s["slots"] // page, :, s["slots"] % page] = _turned(s["k"], cos, sin, case["interleaved"])
            s["v_cache"][s["slots"] // page, :, s["slots"] % page] = s["v"]
        return {k: s[k] for k in ("q_out", "k_cache", "v_cache")}
    if own:
        r_paged.rpaged_attention_launcher(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["out"],
                                          q_start=s["q_start"], max_q_len=s["q_max"], scale=s["scale"],
                                          taps=case["taps"], stride=case["stride"], softcap=case["cap"],
                                          slopes=s["slopes"], lse=s["lse"])
    else:
        _attend_plain(s)
    return {"out": s["out"], "lse": s["lse"]}


# ----------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "tables":
        ctx, new = _lens(case)
        page = case["page"]
        fresh = sum(-(-(c + n) // page) + (-c // page) for c, n in zip(ctx, new))
        # lengths in and out, a table entry read or written for each page that new tokens fall on, slot, position and request of a token
        return {"bytes": 4 * (4 * case["B"] + 1) + 8 * fresh + 4 * case["B"] + 16 * sum(new) + 40, "flops": 0}
    e, d, heads = SIZE[case["dtype"]], case["d"], case["Hq"] + case["Hkv"]
    if kind == "rotary":
        tokens = case["B"] * case["L"]
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * (2 * tokens * heads * d * e + 4 * case["axes"] * tokens),
                "flops": passes * 3 * tokens * heads * case["turned"]}
    if kind == "append":
        T = case["T"]
        return {"bytes": 2 * T * (heads + case["Hkv"]) * d * e + T * (8 + 4 * case["axes"]),
                "flops": 3 * T * heads * case["turned"]}
    ctx, new = _lens(case)
    stride, taps = case["stride"], case["taps"] or 1 << 60
    pairs = keys = 0
    for c, n in zip(ctx, new):
        pairs += sum(min(taps, i // stride + 1) for i in range(c, c + n))
        for r in range(min(stride, n)):                        # keys of a residue class, from the first query's first on
            first, last = c + r, c + r + (n - 1 - r) // stride * stride
            keys += last // stride - max(0, first // stride - taps + 1) + 1
    T = sum(new)
    return {"bytes": 2 * keys * case["Hkv"] * d * e + T * case["Hq"] * (2 * d * e + 4),
            "flops": 4 * pairs * case["Hq"] * d}


# ----------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ----------------------------------------------------------------------------------------------
def _turn_exact(x, places, inv_freq, sections, interleaved, back=False):
    """x (T, H, d) by places (axes, T), as products with complex numbers of modulus one; back: the other way round."""
    out = x.double().clone()
    half, lo = len(inv_freq), 0
    for axis, count in enumerate(sections):
        pairs = slice(lo, lo + count)
        turn = places[axis].double()[:, None] * inv_freq[pairs].double()[None]
        unit = torch.polar(torch.ones_like(turn), -turn if back else turn)[:, None]
        re = torch.arange(lo, lo + count, device="cuda") * (2 if interleaved else 1)
        im = re + (1 if interleaved else half)
        z = torch.complex(out[..., re], out[..., im]) * unit
        out[..., re], out[..., im] = z.real, z.imag
        lo += count
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None                    # whole numbers only
    s = prepare(case, seed)
    if kind == "rotary":
        def all_of(x, back=False):
            rows = [_turn_exact(x[b].detach().transpose(0, 1), s["positions"][:, b], s["inv_freq"], s["sections"],
                                case["interleaved"], back).transpose(0, 1) for b in range(x.shape[0])]
            return torch.stack(rows)
        out = {"q": all_of(s["q"]), "k": all_of(s["k"])}
        if case["backward"]:
            out.update(dq=all_of(s["dq"], True), dk=all_of(s["dk"], True))
        return out
    if kind == "append":
        turn = [_turn_exact(x, s["positions"], s["inv_freq"], s["sections"], case["interleaved"]) for x in (s["q"], s["k"])]
        caches = []
        for cache, rows in ((s["k_cache"], turn[1]), (s["v_cache"], s["v"].double())):
            flat = cache.double().transpose(1, 2).reshape(-1, case["Hkv"], case["d"])
            flat[s["slots"]] = rows
            caches.append(flat.view(-1, case["page"], case["Hkv"], case["d"]).transpose(1, 2))
        return {"q_out": turn[0], "k_cache": caches[0], "v_cache": caches[1]}
    ctx, new = _lens(case)
    g, page, stride = case["Hq"] // case["Hkv"], case["page"], case["stride"]
    out, lse = s["out"].double(), s["lse"].double()
    row = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        j = torch.arange(c + n, device="cuda")
        pages, within = s["table"][b, j // page].long(), j % page
        i = torch.arange(c, c + n, device="cuda")
        behind = (i[:, None] - j[None])
        hidden = (behind < 0) | (behind % stride != 0)
        if case["taps"]:
            hidden |= behind // stride >= case["taps"]
        for h in range(case["Hkv"]):
            k, v = (x[pages, h, within].double() for x in (s["k_cache"], s["v_cache"]))
            for e in range(h * g, (h + 1) * g):
                z = s["q"][row:row + n, e].double() @ k.T * s["scale"]
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if s["slopes"] is not None:
                    z = z - s["slopes"][e].double() * behind
                z[hidden] = -math.inf
                sums = torch.logsumexp(z, -1)
                out[row:row + n, e] = torch.exp(z - sums[:, None]) @ v
                lse[row:row + n, e] = sums
        row += n
    return {"out": out, "lse": lse}
