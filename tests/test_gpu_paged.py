"""GPU: block tables, the paged cache and attention over it, against 64 bits."""
import math
import random

import pytest
import torch

import r_paged
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


# ----------------------------------------------------------------------------------------------
# tables
# ----------------------------------------------------------------------------------------------
def run_tables(ctx, new, page, width, free, span, tokens, table=None):
    B = len(ctx)
    t = {"table": ints(table if table is not None else [[-7] * width for _ in range(B)]).view(B, width),
         "kv_lens": ints([-5] * B), "q_start": ints([-5] * (B + 1)), "slots": ints([-5] * tokens, torch.int64),
         "positions": ints([-5] * tokens), "requests": ints([-5] * tokens), "taken": ints([-5] * 3, torch.int64)}
    r_paged.rpaged_tables_launcher(ints(ctx), ints(new), t["table"], ints(free), ints(span, torch.int64), page, t["kv_lens"],
                                   t["q_start"], t["slots"], t["positions"], t["requests"], t["taken"])
    return {k: v.cpu().tolist() for k, v in t.items()}


@pytest.mark.parametrize("B, page, most_ctx, most_new, short", [
    (1, 1, 0, 1, False), (1, 16, 100, 1, False), (7, 16, 100, 40, False), (7, 3, 50, 9, True), (40, 24, 300, 700, False),
    (513, 16, 200, 3, False), (1100, 8, 60, 20, True), (64, 128, 5000, 1, False)])
def test_tables(B, page, most_ctx, most_new, short):
    rng = random.Random(B * 1000 + page)
    ctx = [rng.randint(0, most_ctx) if rng.random() > 0.2 else -3 * (rng.random() < 0.2) for _ in range(B)]
    new = [rng.randint(0, most_new) if rng.random() > 0.1 else -2 for _ in range(B)]
    new[B // 2] = most_new
    width = -(-(most_ctx + most_new) // page) - (2 if short else 0)
    held = [-(-max(c, 0) // page) for c in ctx]
    table, at = [], 10
    for h in held:
        table.append([at + i if i < h else -7 for i in range(width)])
        at += h
    need = sum(-(-(max(c, 0) + max(n, 0)) // page) - h for c, n, h in zip(ctx, new, held))
    free = list(range(100000, 100000 + max(1, need // 2 if short else need + 3)))
    rng.shuffle(free)
    first = rng.randrange(5 * len(free))
    span = [first, first + len(free) - (1 if short else 0)]
    tokens = sum(max(n, 0) for n in new) + 5
    got = run_tables(ctx, new, page, width, free, span, tokens, table)
    assert got == po.tables(ctx, new, table, free, span, page, tokens)


def test_tables_without_requests_tokens_or_free_pages():
    assert run_tables([], [], 16, 4, [3], [0, 1], 3)["slots"] == [-1, -1, -1]
    got = run_tables([3, 0], [0, 0], 16, 4, [3], [0, 0], 0)
    assert got["kv_lens"] == [3, 0] and got["q_start"] == [0, 0, 0] and got["taken"] == [0, 0, 0]
    got = run_tables([15, 0], [2, 3], 16, 4, [3], [9, 9], 6, [[8, -7, -7, -7], [-7] * 4])
    assert got == po.tables([15, 0], [2, 3], [[8, -7, -7, -7], [-7] * 4], [3], [9, 9], 16, 6)
    # fewer rows than tokens: what is there is right
    got = run_tables([0, 0], [5, 5], 2, 4, list(range(9)), [0, 9], 7)
    assert got["slots"] == po.tables([0, 0], [5, 5], [[-7] * 4] * 2, list(range(9)), [0, 9], 2, 7)["slots"]


@pytest.mark.parametrize("rows", [0, 1, 4, 7, 9, 10, 11])
def test_tables_of_steps_with_more_tokens_than_rows(rows):
    """Pages are taken for all of a step's tokens, so all of them stand in the table: none is lost."""
    args = ([0, 3, 0], [5, 5, 40], 2, 9, list(range(50, 80)), [4, 30], rows, [[-7] * 9, [8, 9] + [-7] * 7, [-7] * 9])
    assert run_tables(*args) == po.tables(args[0], args[1], args[7], args[4], args[5], args[2], rows)
    rng = random.Random(rows)
    ctx, new, page = [rng.randrange(60) for _ in range(700)], [rng.randrange(50) for _ in range(700)], 8
    free = list(range(90000, 90000 + 3000))
    got = run_tables(ctx, new, page, 12, free, [7, 3000], 1000 * rows)
    assert got == po.tables(ctx, new, [[-7] * 12] * 700, free, [7, 3000], page, 1000 * rows)
    # lengths that no table has room for
    top = 2 ** 31 - 1
    assert run_tables([0, 5], [top, top], 4, 3, [5, 6, 7, 8], [0, 4], rows)["table"] == [[5, 6, 7], [-7, -7, 8]]


def test_a_step_with_more_tokens_than_the_module_has_rows_for():
    """The requests that do not fit are not answered; their pages come back when they are released."""
    m = r_paged.PagedAttention(12, 4, 2, 1, 64, 3, 8, 24, 0, BF16, scale=0.125)
    x = [torch.randn(8, h, 64, device="cuda").to(BF16) for h in (2, 1, 1)]
    m.begin_step(ints([0, 0, 0]), ints([5, 13, 1]))
    m.output.fill_(7.0)
    out = m(*x)
    want, _, tol, _ = po.attention(x[0][:5], m.k_cache[0], m.v_cache[0], m.block_table[:1], m.kv_lens[:1], m.q_start[:2], scale=0.125)
    assert bool(((out[:5].double() - want).abs() <= tol).all()) and bool((out[5:] == 7).all())
    assert m.missing_pages() == 0 and m.free_span.tolist() == [7, 12]
    for b, n in enumerate((5, 13, 1)):
        m.release(b, n)
    head, tail = m.free_span.tolist()
    assert sorted(int(m.free_pages[i % 12]) for i in range(head, tail)) == list(range(12))


def test_tables_of_the_longest_lengths():
    top = 2 ** 31 - 1
    got = run_tables([top, top], [1, 2], 1, 3, [5, 6], [0, 2], 3)
    assert got["slots"] == [-1, -1, -1] and got["kv_lens"] == [top, top] and got["table"] == [[-7] * 3] * 2


def test_tables_for_the_most_requests():
    B = 16384
    got = run_tables([0] * B, [1] * B, 4, 2, list(range(B)), [0, B], B)
    assert got["slots"] == [4 * b for b in range(B)] and got["requests"] == list(range(B))


# ----------------------------------------------------------------------------------------------
# a batch over a cache whose every row that no token stands in is NaN
# ----------------------------------------------------------------------------------------------
def batch(dtype, lens, heads, kv_heads, d, page, seed=0, rows_first=False, spare=2, pad=0, shift=0):
    """lens: (tokens in all, new ones) of every request.  pad: rows of q in front of and behind the requests'."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = [-(-max(kv, 0) // page) for kv, _ in lens]
    pages, width = sum(held) + spare, max([1] + held) + 1
    whole = d + shift
    shape = (pages, page, kv_heads, whole) if rows_first else (pages, kv_heads, page, whole)
    caches = [torch.full(shape, float("nan"), device="cuda", dtype=dtype)[..., shift:] for _ in range(2)]
    if rows_first:
        caches = [c.transpose(1, 2) for c in caches]
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, ((kv, _), h) in enumerate(zip(lens, held)):
        table[b, :h] = order[at:at + h]
        at += h
        j = torch.arange(max(kv, 0), device="cuda")
        for c in caches:
            c[table[b, j // page].long(), :, j % page] = torch.randn(len(j), kv_heads, d, device="cuda", generator=g).to(dtype)
    start = [pad]
    for _, n in lens:
        start.append(start[-1] + n)
    q = torch.randn(start[-1] + pad, heads, whole, device="cuda", generator=g).to(dtype)[..., shift:]
    return dict(q=q, k_cache=caches[0], v_cache=caches[1], block_table=table, kv_lens=ints([kv for kv, _ in lens]), q_start=ints(start))


def attend(x, **kw):
    out = torch.full(x["q"].shape, 7.0, device="cuda", dtype=x["q"].dtype)
    lse = torch.full(x["q"].shape[:2], 7.0, device="cuda")
    got = r_paged.rpaged_attention_launcher(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], out,
                                            q_start=x["q_start"], lse=lse, **kw)
    assert got is out
    return out, lse


def check(x, want=None, **kw):
    out, lse = attend(x, **kw)
    kw.pop("max_q_len", None)
    want, want_lse, tol, lse_tol = want or po.attention(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], x["q_start"], **kw)
    rows = ~want_lse.isnan().all(1) | want[:, 0, 0].isfinite()
    if not bool(rows.all()):
        assert bool((out[~rows] == 7).all()) and bool((lse[~rows] == 7).all())
    off = (out[rows].double() - want[rows]).abs()
    assert bool((off <= tol[rows]).all()), (float(off.nan_to_num(1e9).max()), float((off / tol[rows]).nan_to_num(1e9).max()))
    empty = want_lse[rows] == float("-inf")
    assert torch.equal(lse[rows] == float("-inf"), empty)
    off = (lse[rows].double() - want_lse[rows]).abs()[~empty]
    assert bool((off <= lse_tol[rows][~empty]).all()), float((off / lse_tol[rows][~empty]).max())


LENS = [(1, 1), (0, 0), (700, 1), (64, 1), (65, 2), (130, 0), (33, 5), (257, 3)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads, kv_heads, d, page", [(4, 2, 64, 16), (8, 8, 128, 64), (16, 1, 128, 16), (6, 2, 80, 24),
                                                      (3, 1, 40, 7), (10, 2, 128, 1), (7, 7, 33, 8), (4, 2, 256, 32), (24, 1, 64, 128)])
def test_a_few_tokens_of_each_request(dtype, heads, kv_heads, d, page):
    check(batch(dtype, LENS, heads, kv_heads, d, page, pad=2), scale=d ** -0.5)
    check(batch(dtype, [(kv, 1) for kv, _ in LENS if kv], heads, kv_heads, d, page, rows_first=True), scale=d ** -0.5, max_q_len=1)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kw", [dict(taps=1), dict(taps=64), dict(taps=100, stride=2), dict(stride=3), dict(stride=64), dict(taps=5, stride=1000),
                                dict(softcap=5.0), dict(slopes=True), dict(taps=77, softcap=3.0, slopes=True), dict(stride=4, slopes=True, softcap=10.0)],
                         ids=lambda kw: " ".join(f"{k}{v}" for k, v in kw.items()))
def test_patterns_caps_and_bias(dtype, kw):
    kw = dict(kw)
    if kw.get("slopes"):
        kw["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(8)], device="cuda")
    x = batch(dtype, [(300, 1), (1, 1), (129, 40), (513, 150), (64, 64)], 8, 2, 64, 16, seed=3)
    check(x, scale=0.125, **kw)
    x = batch(dtype, [(1000, 1), (65, 1), (64, 1), (3, 1)], 8, 4, 128, 32, seed=4)
    check(x, scale=0.2, max_q_len=1, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("softcap", [0.5, 50.0, 1e3, 1e5, 1e7, 1e30])
def test_caps_far_from_the_scores(dtype, softcap):
    """A capped score is as exact as its own size asks for, whatever the cap: single tokens, a few, and chunks."""
    for d, heads in ((64, 8), (128, 4)):
        check(batch(dtype, [(700, 1), (65, 1), (1, 1)], heads, 2, d, 16, seed=6), scale=d ** -0.5, softcap=softcap, max_q_len=1)
        check(batch(dtype, [(300, 3), (257, 150)], heads, 2, d, 16, seed=7), scale=d ** -0.5, softcap=softcap)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lens, heads, kv_heads, d, page", [
    ([(128, 128)], 2, 2, 64, 16), ([(200, 129), (257, 31)], 4, 1, 128, 64), ([(640, 130), (1, 1), (90, 90), (700, 1)], 6, 2, 128, 32),
    ([(333, 77)], 8, 1, 80, 24), ([(150, 150)], 5, 5, 96, 128), ([(300, 140)], 3, 1, 120, 8), ([(260, 130)], 2, 1, 48, 12)])
def test_chunks(dtype, lens, heads, kv_heads, d, page):
    x = batch(dtype, lens, heads, kv_heads, d, page, pad=1)
    for kw in (dict(), dict(taps=100), dict(stride=2, taps=40)):
        check(x, scale=d ** -0.5, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_context_is_divided_and_joined(dtype):
    x = batch(dtype, [(20000, 1), (9000, 3)], 8, 2, 128, 16)
    check(x, scale=0.3)
    x = batch(dtype, [(12000, 40)], 4, 1, 64, 64)
    check(x, scale=0.3)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_queries_without_a_key(dtype):
    """More queries than tokens, lengths of nothing, pages that are missing."""
    x = batch(dtype, [(3, 3), (40, 2), (5, 5), (70, 70)], 4, 2, 64, 16)
    x["kv_lens"].copy_(ints([1, 0, -4, 70]))               # the first request's first two queries stand in front of its start
    check(x, scale=0.2)
    x = batch(dtype, [(100, 100), (50, 1), (20, 20)], 4, 2, 64, 16)
    x["block_table"][0, 2] = -1
    x["block_table"][0, 0] = x["k_cache"].shape[0]
    x["block_table"][1, :] = 2 ** 31 - 1
    x["block_table"][2, 0] = -2 ** 31
    check(x, scale=0.2)
    check(x, scale=0.2, taps=3)
    x["kv_lens"][1] = 2 ** 31 - 1                          # (far beyond its table)
    check_rows = attend(x, scale=0.2)
    assert bool((check_rows[0][100] == 0).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 3, 200])
@pytest.mark.parametrize("page", [16, 7])
def test_lengths_far_beyond_the_table(dtype, new, page):
    """What a length claims behind the table's end is not there, and nothing walks over it: 2^30 keys would take seconds."""
    full, T = -(-130 // page) * page, new + 1              # (rows that no token was written to would be seen, too)
    x = batch(dtype, [(full, new), (40, 1)], 4, 2, 64, page, seed=9)
    alone = {**x, "block_table": torch.cat((x["block_table"][:1].expand(new, -1), x["block_table"][1:])).contiguous(),
             "kv_lens": ints([full] * new + [40]), "q_start": ints(list(range(T + 1)))}
    want = po.attention(*(alone[k] for k in ("q", "k_cache", "v_cache", "block_table", "kv_lens", "q_start")), scale=0.2)
    attend(x, scale=0.2), attend(x, scale=0.2, max_q_len=new)      # (the first calls load the kernels)
    events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    for length in (10 ** 6, 2 ** 30 - 5, 2 ** 31 - 1):
        x["kv_lens"][0] = length
        for kw in (dict(), dict(max_q_len=new)):
            torch.cuda.synchronize()
            events[0].record()
            out, lse = attend(x, scale=0.2, **kw)
            events[1].record()
            torch.cuda.synchronize()
            assert events[0].elapsed_time(events[1]) < 20
            assert bool(((out.double() - want[0]).abs() <= want[2]).all()) and bool(((lse.double() - want[1]).abs() <= want[3]).all())
        out, lse = attend(x, scale=0.2, taps=60)           # a window behind everything that is there
        assert bool((out[:new] == 0).all()) and bool((lse[:new] == float("-inf")).all()) and bool(lse[new:].isfinite().all())
        for stride in (2, 64):
            out, lse = attend(x, scale=0.2, stride=stride)
            assert bool(lse.isfinite().all())


def test_rows_of_no_request():
    x = batch(BF16, [(40, 7), (30, 1)], 4, 2, 64, 16, pad=9)
    check(x, scale=0.2)
    # requests whose rows do not lie within q are left alone, and so is q
    x["q_start"].copy_(ints([9, 16, 200]))
    out, _ = attend(x)
    assert bool((out[16:] == 7).all()) and not bool((out[9:16] == 7).any())
    x["q_start"].copy_(ints([-3, 4, 2]))
    out, _ = attend(x)
    assert bool((out == 7).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_masked_keys_hold_does_not_matter(dtype, bad):
    """K and V of later tokens, of keys outside the pattern and of other requests."""
    for lens, kw, hurt in (([(90, 30), (200, 1)], dict(), 75), ([(200, 150)], dict(taps=9), 100), ([(300, 200)], dict(stride=4, taps=20), 160)):
        x = batch(dtype, lens, 4, 2, 64, 16)
        want = po.attention(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], x["q_start"], scale=0.2, **kw)
        page, row = int(x["block_table"][0, hurt // 16]), hurt % 16
        x["k_cache"][page, :, row] = bad
        x["v_cache"][page, :, row] = bad
        out, lse = attend(x, scale=0.2, **kw)
        kv, n = lens[0]
        for t in range(out.shape[0]):
            i = kv - n + t
            away = i - hurt
            sees = t < n and away >= 0 and away % kw.get("stride", 1) == 0 and away // kw.get("stride", 1) < kw.get("taps", 1 << 30)
            if not sees:
                assert bool(((out[t].double() - want[0][t]).abs() <= want[2][t]).all()), (t, i)
                assert bool(((lse[t].double() - want[1][t]).abs() <= want[3][t]).all()), (t, i)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [dict(softcap=30.0), dict(softcap=30.0, taps=50), dict(softcap=30.0, stride=2), dict(softcap=3.0), dict()],
                         ids=lambda kw: " ".join(f"{k}{v}" for k, v in kw.items()))
def test_keys_that_no_query_sees_do_not_change_a_bit(dtype, d, kw):
    """Rows of the cache behind the last token, keys in front of every window and pages that are missing."""
    x = batch(dtype, [(200, 100), (75, 40), (330, 1)], 4, 2, d, 16)
    x["block_table"][0, 9] = -1                            # 144 to 159
    rows = []                                              # (page, row) that no query sees
    for b, (kv, n) in enumerate(((200, 100), (75, 40), (330, 1))):
        seen = {j for i in range(kv - n, kv) for j in list(range(i, -1, -kw.get("stride", 1)))[:kw.get("taps") or None]}
        for j in range(-(-kv // 16) * 16):
            if j not in seen and int(x["block_table"][b, j // 16]) >= 0:
                rows.append((int(x["block_table"][b, j // 16]), j % 16))
    pages, at = (ints(v, torch.int64) for v in zip(*rows))
    first = None
    for held in (float("nan"), 0.0, 300.0, -6e4, float("inf"), 0.0):
        x["k_cache"][pages, :, at] = held
        x["v_cache"][pages, :, at] = held if math.isfinite(held) else 1.0      # (a row that meets infinity is computed again, otherwise)
        got = attend(x, scale=d ** -0.5, **kw)
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1]), held


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_seen_keys_hold_matters(dtype):
    x = batch(dtype, [(40, 20)], 2, 1, 64, 16)
    page, row = int(x["block_table"][0, 1]), 3             # token 19: all 20 queries see it
    x["v_cache"][page, 0, row, 5] = float("inf")
    out, lse = attend(x, scale=0.1)
    assert bool((out[..., 5] == float("inf")).all()) and bool(lse.isfinite().all())
    assert bool(out[..., :5].isfinite().all()) and bool(out[..., 6:].isfinite().all())
    x["k_cache"][page, 0, row, 0] = float("nan")
    out, lse = attend(x, scale=0.1)
    assert bool(out.isnan().all()) and bool(lse.isnan().all())


def test_large_scores():
    for dtype in (F32, F16, BF16):
        x = batch(dtype, [(400, 60), (300, 1)], 4, 2, 64, 16)
        check(x, scale=8.0)
        check(x, scale=-8.0)
        check(x, scale=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_offsets_and_strides_of_the_operands(dtype):
    """Rows that do not start on 16 bytes, q as a slice of a fused projection, K and V as halves of one array."""
    x = batch(dtype, [(130, 3), (70, 1), (200, 140)], 4, 2, 64, 16, shift=3)
    check(x, scale=0.2)
    x = batch(dtype, [(130, 3), (70, 1), (200, 140)], 4, 2, 64, 16)
    wide = torch.randn(x["q"].shape[0], 8, 64, device="cuda").to(dtype)
    wide[:, :4] = x["q"]
    both = torch.stack((x["k_cache"], x["v_cache"]), 1)
    y = {**x, "q": wide[:, :4], "k_cache": both[:, 0], "v_cache": both[:, 1]}
    check(y, scale=0.2)
    table = torch.full((3, x["block_table"].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    table[:, :-5] = x["block_table"]
    check({**y, "block_table": table[:, :-5]}, scale=0.2)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 elements: pages at its far end."""
    pages, page, d = (1 << 32) // (64 * 2 * 128) + 8, 64, 128
    caches = [torch.zeros(pages, 2, page, d, device="cuda", dtype=BF16) for _ in range(2)]
    x = batch(BF16, [(300, 1), (200, 140)], 4, 2, d, page)
    far = torch.tensor([pages - 1 - i for i in range(x["k_cache"].shape[0])], device="cuda")
    for c, name in zip(caches, ("k_cache", "v_cache")):
        c[far] = x[name]
    want = po.attention(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], x["q_start"], scale=0.1)
    x["block_table"] = torch.where(x["block_table"] >= 0, far[x["block_table"].clamp(min=0).long()].to(torch.int32), -1)
    check({**x, "k_cache": caches[0], "v_cache": caches[1]}, want=want, scale=0.1)
    slots = far[:3] * page + 5
    new = torch.randn(3, 2, d, device="cuda").to(BF16)
    r_paged.rpaged_append_launcher(None, new, new, caches[0], caches[1], slots)
    assert torch.equal(caches[0][far[:3], :, 5], new) and torch.equal(caches[1][far[:3], :, 5], new)


@pytest.mark.parametrize("requests", [129, 700])
def test_many_requests(requests):
    rng = random.Random(requests)
    lens = [(rng.randint(1, 50), 1) if rng.random() < 0.9 else (0, 0) for _ in range(requests)]
    check(batch(F16, lens, 4, 4, 64, 16), scale=0.2)


def test_many_requests_with_chunks():
    rng = random.Random(8)
    lens = [(rng.randint(20, 60), 20) if rng.random() < 0.7 else (rng.randint(1, 60), 1) for _ in range(300)]
    check(batch(BF16, lens, 4, 1, 64, 16), scale=0.2)
    check(batch(F16, [(24, 8)] * 40, 4, 1, 128, 32), scale=0.2, max_q_len=8)


def test_a_bound_on_the_lengths_that_does_not_hold():
    """max_q_len chooses the kernel; requests that bring more, or fewer as the number of rows suggests, are right all the same."""
    x = batch(BF16, [(300, 150), (40, 1), (70, 9)], 4, 1, 64, 16)
    want = po.attention(*(x[k] for k in ("q", "k_cache", "v_cache", "block_table", "kv_lens", "q_start")), scale=0.2)
    for most in (0, 1, 5, 53, 54, 160, 1 << 40):
        check(x, want=want, scale=0.2, max_q_len=most)


def test_cache_without_pages_and_tables_without_columns():
    x = batch(BF16, [(20, 3), (5, 1)], 4, 2, 64, 16)
    none = x["k_cache"][:0]
    out, lse = attend({**x, "k_cache": none, "v_cache": none.clone()})
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    out, lse = attend({**x, "block_table": x["block_table"][:, :0].contiguous()})
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())


def test_large_strides():
    """Strides and windows beyond every length: a query's own key alone."""
    x = batch(BF16, [(50, 20), (9, 1)], 4, 2, 64, 16)
    for kw in (dict(stride=1 << 40), dict(taps=1), dict(stride=2 ** 31, taps=2 ** 40)):
        check(x, scale=0.2, **({"stride": 1 << 20} if "taps" not in kw else {"taps": 1}))
        a, b = attend(x, scale=0.2, **kw), attend(x, scale=0.2, taps=1)
        assert torch.equal(a[0], b[0])
    check(x, scale=0.2, taps=2 ** 40)


@pytest.mark.parametrize("heads, kv_heads", [(64, 1), (130, 2), (33, 3)])
def test_many_heads_to_a_group(heads, kv_heads):
    check(batch(F16, [(200, 1), (40, 3)], heads, kv_heads, 64, 16), scale=0.2)


def test_a_reported_wait_stops_the_kernels_and_is_raised():
    """While the status word is set the tensor-core kernels do nothing; the next call raises and clears it."""
    import splat_native as n
    dev = torch.device("cuda", torch.cuda.current_device())
    x, y = batch(BF16, [(200, 1)], 4, 2, 64, 16), batch(BF16, [(200, 100)], 4, 2, 64, 16)
    attend(x), attend(y)
    for z, kw in ((x, dict(max_q_len=1)), (y, {})):
        n.status_word(dev).fill_(81)
        torch.cuda.synchronize()
        out, lse = attend(z, **kw)
        torch.cuda.synchronize()
        assert bool((out == 7).all()) and bool((lse == 7).all())
        with pytest.raises(RuntimeError, match="code 81"):
            attend(z, **kw)
        check(z, scale=0.2, **kw)


def test_first_call_of_a_process_is_captured():
    """No status word yet, and none can be set up: kernels without bounded waits run, with the same results."""
    import os
    import subprocess
    import sys
    import textwrap
    from conftest import ROOT, SPLAT_DIR
    code = """
        import torch
        import test_gpu_paged as t
        from oracle import paged_oracle as po
        for lens in ([(300, 1), (40, 1)], [(200, 90), (30, 3)]):
            x = t.batch(torch.bfloat16, lens, 4, 2, 64, 16)
            out = torch.full(x["q"].shape, 7.0, device="cuda", dtype=x["q"].dtype)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                t.r_paged.rpaged_attention_launcher(x["q"], x["k_cache"], x["v_cache"], x["block_table"], x["kv_lens"], out,
                                                    q_start=x["q_start"], scale=0.2)
            graph.replay()
            want, _, tol, _ = po.attention(*(x[k] for k in ("q", "k_cache", "v_cache", "block_table", "kv_lens", "q_start")), scale=0.2)
            assert bool(((out.double() - want).abs() <= tol).all())
        print("alive")
        """
    head = f"import sys; sys.path[:0] = [{ROOT!r}, {SPLAT_DIR!r}, {os.path.join(ROOT, 'tests')!r}]\n"
    r = subprocess.run([sys.executable, "-c", head + textwrap.dedent(code)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "alive" in r.stdout, r.stderr[-2000:]


def test_results_do_not_depend_on_timing():
    x = batch(BF16, [(9000, 1), (5000, 200), (17, 1)], 8, 2, 128, 16)
    first = attend(x, scale=0.1)
    for _ in range(5):
        again = attend(x, scale=0.1)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_streams_and_graphs():
    """Two captured graphs and an eager call at once, each with scratch of its own; lengths that change between replays."""
    xs = [batch(BF16, [(6000, 1), (900, 1), (50, 1)], 8, 2, 128, 16, seed=s) for s in range(3)]
    want = [attend(x, scale=0.1, max_q_len=1) for x in xs]
    outs, graphs, streams = [], [], [torch.cuda.Stream() for _ in xs]
    for x in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attend(x, scale=0.1, max_q_len=1))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = attend(xs[2], scale=0.1, max_q_len=1)
    torch.cuda.synchronize()
    for got, expected in zip(outs + [eager], want):
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
    xs[0]["kv_lens"].copy_(ints([5000, 20, 48]))
    graphs[0].replay()
    check_against = po.attention(*(xs[0][k] for k in ("q", "k_cache", "v_cache", "block_table", "kv_lens", "q_start")), scale=0.1)
    assert bool(((outs[0][0].double() - check_against[0]).abs() <= check_against[2]).all())


# ----------------------------------------------------------------------------------------------
# append
# ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T, heads, kv_heads, d, half, axes, interleaved, page", [
    (1, 4, 2, 64, 32, 1, False, 16), (37, 8, 8, 128, 64, 3, False, 16), (300, 6, 2, 80, 20, 2, True, 24), (19, 3, 1, 33, 16, 2, False, 7)])
def test_append(dtype, T, heads, kv_heads, d, half, axes, interleaved, page):
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = torch.randn(T, heads + 2 * kv_heads, d, device="cuda", generator=g).to(dtype)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    slots[T // 2] = -1
    if T > 10:
        slots[3], slots[5] = pages * page, 2 ** 40
    pos = torch.randint(0, 9999, (axes, T), device="cuda", generator=g)
    freq = torch.rand(half, device="cuda", generator=g)
    cut = (half - (axes - 1) * (half // 4), *[half // 4] * (axes - 1))
    for rows_first in (False, True):
        caches = [torch.full((pages, page, kv_heads, d) if rows_first else (pages, kv_heads, page, d), 7.0, device="cuda", dtype=dtype) for _ in range(2)]
        views = [c.transpose(1, 2) if rows_first else c for c in caches]
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        r_paged.rpaged_append_launcher(q, k, v, *views, slots, q_out, positions=pos, inv_freq=freq, sections=cut, interleaved=interleaved)
        turned = [po.rotary(x.transpose(0, 1)[None], pos[:, None], freq, cut, interleaved)[0].transpose(0, 1) for x in (q, k)]
        u = torch.finfo(dtype).eps / 2

        def near(got, want, x):      # as in test_gpu_rotary.py
            size = x.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
            return bool(((got.double() - want).abs() <= u * want.abs() + 4 * 2.0 ** -22 * size * (1 + u) + torch.finfo(dtype).smallest_normal).all())
        assert near(q_out, turned[0], q)
        kept = (slots >= 0) & (slots < pages * page)
        at = slots[kept]
        rows = [c.transpose(1, 2).reshape(pages * page, kv_heads, d) for c in views]
        assert near(rows[0][at], turned[1][kept], k[kept]) and torch.equal(rows[1][at], v[kept])
        rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert bool((rows[0][rest] == 7).all()) and bool((rows[1][rest] == 7).all())
        # without positions: copies
        r_paged.rpaged_append_launcher(q, k, v, *views, slots, q_out)
        rows = [c.transpose(1, 2).reshape(pages * page, kv_heads, d) for c in views]
        assert torch.equal(q_out, q) and torch.equal(rows[0][at], k[kept]) and torch.equal(rows[1][at], v[kept])


def test_append_of_nothing():
    cache = torch.zeros(2, 2, 16, 64, device="cuda")
    none = torch.zeros(0, 2, 64, device="cuda")
    r_paged.rpaged_append_launcher(None, none, none, cache, cache.clone(), torch.zeros(0, dtype=torch.int64, device="cuda"))
    out = torch.zeros(0, 4, 64, device="cuda")
    r_paged.rpaged_attention_launcher(out, cache, cache.clone(), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), ints([1, 2, 3]), out,
                                      q_start=ints([0, 0, 0, 0]))


# ----------------------------------------------------------------------------------------------
# all of them together
# ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kw", [dict(), dict(taps=20), dict(stride=3, taps=9)], ids=["causal", "window", "dilated"])
def test_serving_steps(dtype, kw):
    """Prompts in chunks, decoding beside them, a request that leaves and one that takes its place; every step's output is that
    of attention over the whole sequences, turned to their positions."""
    heads, kv_heads, d, page, B, T = 4, 2, 64, 8, 3, 40
    half = 24
    freq = torch.tensor([100.0 ** (-i / half) for i in range(half)], device="cuda")
    m = r_paged.PagedAttention(24, page, heads, kv_heads, d, B, T, 96, 0, dtype, num_layers=2, scale=d ** -0.5, inv_freq=freq,
                               sections=(16, 8), lse=True, **kw)
    g = torch.Generator(device="cuda").manual_seed(2)
    seqs = [{"k": [], "v": []} for _ in range(B)]
    lens = [0] * B
    steps = [[30, 7, 0], [1, 20, 5], [1, 1, 1], [1, 1, 33], None, [1, 25, 1], [1, 1, 1]]
    for step in steps:
        if step is None:                                   # request 1 is done
            m.release(1, lens[1])
            lens[1], seqs[1] = 0, {"k": [], "v": []}
            continue
        n = sum(step)
        q, k, v = (torch.randn(T, h, d, device="cuda", generator=g).to(dtype) for h in (heads, kv_heads, kv_heads))
        m.begin_step(ints(lens), ints(step), max(step))
        places = torch.stack((m.positions, m.positions // 7)).contiguous()
        m.output.fill_(7.0)
        for layer in (1, 0):
            out = m(q, k, v, layer=layer, positions=places)
        assert m.missing_pages() == 0
        row = 0
        for b, new in enumerate(step):
            pos = torch.arange(lens[b], lens[b] + new, device="cuda")
            where = torch.stack((pos, pos // 7))[:, None]
            # keys as the cache holds them: turned in 64 bits and rounded to the type (to the neighbour, where the kernel's differ)
            seqs[b]["k"].append(k[row:row + new].transpose(0, 1)[None])
            seqs[b]["v"].append(v[row:row + new])
            lens[b] += new
            kv = lens[b]
            have = [m.k_cache[0], m.v_cache[0]]
            j = torch.arange(kv, device="cuda")
            at = m.block_table[b, j // page].long()
            assert torch.equal(have[1][at, :, j % page], torch.cat(seqs[b]["v"]))
            both = torch.stack((j, j // 7))[:, None]
            exact = po.rotary(torch.cat(seqs[b]["k"], 2), both, freq, (16, 8))[0].transpose(0, 1) if kv else None
            if kv:
                u = torch.finfo(dtype).eps / 2
                size = exact.abs().amax(-1, keepdim=True) * 2
                assert bool(((have[0][at, :, j % page].double() - exact).abs() <= u * exact.abs() + 2.0 ** -19 * size).all())
            if new:
                turned = po.rotary(q[row:row + new].transpose(0, 1)[None], where, freq, (16, 8))[0].transpose(0, 1)
                assert bool(((m.q_turned[row:row + new].double() - turned).abs() <= u * turned.abs() + 2.0 ** -19 * 8).all())
            row += new
        want, want_lse, tol, lse_tol = po.attention(m.q_turned, m.k_cache[0], m.v_cache[0], m.block_table, m.kv_lens, m.q_start,
                                                    scale=d ** -0.5, **kw)
        assert out is m.output and bool(((out[:n].double() - want[:n]).abs() <= tol[:n]).all())
        assert bool(((m.lse[:n].double() - want_lse[:n]).abs() <= lse_tol[:n]).all())
        assert bool((out[n:] == 7).all())
        assert torch.equal(m.k_cache[0], m.k_cache[1])
    m.check_status()


def test_drafted_tokens_that_are_refused():
    """Steps of up to six drafted tokens of which some are kept: no page is lost, and what is kept is attended to."""
    heads, kv_heads, d, page, B = 4, 2, 64, 4, 3
    m = r_paged.PagedAttention(180, page, heads, kv_heads, d, B, 6 * B, 240, 0, BF16, scale=d ** -0.5)
    rng, lens = random.Random(4), [0] * B
    graph = None
    lengths, drafts = ints([0] * B), ints([0] * B)
    q, k, v = (torch.zeros(6 * B, h, d, device="cuda", dtype=BF16) for h in (heads, kv_heads, kv_heads))

    def step():
        m.rewind(lengths)
        m.begin_step(lengths, drafts, 6)
        m(q, k, v)
    values = [[] for _ in range(B)]
    for i in range(40):
        new = [rng.randint(1, 6) for _ in range(B)]
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda"))
        lengths.copy_(ints(lens))
        drafts.copy_(ints(new))
        if i < 3:
            step()
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            graph.replay()
        assert m.missing_pages() == 0
        head, tail = m.free_span.tolist()
        entries = [e for row in m.block_table.tolist() for e in row if e >= 0]
        free = [int(m.free_pages[j % 180]) for j in range(head, tail)]
        assert sorted(entries + free) == list(range(180))
        assert len(entries) == sum(-(-(a + b) // page) for a, b in zip(lens, new))
        want, _, tol, _ = po.attention(q, m.k_cache[0], m.v_cache[0], m.block_table, m.kv_lens, m.q_start, scale=d ** -0.5)
        n = sum(new)
        assert bool(((m.output[:n].double() - want[:n]).abs() <= tol[:n]).all())
        row = 0
        for b in range(B):
            kept = rng.randint(1, new[b])
            values[b].append(v[row:row + kept].clone())
            row += new[b]
            lens[b] += kept
            j = torch.arange(lens[b], device="cuda")
            assert torch.equal(m.v_cache[0][m.block_table[b, j // page].long(), :, j % page], torch.cat(values[b]))


def test_captured_serving_step():
    """A decoding step recorded once and replayed as the requests grow."""
    heads, kv_heads, d, page, B = 8, 2, 128, 16, 4
    m = r_paged.PagedAttention(64, page, heads, kv_heads, d, B, B, 200, 0, BF16, scale=d ** -0.5)
    lens, ones = ints([0] * B), ints([1] * B)
    q, k, v = (torch.randn(B, h, d, device="cuda").to(BF16) for h in (heads, kv_heads, kv_heads))

    def step():
        m.begin_step(lens, ones, 1)
        m(q, k, v)
        lens.add_(1)
    step()
    lens.zero_()
    m.free_span.copy_(ints([0, 64], torch.int64))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens.zero_()
    m.free_span.copy_(ints([0, 64], torch.int64))
    for i in range(40):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        if i % 13 == 0 or i == 39:
            want, _, tol, _ = po.attention(q, m.k_cache[0], m.v_cache[0], m.block_table, m.kv_lens, m.q_start, scale=d ** -0.5)
            assert bool(((m.output.double() - want).abs() <= tol).all())
    assert m.kv_lens.tolist() == [40] * B and m.missing_pages() == 0


def test_log_sums_in_another_operands_place_are_refused():
    q, cache = torch.zeros(2, 4, 4, device="cuda"), torch.zeros(3, 4, 2, 4, device="cuda")
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    out, other = torch.zeros_like(q), torch.zeros_like(cache)
    for lse in (q.view(-1)[:8].view(2, 4), out.view(-1)[:8].view(2, 4), cache.view(-1)[:8].view(2, 4)):
        with pytest.raises(ValueError, match="share memory"):
            r_paged.rpaged_attention_launcher(q, cache, other, table, lens, out, lse=lse)


def joined(rows_of, begins, rows=4, d=8, tokens=3, heads=2, status=0):
    """splat_selftest_paged_join over the parts (part, row) -> (maximum, sum, token, head, value), in an output with room around it."""
    import ctypes
    import splat_native as n

    class Args(ctypes.Structure):
        _fields_ = [(f, ctypes.c_void_p) for f in ("q", "k_cache", "v_cache", "o", "lse")] + \
                   [(f, ctypes.c_int64) for f in ("q_row", "q_head", "o_row", "o_head", "k_page", "k_head", "k_row", "v_page", "v_head", "v_row")] + \
                   [("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_width", ctypes.c_int64)] + \
                   [(f, ctypes.c_void_p) for f in ("kv_lens", "q_start", "slopes")] + \
                   [(f, ctypes.c_int64) for f in ("tokens", "requests", "pages", "page", "heads", "kv_heads", "d", "taps", "stride", "max_q_len")] + \
                   [("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("dtype", ctypes.c_int32), ("status_word", ctypes.c_void_p),
                    ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)]

    ctas, at = len(begins), -(-len(begins) * 8 // 16) * 16
    work = torch.zeros(at + 2 * ctas * rows * 16 + 2 * ctas * rows * 64 * 4, dtype=torch.uint8, device="cuda")
    work[:ctas * 8].view(torch.int64).copy_(ints(begins, torch.int64))
    ends = work[at:at + 2 * ctas * rows * 16].view(torch.float32).view(2 * ctas, rows, 4)
    sums = work[at + 2 * ctas * rows * 16:].view(torch.float32).view(2 * ctas, rows, 64)
    ends[:, :, 2:].view(torch.int32).fill_(-1)
    for (part, row), (top, total, token, head, value) in rows_of.items():
        ends[part, row, :2] = torch.tensor([top, total], device="cuda")
        ends[part, row, 2:].view(torch.int32).copy_(ints([token, head]))
        sums[part, row, :d] = value
    around = torch.full((50, heads, d), 7.0, device="cuda")
    lse = torch.full((50, heads), 7.0, device="cuda")
    word = ints([status])
    out, out_lse = around[20:20 + tokens], lse[20:20 + tokens]
    x = Args(o=out.data_ptr(), lse=out_lse.data_ptr(), o_row=heads * d, o_head=d, tokens=tokens, requests=1, pages=1, page=16, heads=heads,
             kv_heads=1, d=d, stride=1, status_word=word.data_ptr(), workspace=work.data_ptr(), workspace_bytes=work.numel())
    assert n._lib.splat_selftest_paged_join(ctypes.byref(x), ctas, rows, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    rest = torch.ones(50, dtype=torch.bool)
    rest[20:20 + tokens] = False
    assert bool((around[rest] == 7).all()) and bool((lse[rest] == 7).all())
    return out.cpu(), out_lse.cpu()


def test_joining_of_parts_that_a_kernel_never_wrote():
    """A kernel that gives up has announced parts that it does not write: the workspace holds anything.  Rows that the call does not have
    are not written, and none is while the status word is set."""
    good = {(1, 0): (0.0, 1.0, 0, 1, 2.0), (2, 0): (1.0, 1.0, 0, 1, 8.0)}
    # (0 + 2^0 2 + 2^1 8) / (2^0 + 2^1), and its log-sum-exp
    out, lse = joined(good, [-1, 0, -1])
    assert bool(((out[0, 1] - 6.0).abs() < 1e-5).all()) and abs(float(lse[0, 1]) - math.log(3)) < 1e-6 and bool((out[0, 0] == 7).all())
    for token, head in ((3, 0), (5, 1), (-1, 0), (-17, 0), (1, 2), (1, -1), (0, 9), (29, 0)):
        bad = {**good, (1, 1): (0.0, 1.0, token, head, 3.0), (2, 1): (0.0, 1.0, token, head, 3.0)}
        for begins in ([-1, 0, -1], [-1, 0, -1, -1, -1]):  # a warp to a row, and four
            out, lse = joined(bad, begins)
            assert bool(((out[0, 1] - 6.0).abs() < 1e-5).all())
            out[0, 1], lse[0, 1] = 7.0, 7.0
            assert bool((out == 7).all()) and bool((lse == 7).all()), (token, head)
    for begins in ([-1, 0, -1], [-1, 0, -1, -1, -1]):
        out, lse = joined(good, begins, status=81)
        assert bool((out == 7).all()) and bool((lse == 7).all())
    # tiles of 32 rows: a warp to a row
    out, lse = joined({**good, (1, 30): (0.0, 1.0, 29, 0, 3.0), (2, 31): (0.0, 1.0, 3, 0, 3.0)}, [-1, 0, -1], rows=32)
    assert bool(((out[0, 1] - 6.0).abs() < 1e-5).all()) and bool((out[1:] == 7).all())
