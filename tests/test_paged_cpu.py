"""CPU: what the paged cache's and the rotary positions' launchers refuse, and their oracle against itself."""
import random

import pytest
import torch

import r_paged
import r_rotary
from oracle import paged_oracle as po


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def i64(*shape):
    return torch.zeros(shape, dtype=torch.int64)


def refused(call, kw, change, words, error=ValueError):
    kw = {**kw, **change}
    with pytest.raises(error, match=words):
        call(**kw)


def tables_args():
    return dict(ctx_lens=i32(3), q_lens=i32(3), block_table=i32(3, 5), free_pages=i32(9), free_span=i64(2), page_size=16,
                kv_lens=i32(3), q_start=i32(4), slots=i64(7), positions=i32(7), requests=i32(7), free_span_out=i64(3))


@pytest.mark.parametrize("change, words, error", [
    (dict(), "CUDA devices only", ValueError),
    (dict(q_lens=i32(2)), "q_lens and ctx_lens", ValueError),
    (dict(ctx_lens=i64(3)), "ctx_lens must be int32", TypeError),
    (dict(slots=i32(7)), "slots must be int64", TypeError),
    (dict(q_start=i32(3)), "q_start", ValueError),
    (dict(block_table=i32(2, 5)), "a row for each request", ValueError),
    (dict(block_table=i32(1, 5).expand(3, 5)), "must not overlap", ValueError),
    (dict(block_table=i32(5, 3).t()), "last dimension", ValueError),
    (dict(page_size=0), "page_size must be at least 1", ValueError),
    (dict(page_size=1.5), "integer", TypeError),
    (dict(free_pages=i32(0)), "must not be empty", ValueError),
    (dict(free_span=i64(3)), "2 entries", ValueError),
    (dict(free_span_out=i64(2)), "3 entries", ValueError),
    (dict(positions=i32(6)), "differ in length", ValueError),
    (dict(ctx_lens=i32(6)[::2]), "contiguous", ValueError),
    (dict(ctx_lens=[1, 2, 3]), "must be a tensor", TypeError),
    (dict(ctx_lens=i32(20000), q_lens=i32(20000), kv_lens=i32(20000), q_start=i32(20001), block_table=i32(20000, 1)),
     "at most", ValueError),
])
def test_tables_refusals(change, words, error):
    refused(r_paged.rpaged_tables_launcher, tables_args(), change, words, error)


def rotary_args():
    return dict(q=torch.zeros(2, 4, 6, 16), k=torch.zeros(2, 2, 6, 16), positions=i32(3, 2, 6), inv_freq=torch.zeros(8),
                sections=(4, 2, 2))


@pytest.mark.parametrize("change, words, error", [
    (dict(), "CUDA devices only", ValueError),
    (dict(k=torch.zeros(2, 2, 5, 16)), "must agree", ValueError),
    (dict(k=torch.zeros(2, 2, 6, 16).half()), "dtype", TypeError),
    (dict(q=torch.zeros(2, 4, 6, 16).double()), "unsupported dtype", TypeError),
    (dict(q=torch.zeros(4, 6, 16)), "4-dimensional", ValueError),
    (dict(q=torch.zeros(2, 4, 16, 6).transpose(2, 3)), "last dimension", ValueError),
    (dict(positions=i32(3, 2, 5)), "differ in length", ValueError),
    (dict(positions=i32(3, 1, 6)), "differ in batch", ValueError),
    (dict(positions=torch.zeros(3, 2, 6)), "int32 or int64", TypeError),
    (dict(positions=i32(5, 2, 6), sections=(2, 2, 2, 1, 1)), "1 to 4 axes", ValueError),
    (dict(sections=(4, 4)), "an entry for each axis", ValueError),
    (dict(sections=(4, 2, 1)), "add up", ValueError),
    (dict(sections=(10, -1, -1)), "at least 0", ValueError),
    (dict(sections=None), "must be given", ValueError),
    (dict(inv_freq=torch.zeros(9), sections=(5, 2, 2)), "only 16 elements", ValueError),
    (dict(inv_freq=torch.zeros(8).double()), "float32", TypeError),
])
def test_rotary_refusals(change, words, error):
    refused(r_rotary.rrotary_launcher, rotary_args(), change, words, error)
    refused(r_rotary.rrotary, rotary_args(), change, words, error)


def test_rotary_refuses_gradients_of_the_frequencies_and_expanded_outputs():
    kw = rotary_args()
    kw["inv_freq"].requires_grad_(True)
    refused(r_rotary.rrotary, kw, {}, "no.* for the frequencies")
    refused(r_rotary.rrotary_launcher, rotary_args(), dict(q_out=torch.zeros(1, 4, 6, 16).expand(2, 4, 6, 16)), "expanded")
    refused(r_rotary.rrotary_launcher, rotary_args(), dict(q_out=torch.zeros(2, 4, 6, 8)), "shape")


def append_args():
    return dict(q=torch.zeros(5, 4, 16), k=torch.zeros(5, 2, 16), v=torch.zeros(5, 2, 16), k_cache=torch.zeros(3, 2, 8, 16),
                v_cache=torch.zeros(3, 2, 8, 16), slots=i64(5), q_out=torch.zeros(5, 4, 16), positions=i32(2, 5),
                inv_freq=torch.zeros(8), sections=(5, 3))


@pytest.mark.parametrize("change, words, error", [
    (dict(), "CUDA devices only", ValueError),
    (dict(slots=i64(4)), "differ in length", ValueError),
    (dict(slots=i32(5)), "int64", TypeError),
    (dict(v=torch.zeros(5, 3, 16)), "same shape", ValueError),
    (dict(k_cache=torch.zeros(3, 1, 8, 16), v_cache=torch.zeros(3, 1, 8, 16)), "differ in heads", ValueError),
    (dict(k_cache=torch.zeros(3, 2, 8, 8), v_cache=torch.zeros(3, 2, 8, 8)), "differ in length", ValueError),
    (dict(k_cache=torch.zeros(3, 2, 8, 16).half()), "dtype", TypeError),
    (dict(k_cache=torch.zeros(1, 2, 8, 16).expand(3, 2, 8, 16)), "expanded", ValueError),
    (dict(k_cache=torch.zeros(3, 2, 16, 8).transpose(2, 3)), "last dimension", ValueError),
    (dict(q_out=None), "q_out must be a tensor", TypeError),
    (dict(q=None), "q_out without q", ValueError),
    (dict(q_out=torch.zeros(5, 4, 8)), "shape of q", ValueError),
    (dict(positions=None), "inv_freq without positions", ValueError),
    (dict(inv_freq=None), "positions without inv_freq", ValueError),
    (dict(positions=i32(2, 4)), "differ in length", ValueError),
    (dict(positions=i32(2, 1, 5)), "axes, tokens", ValueError),
])
def test_append_refusals(change, words, error):
    refused(r_paged.rpaged_append_launcher, append_args(), change, words, error)


def attention_args():
    return dict(q=torch.zeros(5, 4, 16), k_cache=torch.zeros(3, 2, 8, 16), v_cache=torch.zeros(3, 2, 8, 16),
                block_table=i32(2, 4), kv_lens=i32(2), output=torch.zeros(5, 4, 16), q_start=i32(3))


@pytest.mark.parametrize("change, words, error", [
    (dict(), "CUDA devices only", ValueError),
    (dict(q_start=None), "one token for each request", ValueError),
    (dict(q_start=i32(2)), "one entry more", ValueError),
    (dict(q_start=i64(3)), "int32", TypeError),
    (dict(q=torch.zeros(5, 3, 16), output=torch.zeros(5, 3, 16)), "multiple", ValueError),
    (dict(output=torch.zeros(5, 4, 8)), "shape of q", ValueError),
    (dict(output=torch.zeros(5, 4, 32)[..., ::2]), "output must be contiguous", ValueError),
    (dict(output=torch.zeros(5, 4, 16).half()), "dtype", TypeError),
    (dict(v_cache=torch.zeros(3, 2, 4, 16)), "same shape", ValueError),
    (dict(block_table=i32(1, 4)), "a row for each request", ValueError),
    (dict(kv_lens=i64(2)), "int32", TypeError),
    (dict(taps=-1), "taps must be at least 0", ValueError),
    (dict(stride=0), "stride must be at least 1", ValueError),
    (dict(softcap=-1.0), "softcap must not be negative", ValueError),
    (dict(softcap=1e-40), "too small for the scale", ValueError),
    (dict(softcap=1e-30, scale=1e10), "too small for the scale", ValueError),
    (dict(scale=float("nan")), "scale must be finite", ValueError),
    (dict(scale=1e300), "scale must be finite", ValueError),
    (dict(slopes=torch.zeros(2)), "an entry for each head", ValueError),
    (dict(slopes=torch.zeros(4).half()), "float32", TypeError),
    (dict(lse=torch.zeros(4, 5)), "lse must have shape", ValueError),
    (dict(max_q_len=-1), "max_q_len must be at least 0", ValueError),
    (dict(q=torch.zeros(5, 4, 257), output=torch.zeros(5, 4, 257), k_cache=torch.zeros(3, 2, 8, 257),
          v_cache=torch.zeros(3, 2, 8, 257)), "1 to 256", ValueError),
    (dict(k_cache=torch.zeros(1, 2, 1, 16).expand(1, 2, 1 << 29, 16), v_cache=torch.zeros(1, 2, 1, 16).expand(1, 2, 1 << 29, 16)),
     "beyond what the kernels count", ValueError),
])
def test_attention_refusals(change, words, error):
    refused(r_paged.rpaged_attention_launcher, attention_args(), change, words, error)


@pytest.mark.parametrize("change, words", [
    (dict(scale=3e38), "scale must be at most 2e38"), (dict(scale=-3e38), "scale must be at most 2e38"), (dict(scale=2e38), "CUDA devices only"),
    (dict(softcap=3e38), "too large for the scale"), (dict(softcap=1e38, scale=1e-3), "too large for the scale"),
    (dict(softcap=1e38, scale=-1e-3), "too large for the scale"), (dict(softcap=1e38, scale=0.0), "CUDA devices only"),
    (dict(softcap=1e30, scale=0.125), "CUDA devices only")])
def test_scales_and_caps_whose_products_overflow_are_refused(change, words):
    """2 log2 e softcap, log2 e scale and scale / softcap are what the kernels multiply with: infinite ones made NaN, tiny ones lost bits."""
    refused(r_paged.rpaged_attention_launcher, attention_args(), change, words)


def test_c_entry_points_refuse_bad_arguments():
    """Statuses of the C ABI for calls that launch nothing: null pointers, sizes that do not agree."""
    import ctypes
    import splat_native as n
    lib, none = n._lib, None
    assert lib.splat_paged_attention(none, none) == -1 and lib.splat_paged_attention_workspace(none) == 0
    sections, rows = (ctypes.c_int64 * 2)(3, 4), (ctypes.c_int64 * 10)()
    assert lib.splat_rotary(none, 1, none, 0, 0, 0, 0, none, 0, none, 0, 0, 0, 1, 1, 8, 0, none, 1, 0, none) == -1
    assert lib.splat_rotary(rows, 1, none, 0, 0, 0, 0, none, 0, none, 0, 0, 0, 1, 1, 8, 7, none, 1, 0, none) == -2      # dtype
    assert lib.splat_rotary(rows, 1, none, 0, 0, 0, 0, none, 5, sections, 2, 0, 0, 1, 1, 8, 0, none, 1, 0, none) == -1  # half > d / 2
    assert lib.splat_rotary(rows, 1, none, 0, 0, 0, 0, none, 0, none, 0, 0, 0, 1, 1, 8, 0, none, 1, 0, none) == 0       # no heads: nothing to do
    assert lib.splat_paged_tables(none, none, none, 0, none, 1, none, 16, 0, 0, 0, none, none, none, none, none, none, none) == -1
    assert lib.splat_paged_tables(none, none, none, 0, none, 1, none, 16, 20000, 0, 0, none, none, none, none, none, none, none) == -6


def test_more_tokens_than_the_kernel_counts():
    """Rows of 2^31 - 100 tokens and more: the last block's count passes 2^31 - 1.  (Nothing is launched, so any addresses do.)"""
    import ctypes
    import splat_native as n

    class Rows(ctypes.Structure):
        _fields_ = [("src", ctypes.c_void_p), ("dst", ctypes.c_void_p)] + [(f, ctypes.c_int64) for f in ("heads", "sb", "sh", "sl", "db", "dh", "dl")] + \
                   [("turned", ctypes.c_int32), ("paged", ctypes.c_int32)]
    rows = Rows(src=16, dst=16, heads=1, sl=2, dl=2)
    for batch, length in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 100), (2 ** 20, 2 ** 11), (3, 2 ** 30), (1, 2 ** 33)):
        assert n._lib.splat_rotary(ctypes.byref(rows), 1, None, 0, 0, 0, 0, None, 0, None, 0, 0, 0, batch, length, 2, 0, None, 1, 0, None) == -6


def test_module_refuses_the_cpu():
    with pytest.raises(ValueError, match="CUDA devices only"):
        r_paged.PagedAttention(4, 16, 4, 2, 64, 2, 8, 64, "cpu", torch.float16)


def test_oracle_tables_hand_out_each_page_once():
    rng = random.Random(5)
    for _ in range(50):
        page, B = rng.choice([1, 3, 16]), rng.randrange(1, 6)
        ctx = [rng.randrange(40) for _ in range(B)]
        new = [rng.randrange(-2, 30) for _ in range(B)]
        width = 80
        held = [-(-c // page) for c in ctx]
        free = list(range(1000, 1000 + rng.randrange(1, 120)))
        table, at = [], 0
        for h in held:
            table.append([at + i if i < h else -7 for i in range(width)])
            at += h
        got = po.tables(ctx, new, table, free, [11, 11 + len(free)], page, 200)
        used = [p for row, c, n in zip(got["table"], ctx, new) for p in row[:-(-(c + max(n, 0)) // page)] if p >= 0]
        assert len(used) == len(set(used))
        live = [s for s in got["slots"] if s >= 0]
        assert len(live) == len(set(live))
        assert got["taken"][0] - 11 + got["taken"][2] == sum(-(-(c + max(n, 0)) // page) - h for c, n, h in zip(ctx, new, held))


def test_oracle_rotary_turns_back():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 5, 12, generator=g, dtype=torch.float64)
    pos = torch.randint(0, 50000, (2, 2, 5), generator=g)
    freq = torch.rand(5, generator=g)
    for interleaved in (False, True):
        y = po.rotary(x, pos, freq, (2, 3), interleaved)
        assert torch.allclose(po.rotary(y, pos, freq, (2, 3), interleaved, inverse=True), x)
        assert torch.equal(y[..., 10:], x[..., 10:])


@pytest.mark.parametrize("row, length, freed", [([4, 2, -1, -1, -1, -1, -1], 17, [4, 2]), ([4, -1, 2, -1, -1, -1, -1], 17, [4, 2]),
                                                ([-1] * 7, 28, []), ([0, 1, 2, 3, 4, -1, -1], 28, [0, 1, 2, 3, 4]), ([-1] * 7, 0, [])])
def test_release_of_a_request_that_was_short_of_pages(row, length, freed):
    """Pages that were missing are no pages to hand out again, and a request that is released twice has none to give."""
    m = r_paged.PagedAttention.__new__(r_paged.PagedAttention)
    torch.nn.Module.__init__(m)
    m.device, m.page_size = torch.device("cpu"), 4
    m.block_table = torch.tensor([[-1] * 7, row], dtype=torch.int32)
    held = [p for p in range(5) if p not in freed]
    m.free_pages = torch.full((5,), 77, dtype=torch.int32)
    m.free_span = torch.tensor([8, 8 + len(held)])
    for i, p in enumerate(held):
        m.free_pages[(8 + i) % 5] = p
    for _ in range(2):
        m.release(1, length)
        assert m.free_span.tolist() == [8, 13]
        assert [int(m.free_pages[i % 5]) for i in range(8, 13)] == held + freed
        assert m.block_table.eq(-1).all()


def module_on_the_cpu(table, page_size, pages, held):
    """The tables of a PagedAttention that has handed out all but `held` of its pages, which lie in its ring from 8 on."""
    m = r_paged.PagedAttention.__new__(r_paged.PagedAttention)
    torch.nn.Module.__init__(m)
    m.device, m.page_size = torch.device("cpu"), page_size
    m.block_table = torch.tensor(table, dtype=torch.int32)
    m.free_pages = torch.full((pages,), 77, dtype=torch.int32)
    m.free_span = torch.tensor([8, 8 + len(held)])
    for i, p in enumerate(held):
        m.free_pages[(8 + i) % pages] = p
    return m


@pytest.mark.parametrize("length", [0, 3, 5, 8, 9, 28])
def test_release_gives_all_pages_back_whatever_the_length(length):
    """A request that dropped tokens has pages behind its length."""
    m = module_on_the_cpu([[3, 1, -1, 4, -1, -1, -1], [0, 2, -1, -1, -1, -1, -1]], 4, 5, [])
    m.release(0, length)
    assert m.free_span.tolist() == [8, 11] and [int(m.free_pages[i % 5]) for i in range(8, 11)] == [3, 1, 4]
    assert m.block_table.tolist() == [[-1] * 7, [0, 2, -1, -1, -1, -1, -1]]


@pytest.mark.parametrize("ctx, freed, left", [
    ([16, 8], [], [[3, 1, -1, 4, -1], [0, 2, -1, -1, -1]]), ([13, 5], [], [[3, 1, -1, 4, -1], [0, 2, -1, -1, -1]]),
    ([12, 5], [4], [[3, 1, -1, -1, -1], [0, 2, -1, -1, -1]]), ([4, 4], [1, 4, 2], [[3, -1, -1, -1, -1], [0, -1, -1, -1, -1]]),
    ([0, -3], [3, 1, 4, 0, 2], [[-1] * 5] * 2), ([2 ** 31 - 1, 1], [2], [[3, 1, -1, 4, -1], [0, -1, -1, -1, -1]])])
def test_rewind_gives_back_the_pages_behind_what_is_left(ctx, freed, left):
    held = [5, 6]
    m = module_on_the_cpu([[3, 1, -1, 4, -1], [0, 2, -1, -1, -1]], 4, 7, held)
    for _ in range(2):                                     # (once more: nothing)
        m.rewind(torch.tensor(ctx, dtype=torch.int32))
        assert m.block_table.tolist() == left and m.free_span.tolist() == [8, 10 + len(freed)]
        assert [int(m.free_pages[i % 7]) for i in range(8, 10 + len(freed))] == held + freed


def test_operands_that_are_not_what_their_memory_holds_are_refused():
    """Views with a sign to be turned, and zeros without memory."""
    for odd in (torch._neg_view(torch.ones(2, 4, 6, 16)), torch._efficientzerotensor((2, 4, 6, 16))):
        for call in (r_rotary.rrotary, r_rotary.rrotary_launcher):
            refused(call, rotary_args(), dict(q=odd), "values in memory", TypeError)
        refused(r_paged.rpaged_attention_launcher, attention_args(), dict(q=odd[0, :, :5].transpose(0, 1)), "values in memory", TypeError)
        refused(r_paged.rpaged_append_launcher, append_args(), dict(k=odd[0, :2, :5].transpose(0, 1)), "values in memory", TypeError)


def test_outputs_are_the_operands_themselves_or_elsewhere():
    """In place means at the same strides: a row written before it is read as another one would be a wrong answer."""
    x = torch.zeros(2, 4, 4, 16)
    turned = x.transpose(1, 2)
    for kw, words in [(dict(q=x, k=None, q_out=turned), "q_out must be q itself"), (dict(q=x, k=x.clone(), q_out=x, k_out=x), "share memory"),
                      (dict(q=x.clone(), k=x, q_out=x), "share memory"), (dict(q=x, k=turned, k_out=x), "share memory"),
                      (dict(q=x, k=None, q_out=x), "CUDA devices only")]:
        refused(r_rotary.rrotary_launcher, dict(positions=i32(4), inv_freq=torch.zeros(8), **kw), {}, words)
    kw = append_args()
    for change, words in [(dict(q_out=kw["q"]), "CUDA devices only"), (dict(q_out=kw["k"].expand(5, 2, 16), q=kw["v"]), "share memory"),
                          (dict(q=kw["q"][:, :2], q_out=kw["v"]), "share memory"),
                          (dict(q=kw["q"].view(4, 5, 16).transpose(0, 1), q_out=kw["q"]), "q_out must be q itself"),
                          (dict(q_out=kw["k_cache"].view(6, 8, 16)[:5, :4]), "share memory"),
                          (dict(q=kw["k_cache"].view(6, 8, 16)[:5, :4]), "share memory")]:
        refused(r_paged.rpaged_append_launcher, kw, change, words)


def test_outputs_that_start_elsewhere_in_an_operand_are_refused():
    wide = torch.zeros(2, 4, 8, 16)
    turn = dict(positions=i32(7), inv_freq=torch.zeros(8))
    for kw, words in [(dict(q=wide[:, :, :-1], k=None, q_out=wide[:, :, 1:]), "q_out must be q itself"),
                      (dict(q=wide[:, :, 1:], k=wide[:, :, :-1].clone(), k_out=wide[:, :, :-1]), "q must not share memory|k_out and q"),
                      (dict(q=wide[:, 2:, 1:], k=wide[:, :2, 1:], q_out=wide[:, 2:, 1:], k_out=wide[:, :2, 1:]), "CUDA devices only"),
                      (dict(q=wide[:, 2:, 1:], k=wide[:, :2, 1:], q_out=wide[:, :2, :-1], k_out=None), "q_out and k must not share")]:
        refused(r_rotary.rrotary_launcher, {**turn, **kw}, {}, words)
    kw = attention_args()
    flat = torch.zeros(5 * 4 * 16 + 20 + 64)
    out = flat[64:64 + 320].view(5, 4, 16)
    f = dict(q=flat[:320].view(5, 4, 16), output=out)
    refused(r_paged.rpaged_attention_launcher, kw, f, "output and q must not share")
    for start in (0, 4, 300):
        refused(r_paged.rpaged_attention_launcher, kw, dict(lse=kw["q"].view(-1)[start:start + 20].view(5, 4)), "lse and q must not share")
        refused(r_paged.rpaged_attention_launcher, kw, dict(lse=kw["output"].view(-1)[start:start + 20].view(5, 4)), "output and lse must not share")
    refused(r_paged.rpaged_attention_launcher, kw, dict(lse=flat[64:84].view(5, 4), slopes=flat[80:84]), "lse and slopes must not share")
    refused(r_paged.rpaged_attention_launcher, kw, dict(block_table=kw["output"].view(torch.int32).view(-1)[3:11].view(2, 4)), "output and block_table")
    kw = append_args()
    refused(r_paged.rpaged_append_launcher, kw, dict(q_out=kw["k_cache"][1:].view(-1)[5 * 16:5 * 16 + 320].view(5, 4, 16)), "q_out and k_cache")
    refused(r_paged.rpaged_append_launcher, kw, dict(v_cache=torch.zeros(5, 2, 8, 16)[1:4], k_cache=kw["k_cache"]), "CUDA devices only")
    both = torch.zeros(4, 2, 8, 16)
    refused(r_paged.rpaged_append_launcher, kw, dict(k_cache=both[:3], v_cache=both[1:]), "k_cache and v_cache must not share")
    kw = tables_args()
    line = i32(40)
    refused(r_paged.rpaged_tables_launcher, kw, dict(kv_lens=line[:3], q_start=line[2:6]), "kv_lens and q_start must not share")
    refused(r_paged.rpaged_tables_launcher, kw, dict(block_table=line[:24].view(3, 8)[:, :5], requests=line[10:17]), "block_table and requests")
    refused(r_paged.rpaged_tables_launcher, kw, dict(block_table=line[:24].view(3, 8)[:, :5], kv_lens=line[5:8]), "CUDA devices only")


def test_outputs_between_the_elements_of_operands_are_not_refused():
    """Heads of a fused projection turned in place, K and V as halves of one array, rows of one page beside the others'."""
    qkv = torch.zeros(5, 8, 16)
    kw = {**append_args(), "q": qkv[:, :4], "k": qkv[:, 4:6], "v": qkv[:, 6:], "q_out": qkv[:, :4]}
    both = torch.zeros(3, 2, 2, 8, 16)
    rows = torch.zeros(3, 8, 4, 16)
    for caches in ((both[:, 0], both[:, 1]), (rows[:, :, :2].transpose(1, 2), rows[:, :, 2:].transpose(1, 2))):
        refused(r_paged.rpaged_append_launcher, kw, dict(k_cache=caches[0], v_cache=caches[1]), "CUDA devices only")
    refused(r_paged.rpaged_append_launcher, kw, dict(q_out=qkv[:, 1:5]), "q_out must be q itself|q_out and k")
    x = torch.zeros(2, 6, 7, 16)
    refused(r_rotary.rrotary_launcher, dict(q=x[:, :4], k=x[:, 4:], q_out=x[:, :4], k_out=x[:, 4:], positions=i32(7), inv_freq=torch.zeros(8)), {},
            "CUDA devices only")


def test_shared_elements_against_sets_of_them():
    """Random strided views of one small buffer, as operand and output: refused if and only if an element is both, or twice in the output."""
    rng = random.Random(3)
    buffer, where = torch.zeros(300), torch.arange(300)
    seen = {"apart": 0, "itself": 0, "twice": 0, "shared": 0}
    for _ in range(3000):
        d = rng.choice([1, 2, 3])
        size = [rng.randrange(1, 4) for _ in range(3)] + [d]

        def view():
            strides = [rng.choice([1, 2, 3, 4, 6, 9, 12, 18, 24, 36]) for _ in range(3)] + [1]
            return size, strides, rng.randrange(0, 60)
        a = view()
        b = a if rng.random() < 0.1 else (a[0], a[1], rng.randrange(0, 60)) if rng.random() < 0.5 else view()
        q, out = (buffer.as_strided(*v) for v in (a, b))
        of_q, of_out = (where.as_strided(*v).reshape(-1).tolist() for v in (a, b))
        real = [i for i in range(4) if size[i] > 1]
        words = "CUDA devices only"
        if len(set(of_out)) < len(of_out):
            words, kind = "overlap itself", "twice"
        elif not set(of_q) & set(of_out):
            kind = "apart"
        elif a[2] == b[2] and all(a[1][i] == b[1][i] for i in real):
            kind = "itself"
        else:
            words, kind = "q_out must be q itself", "shared"
        seen[kind] += 1
        with pytest.raises(ValueError, match=words):
            r_rotary.rrotary_launcher(q, None, i32(size[2]), torch.zeros(0), q_out=out)
    assert min(seen.values()) > 50, seen
