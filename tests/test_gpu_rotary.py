"""GPU: rotary positions of several axes against 64 bits, and their gradients."""
import pytest
import torch

import r_rotary
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


def inputs(dtype, B, H, L, d, half, axes, seed=0, far=30000):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, L, H, d, device="cuda", generator=g).to(dtype).transpose(1, 2)
    pos = torch.randint(-far, far, (axes, B, L), device="cuda", generator=g, dtype=torch.int32)
    freq = torch.tensor([10000.0 ** (-i / max(half, 1)) for i in range(half)], device="cuda")
    cut = [half // axes] * (axes - 1)
    return x, pos, freq, (half - sum(cut), *cut)


def close(got, want, x):
    """Two products and a sum in fp32 with cosines that are off by 2^-21 at most, of pairs whose length is the rows' own, then
    one rounding; the pair's length is bounded by the row's largest element times sqrt 2."""
    u = torch.finfo(got.dtype).eps / 2
    size = x.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
    bound = u * want.abs() + 4 * 2.0 ** -22 * size * (1 + u) + torch.finfo(got.dtype).smallest_normal
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B, H, Hk, L, d, half, axes, interleaved", [
    (1, 1, 1, 1, 2, 1, 1, False),
    (2, 4, 2, 33, 64, 32, 1, False),
    (2, 4, 2, 33, 64, 32, 2, True),
    (1, 3, 1, 17, 128, 32, 3, False),          # half of the row turns
    (3, 5, 5, 7, 80, 40, 3, True),
    (1, 2, 2, 65, 96, 48, 4, False),
    (2, 2, 1, 9, 33, 11, 3, False),            # no 16-byte pieces
    (2, 2, 1, 9, 34, 17, 2, True),
    (1, 2, 2, 5, 48, 0, 1, False),             # nothing turns
    (1, 48, 16, 700, 64, 32, 2, False),
])
def test_rotary_against_64_bits(dtype, B, H, Hk, L, d, half, axes, interleaved):
    q, pos, freq, cut = inputs(dtype, B, H, L, d, half, axes)
    k = inputs(dtype, B, Hk, L, d, half, axes, seed=1)[0]
    for inverse in (False, True):
        a, b = r_rotary.rrotary_launcher(q, k, pos, freq, cut, interleaved=interleaved, inverse=inverse)
        assert a.shape == q.shape and b.shape == k.shape and a.is_contiguous() and a.dtype == dtype
        close(a, po.rotary(q, pos, freq, cut, interleaved, inverse), q)
        close(b, po.rotary(k, pos, freq, cut, interleaved, inverse), k)
    alone, none = r_rotary.rrotary_launcher(q, None, pos, freq, cut, interleaved=interleaved)
    assert none is None
    close(alone, po.rotary(q, pos, freq, cut, interleaved), q)


def test_layouts_positions_and_places():
    """Positions of one batch for all, 64-bit ones, strided operands, offsets from a 16-byte boundary, in place."""
    q, pos, freq, cut = inputs(torch.bfloat16, 2, 3, 21, 64, 32, 2)
    want = po.rotary(q, pos[:, :1].expand(-1, 2, -1), freq, cut)
    for p in (pos[:, 0], pos[:, :1].expand(-1, 2, -1), pos[:, 0].long(), pos[:, 0].t().contiguous().t()):
        close(r_rotary.rrotary_launcher(q, None, p, freq, cut)[0], want, q)
    one = po.rotary(q, pos[:1, :1].expand(-1, 2, -1), freq, (32,))
    close(r_rotary.rrotary_launcher(q, None, pos[0, 0], freq)[0], one, q)
    wide = torch.zeros(2, 3, 21, 80, device="cuda", dtype=torch.bfloat16)
    for shift in (0, 3, 8):
        view = wide[..., shift:shift + 64]
        view.copy_(q)
        out = torch.full((2, 3, 21, 90), 7.0, device="cuda", dtype=torch.bfloat16)
        r_rotary.rrotary_launcher(view, None, pos[:, 0], freq, cut, q_out=out[..., 5:69])
        close(out[..., 5:69], want, q)
        assert bool((out[..., :5] == 7).all()) and bool((out[..., 69:] == 7).all())
        got, _ = r_rotary.rrotary_launcher(view, None, pos[:, 0], freq, cut, q_out=view)
        assert got is view
        close(view, want, q)
    broadcast = q[:1].expand(4, -1, -1, -1)
    close(r_rotary.rrotary_launcher(broadcast, None, pos[:, 0], freq, cut)[0], po.rotary(broadcast, pos[:, :1].expand(-1, 4, -1), freq, cut), broadcast)


def test_far_positions():
    """Angles of positions beyond fp32's 24 bits."""
    q, _, freq, cut = inputs(torch.float32, 1, 2, 8, 64, 32, 1)
    pos = torch.tensor([2 ** 24 + 1, 2 ** 30 + 3, 2 ** 31 - 1, -2 ** 31, -1, 0, 123456789, 99999999], device="cuda", dtype=torch.int32)
    close(r_rotary.rrotary_launcher(q, None, pos, freq)[0], po.rotary(q, pos[None, None], freq, cut), q)


def test_cosines_and_sines_as_exact_as_fp32_has_them():
    """The pairs (1, 0) come out as (cos, sin).  Functions off by one last place at most, 2^-24 below 1; one rounding more, half of one;
    angles of up to 30000 radians in 64 bits, 2^-38."""
    pos = torch.arange(30000, device="cuda", dtype=torch.int32)
    freq = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], device="cuda")
    x = torch.cat((torch.ones(1, 1, 30000, 32, device="cuda"), torch.zeros(1, 1, 30000, 32, device="cuda")), -1)
    got = r_rotary.rrotary_launcher(x, None, pos, freq)[0]
    off = (got.double() - po.rotary(x, pos[None, None], freq, (32,))).abs()
    assert float(off.max()) <= 1.5 * 2.0 ** -24 + 2.0 ** -38, float(off.max()) * 2 ** 24


def test_empty_operands():
    freq = torch.ones(4, device="cuda")
    for shape in ((0, 2, 3, 8), (2, 0, 3, 8), (2, 2, 0, 8)):
        q = torch.zeros(shape, device="cuda")
        pos = torch.zeros(shape[2], device="cuda", dtype=torch.int32)
        out, _ = r_rotary.rrotary(q, None, pos, freq)
        assert out.shape == shape
    # no heads of q, some of k
    k = torch.randn(2, 2, 3, 8, device="cuda")
    _, b = r_rotary.rrotary(torch.zeros(2, 0, 3, 8, device="cuda"), k, torch.zeros(3, device="cuda", dtype=torch.int32), freq)
    assert torch.equal(b, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(dtype, interleaved):
    q, pos, freq, cut = inputs(dtype, 2, 4, 19, 80, 32, 3)
    k = inputs(dtype, 2, 2, 19, 80, 32, 3, seed=1)[0]
    dq = inputs(dtype, 2, 4, 19, 80, 32, 3, seed=2)[0]
    dk = inputs(dtype, 2, 2, 19, 80, 32, 3, seed=3)[0]
    q.requires_grad_(True)
    k.requires_grad_(True)
    a, b = r_rotary.rrotary(q, k, pos, freq, cut, interleaved=interleaved)
    gq, gk = torch.autograd.grad((a, b), (q, k), (dq, dk))
    close(gq, po.rotary(dq, pos, freq, cut, interleaved, inverse=True), dq)
    close(gk, po.rotary(dk, pos, freq, cut, interleaved, inverse=True), dk)
    # one of the two alone, and gradients that come expanded
    a, b = r_rotary.rrotary(q, k.detach(), pos, freq, cut, interleaved=interleaved)
    ones = torch.ones_like(q)
    close(torch.autograd.grad(a.sum(), q)[0], po.rotary(ones, pos, freq, cut, interleaved, inverse=True), ones)
    a, b = r_rotary.rrotary(q.detach(), k, pos, freq, cut, interleaved=interleaved)
    assert not torch.autograd.grad(b, k, dk)[0].isnan().any()
    a, b = r_rotary.rrotary(q, k, pos, freq, cut, interleaved=interleaved)
    gk, = torch.autograd.grad(b, k, dk)                    # q's gradient is not asked for, nor is there one
    close(gk, po.rotary(dk, pos, freq, cut, interleaved, inverse=True), dk)
    # a batch that shares its rows: the gradients add up
    shared = q.detach()[:1].clone().requires_grad_(True)
    a, _ = r_rotary.rrotary(shared.expand(2, -1, -1, -1), None, pos, freq, cut, interleaved=interleaved)
    g, = torch.autograd.grad(a, shared, dq)
    each = po.rotary(dq, pos, freq, cut, interleaved, inverse=True)
    u = torch.finfo(dtype).eps / 2
    room = u * (2 * each.abs().sum(0, keepdim=True) + each.sum(0, keepdim=True).abs()) + 1e-5
    assert bool(((g.double() - each.sum(0, keepdim=True)).abs() <= room).all())


def test_gradients_with_a_sign_to_be_turned():
    """The imaginary part of a conjugate is a view whose sign is not in memory."""
    q, pos, freq, cut = inputs(torch.float32, 1, 2, 5, 16, 8, 1)
    q.requires_grad_(True)
    a, _ = r_rotary.rrotary(q, None, pos, freq, cut)
    dq = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    g, = torch.autograd.grad(a, q, torch._neg_view(dq))
    close(g, po.rotary(-dq, pos, freq, cut, inverse=True), dq)


def test_gradient_against_differences():
    q, pos, freq, cut = inputs(torch.float32, 1, 2, 3, 16, 6, 2, far=50)
    q = q.contiguous().requires_grad_(True)
    weight = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))

    def loss(x):
        return (r_rotary.rrotary(x, None, pos, freq, cut)[0].double() * weight).sum()
    g, = torch.autograd.grad(loss(q), q)
    for at in range(0, q.numel(), 7):
        step = torch.zeros(q.numel(), device="cuda")
        step[at] = 0.5                                     # (linear: any step will do)
        up, down = (loss((q.detach().view(-1) + s * step).view_as(q)) for s in (1, -1))
        # values up to 5 in fp32, 96 of them, turned with 2^-21: a difference is off by less than this
        assert abs(float(up - down) - float(g.view(-1)[at])) < 96 * 5 * 5 * 2.0 ** -21


def test_second_gradient():
    q, pos, freq, cut = inputs(torch.float32, 1, 2, 5, 16, 8, 2)
    q.requires_grad_(True)
    dq = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).requires_grad_(True)
    a, _ = r_rotary.rrotary(q, None, pos, freq, cut)
    g, = torch.autograd.grad(a, q, dq, create_graph=True)
    again, = torch.autograd.grad(g, dq, q.detach())
    close(again, po.rotary(q.detach(), pos, freq, cut), q.detach())


def test_captured_forward_and_backward():
    q, pos, freq, cut = inputs(torch.bfloat16, 1, 4, 40, 64, 32, 2)
    q.requires_grad_(True)
    dq = torch.randn(q.shape, device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(r_rotary.rrotary(q, None, pos, freq, cut)[0], q, dq)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, _ = r_rotary.rrotary(q, None, pos, freq, cut)
        g, = torch.autograd.grad(a, q, dq)
    with torch.no_grad():
        q.copy_(torch.randn(q.shape, device="cuda"))
    pos.add_(5)
    graph.replay()
    close(a, po.rotary(q.detach(), pos, freq, cut), q.detach())
    close(g, po.rotary(dq, pos, freq, cut, inverse=True), dq)


def test_tangents_in_forward_mode():
    """The derivative along a tangent is the tangent, turned: of q, of k, of both, and with a gradient behind it."""
    import torch.autograd.forward_ad as fwd
    q, pos, freq, cut = inputs(torch.float32, 2, 4, 9, 32, 12, 2)
    k = inputs(torch.float32, 2, 2, 9, 32, 12, 2, seed=1)[0]
    dq, dk = (inputs(torch.float32, 2, h, 9, 32, 12, 2, seed=5 + h)[0].contiguous() for h in (4, 2))
    want = [po.rotary(x, pos, freq, cut) for x in (q, k, dq, dk)]
    with fwd.dual_level():
        for with_q, with_k in ((True, True), (True, False), (False, True)):
            a = fwd.make_dual(q, dq) if with_q else q
            b = fwd.make_dual(k, dk) if with_k else k
            for no_grad in (False, True):
                with torch.set_grad_enabled(not no_grad):
                    ya, yb = (fwd.unpack_dual(y) for y in r_rotary.rrotary(a, b, pos, freq, cut))
                close(ya.primal, want[0], q)
                close(yb.primal, want[1], k)
                assert (ya.tangent is not None) == with_q and (yb.tangent is not None) == with_k
                if with_q:
                    close(ya.tangent, want[2], dq)
                if with_k:
                    close(yb.tangent, want[3], dk)
        alone, none = r_rotary.rrotary(fwd.make_dual(q, dq), None, pos, freq, cut)
        assert none is None
        close(fwd.unpack_dual(alone).tangent, want[2], dq)
        turned = r_rotary.rrotary(fwd.make_dual(q.contiguous(), torch._neg_view(dq)), None, pos, freq, cut)[0]      # (a sign that is not in memory)
        close(fwd.unpack_dual(turned).tangent, po.rotary(-dq, pos, freq, cut), dq)
        # a tangent of nothing but zeros, and one that has a gradient itself
        zero = fwd.unpack_dual(r_rotary.rrotary(fwd.make_dual(q, torch._efficientzerotensor(q.shape, device="cuda")), None, pos, freq, cut)[0])
        assert zero.tangent is None or not zero.tangent.any()
        x, t = q.detach().clone().requires_grad_(True), dq.clone().requires_grad_(True)
        y = fwd.unpack_dual(r_rotary.rrotary(fwd.make_dual(x, t), None, pos, freq, cut)[0])
        gx, = torch.autograd.grad(y.primal, x, dq, retain_graph=True)
        gt, = torch.autograd.grad(y.tangent, t, q)
        close(gx, po.rotary(dq, pos, freq, cut, inverse=True), dq)
        close(gt, po.rotary(q, pos, freq, cut, inverse=True), q)
        with pytest.raises(ValueError, match="none for the frequencies"):
            r_rotary.rrotary(q, None, pos, fwd.make_dual(freq, freq.clone()), cut)
