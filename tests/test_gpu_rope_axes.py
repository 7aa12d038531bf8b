"""Rotary positions with several axes (uniception RoPEAxes / mapa_rope_axes) against the formula in 64 bits."""

import pytest
import torch

from streaming_ref import half_step, rope, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def RoPEAxes():
    from uniception.models.libs.croco.pos_embed import RoPEAxes as cls

    return cls


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _data(B, H, N, D, dtype, seed, order="token"):
    """(B, H, N, D): a view of packed (B, N, 3, H, D) rows ("token"), or heads outside tokens ("head")."""
    if order == "token":
        return torch.randn(B, N, 3, H, D, generator=_gen(seed), device="cuda").to(dtype)[:, :, 1].transpose(1, 2)
    return torch.randn(B, H, N, D, generator=_gen(seed), device="cuda").to(dtype)


def _positions(B, N, axes, far, seed, kind=torch.int64):
    p = torch.randint(-3, far, (B, N, axes), generator=_gen(seed), device="cuda")
    return p if kind == torch.int64 else p.to(kind) + 0.375


def _check(got, x, pos, what, **kw):
    want, bound = rope(x, pos, **kw)
    tol = bound if x.dtype == torch.float32 else bound + half_step(x.dtype) * (want.abs() + bound) + 2.0 ** -25
    within(got, want, tol, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["axial", "half", "interleaved"])
@pytest.mark.parametrize("B,Hq,Hk,N,D,sections,spectrum,far,order", [
    (1, 12, 12, 1, 64, (8, 12, 12), "axis", 100000, "token"),   # one token, far
    (2, 12, 12, 1370, 64, (8, 12, 12), "axis", 400, "token"),
    (3, 16, 4, 37, 64, (10, 11, 11), "shared", 1000000, "head"),  # odd sections, fewer key heads
    (1, 5, 1, 65, 64, (32,), "axis", 5000, "token"),             # one axis
    (2, 3, 2, 9, 80, (7, 1, 5, 3), "shared", 50, "head"),        # four axes, dims that pass through
    (1, 1, 1, 8200, 16, (4, 4), "axis", 4096, "token"),          # more tokens than workgroups take one by one
    (1, 2, 2, 5, 256, (64, 32, 32), "axis", 70, "head"),         # widest head
])
def test_rope_axes_matches_formula(RoPEAxes, dtype, layout, B, Hq, Hk, N, D, sections, spectrum, far, order):
    r = RoPEAxes(sections, freq=10000.0, F0=1.25, layout=layout, spectrum=spectrum)
    q, k = _data(B, Hq, N, D, dtype, 1, order), _data(B, Hk, N, D, dtype, 2, order)
    pos = _positions(B, N, len(sections), far, 3)
    kw = dict(sections=sections, freq=10000.0, f0=1.25, layout=layout, spectrum=spectrum)
    q0, k0 = q.clone(), k.clone()
    gq, gk = r(q, pos, k)
    assert torch.equal(q, q0) and torch.equal(k, k0)
    _check(gq, q, pos, "q", **kw)
    _check(gk, k, pos, "k", **kw)
    rest = 2 * sum(sections)
    assert torch.equal(gq[..., rest:], q[..., rest:]) and torch.equal(gk[..., rest:], k[..., rest:])
    assert torch.equal(r(k, pos), gk)  # alone as beside the queries
    out = r(q, pos, k, inplace=True)
    assert out[0].data_ptr() == q.data_ptr() and torch.equal(q, gq) and torch.equal(k, gk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_axes_float_and_shared_positions(RoPEAxes, dtype):
    """fp32 positions between the grid's points, one (N, axes) table for every batch entry, int32 positions."""
    r = RoPEAxes((8, 12, 12), freq=100.0)
    x = _data(3, 12, 77, 64, dtype, 4)
    pos = _positions(1, 77, 3, 900, 5, torch.float32)
    kw = dict(sections=(8, 12, 12), freq=100.0)
    _check(r(x, pos[0]), x, pos.expand(3, -1, -1), "fp32 positions", **kw)
    whole = _positions(1, 77, 3, 900, 6)
    a = r(x, whole.expand(3, -1, -1))
    _check(a, x, whole.expand(3, -1, -1), "expanded", **kw)
    assert torch.equal(a, r(x, whole.to(torch.int32)))


def test_rope_axes_two_axes_are_rope2d(RoPEAxes):
    """(D/4, D/4) pairs are RoPE2D: its own frequencies and angles are fp32, an ulp of the angle apart."""
    from uniception.models.libs.croco.pos_embed import RoPE2D

    x = _data(2, 4, 50, 64, torch.float32, 7, "head")
    pos = torch.randint(0, 37, (2, 50, 2), generator=_gen(8), device="cuda")
    want = RoPE2D(freq=100.0)(x.clone(), pos)
    got = RoPEAxes((16, 16), freq=100.0)(x, pos)
    # angles up to 37 in fp32: 37 2^-23, and both kernels' own bound
    assert ((got - want).abs() <= x.abs().max() * 2 * (37 * 2.0 ** -23 + 2.0 ** -20)).all()


@pytest.mark.parametrize("offset,stride", [(1, 67), (2, 66), (4, 68)])
@pytest.mark.parametrize("layout", ["axial", "half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_axes_unaligned_views(RoPEAxes, dtype, layout, offset, stride):
    """Bases and strides that allow narrower accesses only; what lies between the rows stays as it is."""
    B, H, N = 2, 3, 11
    flat = torch.randn(B * N * H * stride + 8, generator=_gen(9), device="cuda").to(dtype)
    x = flat[offset:].as_strided((B, H, N, 64), (N * H * stride, stride, H * stride, 1))
    pos = _positions(B, N, 3, 100, 10)
    r = RoPEAxes((8, 12, 12), freq=100.0, layout=layout)
    want = r(x.contiguous(), pos)
    _check(want, x, pos, "contiguous", sections=(8, 12, 12), freq=100.0, layout=layout)
    assert torch.equal(r(x, pos), want)
    before = flat.clone()
    r(x, pos, inplace=True)
    assert torch.equal(x, want)
    before[offset:].as_strided(x.shape, x.stride()).copy_(want)
    assert torch.equal(flat, before)


@pytest.mark.parametrize("layout", ["axial", "half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_axes_gradients(RoPEAxes, layout, dtype):
    """The backward pass is the turn by the opposite angle: against the formula, and against differences (the map is
    linear, so <g, R d> = <R' g, d> for any direction d, in exact arithmetic)."""
    r = RoPEAxes((10, 11, 11), freq=10000.0, layout=layout, spectrum="shared")
    kw = dict(sections=(10, 11, 11), freq=10000.0, layout=layout, spectrum="shared")
    q, k = (_data(2, h, 33, 64, dtype, 11 + h).detach().requires_grad_() for h in (6, 2))
    pos = _positions(2, 33, 3, 3000, 13)
    gq, gk = _data(2, 6, 33, 64, dtype, 14, "head"), _data(2, 2, 33, 64, dtype, 15)
    oq, ok = r(q, pos, k)
    _check(oq.detach(), q.detach(), pos, "forward", **kw)
    dq, dk = torch.autograd.grad([oq, ok], [q, k], [gq, gk])
    _check(dq, gq, pos, "dq", inverse=True, **kw)
    _check(dk, gk, pos, "dk", inverse=True, **kw)
    d = _data(2, 6, 33, 64, dtype, 16)
    moved = r(q.detach() + d, pos).double() - r(q.detach(), pos).double()
    left, right = (gq.double() * moved).sum(), (dq.double() * d.double()).sum()
    # every term is off by a few roundings of values of about one: 2 * 3 * half a step each, as a random sum
    n = d.numel()
    assert (left - right).abs() <= 8 * 6 * max(half_step(dtype), 2.0 ** -20) * n ** 0.5


def test_rope_axes_gradients_of_shared_inputs(RoPEAxes):
    """Expanded keys (one head seen as many) sum their gradient; an output that nothing uses gives none; a gradient
    that comes expanded (from a sum) is read as it is; a second derivative turns forward again."""
    r = RoPEAxes((8, 12, 12), freq=100.0)
    kw = dict(sections=(8, 12, 12), freq=100.0)
    pos = _positions(1, 20, 3, 50, 17)
    base = torch.randn(1, 1, 20, 64, generator=_gen(18), device="cuda", requires_grad=True)
    q = torch.randn(1, 4, 20, 64, generator=_gen(19), device="cuda", requires_grad=True)
    oq, ok = r(q, pos, base.expand(1, 4, 20, 64))
    ok.sum().backward(retain_graph=True)
    assert q.grad is None
    want, bound = rope(torch.ones(1, 4, 20, 64, device="cuda"), pos, inverse=True, **kw)
    within(base.grad, want.sum(1, keepdim=True), bound.sum(1, keepdim=True) * 2, "expanded keys")
    g = torch.randn(1, 4, 20, 64, generator=_gen(20), device="cuda", requires_grad=True)
    (dq,) = torch.autograd.grad(oq, q, g, create_graph=True)
    up = torch.randn(1, 4, 20, 64, generator=_gen(21), device="cuda")
    (dg,) = torch.autograd.grad(dq, g, up)
    _check(dg, up, pos, "second derivative", **kw)


def test_rope_axes_on_a_stream_and_in_a_graph(RoPEAxes):
    r = RoPEAxes((8, 12, 12), freq=100.0)
    x = _data(2, 12, 300, 64, torch.bfloat16, 22)
    pos = _positions(2, 300, 3, 500, 23)
    want = r(x, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = r(x, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = r(x, pos)
    for i in range(3):
        x.copy_(_data(2, 12, 300, 64, torch.bfloat16, 30 + i))
        pos.add_(17)
        eager = r(x, pos)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_rope_axes_empty_and_refused(RoPEAxes):
    from mapanything import _native as nat

    r = RoPEAxes((8, 12, 12), freq=100.0)
    e = torch.empty(2, 3, 0, 64, device="cuda")
    assert r(e, torch.empty(2, 0, 3, dtype=torch.int64, device="cuda")).shape == e.shape
    x = torch.randn(1, 2, 4, 64, device="cuda")
    pos = torch.zeros(1, 4, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        r(x, pos[..., :2])
    with pytest.raises(ValueError):
        r(x, pos.double())
    with pytest.raises(ValueError):
        r(x, pos.float().requires_grad_())
    with pytest.raises(ValueError):
        r(x[..., ::2], pos)
    with pytest.raises(ValueError):
        r(x[:, :1].expand(1, 2, 4, 64), pos, inplace=True)
    with pytest.raises(ValueError):
        r(x.clone().requires_grad_(), pos, inplace=True)
    with pytest.raises(ValueError):
        r(x, pos, x.to(torch.bfloat16))
    with pytest.raises(nat.NativeError):
        r(x.double(), pos)
    with pytest.raises(nat.NativeError):
        r(x.cpu(), pos.cpu())


def test_rope_axes_inplace_twice_refused_and_seen_by_autograd(RoPEAxes):
    r = RoPEAxes((8, 12, 12), freq=100.0)
    x = torch.randn(1, 2, 4, 64, device="cuda")
    pos = torch.ones(1, 4, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        r(x, pos, x, inplace=True)
    assert all(torch.equal(t, r(x, pos)) for t in r(x, pos, x))
    w = torch.ones((), device="cuda", requires_grad=True)
    y = w * x  # keeps x for w's gradient
    r(x, pos, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_rope_axes_gradient_in_a_graph(RoPEAxes):
    """Forward and backward captured, replayed with other inputs between eager work; no eager graph of the captured
    leaf lives meanwhile (torch cannot capture a backward pass then)."""
    r = RoPEAxes((8, 12, 12), freq=100.0)
    pos = _positions(2, 70, 3, 500, 51)
    leaf = _data(2, 3, 70, 64, torch.bfloat16, 50).requires_grad_()
    up = _data(2, 3, 70, 64, torch.bfloat16, 52)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(r(leaf, pos), leaf, up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = r(leaf, pos)
        (grad,) = torch.autograd.grad(out, leaf, up)
    for i in range(3):
        with torch.no_grad():
            leaf.copy_(_data(2, 3, 70, 64, torch.bfloat16, 60 + i))
            up.copy_(_data(2, 3, 70, 64, torch.bfloat16, 70 + i))
            pos.add_(5)
        graph.replay()
        x = leaf.detach().clone().requires_grad_()
        y = r(x, pos)
        (g,) = torch.autograd.grad(y, x, up)
        torch.cuda.synchronize()
        assert torch.equal(out, y) and torch.equal(grad, g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("layout", ["axial", "half", "interleaved"])
@pytest.mark.parametrize("sections,D", [((32,), 64), ((16, 2, 2, 8), 56), ((8, 4), 26), ((2,), 4)])
def test_rope_axes_alignment_does_not_change_results(RoPEAxes, dtype, layout, sections, D):
    """Bit for bit the same from aligned rows, from rows one value further and in place in rows of odd length."""
    r = RoPEAxes(sections, freq=100.0, layout=layout)
    x = _data(2, 3, 1500, D, dtype, 80)
    pos = _positions(2, 1500, len(sections), 50, 81)
    want = r(x, pos)
    odd = torch.zeros(2, 3, 1500, D + 9, dtype=dtype, device="cuda")
    odd[..., 1: D + 1] = x
    assert torch.equal(r(odd[..., 1: D + 1], pos), want)
    r(odd[..., 1: D + 1], pos, inplace=True)
    assert torch.equal(odd[..., 1: D + 1], want)
    assert (odd[..., 0] == 0).all() and (odd[..., D + 1:] == 0).all()
