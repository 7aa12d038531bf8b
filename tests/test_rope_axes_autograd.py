"""RoPEAxes under autograd's other modes.  On the CPU the kernel's launch is replaced by the plain rotation (what is tested is
the Python around it); on the GPU the same tests run the kernel."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from streaming_ref import half_step, rope, within

SECTIONS, FREQ = (8, 12, 12), 100.0
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture(params=DEVICES)
def device(request, monkeypatch):
    if request.param == "cpu":
        from uniception.models.libs.croco.pos_embed import RoPEAxes

        def run(self, a, b, positions, inverse, ya, yb):
            for x, y in ((a, ya), (b, yb)):
                if x is not None:
                    x.data_ptr()  # as the launch takes it: a wrapper without memory raises
                    y.copy_(rope(x.detach(), positions.expand(x.shape[0], -1, -1), self.sections, self.base,
                                 inverse=inverse)[0])

        monkeypatch.setattr(RoPEAxes, "_run", run)
    return request.param


@pytest.fixture()
def turn():
    from uniception.models.libs.croco.pos_embed import RoPEAxes

    return RoPEAxes(SECTIONS, freq=FREQ)


def _x(device, heads, seed):
    return torch.randn(2, heads, 9, 64, generator=torch.Generator().manual_seed(seed)).to(device)


def _pos(device):
    return torch.randint(0, 50, (2, 9, 3), generator=torch.Generator().manual_seed(3)).to(device)


def _check(got, x, pos, what, inverse=False):
    want, bound = rope(x, pos, SECTIONS, FREQ, inverse=inverse)
    within(got, want, bound + half_step(torch.float32) * want.abs(), what)


def test_forward_mode(turn, device):
    """The tangent of a turn is the turn of the tangent, for tokens, keys or both, beside reverse mode or alone."""
    q, k, pos = _x(device, 3, 1), _x(device, 2, 2), _pos(device)
    tq, tk = _x(device, 3, 4), _x(device, 2, 5)
    plain = turn(q, pos, k)
    with fwd.dual_level():
        dq, dk = fwd.make_dual(q, tq), fwd.make_dual(k, tk)
        _check(fwd.unpack_dual(turn(dq, pos)).tangent, tq, pos, "alone")
        both = [fwd.unpack_dual(o) for o in turn(dq, pos, dk)]
        _check(both[0].tangent, tq, pos, "both, tokens")
        _check(both[1].tangent, tk, pos, "both, keys")
        assert all(torch.equal(a.primal, b) for a, b in zip(both, plain))
        first = [fwd.unpack_dual(o) for o in turn(dq, pos, k)]
        _check(first[0].tangent, tq, pos, "tokens")
        assert first[1].tangent is None or not first[1].tangent.any()
        second = [fwd.unpack_dual(o) for o in turn(q, pos, dk)]
        _check(second[1].tangent, tk, pos, "keys")
        assert second[0].tangent is None or not second[0].tangent.any()
        with torch.no_grad():
            _check(fwd.unpack_dual(turn(dq, pos)).tangent, tq, pos, "no_grad")
        leaf = q.clone().requires_grad_()
        y = fwd.unpack_dual(turn(fwd.make_dual(leaf, tq), pos))
        _check(y.tangent, tq, pos, "beside a leaf")
        (g,) = torch.autograd.grad(y.primal, leaf, tq)
        _check(g, tq, pos, "its gradient", inverse=True)


def test_gradient_of_a_tangent(turn, device):
    """Reverse over forward: the tangent's own gradient is turned back."""
    q, t, pos = _x(device, 3, 1), _x(device, 3, 4).requires_grad_(), _pos(device)
    up = _x(device, 3, 6)
    with fwd.dual_level():
        out = fwd.unpack_dual(turn(fwd.make_dual(q, t), pos)).tangent
        (g,) = torch.autograd.grad(out, t, up)
    _check(g, up, pos, "gradient of the tangent", inverse=True)


def test_function_transforms_raise(turn, device):
    q, pos, up = _x(device, 3, 1), _pos(device), _x(device, 3, 6)
    for call in (lambda: torch.func.grad(lambda x: (turn(x, pos) * up).sum())(q),
                 lambda: torch.func.jvp(lambda x: turn(x, pos), (q,), (up,)),
                 lambda: torch.func.vjp(lambda x: turn(x, pos), q)[1](up),
                 lambda: torch.func.vmap(lambda x: turn(x[None], pos[:1]))(q)):
        with pytest.raises(RuntimeError):
            call()


def test_what_has_no_derivative_is_refused(turn, device):
    q, k, pos = _x(device, 3, 1), _x(device, 2, 2), _pos(device)
    before = q.clone()
    with fwd.dual_level():
        for args in ((fwd.make_dual(q, torch.ones_like(q)), pos), (q, pos, fwd.make_dual(k, torch.ones_like(k)))):
            with pytest.raises(ValueError, match="inplace"):
                turn(*args, inplace=True)
        where = pos.float()
        with pytest.raises(ValueError, match="positions"):
            turn(q, fwd.make_dual(where, torch.ones_like(where)))
    assert torch.equal(q, before)


@pytest.mark.parametrize("which", [0, 1])
def test_only_what_needs_a_gradient_gets_one(turn, device, which):
    """Keys that need no gradient come back so beside tokens that do (a cache takes them), and the other way round."""
    x = [_x(device, 3, 1), _x(device, 2, 2)]
    pos, up = _pos(device), _x(device, 3 - which, 6)
    x[which].requires_grad_()
    out = turn(x[0], pos, x[1])
    assert out[which].requires_grad and not out[1 - which].requires_grad
    (g,) = torch.autograd.grad(out[which], x[which], up)
    _check(g, up, pos, "gradient", inverse=True)
    with fwd.dual_level():  # a tangent beside the gradient stays
        x[1 - which] = fwd.make_dual(x[1 - which], torch.ones_like(x[1 - which]))
        t = fwd.unpack_dual(turn(x[0], pos, x[1])[1 - which]).tangent
        _check(t, torch.ones_like(t), pos, "tangent")
