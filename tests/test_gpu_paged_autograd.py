"""The paged cache beside autograd."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_paged import E4M3, Scene, _ints, _randn, nat, no_fault  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [torch.bfloat16, torch.float16, E4M3, torch.int8], ids=str)
def test_write_is_seen_by_autograd(nat, pages):
    """A graph that keeps the pages (or their exponents) does not go backward over what a later write left in them."""
    s = Scene([(2, 40)], 2, 16, pages)
    s.fill(1)
    rows = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16)
    tensors = [t for t in (s.cache.k, s.cache.v, s.cache.k_exp, s.cache.v_exp) if t is not None]
    before = [t._version for t in tensors]
    s.cache.write(rows, rows, s.batch)
    assert all(t._version > b for t, b in zip(tensors, before))
    if pages == torch.bfloat16:
        w = torch.ones((), dtype=pages, device="cuda", requires_grad=True)
        y = (w * s.cache.k[0]).sum()
        s.cache.write(rows, rows, s.batch)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():  # pages without a version counter of their own
        t = Scene([(2, 40)], 2, 16, pages)
        t.cache.write(rows, rows, t.batch)
        s.cache.write(rows, rows, s.batch)


@pytest.mark.parametrize("which", ["k", "v"])
def test_pages_that_need_a_gradient_are_refused(nat, which):
    from mapanything.kv_cache import PagedKVCache

    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    s.fill(1)
    pages = {x: getattr(s.cache, x).detach().clone() for x in ("k", "v")}
    leaf = pages[which].requires_grad_()
    rows = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16)
    cu = _ints([0, 40])
    for held in (pages, {**pages, which: leaf * 1}):  # a leaf, and what was computed from one
        cache = PagedKVCache.wrap(held["k"], held["v"])
        for call in (lambda: cache.attend(rows, s.batch), lambda: cache.read(s.batch, cu, 40),
                     lambda: cache.write(rows, rows, s.batch)):
            with pytest.raises(nat.NativeError, match="gradient"):
                call()
            with torch.no_grad():
                call()


def test_forward_mode_derivatives_are_refused(nat):
    from mapanything.kv_cache import PagedKVCache

    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    s.fill(1)
    rows = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16)
    cu = _ints([0, 40])
    bufs = [torch.zeros(40, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    want = s.cache.attend(rows, s.batch)
    with fwd.dual_level():
        dual = fwd.make_dual(rows, torch.ones_like(rows))
        wide = fwd.make_dual(bufs[1], torch.ones_like(bufs[1]))
        held = PagedKVCache.wrap(fwd.make_dual(s.cache.k, torch.ones_like(s.cache.k)), s.cache.v)
        for call in (lambda: s.cache.attend(dual, s.batch), lambda: s.cache.write(dual, rows, s.batch),
                     lambda: s.cache.write(rows, dual, s.batch), lambda: s.cache.attend(rows, s.batch, out=dual),
                     lambda: s.cache.read(s.batch, cu, 40, out=(bufs[0], wide)), lambda: held.attend(rows, s.batch),
                     lambda: held.read(s.batch, cu, 40)):
            with pytest.raises(nat.NativeError, match="forward-mode"):
                call()
        assert torch.equal(s.cache.attend(rows, s.batch), want)  # tensors without one, at the same level
