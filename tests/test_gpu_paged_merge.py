"""Two attentions over the parts of a sequence, joined by their log-sum-exps, held to the bound that the parts' own bounds
give."""

import pytest
import torch

import streaming_ref as ref
from test_gpu_paged import E4M3, Scene, _ints, _randn, nat, no_fault  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,pages", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, E4M3), (torch.bfloat16, torch.int8)],
                         ids=str)
@pytest.mark.parametrize("new,old,later", [(1, 512, 100), (5, 64, 2000), (96, 1024, 96), (200, 3008, 450)])
def test_two_parts_join(nat, kind, pages, new, old, later):
    """out = w1 o1 + w2 o2 with w1 = 1 / (1 + exp(l2 - l1)): off by w1 and w2 times the parts' errors (their roundings to 16
    bits among them), by |o1 - o2| w1 w2 times the errors of l1 and l2, and by the kernel's own arithmetic: the weights,
    exponentials of a difference, within 2^-20 of themselves, and one rounding."""
    from mapanything.kv_cache import KVBatch

    H, page = 4, 64
    s = Scene([(new, old + later)], H, page, pages)
    s.fill(4)
    q = _randn(new, H, 64, seed=6, dtype=kind)
    cu = _ints([0, new])
    first = KVBatch(s.table[:, : old // page].contiguous(), _ints([old]), cu, max_new=new, max_kv=old)
    second = KVBatch(s.table[:, old // page:].contiguous(), _ints([later]), cu, max_new=new, max_kv=later)
    (o1, l1), (o2, l2) = (s.cache.attend(q, b, return_lse=True) for b in (first, second))
    out = torch.empty_like(o1)
    nat.attn_merge(o1, l1, o2, l2, out, new, H, H * 64)
    k, v = s.held(0)
    a, la, ta, lta = ref.attention(q, k[:old], v[:old], [old] * new, 0.125)
    b, lb, tb, ltb = ref.attention(q, k[old:], v[old:], [later] * new, 0.125)
    want, _, _, _ = ref.attention(q, k, v, [old + later] * new, 0.125)
    w = torch.sigmoid(la - lb).t()[..., None]
    err = (lta + ltb).t()[..., None]
    half = ref.half_step(kind)
    tol = w * ta + (1 - w) * tb + (a - b).abs() * w * (1 - w) * err + (a.abs() + b.abs()) * 2.0 ** -20
    ref.within(out, want, tol + half * (want.abs() + tol), "joined")


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_parts_that_see_nothing(nat, kind):
    """A row that sees nothing in one part is the other part's; in both, zeros and -inf, as attend gives them."""
    rows, H = 6, 4
    o = [_randn(rows, H, 64, seed=i, dtype=kind) for i in range(2)]
    l = [_randn(H, rows, seed=7 + i) for i in range(2)]
    for i, hidden in enumerate(((0, 1), (1, 2))):  # row 0: hidden in the first part, 1 in both, 2 in the second
        for r in hidden:
            o[i][r] = 0
            l[i][:, r] = -float("inf")
    out, lse = torch.empty_like(o[0]), torch.empty_like(l[0])
    nat.attn_merge(o[0], l[0], o[1], l[1], out, rows, H, H * 64, lse_out=lse)
    assert torch.equal(out[0], o[1][0]) and torch.equal(out[2], o[0][2]) and not out[1].any()
    assert torch.equal(lse[:, 0], l[1][:, 0]) and torch.equal(lse[:, 2], l[0][:, 2])
    assert (lse[:, 1] == -float("inf")).all()
    assert torch.isfinite(out.float()).all()
