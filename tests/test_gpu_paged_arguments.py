"""Numbers that do not fit the descriptors' fields are refused, not cut to other ones."""

import pytest
import torch

from test_gpu_paged import Scene, _randn, nat, no_fault  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [{"mask_block": 1 << 31}, {"mask_block": (1 << 32) + 1}, {"mask_block": -1}, {"scale": 1e-50},
                                {"scale": -0.5}, {"scale": 1e40}, {"scale": float("nan")}])
def test_attend_refuses(nat, kw):
    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    s.fill(1)
    with pytest.raises(nat.NativeError):
        s.cache.attend(_randn(2, 2, 64, seed=2, dtype=torch.bfloat16), s.batch, **kw)


@pytest.mark.parametrize("kw", [{"max_new": (1 << 32) + 2, "max_kv": 40}, {"max_new": 2, "max_kv": (1 << 32) + 40},
                                {"max_new": 2, "max_kv": (1 << 30) + 1}, {"max_new": -1, "max_kv": 40},
                                {"max_new": 2, "max_kv": -1}])
def test_batch_refuses(nat, kw):
    from mapanything.kv_cache import KVBatch

    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    with pytest.raises(nat.NativeError):
        KVBatch(s.table, s.lens, s.cu, **kw)


def test_the_largest_that_fit(nat):
    from mapanything.kv_cache import KVBatch

    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    s.fill(1)
    q = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16)
    want = s.cache.attend(q, s.batch)
    assert torch.equal(s.cache.attend(q, s.batch, mask_block=(1 << 31) - 1), want)
    wide = KVBatch(s.table, s.lens, s.cu, max_new=2, max_kv=1 << 30)
    assert torch.equal(s.cache.attend(q, wide, scale=0), want) and torch.equal(s.cache.attend(q, wide, scale=0.125), want)


def test_strides_of_single_rows_heads_and_sequences_do_not_matter(nat):
    """torch gives a dimension of one element any stride: it is not held against the tensor."""
    from mapanything.kv_cache import KVBatch, PagedKVCache

    c = PagedKVCache(4, 16, 1, torch.bfloat16)
    c.k.zero_()
    c.v.zero_()

    def odd(t):  # (1, 1, 64) with strides (7, 3, 1)
        return torch.empty(64, dtype=t.dtype, device="cuda").as_strided((1, 1, 64), (7, 3, 1)).copy_(t)

    i = torch.tensor([1, 9, 2, 9, 0, 9, 1, 9], dtype=torch.int32, device="cuda")
    table, lens, cu = i[2:3][None], i[6:8][::2], torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    column = torch.tensor([[2, 3]], dtype=torch.int32, device="cuda").t()[:1]  # (1, 1) with strides (1, 2)
    q, k, v = (_randn(1, 1, 64, seed=s, dtype=torch.bfloat16) for s in (1, 2, 3))
    for t in (table, column):
        b = KVBatch(t, lens, cu, max_new=1, max_kv=1)
        c.write(odd(k), odd(v), b)
        assert torch.equal(c.k[2, :, :1].transpose(0, 1), k) and torch.equal(c.v[2, :, :1].transpose(0, 1), v)
        out = odd(torch.zeros_like(q))
        assert torch.equal(c.attend(odd(q), b, out=out), v) and torch.equal(out, v)
        bufs = odd(torch.zeros_like(k)), odd(torch.zeros_like(v))
        c.read(b, cu, 1, out=bufs)
        assert torch.equal(bufs[0], k) and torch.equal(bufs[1], v)
    two = torch.randn(5, 64, 1, device="cuda").to(torch.bfloat16).transpose(1, 2)  # (5, 1, 64), strides (64, 1, 1)
    b = KVBatch(table, torch.full_like(lens, 5), torch.tensor([0, 5], dtype=torch.int32, device="cuda"), max_new=5, max_kv=5)
    c.write(two, two, b)
    assert torch.equal(c.k[2, :, :5].transpose(0, 1), two)
