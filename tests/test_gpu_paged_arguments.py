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
