"""What the paged cache's C entries refuse because two of a call's tensors are one: shown before any launch, so no GPU is
needed."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def nat():
    from mapanything import _native

    _native.load_library()
    return _native


def _cache(nat, **over):
    c = nat.KVCacheDesc(nat.BF16, 12, 64, 8, 4096, 8192, None, None)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def test_read_refuses_one_output_for_keys_and_values(nat):
    L = nat.load_library()
    c, b = _cache(nat), nat.KVBatchDesc(2, 4, 4096, 4096, 4096, 10, 5, 200)
    strides = (768, 64, 768, 64, None)
    assert L.mapa_kv_cache_read(ctypes.byref(c), ctypes.byref(b), 4096, 10, 4096, 4096, nat.BF16, *strides) != 0
    assert b"one output" in L.mapa_last_error(), L.mapa_last_error()
    # nothing to write: not an error
    assert L.mapa_kv_cache_read(ctypes.byref(c), ctypes.byref(b), 4096, 0, 4096, 4096, nat.BF16, *strides) == 0


@pytest.mark.parametrize("over", [{"v": 4096}, {"dtype": 6, "k_exp": 64, "v_exp": 64}, {"dtype": 5, "v": 4096, "k_exp": 64, "v_exp": 128}])
def test_write_refuses_one_place_for_keys_and_values(nat, over):
    """Pages (or exponents) that keys and values share may be read, not written."""
    L = nat.load_library()
    c, b = _cache(nat, **over), nat.KVBatchDesc(2, 4, 4096, 4096, 4096, 10, 5, 200)
    rows = (4096, 8192, nat.BF16, 768, 64, 768, 64, None)
    assert L.mapa_kv_cache_write(ctypes.byref(c), ctypes.byref(b), *rows) != 0
    assert b"share" in L.mapa_last_error(), L.mapa_last_error()


@pytest.mark.gpu
def test_class_refuses_one_output_and_takes_two_halves(nat):
    from test_gpu_paged import Scene, _ints, _randn

    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    s.fill(1)
    cu = _ints([0, 40])
    want = s.cache.read(s.batch, cu, 40)
    x = torch.zeros(40, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(nat.NativeError, match="one output"):
        s.cache.read(s.batch, cu, 40, out=(x, x))
    assert not x.any()
    both = torch.zeros(40, 2, 2, 64, dtype=torch.bfloat16, device="cuda")  # side by side in one buffer
    got = s.cache.read(s.batch, cu, 40, out=(both[:, 0], both[:, 1]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    from mapanything.kv_cache import PagedKVCache

    shared = PagedKVCache.wrap(s.cache.k, s.cache.k)
    rows = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16)
    before = s.cache.k.clone()
    with pytest.raises(nat.NativeError, match="share"):
        shared.write(rows, rows, s.batch)
    assert torch.equal(s.cache.k.view(torch.int16), before.view(torch.int16))
    k, v = shared.read(s.batch, cu, 40)
    assert torch.equal(k, want[0]) and torch.equal(v, want[0])
    shared.attend(rows, s.batch)
