"""One fault word per thread, several users: what a paged K/V cache call reports outlives the model's forwards (which
clear and publish their own bits), and does not stop them."""

import pytest
import torch

from tests_helpers import CASES, make_views, released_config

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from mapanything import _native

    _native.lib()
    return _native


@pytest.fixture(autouse=True)
def clean(nat):
    nat.fault_status(reset=True)
    yield
    nat.fault_status(reset=True)


@pytest.fixture(scope="module")
def model():
    from mapanything.models import MapAnything

    m = MapAnything(**released_config()).load_synthetic_weights().to("cuda").eval()
    yield m
    m._graphs.clear()


def _bad_write():
    """A write whose table names a page outside the cache: skipped and reported by the kernel."""
    from mapanything.kv_cache import KVBatch, PagedKVCache

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    cache = PagedKVCache(4, 16, 2, torch.bfloat16)
    rows = torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    cache.write(rows, rows, KVBatch(ints([[9]]), ints([3]), ints([0, 3]), max_new=3, max_kv=3))


def _raises_kv(nat):
    with pytest.raises(nat.DeviceFault) as e:
        nat.check_faults()
    assert e.value.bits == nat.FAULT_KV_RANGE
    nat.check_faults()  # told once


@pytest.mark.parametrize("graphs", [False, True])
def test_cache_fault_outlives_a_forward(nat, model, graphs):
    views = make_views(CASES["cfg1_224"])
    model.hip_graphs = graphs
    try:
        want = [v["pts3d"].clone() for v in model.infer(views, use_amp=True, apply_mask=False)]
        _bad_write()
        got = [v["pts3d"].clone() for v in model.infer(views, use_amp=True, apply_mask=False)]
    finally:
        model.hip_graphs = True
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    _raises_kv(nat)


def test_cache_fault_between_reset_and_publish(nat):
    """A fault that a paged call raises while a forward is under way is not the forward's."""
    slot = nat.FaultSlot()
    slot.arm()
    slot.reset()
    _bad_write()
    slot.publish()
    slot.wait(timeout_s=60)
    _raises_kv(nat)


def test_forward_fault_is_reported_beside_a_cache_fault(nat):
    """A forward's own bit, beside the cache's: the slot raises with its own alone (the recipe's fallback goes by it), and
    the cache's is still to be told."""
    x = torch.full((4, 64), 1e6, device="cuda")
    y = torch.empty(4, 128, dtype=torch.float16, device="cuda")
    slot = nat.FaultSlot()
    slot.arm()
    slot.reset()
    _bad_write()
    nat.split_rows(x, 4, 64, 64, y)
    slot.publish()
    with pytest.raises(nat.DeviceFault) as e:
        slot.wait(timeout_s=60)
    assert e.value.bits == nat.FAULT_F16_RANGE and e.value.range_only
    _raises_kv(nat)


def test_module_check_leaves_the_cache_fault(nat):
    """check_faults for the engine's bits alone neither raises for the cache's nor clears it."""
    _bad_write()
    nat.check_faults(nat.ENGINE_FAULTS)
    _raises_kv(nat)
