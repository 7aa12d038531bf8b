"""Attention over a paged cache under its plans: most tasks whole and the rest of one sequence's cut into key ranges; four
or eight waves a workgroup."""

import ctypes

import pytest
import torch

import streaming_ref as ref
from test_gpu_paged import E4M3, Scene, _randn, nat, no_fault  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,pages,waves", [(torch.bfloat16, torch.bfloat16, 4), (torch.float16, torch.float16, 4),
                                              (torch.bfloat16, E4M3, 8), (torch.float16, torch.int8, 8)], ids=str)
@pytest.mark.parametrize("block", [0, 1, 370])
@pytest.mark.parametrize("new,total,heads,kv_heads", [(1370, 3000, 48, 48), (685, 2100, 104, 52)])
def test_whole_and_split_tasks_of_one_sequence(nat, kind, pages, waves, block, new, total, heads, kv_heads):
    s = Scene([(new, total)], kv_heads, 16, pages)
    s.fill(3, kind)
    q = _randn(new, heads, 64, seed=5, dtype=kind)
    # the plan, by its workspace: slots of (rows of a workgroup) x (64 + 1) floats; all tasks split would take two each
    rows = new * heads // kv_heads
    tasks = -(-rows // (32 * waves)) * kv_heads
    resident = 512 if waves == 4 else 256  # two workgroups of four waves per CU
    d = nat.AttnPagedDesc(cache=s.cache.desc, batch=s.batch._rows(new), dtype=nat.dt_code(kind), heads=heads)
    slots = nat.lib().mapa_attention_paged_workspace_bytes(ctypes.byref(d)) / (32 * waves * 65 * 4)
    rest = tasks % resident
    assert tasks > resident and slots == int(slots) and slots >= 2 * rest and slots % rest == 0 and slots < 2 * tasks
    got, lse = s.cache.attend(q, s.batch, mask_block=block, return_lse=True)
    want, wlse, tol, ltol = s.expect(q, block)
    ref.within(got, want, tol, "out")
    ref.within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("kind,pages", [(torch.bfloat16, E4M3), (torch.float16, torch.int8)], ids=str)
@pytest.mark.parametrize("new", [100, 130, 300, 500, 600, 860, 1100])
def test_either_number_of_waves(nat, kind, pages, new):
    """Rows that pad to as many, a few or many more in workgroups of 256 than of 128, on both sides of the rule."""
    s = Scene([(new, 2500)], 2, 64, pages)
    s.fill(3, kind)
    q = _randn(new, 2, 64, seed=5, dtype=kind)
    got, lse = s.cache.attend(q, s.batch, mask_block=1, return_lse=True)
    want, wlse, tol, ltol = s.expect(q, 1)
    ref.within(got, want, tol, "out")
    ref.within(lse, wlse, ltol, "lse")
