"""Attention over a paged cache where values are extreme."""

import ctypes
import math

import pytest
import torch

import streaming_ref as ref
from test_gpu_paged import Scene, _randn, nat, no_fault  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


def _attend(nat, s, q, block, split):
    """(out, lse) through the class, or through the C entry without a workspace (every row's keys in one workgroup)."""
    if split:
        return s.cache.attend(q, s.batch, mask_block=block, return_lse=True)
    out, lse = torch.empty_like(q), torch.empty(q.shape[1], q.shape[0], device="cuda")
    d = nat.AttnPagedDesc(cache=s.cache.desc, batch=s.batch._rows(s.rows), dtype=nat.dt_code(q.dtype), heads=q.shape[1],
                          q=q.data_ptr(), o=out.data_ptr(), q_rstride=q.stride(0), q_hstride=64, o_rstride=out.stride(0),
                          o_hstride=64, lse=lse.data_ptr(), mask_block=block)
    nat.check(nat.lib().mapa_attention_paged(ctypes.byref(d), nat.stream()), "mapa_attention_paged")
    return out, lse


# (new, cached) of one sequence, query heads, K/V heads: single tokens, a few, chunks
ONE = [([(1, 9000)], 4, 4), ([(5, 3000)], 6, 2), ([(200, 3000)], 4, 4), ([(45, 2500)], 15, 5)]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("dead", [(0, 0.5), (0.3, 0.8), (0.6, 0.95), (0, 1)])
@pytest.mark.parametrize("shape", range(len(ONE)))
def test_ranges_of_minus_infinity(nat, kind, split, dead, shape):
    """Keys [a, b) of the sequence have scores of -inf: they weigh nothing, whether or not they fill whole ranges of the
    plan.  A row that sees no other keys is NaN (0 / 0), in its output and its log-sum-exp."""
    seqs, heads, kv_heads = ONE[shape]
    new, total = seqs[0]
    a, b = int(dead[0] * (total - new)), int(dead[1] * (total - new))
    if dead[1] == 1:
        b = total - 1 if shape % 2 else total  # the last token alone is alive, or none

    def spoil(batch, k, v):
        k[a:b, :, 3] = -math.inf

    s = Scene(seqs, kv_heads, 16, kind)
    s.fill(40 + shape, kind, change=spoil)
    q = _randn(new, heads, 64, seed=2, dtype=kind)
    q[:, :, 3] = q[:, :, 3].abs() + 0.25
    got, lse = _attend(nat, s, q, 1, split)
    k, v = s.held(0)
    alive = torch.cat([torch.arange(a, device="cuda"), torch.arange(b, total, device="cuda")])
    limit = [int((alive < x).sum()) for x in ref.limits(new, total, 1)]
    want, wlse, tol, ltol = ref.attention(q, k[alive], v[alive], limit, 0.125)
    none = torch.tensor(limit, device="cuda") == 0
    want[none] = math.nan
    wlse[:, none] = math.nan
    ref.within(got, want, tol, "out")
    ref.within(lse, wlse, ltol, "lse")
