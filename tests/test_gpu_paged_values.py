"""Attention over a paged cache where values are extreme."""

import ctypes
import math

import pytest
import torch

import streaming_ref as ref
from test_gpu_paged import E4M3, Scene, _randn, nat, no_fault  # noqa: F401  (fixtures)

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


@pytest.mark.parametrize("gap", [12, 14, 16, 17, 18])
@pytest.mark.parametrize("shape", [([(1, 20000)], 2, 2), ([(3, 20000)], 8, 2), ([(70, 20000)], 2, 2)])
def test_small_probabilities_in_fp16(nat, gap, shape):
    """One key `gap` above 20 thousand others, its value 0 and theirs about 1: what the small ones add up to is not lost.
    P carries a factor of 2^7, so that one under fp16's smallest steps is off by 2^-25 2^-7 of the row's largest at
    most, n of them against a sum of at least one."""
    seqs, heads, kv_heads = shape
    n = seqs[0][1]

    def peak(batch, k, v):
        k.zero_()
        k[0, :, 0] = gap
        v.uniform_(0.5, 1, generator=torch.Generator(device="cuda").manual_seed(1))
        v[1] = 1
        v[0] = 0

    s = Scene(seqs, kv_heads, 64, torch.float16)
    s.fill(1, torch.float16, change=peak)
    q = torch.zeros(s.rows, heads, 64, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 8
    want, wlse, tol, ltol = s.expect(q, 1)
    tol = tol - n * 2.0 ** -25 + n * 2.0 ** -32
    for split in (True, False):
        got, lse = _attend(nat, s, q, 1, split)
        ref.within(got, want, tol, "out")
        ref.within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("seqs,heads,kv_heads", [([(1, 5000), (1, 80)], 12, 12), ([(200, 900)], 4, 4), ([(4, 700)], 8, 2)])
@pytest.mark.parametrize("pages", [torch.float16, torch.int8], ids=str)
@pytest.mark.parametrize("top", [1, 12, 30])
def test_growing_scores_in_fp16(nat, seqs, heads, kv_heads, pages, top):
    """Keys that grow along the sequence, slowly and fast: probabilities pass the reference's again and again and stay
    within fp16."""
    s = Scene(seqs, kv_heads, 32, pages)

    def grow(batch, k, v):
        at = batch.cu_new.tolist()
        for a, b in zip(at, at[1:]):
            k[a:b] *= torch.linspace(0.1, top, b - a, device="cuda")[:, None, None].to(k.dtype)
        v *= 100

    s.fill(3, torch.float16, change=grow)
    q = _randn(s.rows, heads, 64, seed=9, dtype=torch.float16)
    for split in (True, False):
        got, lse = _attend(nat, s, q, 1, split)
        want, wlse, tol, ltol = s.expect(q, 1)
        ref.within(got, want, tol, "out")
        ref.within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("kind,pages", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                        (torch.bfloat16, E4M3), (torch.float16, torch.int8)], ids=str)
@pytest.mark.parametrize("seqs,heads,kv_heads", [([(6, 70), (3, 3)], 4, 2), ([(100, 260), (40, 40)], 4, 2),
                                                 ([(300, 900)], 2, 2), ([(500, 3000)], 2, 1)])
@pytest.mark.parametrize("block", [1, 5])
@pytest.mark.parametrize("split", [True, False])
def test_results_do_not_depend_on_what_is_hidden(nat, kind, pages, seqs, heads, kv_heads, block, split):
    """Bit for bit the same for the rows that do not see a token, whatever its key and value are: a score that moves its
    neighbours' reference, a NaN, an infinite value.  The first keys' scores are small, so that the rows' references lie
    below what follows and a step that moved them all would show."""
    at = [0]
    for _, t in seqs:
        at.append(at[-1] + t)
    which = [t - 1 - min(n // 2, 20) for n, t in seqs]  # the token of each sequence that changes

    def run(change):
        def spoil(batch, k, v):
            k *= 0.4
            for a, i in zip(at, which):
                k[a: a + min(64, i)] *= 0.1
                if change:
                    change(k, v, a + i)

        s = Scene(seqs, kv_heads, 16, pages)
        s.fill(21, kind, change=spoil)
        return _attend(nat, s, q, block, split)

    q = _randn(sum(n for n, _ in seqs), heads, 64, seed=2, dtype=kind)
    hidden = torch.cat([torch.tensor([x <= i for x in ref.limits(n, t, block)]) for (n, t), i in zip(seqs, which)]).cuda()
    assert hidden.any()
    want, wlse = run(None)

    def large(k, v, i):  # the rows that see it move their reference by dozens
        k[i] *= 150

    def nan_key(k, v, i):
        k[i, :, 7] = math.nan

    def infinite(k, v, i):
        v[i, :, 5] = math.inf
        v[i, :, 9] = math.nan

    for change in (large, nan_key, infinite):
        got, lse = run(change)
        assert torch.equal(got[hidden], want[hidden]), change.__name__
        assert torch.equal(lse[:, hidden], wlse[:, hidden]), change.__name__
        if change is large:
            assert not torch.equal(got[~hidden], want[~hidden])


@pytest.mark.parametrize("kind,pages", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                        (torch.bfloat16, E4M3), (torch.float16, torch.int8)], ids=str)
@pytest.mark.parametrize("new,heads,first", [(100, 1, 256), (100, 3, 256), (8, 2, 288), (300, 1, 256)])
def test_a_special_value_anywhere_in_a_tile_stays_hidden(nat, kind, pages, new, heads, first):
    """A NaN in every dim, or an infinity in one, of each key of a tile in turn: the rows that do not see the key keep their
    bits, whatever else of the tile they see."""
    total = first + 100 if new > 8 else first + 8
    q = _randn(new, heads, 64, seed=2, dtype=kind)

    def run(key=None, dim=None):
        def spoil(batch, k, v):
            if key is not None:
                v[key, :, slice(None) if dim is None else dim] = math.nan if dim is None else math.inf

        s = Scene([(new, total)], 1, 16, pages, seed=1)
        s.fill(1, kind, change=spoil)
        return _attend(nat, s, q, 1, False)[0]

    want = run()
    limit = torch.tensor(ref.limits(new, total, 1), device="cuda")
    for key in range(first, min(first + 64, total)):
        hidden = limit <= key
        for dim in (None, (7 * key) % 64):
            got = run(key, dim)
            assert torch.equal(got[hidden], want[hidden]), (key - first, dim)
            assert not torch.isfinite(got[~hidden].float()).all(-1).any() or not (~hidden).any()
