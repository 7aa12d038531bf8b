"""The paged K/V cache (mapanything.kv_cache: mapa_kv_cache_write / _read) and attention over it
(mapa_attention_paged) against their definitions in 64 bits."""

import math

import pytest
import torch

import streaming_ref as ref

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
PAGE_TYPES = [torch.bfloat16, torch.float16, E4M3, torch.int8]


@pytest.fixture(scope="module")
def nat():
    from mapanything import _native

    _native.lib()
    return _native


@pytest.fixture(autouse=True)
def no_fault(nat):
    nat.fault_status(reset=True)
    yield
    assert nat.fault_status(reset=True) == 0, "a fault bit was left behind"


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=_gen(seed), device="cuda").to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Scene:
    """Sequences [(new, cached with them)], a shuffled page table, garbage (NaN bit patterns among it) in every page."""

    def __init__(self, seqs, heads, page, dtype, seed=0, spare=3, shuffle=True, extra_columns=2):
        from mapanything.kv_cache import KVBatch, PagedKVCache

        self.seqs, self.page = seqs, page
        need = [-(-t // page) for _, t in seqs]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist() if shuffle else list(range(pages))[::-1]
        cols = max(need + [0]) + extra_columns
        self.table = _ints([[order.pop() for _ in range(n)] + [-7] * (cols - n) for n in need]).view(len(seqs), cols)
        self.lens = _ints([t for _, t in seqs])
        cu = [0]
        for n, _ in seqs:
            cu.append(cu[-1] + n)
        self.cu, self.rows = _ints(cu), cu[-1]
        self.cache = PagedKVCache(pages, page, heads, dtype)
        for t in (self.cache.k, self.cache.v, self.cache.k_exp, self.cache.v_exp):
            if t is not None:
                t.view(torch.uint8).fill_(0xFF)  # NaN in every float type, and as an exponent
        self.batch = KVBatch(self.table, self.lens, self.cu, max_new=max(n for n, _ in seqs), max_kv=max(t for _, t in seqs))

    def whole(self):
        """The batch that writes every cached token."""
        from mapanything.kv_cache import KVBatch

        cu = [0]
        for _, t in self.seqs:
            cu.append(cu[-1] + t)
        most = max(t for _, t in self.seqs)
        return KVBatch(self.table, self.lens, _ints(cu), max_new=most, max_kv=most), cu[-1]

    def fill(self, seed, dtype=torch.bfloat16, change=None):
        batch, rows = self.whole()
        heads = self.cache.k.shape[1]
        kv = [_randn(rows, heads, 64, seed=seed + i, dtype=dtype) for i in range(2)]
        if change:
            change(batch, *kv)
        self.cache.write(kv[0], kv[1], batch)
        return kv

    def held(self, b):
        """(k, v) of sequence b in 64 bits, out of the pages."""
        c = self.cache
        t = self.seqs[b][1]
        return (ref.sequence_rows(c.k, c.k_exp, self.table[b], t), ref.sequence_rows(c.v, c.v_exp, self.table[b], t))

    def expect(self, q, block, scale=0.125, hidden_ok=True):
        outs = [[], [], [], []]
        at = 0
        for b, (n, t) in enumerate(self.seqs):
            k, v = self.held(b)
            got = ref.attention(q[at: at + n], k, v, ref.limits(n, t, block), scale)
            for o, g in zip(outs, got):
                o.append(g)
            at += n
        return torch.cat(outs[0]), torch.cat(outs[1], 1), torch.cat(outs[2]), torch.cat(outs[3], 1)


# --------------------------------------------------------------------------------------------- write and read back
@pytest.mark.parametrize("pages", PAGE_TYPES, ids=str)
@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("seqs,heads,page", [
    ([(1, 1)], 1, 16),
    ([(1, 64), (1, 65), (1, 1), (0, 7), (0, 0), (3, 200)], 12, 64),
    ([(17, 17), (1370, 2900), (33, 1000)], 3, 32),
    ([(40, 40)] * 300, 2, 16),  # more sequences than a workgroup has threads
])
def test_cache_write_and_read(nat, pages, src, seqs, heads, page):
    s = Scene(seqs, heads, page, pages)
    c = s.cache
    pad = 5
    packed = _randn(s.rows + pad, 3, heads, 64, seed=1, dtype=src)  # strided rows of a projection, padding behind
    k, v = packed[:, 1], packed[:, 2]
    if pad:
        packed[s.rows:] = math.nan  # not to be read
    before = [None if t is None else t.clone() for t in (c.k, c.v, c.k_exp, c.v_exp)]
    c.write(k, v, s.batch)
    for x, t, e, t0, e0 in ((k, c.k, c.k_exp, before[0], before[2]), (v, c.v, c.v_exp, before[1], before[3])):
        want = t0.clone()
        wexp = None if e0 is None else e0.clone()
        at = 0
        for b, (n, total) in enumerate(seqs):
            pos = torch.arange(total - n, total, device="cuda")
            p, r = s.table[b, pos // page].long(), pos % page
            rows = x[at: at + n]
            if e is None:
                want.view(torch.int16)[p, :, r] = rows.to(pages).view(torch.int16)
            else:
                codes, exps = ref.quantise(rows, pages)
                want.view(torch.uint8)[p, :, r] = codes.float().to(pages).view(torch.uint8)
                wexp[p, :, r] = exps
            at += n
        assert torch.equal(t.view(torch.uint8), want.view(torch.uint8))  # new rows exact, everything else untouched
        assert e is None or torch.equal(e, wexp)

    whole, rows = s.whole()
    s.fill(7, src)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        buf = [torch.full((rows + 4, heads, 64), 7.0, dtype=out, device="cuda") for _ in range(2)]
        gk, gv = c.read(s.batch, whole.cu_new, rows + 4, out=buf)
        at = 0
        for b, (_, total) in enumerate(seqs):
            for got, want in zip((gk, gv), s.held(b)):
                assert torch.equal(got[at: at + total], want.to(out))
            at += total
        assert (gk[rows:] == 7).all() and (gv[rows:] == 7).all()


def test_cache_reads_past_the_length_as_zero(nat):
    s = Scene([(0, 20), (0, 0), (0, 33)], 2, 16, E4M3)
    s.fill(3)
    k, v = s.cache.read(s.batch, _ints([0, 50, 60, 93]), 93, dtype=torch.float32)
    assert (k[20:60] == 0).all() and (v[20:60] == 0).all()
    assert torch.equal(k[60:93].double(), s.held(2)[0])


@pytest.mark.parametrize("pages", [E4M3, torch.int8], ids=str)
def test_cache_codes_at_the_edges(nat, pages):
    """Zero rows, one large value among small ones, values at the codes' largest times a power of two and just past it,
    subnormal and huge rows, ties, and rows with an infinity or a NaN (held as NaN)."""
    top = ref.CODE_MAX[pages]
    rows = []
    for base in (0.0, 1.0, top, top * (1 + 2.0 ** -23), 2.0 ** -140, 2.0 ** -100, 2.0 ** 127, 3.0e38, 2.0 ** -126):
        r = torch.linspace(-1, 1, 64) * base
        rows += [r, torch.cat([torch.tensor([base]), r[1:] * 2.0 ** -12])]
    rows.append(torch.arange(64) * 2.0 + 0.5 * (torch.arange(64) % 2))  # ties of whole numbers
    rows[-1][0] = top
    for bad in (math.inf, -math.inf, math.nan):
        r = torch.ones(64)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows)[:, None].cuda()
    s = Scene([(x.shape[0], x.shape[0])], 1, 16, pages)
    s.cache.write(x, -x, s.batch)
    k, v = s.cache.read(s.batch, s.cu, x.shape[0], dtype=torch.float32)
    codes, exps = ref.quantise(x, pages)
    want = ref.values(codes, exps)
    got = k.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    assert torch.equal(v.double().nan_to_num(0), -want.nan_to_num(0))
    # one rounding: at most half a step of the row's scale (int8), half a step of the value or of the smallest (e4m3)
    unit = torch.exp2(exps.double() - 127)[..., None].expand_as(want)
    step = unit / 2 if pages == torch.int8 else torch.maximum(x.double().abs() * 2.0 ** -4, unit * 2.0 ** -10)
    ok = torch.isfinite(want)
    assert ((got - x.double()).abs()[ok] <= step[ok]).all()


def test_cache_shared_prefix_pages(nat):
    """Two sequences that share their first pages read the same rows; each writes its own last page."""
    from mapanything.kv_cache import KVBatch, PagedKVCache

    c = PagedKVCache(8, 16, 2, torch.bfloat16)
    table = _ints([[5, 2, 7], [5, 2, 0]])
    first = KVBatch(table[:1].contiguous(), _ints([32]), _ints([0, 32]), max_new=32, max_kv=32)
    k, v = _randn(32, 2, 64, seed=1, dtype=torch.bfloat16), _randn(32, 2, 64, seed=2, dtype=torch.bfloat16)
    c.write(k, v, first)
    both = KVBatch(table, _ints([40, 37]), _ints([0, 8, 13]))
    assert (both.max_new, both.max_kv) == (8, 40)
    kn, vn = _randn(13, 2, 64, seed=3, dtype=torch.bfloat16), _randn(13, 2, 64, seed=4, dtype=torch.bfloat16)
    c.write(kn, vn, both)
    gk, _ = c.read(both, _ints([0, 40, 77]), 77)
    assert torch.equal(gk[:32], k) and torch.equal(gk[40:72], k)
    assert torch.equal(gk[32:40], kn[:8]) and torch.equal(gk[72:], kn[8:])
    q = _randn(13, 4, 64, seed=5, dtype=torch.bfloat16)
    out, lse = c.attend(q, both, mask_block=1, return_lse=True)
    at = 0
    for b, (n, t) in enumerate([(8, 40), (5, 37)]):
        kk, vv = (ref.sequence_rows(x, None, table[b], t) for x in (c.k, c.v))
        o, l, ot, lt = ref.attention(q[at: at + n], kk, vv, ref.limits(n, t, 1), 0.125)
        ref.within(out[at: at + n], o, ot, "out")
        ref.within(lse[:, at: at + n], l, lt, "lse")
        at += n


# --------------------------------------------------------------------------------------------- attention
SHAPES = [
    # (new, cached) per sequence, query heads, K/V heads, page
    ([(1, 1)], 1, 1, 16),
    ([(1, 10960)], 12, 12, 64),                                     # one token, keys cut into ranges
    ([(1, n) for n in (1, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 1000)], 16, 4, 16),
    ([(2, 300), (1, 1), (0, 50), (5, 5), (3, 2000), (0, 0)], 6, 2, 32),  # few tokens, empty sequences
    ([(2, 3000), (1, 40)], 16, 1, 128),                             # 32 rows
    ([(7, 3), (4, 0), (1, 9)], 4, 4, 16),                           # more new tokens than cached ones
    ([(33, 33), (64, 64), (1, 700), (129, 500), (0, 12), (127, 128)], 4, 4, 64),
    ([(200, 150), (31, 31), (90, 4000)], 6, 2, 32),
    ([(45, 2500)], 15, 5, 16),                                      # three heads of a group: 126 of a tile's 128 rows
    ([(300, 5000)], 12, 12, 64),
    ([(1370, 2740)], 2, 2, 64),
    ([(250, 1111)], 4, 4, 16),                                      # one sequence that fills workgroups of 256 rows
    ([(500, 3000)], 2, 1, 32),
    ([(5, 100)] * 70, 8, 8, 16),                                    # more sequences than a wave has lanes
    ([(9, 60)] * 70, 16, 2, 16),
    ([(1, 3000), (2, 1100)], 40, 1, 16),                            # 40 heads of a group: three tokens a tile
    ([(3, 500), (1, 1)], 128, 1, 64),                               # 128: one token a tile
    ([(1, 3000), (3, 1024), (2, 1025)], 4, 4, 1024),                # the largest pages
    ([(150, 2100)], 4, 4, 1024),
    ([(1, 4000), (1, 2500)] * 30, 8, 8, 16),                        # ranges of more pages than a wave's window holds
]


@pytest.mark.parametrize("kind,pages", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                        (torch.bfloat16, E4M3), (torch.float16, E4M3),
                                        (torch.bfloat16, torch.int8), (torch.float16, torch.int8)], ids=str)
@pytest.mark.parametrize("block", [0, 1, 37])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_paged_matches_formula(nat, kind, pages, block, shape):
    seqs, heads, kv_heads, page = SHAPES[shape]
    s = Scene(seqs, kv_heads, page, pages, seed=shape)
    s.fill(10 * shape, kind)
    pad = 3
    packed = _randn(s.rows + pad, 3, heads, 64, seed=5, dtype=kind)
    q = packed[:, 0]
    out = torch.full((s.rows + pad, heads, 64), 7.0, dtype=kind, device="cuda")
    got, lse = s.cache.attend(q, s.batch, mask_block=block, out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    want, wlse, tol, ltol = s.expect(q[: s.rows], block)
    ref.within(got[: s.rows], want, tol, "out")
    ref.within(lse[:, : s.rows], wlse, ltol, "lse")
    assert (out[s.rows:] == 7).all()  # rows behind the last sequence
    again, lse2 = s.cache.attend(q, s.batch, mask_block=block, return_lse=True)
    assert torch.equal(again[: s.rows], got[: s.rows]) and torch.equal(lse2[:, : s.rows], lse[:, : s.rows])


@pytest.mark.parametrize("seqs,heads,kv_heads", [([(1, 5000), (1, 80)], 12, 12), ([(200, 900)], 4, 4)])
def test_attention_paged_scale_strides_and_growing_scores(nat, seqs, heads, kv_heads):
    """Another scale; queries and outputs as column blocks of wider rows; keys that grow along the sequence, so that the
    running maximum moves in every tile; strongly peaked rows."""
    s = Scene(seqs, kv_heads, 32, torch.bfloat16)

    def grow(batch, k, v):
        at = batch.cu_new.tolist()
        for a, b in zip(at, at[1:]):
            k[a:b] *= torch.linspace(0.1, 30, b - a, device="cuda")[:, None, None].to(k.dtype)

    s.fill(3, change=grow)
    wide = _randn(s.rows, 5 * heads * 64, seed=9, dtype=torch.bfloat16)
    q = wide[:, heads * 64: 2 * heads * 64].unflatten(1, (heads, 64))
    owide = torch.zeros(s.rows, heads * 128, dtype=torch.bfloat16, device="cuda")
    out = owide.unflatten(1, (heads, 128))[:, :, 64:]
    s.cache.attend(q, s.batch, scale=0.3, out=out)
    want, _, tol, _ = s.expect(q, 0, scale=torch.tensor(0.3, dtype=torch.float32).item())
    ref.within(out, want, tol, "out")
    assert (owide.unflatten(1, (heads, 128))[:, :, :64] == 0).all()


@pytest.mark.parametrize("pages", [torch.bfloat16, E4M3], ids=str)
@pytest.mark.parametrize("seqs,heads,kv_heads,page", [([(1, 9000)], 12, 12, 16), ([(5, 3000), (2, 100)], 6, 2, 32),
                                                       ([(140, 5000)], 4, 4, 16), ([(33, 40), (70, 2500)], 4, 2, 16)])
def test_attention_paged_without_workspace(nat, pages, seqs, heads, kv_heads, page):
    """The C entry without a workspace (or with one too small): every row's keys in one workgroup, over many page windows."""
    import ctypes

    s = Scene(seqs, kv_heads, page, pages)
    s.fill(17)
    q = _randn(s.rows, heads, 64, seed=18, dtype=torch.bfloat16)
    want, wlse, tol, ltol = s.expect(q, 1)
    small = torch.empty(64, dtype=torch.uint8, device="cuda")
    for ws in (None, small):
        out, lse = torch.empty_like(q), torch.empty(heads, s.rows, device="cuda")
        d = nat.AttnPagedDesc(cache=s.cache.desc, batch=s.batch._rows(s.rows), dtype=nat.BF16, heads=heads,
                              q=q.data_ptr(), o=out.data_ptr(), q_rstride=q.stride(0), q_hstride=64,
                              o_rstride=out.stride(0), o_hstride=64, lse=lse.data_ptr(), mask_block=1)
        assert nat.lib().mapa_attention_paged_workspace_bytes(ctypes.byref(d)) > 64
        if ws is not None:
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        nat.check(nat.lib().mapa_attention_paged(ctypes.byref(d), nat.stream()), "mapa_attention_paged")
        ref.within(out, want, tol, "out")
        ref.within(lse, wlse, ltol, "lse")


@pytest.mark.parametrize("block", [1, 37])
def test_attention_paged_several_streams_at_once(nat, block):
    """Calls of different shapes in flight on three streams at once: each has partials of its own."""
    work = []
    for i, seqs in enumerate(([(1, 9000)], [(200, 3000), (40, 600)], [(3, 800)] * 9)):
        s = Scene(seqs, 4, 32, torch.bfloat16, seed=i)
        s.fill(60 + i)
        q = _randn(s.rows, 8, 64, seed=70 + i, dtype=torch.bfloat16)
        work.append((s, q, s.cache.attend(q, s.batch, mask_block=block), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        outs = []
        for s, q, _, st in work:
            with torch.cuda.stream(st):
                outs.append([s.cache.attend(q, s.batch, mask_block=block) for _ in range(4)])
        torch.cuda.synchronize()
        for (_, _, want, _), got in zip(work, outs):
            assert all(torch.equal(o, want) for o in got)


@pytest.mark.parametrize("pages", [torch.bfloat16, E4M3, torch.int8], ids=str)
@pytest.mark.parametrize("seqs,heads,kv_heads", [([(6, 70), (3, 3)], 4, 2), ([(100, 260), (40, 40)], 4, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_paged_hidden_values_do_not_leak(nat, pages, seqs, heads, kv_heads, bad, which):
    """Tokens whose keys or values are not finite change the rows that see them, and no others."""
    s = Scene(seqs, kv_heads, 16, pages)
    at = [0]
    for _, t in seqs:
        at.append(at[-1] + t)

    def spoil(batch, k, v):
        for a, b in zip(at, at[1:]):
            (k if which == "k" else v)[b - 2, :, 5] = bad  # the last token but one of every sequence

    s.fill(21, change=spoil)
    q = _randn(s.rows, heads, 64, seed=2, dtype=torch.bfloat16).abs() * 0.5  # q.k of an infinity: the same sign
    got, lse = s.cache.attend(q, s.batch, mask_block=1, return_lse=True)
    sees = torch.cat([torch.tensor([x >= t - 1 for x in ref.limits(n, t, 1)]) for n, t in seqs]).cuda()
    assert torch.isfinite(got[~sees].float()).all() and torch.isfinite(lse[:, ~sees]).all()
    clean = Scene(seqs, kv_heads, 16, pages)
    clean.fill(21)
    want, wlse, tol, ltol = clean.expect(q, 1)
    ref.within(got[~sees], want[~sees], tol[~sees], "rows that do not see it")
    ref.within(lse[:, ~sees], wlse[:, ~sees], ltol[:, ~sees], "lse of rows that do not see it")
    if which == "v" and pages == torch.bfloat16:  # the formula's own NaN and infinities, in the same columns
        full, _, ftol, _ = s.expect(q, 1)
        ref.within(got, full, ftol, "all rows")
    elif math.isnan(bad) or pages != torch.bfloat16:
        assert torch.isnan(got[sees].float()).any(-1).all()


def test_attention_paged_merges_with_dense_attention(nat):
    """Paged attention over the earlier tokens and mapa_attention over the new ones, joined by mapa_attn_merge, is
    attention over all of them."""
    from mapanything.kv_cache import KVBatch

    H, old, new = 12, 500, 96
    s = Scene([(new, old + new)], H, 64, torch.bfloat16)
    k, v = s.fill(4)
    q = _randn(new, H, 64, seed=6, dtype=torch.bfloat16)
    want, wlse, tol, ltol = s.expect(q, 0)
    earlier = KVBatch(s.table, _ints([old]), _ints([0, new]), max_new=new, max_kv=old)
    o1, l1 = s.cache.attend(q, earlier, return_lse=True)
    o2, l2 = torch.empty_like(o1), torch.empty_like(l1)
    kn, vn = k[old:].contiguous(), v[old:].contiguous()
    C = H * 64
    nat.attention(q, kn, vn, o2, batch=1, heads=H, seq_q=new, seq_kv=new, q_bstride=new * C, q_rstride=C,
                  k_bstride=new * C, k_rstride=C, v_bstride=new * C, v_rstride=C, o_bstride=new * C, o_rstride=C, lse=l2)
    out = torch.empty_like(o1)
    nat.attn_merge(o1, l1, o2, l2, out, new, H, C)
    # three roundings to bf16 more than one call has, and the dense kernel's rounding of its scaled queries: half a step
    # of every product, |s| of them under 8 here
    half = ref.half_step(torch.bfloat16)
    a = (tol / half).clamp_min(1e-30)
    ref.within(out, want, tol + half * 3 * want.abs() + half * (3 + 8) * a * half / half, "merged")


@pytest.mark.parametrize("step", [True, False])
def test_attention_paged_on_streams_and_in_graphs(nat, step):
    """A side stream; two graphs captured on one stream, replayed in turn and at once on two streams with lengths,
    tables and tokens that change in place between replays, against eager calls."""
    seqs = [(1, 3000), (1, 90)] if step else [(140, 3000), (33, 90)]
    scenes = [Scene(seqs, 4, 16, torch.bfloat16, seed=i) for i in range(2)]
    qs = []
    for i, s in enumerate(scenes):
        s.fill(30 + i)
        qs.append(_randn(s.rows, 8, 64, seed=40 + i, dtype=torch.bfloat16))
    eager = [s.cache.attend(q, s.batch, mask_block=1) for s, q in zip(scenes, qs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = scenes[0].cache.attend(qs[0], scenes[0].batch, mask_block=1)
    torch.cuda.synchronize()
    assert torch.equal(other, eager[0])
    graphs, outs = [], []
    for s, q in zip(scenes, qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.cache.attend(q, s.batch, mask_block=1))
        graphs.append(g)
    for turn in range(3):
        for s, q in zip(scenes, qs):
            q.copy_(_randn(*q.shape, seed=50 + turn, dtype=q.dtype))
            s.lens.sub_(1)  # shorter scenes under the same bounds
        want = [s.cache.attend(q, s.batch, mask_block=1) for s, q in zip(scenes, qs)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_cache_in_a_graph(nat):
    s = Scene([(1, 40), (1, 17)], 2, 16, E4M3)
    s.fill(1)
    k, v = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16), _randn(2, 2, 64, seed=3, dtype=torch.bfloat16)
    whole, rows = s.whole()
    graph = torch.cuda.CUDAGraph()
    s.cache.write(k, v, s.batch)
    with torch.cuda.graph(graph):
        s.cache.write(k, v, s.batch)
        gk, gv = s.cache.read(s.batch, whole.cu_new, rows)
    for i in range(3):
        k.copy_(_randn(2, 2, 64, seed=10 + i, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        codes, exps = ref.quantise(k, E4M3)
        assert torch.equal(gk[39].double(), ref.values(codes, exps)[0])
        assert torch.equal(gk[56].double(), ref.values(codes, exps)[1])


@pytest.mark.parametrize("pages", [torch.bfloat16, E4M3], ids=str)
def test_paged_offsets_past_32_bits(nat, pages):
    """A cache of more than 2^32 bytes (and 2^31 values) per tensor, the sequence in its last pages."""
    heads, page = 16, 64
    count = (1 << 32) // (heads * page * 64 * (2 if pages == torch.bfloat16 else 1)) + 40
    from mapanything.kv_cache import KVBatch, PagedKVCache

    c = PagedKVCache(count, page, heads, pages)
    total = 30 * page - 5
    table = torch.arange(count - 1, count - 31, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    batch = KVBatch(table, _ints([total]), _ints([0, total]))
    k, v = (_randn(total, heads, 64, seed=i, dtype=torch.bfloat16) for i in range(2))
    c.write(k, v, batch)
    gk, gv = c.read(batch, _ints([0, total]), total)
    if pages == torch.bfloat16:
        assert torch.equal(gk, k) and torch.equal(gv, v)
    for new in (1, 200):
        q = _randn(new, heads, 64, seed=7, dtype=torch.bfloat16)
        b2 = KVBatch(table, _ints([total]), _ints([0, new]))
        out = c.attend(q, b2, mask_block=1)
        want, _, tol, _ = ref.attention(q, gk.double(), gv.double(), ref.limits(new, total, 1), 0.125)
        ref.within(out, want, tol, f"{new} tokens")


# --------------------------------------------------------------------------------------------- what is not sound
def test_paged_faults_are_reported(nat):
    """Page numbers, lengths and offsets outside what the host stated raise the fault bit; the sequences that are sound
    keep their results, and nothing outside the cache is touched."""
    from mapanything.kv_cache import KVBatch

    def faulted(call):
        call()
        with pytest.raises(nat.DeviceFault) as e:
            nat.check_faults()
        assert e.value.bits == nat.FAULT_KV_RANGE

    s = Scene([(1, 40), (1, 60)], 2, 16, torch.bfloat16)
    s.fill(1)
    q = _randn(2, 2, 64, seed=2, dtype=torch.bfloat16)
    k = _randn(2, 2, 64, seed=3, dtype=torch.bfloat16)
    good = s.cache.attend(q, s.batch)
    pages = s.cache.k.shape[0]
    for bad in (-1, pages, 1 << 30):
        table = s.table.clone()
        table[0, 2] = bad
        b = KVBatch(table, s.lens, s.cu, max_new=1, max_kv=60)
        out = torch.zeros_like(q)
        faulted(lambda: s.cache.attend(q, b, out=out))
        assert torch.equal(out[1], good[1])
        before = s.cache.k.clone()
        faulted(lambda: s.cache.write(k, k, b))
        want = before.clone()
        want[s.table[1, 3], :, 59 % 16] = k[1]
        assert torch.equal(s.cache.k.view(torch.int16), want.view(torch.int16))
        faulted(lambda: s.cache.read(b, _ints([0, 40, 100]), 100))
        s.cache.write(before.new_zeros(0, 2, 64), before.new_zeros(0, 2, 64), s.batch)  # nothing to do
        s.fill(1)
    for lens in ([41 + 16 * 40, 60], [-1, 60], [61, 60]):
        b = KVBatch(s.table, _ints(lens), s.cu, max_new=1, max_kv=60)
        out = torch.zeros_like(q)
        faulted(lambda: s.cache.attend(q, b, out=out))
        assert torch.equal(out[1], good[1])
    for cu in ([0, 3, 2], [0, 1, 3], [0, -1, 1]):
        b = KVBatch(s.table, s.lens, _ints(cu), max_new=1, max_kv=60)
        faulted(lambda: s.cache.attend(q, b))
    b = KVBatch(s.table, s.lens, _ints([0, 1, 3]), max_new=2, max_kv=60)  # offsets behind the rows
    faulted(lambda: s.cache.write(k, k, b))
    many = KVBatch(s.table, s.lens, _ints([0, 2, 2]), max_new=1, max_kv=60)  # more new tokens than stated
    faulted(lambda: s.cache.attend(q, many))
    with pytest.raises(nat.DeviceFault):  # a position before the sequence's first
        s.cache.write(k.new_zeros(41, 2, 64), k.new_zeros(41, 2, 64),
                      KVBatch(s.table[:1].contiguous(), _ints([40]), _ints([0, 41]), max_new=41, max_kv=60))
        nat.check_faults()


def test_paged_class_refusals(nat):
    from mapanything.kv_cache import KVBatch, PagedKVCache

    s = Scene([(1, 40)], 2, 16, torch.bfloat16)
    q = _randn(1, 2, 64, seed=1, dtype=torch.bfloat16)
    for bad in (q[:, :, :32], q.cpu(), q[0], q.float(), q.to(torch.float16), _randn(1, 3, 64, seed=1, dtype=torch.bfloat16),
                _randn(1, 2, 128, seed=1, dtype=torch.bfloat16)[:, :, ::2],
                _randn(1, 2, 65, seed=1, dtype=torch.bfloat16)[:, :, 1:]):
        with pytest.raises(nat.NativeError):
            s.cache.attend(bad, s.batch)
        if bad.dtype == torch.bfloat16:  # rows to write may be fp32 or fp16 too
            with pytest.raises(nat.NativeError):
                s.cache.write(bad, bad, s.batch)
    for k, v in ((q, q.float()), (q.double(), q.double()), (q, q[:0])):
        with pytest.raises(nat.NativeError):
            s.cache.write(k, v, s.batch)
    g = q.clone().requires_grad_()
    for call in (lambda: s.cache.attend(g, s.batch), lambda: s.cache.write(g, q, s.batch)):
        with pytest.raises(nat.NativeError):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(nat.NativeError):
        s.cache.attend(q, s.batch, out=q.float())
    with pytest.raises(nat.NativeError):
        s.cache.attend(q, s.batch, mask_block=-1)
    for args in ((s.table.long(), s.lens, s.cu), (s.table, s.lens, s.cu[:1]), (s.table[0], s.lens, s.cu),
                 (s.table, s.lens.cpu(), s.cu)):
        with pytest.raises(nat.NativeError):
            KVBatch(*args, max_new=1, max_kv=40)
    z = torch.zeros(2, 1, 16, 64, device="cuda")
    for args in ((z, z), (z.bfloat16(), z.half()), (z.bfloat16()[..., :32], z.bfloat16()[..., :32]),
                 (z.to(torch.int8), z.to(torch.int8)), (z.bfloat16(), z.bfloat16(), z[..., 0].byte(), z[..., 0].byte()),
                 (z.to(torch.int8), z.to(torch.int8), z[..., 0], z[..., 0]),
                 (z.bfloat16().transpose(0, 2), z.bfloat16().transpose(0, 2))):
        with pytest.raises(nat.NativeError):
            PagedKVCache.wrap(*args)
    with pytest.raises(nat.NativeError):
        s.cache.read(s.batch, _ints([0]), 1)


@pytest.mark.parametrize("seqs,heads", [([(1, 300)], 4), ([(1, 300), (70, 1300)], 12), ([(300, 2000)], 2)])
def test_attention_paged_over_its_queries(nat, seqs, heads):
    """out may be q itself, with one key range and with several."""
    s = Scene(seqs, 2, 16, torch.bfloat16)
    s.fill(43)
    q = _randn(sum(n for n, _ in seqs), heads, 64, seed=41, dtype=torch.bfloat16)
    want = s.cache.attend(q, s.batch, mask_block=1)
    mine = q.clone()
    assert s.cache.attend(mine, s.batch, mask_block=1, out=mine) is mine
    assert torch.equal(mine, want)


def test_paged_outputs_are_seen_and_tensors_are_kept(nat):
    s = Scene([(2, 40)], 2, 16, torch.bfloat16)
    q = _randn(2, 4, 64, seed=42, dtype=torch.bfloat16)
    with pytest.raises(nat.NativeError):
        s.cache.attend(q, s.batch, out=q[:1].expand(2, 4, 64))
    with pytest.raises(nat.NativeError):
        s.cache.attend(q, s.batch, out=q[:, :1].expand(2, 4, 64))
    cu, k = _ints([0, 40]), torch.zeros(40, 2, 64, device="cuda")
    with pytest.raises(nat.NativeError):
        s.cache.read(s.batch, cu, 40, out=(k, k[:1].expand(40, 2, 64)))
    w = torch.ones((), device="cuda", requires_grad=True)
    for out, call in ((q, lambda: s.cache.attend(q, s.batch, out=q)),
                      (k, lambda: s.cache.read(s.batch, cu, 40, out=(k, torch.empty_like(k))))):
        y = w * out
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    for t, names in ((s.cache, ("k", "v", "k_exp", "v_exp")), (s.batch, ("table", "kv_lens", "cu_new", "max_new", "max_kv"))):
        for name in names:  # the calls go by what they were made with
            with pytest.raises(AttributeError):
                setattr(t, name, getattr(t, name))


# --------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("pages", [torch.bfloat16, E4M3, torch.int8], ids=str)
def test_streaming_run(nat, pages):
    """A scene view by view, then token by token: rotary (time, row, column) positions on queries and keys, the cache
    written, attention of the new view over it.  Every call against the formulas in 64 bits, fed the 16-bit tensors that
    the call before it gave; at the end the calls' outputs against one block-causal pass over the whole scene."""
    from mapanything.kv_cache import KVBatch, PagedKVCache
    from uniception.models.libs.croco.pos_embed import RoPEAxes

    H, side, views, steps, page = 12, 9, 4, 3, 16
    T = side * side + 1
    total = views * T + steps
    rope = RoPEAxes((8, 12, 12), freq=10000.0)
    cache = PagedKVCache(total // page + 5, page, H, pages)
    table = torch.randperm(cache.k.shape[0], generator=_gen(1), device="cuda")[: -(-total // page)].int()[None].contiguous()
    qkv = _randn(total, 3, H, 64, seed=2, dtype=torch.bfloat16)
    i = torch.arange(total, device="cuda")
    t = torch.where(i < views * T, i % T, 0)
    pos = torch.stack([torch.where(i < views * T, i // T, views + i - views * T), t // side, t % side], -1)
    chunks = [(v * T, T) for v in range(views)] + [(views * T + s, 1) for s in range(steps)]
    outs, qs = [], []
    for at, n in chunks:
        rows = qkv[at: at + n]
        q, k = rope(rows[:, 0].transpose(0, 1)[None], pos[at: at + n], rows[:, 1].transpose(0, 1)[None])
        for got, x in ((q, rows[:, 0]), (k, rows[:, 1])):
            want, bound = ref.rope(x.transpose(0, 1)[None], pos[None, at: at + n], (8, 12, 12), 10000.0)
            ref.within(got, want, bound + ref.half_step(torch.bfloat16) * (want.abs() + bound), "rope")
        q, k = (x[0].transpose(0, 1) for x in (q, k))
        batch = KVBatch(table, _ints([at + n]), _ints([0, n]), max_new=n, max_kv=at + n)
        cache.write(k, rows[:, 2], batch)
        out = cache.attend(q, batch)
        kk, vv = (ref.sequence_rows(a, b, table[0], at + n) for a, b in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)))
        want, _, tol, _ = ref.attention(q, kk, vv, [at + n] * n, 0.125)
        ref.within(out, want, tol, f"tokens {at} to {at + n}")
        outs.append(out)
        qs.append(q)
    whole = KVBatch(table, _ints([views * T]), _ints([0, views * T]))
    once = cache.attend(torch.cat(qs[:views]), whole, mask_block=T)
    # the same sums in another order: each side within the bound of the 64-bit result
    kk, vv = (ref.sequence_rows(a, b, table[0], views * T) for a, b in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)))
    want, _, tol, _ = ref.attention(torch.cat(qs[:views]), kk, vv, ref.limits(views * T, views * T, T), 0.125)
    ref.within(once, want, tol, "one pass")
    ref.within(torch.cat(outs[:views]), want, tol, "view by view")
