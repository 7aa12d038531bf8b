"""Argument checks of the streaming operators' C entries and classes: they run before any launch, so no GPU is needed;
ctypes layouts against the C compiler's."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import REPO


@pytest.fixture(scope="module")
def nat():
    from mapanything import _native

    _native.load_library()
    return _native


def _rope(nat, **over):
    d = nat.RopeAxesDesc(dtype=nat.BF16, batch=1, tokens=4, head_dim=64, axes=3, layout=nat.ROPE_AXIAL)
    for i, n in enumerate((8, 12, 12)):
        d.section[i] = n
    d.x[0] = d.y[0] = 4096
    d.heads[0] = 2
    d.x_bstride[0] = d.y_bstride[0] = 512
    d.x_hstride[0] = d.y_hstride[0] = 64
    d.x_nstride[0] = d.y_nstride[0] = 128
    d.positions = 4096
    for k, v in over.items():
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                getattr(d, k)[i] = x
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,word", [
    ({"dtype": 2}, b"dtype"), ({"axes": 0}, b"axes"), ({"axes": 5}, b"axes"), ({"layout": 3}, b"layout"),
    ({"pos_dtype": 2}, b"pos_dtype"), ({"section": (8, 0, 12)}, b"section"), ({"section": (8, 12, 13)}, b"do not fit"),
    ({"section": (120, 9, 1), "head_dim": 512}, b"do not fit"), ({"head_dim": 0}, b"bad shape"),
    ({"tokens": -1}, b"bad shape"), ({"y": (None, None)}, b"null output"), ({"positions": None}, b"null positions"),
    ({"y_nstride": (64, 0)}, b"in place"), ({"x": (4097, None)}, b"aligned"), ({"heads": (-1, 0)}, b"head count"), ({"heads": (2049, 0)}, b"head count"),
    ({"batch": 65536, "tokens": 65536}, b"too many"),
])
def test_rope_axes_refuses(nat, over, word):
    L = nat.load_library()
    assert L.mapa_rope_axes(ctypes.byref(_rope(nat, **over)), None) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()


def test_rope_axes_refuses_one_output_for_both(nat):
    L = nat.load_library()
    assert L.mapa_rope_axes(ctypes.byref(_rope(nat, x=(4096, 4096), y=(4096, 4096), heads=(2, 2),
                                               **{k: (s, s) for k, s in (("x_bstride", 512), ("y_bstride", 512),
                                                  ("x_hstride", 64), ("y_hstride", 64), ("x_nstride", 128),
                                                  ("y_nstride", 128))})), None) != 0
    assert b"one output" in L.mapa_last_error()


def test_rope_axes_nothing_to_do(nat):
    L = nat.load_library()
    assert L.mapa_rope_axes(None, None) != 0
    assert L.mapa_rope_axes(ctypes.byref(_rope(nat, tokens=0, positions=None)), None) == 0
    assert L.mapa_rope_axes(ctypes.byref(_rope(nat, heads=(0, 0))), None) == 0


@pytest.mark.parametrize("kw", [{"sections": ()}, {"sections": (1,) * 5}, {"sections": (4, 0)}, {"sections": (100, 29)},
                                {"sections": (8,), "layout": "quarter"}, {"sections": (8,), "spectrum": "none"},
                                {"sections": (8,), "freq": 0.0}])
def test_rope_axes_class_refuses(kw):
    from uniception.models.libs.croco.pos_embed import RoPEAxes

    with pytest.raises(ValueError):
        RoPEAxes(**kw)


def _cache(nat, **over):
    c = nat.KVCacheDesc(nat.BF16, 12, 64, 8, 4096, 8192, None, None)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def _batch(nat, **over):
    b = nat.KVBatchDesc(2, 4, 4096, 4096, 4096, 10, 5, 200)
    for k, v in over.items():
        setattr(b, k, v)
    return b


CACHE_REFUSALS = [({"dtype": 0}, b"pages must be"), ({"heads": 0}, b"bad cache"), ({"heads": 2049}, b"bad cache"), ({"num_pages": 0}, b"bad cache"),
                  ({"page_size": 8}, b"page size"), ({"page_size": 48}, b"page size"),
                  ({"page_size": 2048}, b"page size"), ({"k": None}, b"aligned"), ({"v": 8200}, b"aligned"),
                  ({"dtype": 5}, b"exponent"), ({"dtype": 6, "k_exp": 64}, b"exponent")]
BATCH_REFUSALS = [({"seqs": -1}, b"bad batch"), ({"new_rows": -1}, b"bad batch"), ({"max_kv": -1}, b"bad batch"),
                  ({"max_kv": (1 << 30) + 1}, b"bad batch"), ({"kv_lens": None}, b"null batch"),
                  ({"cu_new": None}, b"null batch"), ({"table": None}, b"null batch"), ({"seqs": 65536}, b"bad batch")]


@pytest.mark.parametrize("cache,batch,word", [(c, {}, w) for c, w in CACHE_REFUSALS] + [({}, b, w) for b, w in BATCH_REFUSALS])
def test_cache_and_batch_refused_everywhere(nat, cache, batch, word):
    L = nat.load_library()
    c, b = _cache(nat, **cache), _batch(nat, **batch)
    rows = (4096, 4096, nat.BF16, 768, 64, 768, 64, None)
    assert L.mapa_kv_cache_write(ctypes.byref(c), ctypes.byref(b), *rows) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()
    assert L.mapa_kv_cache_read(ctypes.byref(c), ctypes.byref(b), 4096, 10, *rows) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()
    d = nat.AttnPagedDesc(cache=c, batch=b, dtype=nat.BF16, heads=12, q=4096, o=4096, q_rstride=768, q_hstride=64,
                          o_rstride=768, o_hstride=64)
    assert L.mapa_attention_paged(ctypes.byref(d), None) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()


@pytest.mark.parametrize("rows,word", [((None, 4096, 1, 768, 64, 768, 64), b"null rows"),
                                       ((4096, 4096, 5, 768, 64, 768, 64), b"rows must be"),
                                       ((4104, 4096, 1, 768, 64, 768, 64), b"alignment"),
                                       ((4096, 4096, 1, 764, 64, 768, 64), b"alignment"),
                                       ((4096, 4096, 1, 768, 64, 768, 63), b"alignment")])
def test_cache_rows_refused(nat, rows, word):
    L = nat.load_library()
    c, b = _cache(nat), _batch(nat)
    assert L.mapa_kv_cache_write(ctypes.byref(c), ctypes.byref(b), *rows, None) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()
    assert L.mapa_kv_cache_read(ctypes.byref(c), ctypes.byref(b), 4096, 10, *rows, None) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()


@pytest.mark.parametrize("over,word", [({"dtype": 0}, b"queries must be"), ({"dtype": 3}, b"queries' type"),
                                       ({"heads": 13}, b"query heads"), ({"heads": 0}, b"query heads"),
                                       ({"heads": 12 * 129}, b"query heads"), ({"mask_block": -1}, b"mask_block"),
                                       ({"scale": -1.0}, b"scale"), ({"scale": float("nan")}, b"scale"),
                                       ({"q": None}, b"alignment"), ({"o": 4104}, b"alignment"),
                                       ({"q_rstride": 4}, b"alignment"), ({"o_hstride": 65}, b"alignment")])
def test_attention_paged_refuses(nat, over, word):
    L = nat.load_library()
    d = nat.AttnPagedDesc(cache=_cache(nat), batch=_batch(nat), dtype=nat.BF16, heads=12, q=4096, o=4096, q_rstride=768,
                          q_hstride=64, o_rstride=768, o_hstride=64)
    for k, v in over.items():
        setattr(d, k, v)
    assert L.mapa_attention_paged(ctypes.byref(d), None) != 0
    assert word in L.mapa_last_error(), L.mapa_last_error()


def test_nothing_to_do(nat):
    L = nat.load_library()
    c = _cache(nat)
    for over in ({"seqs": 0}, {"new_rows": 0}):
        b = _batch(nat, **over)
        assert L.mapa_kv_cache_write(ctypes.byref(c), ctypes.byref(b), None, None, 1, 0, 0, 0, 0, None) == 0
        d = nat.AttnPagedDesc(cache=c, batch=b, dtype=nat.BF16, heads=12)
        assert L.mapa_attention_paged(ctypes.byref(d), None) == 0
        assert L.mapa_attention_paged_workspace_bytes(ctypes.byref(d)) == 0
    assert L.mapa_kv_cache_read(ctypes.byref(c), ctypes.byref(_batch(nat)), None, 0, None, None, 1, 0, 0, 0, 0, None) == 0
    assert L.mapa_attention_paged(None, None) != 0


def test_cpu_tensors_are_refused(nat):
    from mapanything.kv_cache import KVBatch, PagedKVCache

    with pytest.raises(nat.NativeError):
        PagedKVCache.wrap(torch.zeros(2, 1, 16, 64), torch.zeros(2, 1, 16, 64))
    with pytest.raises(nat.NativeError):
        PagedKVCache(2, 16, 1, device="cpu")
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(nat.NativeError):
        KVBatch(i[None], i, torch.zeros(2, dtype=torch.int32))


def test_descriptor_layouts_match_header(tmp_path, nat):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = {"mapa_rope_axes_desc": nat.RopeAxesDesc, "mapa_kv_cache": nat.KVCacheDesc, "mapa_kv_batch": nat.KVBatchDesc,
              "mapa_attn_paged_desc": nat.AttnPagedDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mapa.h"', "int main(void) {"]
    for cname, cls in fields.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "off.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-I", os.path.join(REPO, "include"), str(tmp_path / "off.c"), "-o", str(tmp_path / "off")], check=True)
    out = subprocess.run([str(tmp_path / "off")], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {(a, b): int(c) for a, b, c in (ln.split() for ln in out if ln)}
    for cname, cls in fields.items():
        assert got[(cname, "sizeof")] == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert got[(cname, f)] == getattr(cls, f).offset, (cname, f)
    from uniception.models.libs.croco import pos_embed

    assert pos_embed._DESC_HEAD.size == nat.RopeAxesDesc.axes.offset  # what RoPEAxes packs at once
    d = nat.RopeAxesDesc()
    pos_embed._DESC_HEAD.pack_into(d, 0, *range(1, 28))
    flat = [d.dtype, d.batch, d.tokens, d.head_dim, *d.x, *d.y, *d.heads, *d.x_bstride, *d.x_hstride, *d.x_nstride,
            *d.y_bstride, *d.y_hstride, *d.y_nstride, d.positions, d.pos_dtype, d.pos_bstride, d.pos_nstride, d.pos_astride]
    assert flat == list(range(1, 28))
