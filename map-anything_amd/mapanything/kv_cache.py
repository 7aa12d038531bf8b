"""Paged K/V cache of the multi-view transformer's attention, and attention of new tokens over it, on the gfx950 kernels
`mapa_kv_cache_write`, `mapa_kv_cache_read` and `mapa_attention_paged` (include/mapa.h).

The engine's global layers attend over all views of one call.  A scene that grows view by view keeps the keys and
values of its earlier views here instead: pages of `page_size` tokens, handed out by the caller (a page table per
sequence), 16-bit or quantised as they are written.  Head width is 64, as in every attention of the library.

    cache = PagedKVCache(num_pages=4096, page_size=64, heads=12, dtype=torch.float8_e4m3fn)
    batch = KVBatch(table, kv_lens, cu_new, max_new=1370, max_kv=20000)     # int32 device tensors, see KVBatch
    cache.write(k, v, batch)                                 # (rows, 12, 64) new keys and values of all sequences
    out = cache.attend(q, batch, mask_block=1370)            # every view sees itself and the earlier ones

No CPU path: a missing library or device raises.  Page numbers, lengths and offsets live in device memory and are
checked there: `_native.check_faults()` raises if a call of its thread (or a graph that the thread captured) met one
outside the cache since the last check, whatever ran in between."""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _native as nat

HEAD_DIM = 64
_PAGE_CODES = {torch.bfloat16: nat.BF16, torch.float16: nat.F16, torch.float8_e4m3fn: nat.FP8, torch.int8: nat.I8}


def _int32(t: torch.Tensor, name: str, ndim: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.ndim != ndim or not t.is_cuda or not t.is_contiguous():
        raise nat.NativeError(f"{name}: a contiguous int32 GPU tensor with {ndim} dimension(s) is needed, got "
                              f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t


class KVBatch:
    """Which tokens a call is about.

    table (seqs, columns): page of every page_size tokens of a sequence; kv_lens (seqs,): tokens in the cache with the
    new ones; cu_new (seqs + 1,): the packed rows cu_new[b] .. cu_new[b + 1] - 1 are sequence b's new tokens, its last
    positions.  max_new / max_kv: upper bounds of the new / cached tokens of one sequence, which size the launch; left
    out, they are read from the device (a synchronisation, so not while a graph is captured).  The tensors' contents may
    change from call to call; other tensors or bounds make another KVBatch."""

    __slots__ = ("_table", "_kv_lens", "_cu_new", "_max_new", "_max_kv", "desc")

    table = property(lambda self: self._table)
    kv_lens = property(lambda self: self._kv_lens)
    cu_new = property(lambda self: self._cu_new)
    max_new = property(lambda self: self._max_new)
    max_kv = property(lambda self: self._max_kv)

    def __init__(self, table: torch.Tensor, kv_lens: torch.Tensor, cu_new: torch.Tensor, *,
                 max_new: Optional[int] = None, max_kv: Optional[int] = None):
        seqs = kv_lens.shape[0] if kv_lens.ndim else 0
        _int32(table, "KVBatch: table", 2)
        _int32(kv_lens, "KVBatch: kv_lens", 1)
        _int32(cu_new, "KVBatch: cu_new", 1)
        if table.shape[0] != seqs or cu_new.shape[0] != seqs + 1:
            raise nat.NativeError(f"KVBatch: table {tuple(table.shape)}, kv_lens {tuple(kv_lens.shape)} and cu_new "
                                  f"{tuple(cu_new.shape)} do not describe the same sequences")
        if table.device != kv_lens.device or table.device != cu_new.device:
            raise nat.NativeError("KVBatch: table, kv_lens and cu_new must be on one device")
        if max_new is None:
            max_new = int((cu_new[1:] - cu_new[:-1]).max()) if seqs else 0
        if max_kv is None:
            max_kv = int(kv_lens.max()) if seqs else 0
        if not (0 <= max_new < 1 << 31 and 0 <= max_kv <= 1 << 30):  # (a C int would take what is left of a larger one)
            raise nat.NativeError(f"KVBatch: max_new {max_new} and max_kv {max_kv} must be 0 to 2^31 - 1 and 0 to 2^30")
        self._table, self._kv_lens, self._cu_new, self._max_new, self._max_kv = table, kv_lens, cu_new, max_new, max_kv
        self.desc = nat.KVBatchDesc(seqs, table.shape[1], table.data_ptr(), kv_lens.data_ptr(), cu_new.data_ptr(), 0,
                                    max_new, max_kv)

    def _rows(self, rows: int) -> nat.KVBatchDesc:
        d = nat.KVBatchDesc.from_buffer_copy(self.desc)
        d.new_rows = rows
        return d


class PagedKVCache:
    """Pages of keys and values: `k`, `v` (num_pages, heads, page_size, 64) in bf16, fp16, e4m3 (torch.float8_e4m3fn)
    or int8; the 8-bit types carry one exponent byte per row in `k_exp`, `v_exp` (num_pages, heads, page_size) (value =
    code * 2^(byte - 127), see include/mapa.h).  page_size: a power of two, 16 to 1024.  The tensors are the cache's
    for its life: their contents may be moved or filled, larger ones make another cache (wrap)."""

    __slots__ = ("_k", "_v", "_k_exp", "_v_exp", "_tensors", "desc")

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_exp = property(lambda self: self._k_exp)
    v_exp = property(lambda self: self._v_exp)

    def __init__(self, num_pages: int, page_size: int = 64, heads: int = 12, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        shape = (num_pages, heads, page_size)
        k, v = (torch.empty(*shape, HEAD_DIM, dtype=dtype, device=device) for _ in range(2))
        codes = dtype in (torch.float8_e4m3fn, torch.int8)
        k_exp, v_exp = (torch.empty(shape, dtype=torch.uint8, device=device) if codes else None for _ in range(2))
        self._hold(k, v, k_exp, v_exp)

    @classmethod
    def wrap(cls, k, v, k_exp=None, v_exp=None) -> "PagedKVCache":
        """A cache over pages that the caller holds."""
        self = cls.__new__(cls)
        self._hold(k, v, k_exp, v_exp)
        return self

    def _hold(self, k, v, k_exp, v_exp):
        code = _PAGE_CODES.get(k.dtype)
        if code is None or v.dtype != k.dtype:
            raise nat.NativeError(f"PagedKVCache: pages must be bf16, fp16, float8_e4m3fn or int8, got {k.dtype} / "
                                  f"{v.dtype}")
        if k.ndim != 4 or k.shape[3] != HEAD_DIM or v.shape != k.shape or not (k.is_contiguous() and v.is_contiguous()):
            raise nat.NativeError(f"PagedKVCache: k {tuple(k.shape)} and v {tuple(v.shape)} must be contiguous "
                                  f"(pages, heads, page_size, {HEAD_DIM})")
        if not k.is_cuda or v.device != k.device:
            raise nat.NativeError("PagedKVCache: pages must be on one GPU; there is no CPU path")
        if (code in (nat.FP8, nat.I8)) != (k_exp is not None) or (k_exp is None) != (v_exp is None):
            raise nat.NativeError("PagedKVCache: 8-bit pages, and only they, come with k_exp and v_exp")
        if k_exp is not None:
            for e in (k_exp, v_exp):
                if e.dtype != torch.uint8 or e.shape != k.shape[:3] or not e.is_contiguous() or e.device != k.device:
                    raise nat.NativeError("PagedKVCache: exponents must be contiguous uint8 (pages, heads, page_size)")
        self._k, self._v, self._k_exp, self._v_exp = k, v, k_exp, v_exp
        self._tensors = (k, v) if k_exp is None else (k, v, k_exp, v_exp)
        self.desc = nat.KVCacheDesc(code, k.shape[1], k.shape[2], k.shape[0], k.data_ptr(), v.data_ptr(),
                                    None if k_exp is None else k_exp.data_ptr(),
                                    None if v_exp is None else v_exp.data_ptr())

    def _rows(self, t: torch.Tensor, name: str, heads: Optional[int] = None):
        shape = t.shape
        if len(shape) != 3 or shape[2] != HEAD_DIM or (heads is not None and shape[1] != heads) or \
                (t.stride(2) != 1 and t.numel()):
            raise nat.NativeError(f"PagedKVCache: {name} {tuple(shape)} must be (rows, "
                                  f"{heads if heads is not None else 'heads'}, {HEAD_DIM}) with a contiguous head dim")
        if t.device != self._k.device:
            raise nat.NativeError(f"PagedKVCache: {name} is on {t.device}, the pages on {self._k.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise nat.NativeError(f"PagedKVCache: {name} needs a gradient, and none passes through the cache "
                                  "(torch.no_grad() or detach())")
        if nat.has_tangent(t):
            raise nat.NativeError(f"PagedKVCache: {name} carries a forward-mode derivative, and none passes through the "
                                  "cache")

    def _out(self, t: torch.Tensor, name: str, heads: int):
        self._rows(t, name, heads)
        if (t.shape[0] > 1 and t.stride(0) == 0) or (heads > 1 and t.stride(1) == 0):
            raise nat.NativeError(f"PagedKVCache: {name} is expanded: its rows share memory")
        increment_version(t)  # autograd sees that the tensor is written

    def _same(self, batch: KVBatch):
        if batch._table.device != self._k.device:
            raise nat.NativeError(f"PagedKVCache: the batch is on {batch._table.device}, the pages on {self._k.device}")
        if (self._k.requires_grad or self._v.requires_grad) and torch.is_grad_enabled():
            raise nat.NativeError("PagedKVCache: the pages need a gradient, and none passes through the cache "
                                  "(torch.no_grad() or detach())")
        if nat.has_tangent(self._k, self._v):
            raise nat.NativeError("PagedKVCache: the pages carry a forward-mode derivative, and none passes through the "
                                  "cache")

    def write(self, k: torch.Tensor, v: torch.Tensor, batch: KVBatch):
        """The batch's new keys and values (rows, heads, 64), fp32, bf16 or fp16, into their pages.  Rows behind the
        last sequence are not read.  Pages that two sequences share, or that stand twice in one sequence's table, must lie
        before what is written (two tokens would take one place, in no order)."""
        heads = self._k.shape[1]
        self._rows(k, "k", heads)
        self._rows(v, "v", heads)
        self._same(batch)
        if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
            raise nat.NativeError("PagedKVCache: k and v must have the same rows and dtype")
        increment_version(self._tensors)  # autograd sees that they are written
        with nat.on_device(self._k.device):
            nat.kv_cache_write(self.desc, batch._rows(k.shape[0]), k, v)

    def read(self, batch: KVBatch, cu_rows: torch.Tensor, rows: int, dtype: torch.dtype = torch.bfloat16, out=None):
        """(k, v), (rows, heads, 64) each: positions 0, 1, ... of sequence b in the rows cu_rows[b] .. cu_rows[b + 1] -
        1, positions past kv_lens[b] as zeros; rows behind the last sequence stay as they are in `out`, a (k, v) pair of
        tensors that share nothing."""
        self._same(batch)
        _int32(cu_rows, "PagedKVCache: cu_rows", 1)
        if cu_rows.shape[0] != batch._cu_new.shape[0] or cu_rows.device != self._k.device:
            raise nat.NativeError(f"PagedKVCache: cu_rows {tuple(cu_rows.shape)} does not fit the batch")
        heads = self._k.shape[1]
        if out is None:
            shape = (rows, heads, HEAD_DIM)
            k, v = self._k.new_empty(shape, dtype=dtype), self._k.new_empty(shape, dtype=dtype)
        else:
            k, v = out
            for t, name in ((k, "k"), (v, "v")):
                self._out(t, name, heads)
                if t.shape[0] != rows or t.dtype != k.dtype:
                    raise nat.NativeError(f"PagedKVCache: out must hold {rows} rows of one dtype")
        with nat.on_device(self._k.device):
            nat.kv_cache_read(self.desc, batch.desc, cu_rows, rows, k, v)
        return k, v

    def attend(self, q: torch.Tensor, batch: KVBatch, *, mask_block: int = 0, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of the batch's new tokens q (rows, query heads, 64), bf16 or fp16, over their sequences' pages,
        which hold the new tokens' keys and values already.  Query heads are a multiple of the cache's heads (query
        head h reads head h // (query heads // heads)).  mask_block: 0, a token sees its whole sequence; n, it sees up
        to the end of its block of n positions (1: causal; tokens per view: each view itself and the earlier ones).
        scale: 1/8 by default (None or 0).  out may be q itself, otherwise it must not overlap it.  No gradient passes.
        A token that sees nothing gets zeros and an lse of -inf; rows behind the last sequence are left as they are.
        return_lse: also (query heads, rows) fp32 log-sum-exp, as `_native.attn_merge` takes it."""
        self._rows(q, "q")
        self._same(batch)
        if not 0 <= mask_block < 1 << 31:
            raise nat.NativeError(f"PagedKVCache: mask_block {mask_block} must be 0 to 2^31 - 1")
        if scale and not 2.0 ** -149 <= scale < 1e30:  # (less is fp32's zero, which means the default)
            raise nat.NativeError(f"PagedKVCache: scale {scale} must be positive, 2^-149 to 1e30, or None")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            self._out(out, "out", q.shape[1])
            if out.shape[0] != q.shape[0] or out.dtype != q.dtype:
                raise nat.NativeError("PagedKVCache: out must have q's shape and dtype")
        lse = q.new_empty(q.shape[1], q.shape[0], dtype=torch.float32) if return_lse else None
        with nat.on_device(self._k.device):
            nat.attention_paged(self.desc, batch._rows(q.shape[0]), q, out, lse=lse, scale=scale, mask_block=mask_block)
        return (out, lse) if return_lse else out
