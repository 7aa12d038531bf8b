"""RoPE-2D of uniception's croco library (uniception/models/libs/croco/pos_embed.py:101-155 and its CUDA twin
curope/curope2d.py + kernels.cu:17-82) on MI355X: the rotation runs in the gfx950 kernel `mapa_rope2d`
(include/mapa.h), in place on the caller's tensor as cuRoPE2D does.  No CPU path: a missing library or device
raises (mapanything._native).

    rope = RoPE2D(freq=100.0, F0=1.0)
    q = rope(q, positions)     # q (B, heads, N, D) bf16/fp32 on the GPU, positions (B, N, 2) int64 (y, x)
"""

import struct

import torch

from mapanything import _native as nat


class RoPE2D:
    """Same constructor and forward contract as the reference's RoPE2D / cuRoPE2D (pos_embed.py:109-155,
    curope2d.py:31-40): tokens (B, H, N, D) with D % 16 == 0 (the reference asserts D % 2; the kernel's 4-wide
    lanes need D/4 % 4 == 0, true for every head width the models use), positions (B, N, 2) integer (y, x).
    The rotation is applied in place (the head dim must be contiguous) and the tensor is returned."""

    def __init__(self, freq: float = 100.0, F0: float = 1.0):
        self.base = float(freq)
        self.F0 = float(F0)

    def __call__(self, tokens: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        return self.forward(tokens, positions)

    def forward(self, tokens: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        assert tokens.size(3) % 2 == 0, "number of dimensions should be a multiple of two"
        assert positions.ndim == 3 and positions.shape[-1] == 2  # Batch, Seq, 2
        B, H, N, D = tokens.shape
        if positions.shape[:2] != (B, N):
            raise ValueError(f"positions {tuple(positions.shape)} do not match tokens (B={B}, N={N})")
        if tokens.stride(3) != 1:
            raise ValueError("RoPE2D: the head dimension must be contiguous")
        pos = positions.to(device=tokens.device, dtype=torch.int64).contiguous()
        nat.rope2d(tokens, pos, B, H, N, D, tokens.stride(0), tokens.stride(1), tokens.stride(2), self.base, self.F0)
        return tokens


cuRoPE2D = RoPE2D  # curope2d.py:31: the CUDA class the reference prefers when its extension is built


class _RoPEAxesTurn(torch.autograd.Function):
    """One turn of one or two tensors, out of place; linear in them, so its forward-mode derivative is the same turn of
    the tangents, and its backward the turn of the gradients the other way."""

    @staticmethod
    def forward(ctx, rope, inverse, positions, tokens, keys, still=None):  # still: the output that needs no gradient
        ctx.rope, ctx.inverse = rope, inverse
        ctx.shapes = [None if t is None else t.shape for t in (tokens, keys)]
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.set_materialize_grads(False)
        out = rope._turn(tokens, keys, positions, inverse)
        if still is not None:
            ctx.mark_non_differentiable(out[still])
        return out

    @staticmethod
    def backward(ctx, g_tokens, g_keys=None):
        (positions,) = ctx.saved_tensors
        return (None, None, None) + ctx.rope._turn_given(g_tokens, g_keys, positions, not ctx.inverse) + (None,)

    @staticmethod
    def jvp(ctx, _rope, _inverse, _positions, t_tokens, t_keys, _still=None):
        (positions,) = ctx.saved_tensors
        out = ctx.rope._turn_given(t_tokens, t_keys, positions, ctx.inverse)
        given = t_tokens if t_tokens is not None else t_keys
        return tuple(given.new_zeros(s) if y is None and s is not None else y for y, s in zip(out, ctx.shapes))


class RoPEAxes:
    """Rotary positions with several axes (time, row, column, ...): RoPE2D's rotation for any split of the head's pairs
    over up to four axes, differentiable, on the gfx950 kernel `mapa_rope_axes` (include/mapa.h).  RoPE2D is
    `RoPEAxes((D // 4, D // 4), freq)`.

        rope = RoPEAxes(sections=(8, 12, 12), freq=10000.0)     # 32 pairs: time, row, column
        q, k = rope(q, positions, k)                            # (B, heads, N, 64) each, positions (B, N, 3)

    sections: pairs per axis; dims behind the last pair pass through.  layout: the columns of a pair (u, v) —
    "axial" (each axis' own block [u | v], RoPE2D's), "half" (u in the first half of the rotated dims, v in the second)
    or "interleaved" (neighbours).  spectrum: pair j of an axis of n pairs turns by F0 / freq^(j / n) per unit of
    position ("axis", RoPE2D's), or one table runs through the pairs of all axes ("shared").

    tokens / keys: (B, H, N, D) fp32, bf16 or fp16 with a contiguous head dim and any other strides (a view of packed
    qkv rows), the head counts of the two may differ.  positions: (B, N, axes) or (N, axes), integer or fp32; angles are
    formed in 64 bits.  Returns new tensors, or with inplace=True (not for tensors that need a gradient or carry a
    forward-mode derivative, nor for two that share elements) the rotated inputs, as RoPE2D does.  Differentiable in
    both modes, any number of times; not in the positions, and not under torch.func's transforms, which raise."""

    _LAYOUTS = {"axial": nat.ROPE_AXIAL, "half": nat.ROPE_HALF, "interleaved": nat.ROPE_INTERLEAVED}

    def __init__(self, sections, freq: float = 100.0, F0: float = 1.0, layout: str = "axial", spectrum: str = "axis"):
        sections = tuple(int(n) for n in sections)
        if not 1 <= len(sections) <= nat.ROPE_MAX_AXES or min(sections) < 1 or sum(sections) > nat.ROPE_MAX_PAIRS:
            raise ValueError(f"RoPEAxes: sections {sections} must be 1 to {nat.ROPE_MAX_AXES} positive pair counts, "
                             f"{nat.ROPE_MAX_PAIRS} pairs at most")
        if layout not in self._LAYOUTS:
            raise ValueError(f"RoPEAxes: layout must be one of {sorted(self._LAYOUTS)}, got {layout!r}")
        if spectrum not in ("axis", "shared"):
            raise ValueError(f"RoPEAxes: spectrum must be 'axis' or 'shared', got {spectrum!r}")
        if not float(freq) > 0:
            raise ValueError(f"RoPEAxes: freq must be positive, got {freq}")
        self.sections, self.base, self.F0 = sections, float(freq), float(F0)
        self.layout, self.spectrum = layout, spectrum
        self._pairs = pairs = sum(sections)
        if spectrum == "axis":
            part = [j / n for n in sections for j in range(n)]
        else:
            part = [i / pairs for i in range(pairs)]
        d = nat.RopeAxesDesc(axes=len(sections), layout=self._LAYOUTS[layout])
        for i, n in enumerate(sections):
            d.section[i] = n
        for i, x in enumerate(part):
            d.freq[i] = self.F0 * self.base ** -x
        self._desc = d

    def __call__(self, tokens, positions, keys=None, inplace: bool = False):
        return self.forward(tokens, positions, keys, inplace)

    def forward(self, tokens, positions, keys=None, inplace: bool = False):
        self._check(tokens, "tokens")
        B, _, N, D = tokens.shape
        if keys is not None:
            self._check(keys, "keys")
            b, _, n, d = keys.shape
            if b != B or n != N or d != D or keys.dtype != tokens.dtype or keys.device != tokens.device:
                raise ValueError("RoPEAxes: tokens and keys must share device, dtype, batch, length and head dim")
        if positions.ndim == 2:
            positions = positions[None]
        if positions.ndim != 3 or positions.shape[0] not in (1, B) or positions.shape[1] != N or \
                positions.shape[2] != len(self.sections):
            raise ValueError(f"RoPEAxes: positions {tuple(positions.shape)} do not match tokens (B={B}, N={N}) and "
                             f"{len(self.sections)} axes")
        if positions.dtype != torch.int64 and positions.dtype != torch.float32:
            if positions.is_floating_point() or positions.is_complex() or positions.dtype == torch.bool:
                raise ValueError(f"RoPEAxes: positions must be integer or fp32, got {positions.dtype}")
            positions = positions.to(torch.int64)
        if positions.requires_grad and torch.is_grad_enabled():
            raise ValueError("RoPEAxes: no gradient passes to the positions")
        if positions.device != tokens.device:
            positions = positions.to(tokens.device)
        if nat.has_tangent(positions):
            raise ValueError("RoPEAxes: no forward-mode derivative passes from the positions")
        tangent = nat.has_tangent(tokens, keys)
        needs = tangent or (torch.is_grad_enabled() and (tokens.requires_grad or (keys is not None and keys.requires_grad)))
        if inplace:
            if needs:
                raise ValueError("RoPEAxes: inplace rotation of a tensor that needs a gradient or has a forward-mode "
                                 "derivative")
            for t in (tokens, keys):
                if t is not None and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
                    raise ValueError("RoPEAxes: inplace rotation of an expanded tensor")
            if keys is not None and keys.numel() and keys.data_ptr() == tokens.data_ptr():
                raise ValueError("RoPEAxes: inplace rotation of one tensor as tokens and keys")
            for t in (tokens, keys):
                if t is not None:
                    torch.autograd.graph.increment_version(t)  # autograd sees that the tensor is written
            self._run(tokens, keys, positions, False, tokens, keys)
            return tokens if keys is None else (tokens, keys)
        if needs:
            still = None  # keys that need no gradient come back so beside tokens that do, and the other way round
            if not tangent and keys is not None and tokens.requires_grad != keys.requires_grad:
                still = 1 if tokens.requires_grad else 0
            out = _RoPEAxesTurn.apply(self, False, positions.detach(), tokens, keys, still)
        else:
            out = self._turn(tokens, keys, positions, False)
        return out[0] if keys is None else out

    def _turn_given(self, tokens, keys, positions, inverse):
        """The turns of two gradients or tangents, either of which may be missing, differentiable themselves."""
        first, second = (tokens, keys) if tokens is not None else (keys, None)
        if first is None:
            return None, None
        if torch.is_grad_enabled() or nat.has_tangent(first, second):  # a second derivative is asked for
            a, b = _RoPEAxesTurn.apply(self, inverse, positions, first, second)
        else:
            a, b = self._turn(first, second, positions, inverse)
        return (a, b) if tokens is not None else (None, a)

    def _check(self, t, name):
        if t.ndim != 4 or 2 * self._pairs > t.shape[3]:
            raise ValueError(f"RoPEAxes: {name} {tuple(t.shape)} must be (B, H, N, D) with D >= {2 * self._pairs}")
        if t.stride(3) != 1 and t.shape[3] > 1:
            raise ValueError("RoPEAxes: the head dimension must be contiguous")

    def _turn(self, tokens, keys, positions, inverse):
        a = tokens if tokens.stride(3) == 1 else tokens.contiguous()  # a gradient may come expanded
        b = keys if keys is None or keys.stride(3) == 1 else keys.contiguous()
        ya, yb = _like(a), None if b is None else _like(b)
        self._run(a, b, positions, inverse, ya, yb)
        return ya, yb

    def _run(self, a, b, positions, inverse, ya, yb):
        if not a.is_cuda:
            raise nat.NativeError("RoPEAxes: tensors must be on the GPU; there is no CPU path")
        B, H, N, D = a.shape
        sa, ta, sp = a.stride(), ya.stride(), positions.stride()
        if b is None:
            second, sb, tb = (0, 0, 0), (0, 0, 0), (0, 0, 0)
        else:
            second, sb, tb = (b.data_ptr(), yb.data_ptr(), b.shape[1]), b.stride(), yb.stride()
        d = nat.RopeAxesDesc.from_buffer_copy(self._desc)
        # the fields from dtype to pos_astride in one packing (setting them one by one costs more than the launch)
        _DESC_HEAD.pack_into(d, 0, nat.dt_code(a.dtype), B, N, D, a.data_ptr(), second[0], ya.data_ptr(), second[1], H,
                             second[2], sa[0], sb[0], sa[1], sb[1], sa[2], sb[2], ta[0], tb[0], ta[1], tb[1], ta[2],
                             tb[2], positions.data_ptr(),
                             nat.POS_F32 if positions.dtype == torch.float32 else nat.POS_I64,
                             sp[0] if positions.shape[0] > 1 else 0, sp[1], sp[2])
        d.inverse = int(inverse)
        with nat.on_device(a.device):
            nat.rope_axes(d)


# include/mapa.h mapa_rope_axes_desc up to pos_astride: 4 ints, x, y, heads, 12 strides, positions, pos_dtype, 3 strides
_DESC_HEAD = struct.Struct("=4i4Q2i12qQi4x3q")


def _like(x):
    """An empty (B, H, N, D) tensor laid out as x is: heads inside tokens, or tokens inside heads."""
    B, H, N, D = x.shape
    if x.stride(1) < x.stride(2):
        return x.new_empty_strided((B, H, N, D), (N * H * D, D, H * D, 1))
    return x.new_empty((B, H, N, D))
