"""Plain 64-bit forms of the streaming operators (rotary positions with several axes, the paged K/V cache, attention over
it) and the error bounds that their tests hold the kernels to."""

import math

import torch

CODE_MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def half_step(dtype):
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------- rotary positions
def rope_frequencies(sections, freq, f0, spectrum):
    total = sum(sections)
    if spectrum == "axis":
        return [[f0 * freq ** -(j / n) for j in range(n)] for n in sections]
    out, at = [], 0
    for n in sections:
        out.append([f0 * freq ** -((at + j) / total) for j in range(n)])
        at += n
    return out


def rope_columns(sections, layout):
    u, v, at, total = [], [], 0, sum(sections)
    for n in sections:
        for j in range(n):
            if layout == "axial":
                u.append(2 * at + j)
                v.append(2 * at + n + j)
            elif layout == "half":
                u.append(at + j)
                v.append(total + at + j)
            else:
                u.append(2 * (at + j))
                v.append(2 * (at + j) + 1)
        at += n
    return u, v


def rope(x, positions, sections, freq, f0=1.0, layout="axial", spectrum="axis", inverse=False):
    """x (B, H, N, D), positions (B, N, axes): (rotated x in 64 bits, bound of an fp32 kernel's error).

    The bound: with cosine and sine each within d of the true ones, u c - v s is off by (|u| + |v|) d and by three
    roundings (two products, one sum; an fma makes it two), each 2^-24 of at most |u| + |v|.  d: the fraction of a turn
    is rounded to fp32 (2^-25 of a turn at most 1/2: pi 2^-24 in the angle), and the library's sincospif is within 2 ulp
    (2^-23).  Together under (|u| + |v|) (pi + 2 + 3) 2^-24 < (|u| + |v|) 2^-20."""
    y, p = x.double(), positions.double()
    f = torch.tensor([w for ws in rope_frequencies(sections, freq, f0, spectrum) for w in ws], dtype=torch.float64,
                     device=x.device)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    angle = (p[..., axis] * f)[:, None]
    if inverse:
        angle = -angle
    u, v = rope_columns(sections, layout)
    a, b = y[..., u], y[..., v]
    out, bound = y.clone(), torch.zeros_like(y)
    out[..., u] = a * angle.cos() - b * angle.sin()
    out[..., v] = b * angle.cos() + a * angle.sin()
    bound[..., u] = bound[..., v] = (a.abs() + b.abs()) * 2.0 ** -20
    return out, bound


# ------------------------------------------------------------------------------------------------- the cache
def quantise(rows, dtype):
    """(codes in 64 bits, exponent bytes) of rows (..., 64) by the definition."""
    x = rows.double()
    top = CODE_MAX[dtype]
    bad = ~torch.isfinite(x).all(-1)
    most = torch.where(bad, 1.0, x.abs().amax(-1)).clamp_min(2.0 ** -100)
    e = torch.ceil(torch.log2(most / top))
    e = torch.where(torch.exp2(e - 1) * top >= most, e - 1, e)  # the least e with most <= top 2^e, whatever log2 rounds
    e = torch.where(torch.exp2(e) * top < most, e + 1, e)
    z = x / torch.exp2(e)[..., None]
    if dtype == torch.int8:
        codes = z.round()
    else:
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
        codes = (z / step).round() * step
    codes = torch.where(bad[..., None], math.nan, codes)
    return codes, torch.where(bad, 255.0, e + 127).to(torch.uint8)


def values(codes, exps):
    """What pages of codes and exponents stand for, in 64 bits."""
    out = codes.double() * torch.exp2(exps.double() - 127)[..., None]
    return torch.where(exps[..., None] == 255, math.nan, out)


def page_values(pages, exps):
    return pages.double() if exps is None else values(pages.float() if pages.dtype != torch.int8 else pages, exps)


def sequence_rows(pages, exps, table_row, length):
    """(length, heads, 64) in 64 bits: a sequence's rows out of its pages."""
    size = pages.shape[2]
    ids = table_row[: -(-length // size)].long()
    raw = pages.view(torch.uint8)[ids].view(pages.dtype)
    x = page_values(raw, None if exps is None else exps[ids])
    return x.transpose(1, 2).flatten(0, 1)[:length]


# ------------------------------------------------------------------------------------------------- attention
def limits(new, length, block):
    """Keys that each of a sequence's new tokens sees."""
    out = []
    for p in range(length - new, length):
        out.append(length if block == 0 else 0 if p < 0 else min(length, (p // block + 1) * block))
    return out


def attention(q, k, v, limit, scale):
    """One sequence: q (new, heads, 64), k / v (length, kv_heads, 64) in 64 bits, limit per token.
    -> out (new, heads, 64), lse (heads, new), and the bounds (out, lse) of a kernel that multiplies in 16 bits and sums
    in 32.

    Relative error of one p_j: its score is a sum of 64 exact products in fp32 (64 2^-24 of sum |q k|), scaled, shifted
    (2^-24 of |c s| and of the shift, both under c sum |q k| plus the largest) and exponentiated (2 ulp: 2^-22): d below.
    Numerator and denominator each carry d and the fp32 summation of n terms (n 2^-24, at least 64); the numerator's p is
    rounded to 16 bits once (half a step of the operand's type, relative to each p v, so to the sum of p |v|; in fp16 a
    p under 2^-14 is rounded by 2^-25 at most, n of them against a sum of at least one); the output once more."""
    dt, n = q.dtype, k.shape[0]
    new, heads = q.shape[0], q.shape[1]
    group = heads // k.shape[1] if k.shape[1] else 1
    out = torch.zeros(new, heads, 64, dtype=torch.float64, device=q.device)
    lse = torch.full((heads, new), -math.inf, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    lim = torch.tensor(limit, device=q.device)
    if not n or not new:
        return out, lse, tol, ltol
    hidden = torch.arange(n, device=q.device) >= lim[:, None]
    none = lim <= 0
    for h in range(heads):
        kk, vv, qq = k[:, h // group], v[:, h // group], q[:, h].double()
        kt = kk.t().contiguous()
        s = (qq @ kt * scale).masked_fill(hidden, -math.inf)
        big = (qq.abs() @ kt.abs() * scale).masked_fill(hidden, 0).amax(-1)
        lse[h] = torch.where(none, -math.inf, torch.logsumexp(s.masked_fill(none[:, None], 0), -1))
        p = torch.where(none[:, None], 0.0, torch.exp(s - lse[h][:, None]))
        for r in range(0, new, 2048):  # rows that see different keys: only the seen ones, whatever the others hold
            rows = slice(r, min(new, r + 2048))
            if torch.isfinite(vv).all():
                out[rows, h] = p[rows] @ vv
                a = p[rows] @ vv.abs()
            else:
                terms = torch.where(hidden[rows, :, None], 0.0, p[rows, :, None] * vv)
                out[rows, h], a = terms.sum(1), terms.abs().sum(1)
            d = (big[rows] * (64 + 4) * 2.0 ** -24 + 2.0 ** -21)[:, None]
            total = max(n, 64) * 2.0 ** -24
            half = half_step(dt)
            floor = n * 2.0 ** -25 * torch.where(torch.isfinite(vv), vv, 0.0).abs().max() if dt == torch.float16 else 0.0
            tol[rows, h] = a * (half + 2 * d + 2 * total) + floor + half * out[rows, h].abs()
            if dt == torch.float16:
                tol[rows, h] += 2.0 ** -25  # the output's own smallest steps
            ltol[h, rows] = d[:, 0] + total + 2.0 ** -22 * (1 + lse[h, rows].nan_to_num(0, 0, 0).abs())
    return out, lse, tol, ltol


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = torch.isfinite(want)
    assert torch.isfinite(got[ok]).all(), f"{what}: not finite where it should be"
    over = ((got - want).abs() - tol)[ok]
    assert over.numel() == 0 or over.max() <= 0, \
        f"{what}: off by {(got - want).abs()[ok].max():.3e}, past the bound by {over.max():.3e}"
