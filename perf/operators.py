"""Cases for timing the streaming operators: rotary positions with several axes, the paged K/V cache's write and read
back, and attention of new tokens over that cache.  Each case runs in two forms on the same inputs: plain torch
operations (`own` false) and the framework's operators (`own` true).

Head width is 64 throughout, as in the encoder (16 heads) and the multi-view transformer (12 heads); a 518 x 518 view
is 37 x 37 = 1369 tokens, 1370 with one extra token per view.
"""

import functools
import math
import os
import random
import sys

import torch

own = False

HEAD = 64
VIEW = 1370  # tokens of one view with its extra token
GRID = 37  # patches per side of a 518 x 518 view
CODE_MAX = {"fp8": 448.0, "int8": 127.0}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one new token in each of 16 running scenes, far into the capture: launch-bound
        {"name": "rope_step", "op": "rope", "batch": 16, "tokens": 1, "q_heads": 12, "k_heads": 12, "type": "bf16",
         "layout": "axial", "spectrum": "axis", "sections": "8,12,12", "far": 100000, "grad": False},
        # queries and keys of one 8-view chunk of a global layer, (time, row, column) positions
        {"name": "rope_views", "op": "rope", "batch": 1, "tokens": 8 * VIEW, "q_heads": 12, "k_heads": 12,
         "type": "bf16", "layout": "axial", "spectrum": "axis", "sections": "8,12,12", "far": 1000, "grad": False},
        # a training step's rotation and its gradient in fp32, two scenes, 16 heads, odd sections, one table of
        # frequencies shared by the axes
        {"name": "rope_train", "op": "rope", "batch": 2, "tokens": 2 * VIEW + 1, "q_heads": 16, "k_heads": 16,
         "type": "f32", "layout": "half", "spectrum": "shared", "sections": "10,11,11", "far": 4000, "grad": True},
        # queries and keys of a 100-view scene
        {"name": "rope_scene", "op": "rope", "batch": 1, "tokens": 100 * VIEW, "q_heads": 12, "k_heads": 12,
         "type": "bf16", "layout": "axial", "spectrum": "axis", "sections": "8,12,12", "far": 1000, "grad": False},
        # one token in each of 32 scenes goes into an e4m3 cache and the latest 64 rows are read back
        {"name": "cache_step_fp8", "op": "cache", "seqs": 32, "new": 1, "old": 63, "ragged": 0, "heads": 12,
         "page": 64, "pages": "fp8", "type": "bf16"},
        # a 1370-token view goes into each of 4 scenes' 16-bit pages, read back whole
        {"name": "cache_view_bf16", "op": "cache", "seqs": 4, "new": VIEW, "old": 7 * VIEW, "ragged": 3, "heads": 12,
         "page": 64, "pages": "bf16", "type": "bf16"},
        # ragged chunks of 16-head scenes in small pages, 8-bit integer codes
        {"name": "cache_ragged_int8", "op": "cache", "seqs": 13, "new": 2 * VIEW, "old": 4 * VIEW, "ragged": 5,
         "heads": 16, "page": 16, "pages": "int8", "type": "bf16"},
        # one token over one 8-view scene: latency
        {"name": "attend_step", "op": "attend", "seqs": 1, "new": 1, "old": 8 * VIEW - 1, "ragged": 0, "q_heads": 12,
         "k_heads": 12, "page": 64, "pages": "bf16", "type": "bf16", "block": 0},
        # one token in each of 64 scenes of very different lengths, grouped heads, e4m3 pages
        {"name": "attend_steps_fp8", "op": "attend", "seqs": 64, "new": 1, "old": 24 * VIEW, "ragged": 7,
         "q_heads": 16, "k_heads": 4, "page": 64, "pages": "fp8", "type": "bf16", "block": 0},
        # ragged causal chunks in fp16 over int8 pages
        {"name": "attend_causal_int8", "op": "attend", "seqs": 5, "new": 700, "old": 6 * VIEW, "ragged": 11,
         "q_heads": 16, "k_heads": 16, "page": 32, "pages": "int8", "type": "f16", "block": 1},
        # an 8-view chunk, each view seeing itself and all earlier ones
        {"name": "attend_views", "op": "attend", "seqs": 1, "new": 8 * VIEW, "old": 8 * VIEW, "ragged": 0,
         "q_heads": 12, "k_heads": 12, "page": 64, "pages": "bf16", "type": "bf16", "block": VIEW},
        # one view over a 100-view scene
        {"name": "attend_scene", "op": "attend", "seqs": 1, "new": VIEW, "old": 99 * VIEW, "ragged": 0,
         "q_heads": 12, "k_heads": 12, "page": 64, "pages": "bf16", "type": "bf16", "block": 0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attend", "attend"])
    if op == "rope":
        layout = rng.choice(["axial", "half", "interleaved"])
        kind = rng.choice(["bf16", "bf16", "f16", "f32"])
        heads = rng.choice([(12, 12), (16, 16), (16, 4), (12, 1)])
        grad = rng.random() < 0.4
        room = 100 * VIEW * 24 // (sum(heads) * (2 if kind == "f32" else 1) * (2 if grad else 1))
        batch = _spread(rng, 1, 64)
        return {"op": "rope", "batch": batch, "tokens": _spread(rng, 1, max(1, room // batch)), "q_heads": heads[0],
                "k_heads": heads[1], "type": kind, "layout": layout, "spectrum": rng.choice(["axis", "shared"]),
                "sections": rng.choice(["8,12,12", "16,16", "10,11,11", "32", "8,8,8", "4,8,8,12"]),
                "far": _spread(rng, 40, 1000000), "grad": grad}
    if op == "cache":
        heads = rng.choice([1, 4, 12, 16])
        room = 280000 * 16 // heads
        seqs = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(1, min(3 * VIEW, room // (4 * seqs))))
        return {"op": "cache", "seqs": seqs, "new": new, "old": _spread(rng, 1, max(1, min(40 * VIEW, room // seqs))),
                "ragged": rng.randrange(1, 1000), "heads": heads, "page": rng.choice([16, 32, 64, 128]),
                "pages": rng.choice(["bf16", "f16", "fp8", "int8"]), "type": rng.choice(["bf16", "f16"])}
    q_heads, k_heads = rng.choice([(12, 12), (16, 16), (16, 4), (16, 1), (12, 4), (6, 2)])
    kind = rng.choice(["bf16", "bf16", "f16"])
    pages = rng.choice([kind, "fp8", "int8"])
    page = rng.choice([16, 32, 64, 128])
    if rng.random() < 0.5:  # single tokens, or a few
        seqs = _spread(rng, 1, 64)
        return {"op": "attend", "seqs": seqs, "new": rng.choice([1, 1, 1, 2, 5]),
                "old": _spread(rng, 1, min(100 * VIEW, 2400000 // (seqs * k_heads))), "ragged": rng.randrange(1, 1000),
                "q_heads": q_heads, "k_heads": k_heads, "page": page, "pages": pages, "type": kind, "block": 1}
    seqs = _spread(rng, 1, 8)
    new = _spread(rng, 6, 2 * VIEW)
    old = _spread(rng, 1, max(2, 100 * VIEW * VIEW * 12 // (seqs * new * q_heads * 2)))
    return {"op": "attend", "seqs": seqs, "new": new, "old": min(old, 60 * VIEW), "ragged": rng.randrange(1, 1000),
            "q_heads": q_heads, "k_heads": k_heads, "page": page, "pages": pages, "type": kind,
            "block": rng.choice([0, 1, 37, VIEW])}


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence: `new` and `old` at most, much shorter ones among
    them where the case is ragged."""
    if not case["ragged"]:
        return [case["new"]] * case["seqs"], [case["old"] + case["new"]] * case["seqs"]
    rng = random.Random(case["ragged"])
    new = [max(1, int(case["new"] * (1 if i == 0 else rng.uniform(0.05, 1)))) for i in range(case["seqs"])]
    old = [int(case["old"] * (1 if i == case["seqs"] - 1 else rng.uniform(0.02, 1))) for i in range(case["seqs"])]
    return new, [a + b for a, b in zip(old, new)]


def _limit_pairs(new, total, block):
    """Query-key pairs of one sequence: a query at position p sees the keys below the end of its block."""
    if block == 0:
        return new * total
    first = total - new
    return sum(min(total, (p // block + 1) * block) for p in range(first, total))


def work(case):
    if case["op"] == "rope":
        rows = case["batch"] * case["tokens"]
        values = rows * (case["q_heads"] + case["k_heads"]) * HEAD
        size = TYPES[case["type"]].itemsize
        passes = 2 if case["grad"] else 1
        axes = len(case["sections"].split(","))
        return {"bytes": passes * (2 * values * size + rows * axes * 8), "flops": passes * 3 * values}
    new, total = _lengths(case)
    page_row = HEAD * PAGE_TYPES[case["pages"]].itemsize + (1 if case["pages"] in CODE_MAX else 0)
    size = TYPES[case["type"]].itemsize
    if case["op"] == "cache":
        into = 2 * sum(new) * case["heads"] * (HEAD * size + page_row)
        back = 2 * sum(total) * case["heads"] * (HEAD * size + page_row)
        return {"bytes": into + back, "flops": 2 * (sum(new) + sum(total)) * case["heads"] * HEAD}
    pairs = sum(_limit_pairs(a, b, case["block"]) for a, b in zip(new, total))
    rows = 2 * sum(new) * case["q_heads"] * HEAD * size + sum(new) * case["q_heads"] * 4
    return {"bytes": rows + 2 * sum(total) * case["k_heads"] * page_row, "flops": 4 * HEAD * case["q_heads"] * pairs}


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(shape, seed, kind):
    """Normal values with a few strong channels, as projections give them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    x[..., ::13] *= 1.7
    return x.to(TYPES[kind])


def _quantise(x, pages):
    """(codes, exponent bytes): the least power of two that brings a row's largest value within the codes' range."""
    largest = x.abs().amax(-1).clamp_min(2.0 ** -100)
    frac, power = torch.frexp(largest.float())  # largest = frac * 2^power, 0.5 <= frac < 1
    top_frac, top_power = math.frexp(CODE_MAX[pages])
    power = power - top_power + (frac > top_frac).to(power.dtype)
    scaled = torch.ldexp(x.float(), -power[..., None])
    codes = scaled.to(torch.float8_e4m3fn) if pages == "fp8" else scaled.round().to(torch.int8)
    return codes, (power + 127).to(torch.uint8)


def _values(codes, exponents):
    return torch.ldexp(codes.float(), exponents[..., None].int() - 127)


def prepare(case, seed):
    if case["op"] == "rope":
        sections = [int(s) for s in case["sections"].split(",")]
        b, n, heads = case["batch"], case["tokens"], case["q_heads"] + case["k_heads"]
        # queries and keys lie side by side in one buffer of rows, as the projection leaves them
        rows = _normal((b, n, heads, HEAD), seed, case["type"])
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        first = torch.randint(0, max(1, case["far"]), (b, 1, 1), generator=g, device="cuda")
        i = torch.arange(n, device="cuda")
        spread = torch.stack([i // (GRID * GRID), i // GRID % GRID, i % GRID, i % 5], -1)[None].repeat(b, 1, 1)
        spread[..., :1] += first
        state = {"q": rows[:, :, : case["q_heads"]].transpose(1, 2), "k": rows[:, :, case["q_heads"]:].transpose(1, 2),
                 "positions": spread[..., : len(sections)].contiguous(), "sections": sections}
        if case["grad"]:
            up = _normal((b, n, heads, HEAD), seed + 2, case["type"])
            state["gq"] = up[:, :, : case["q_heads"]].transpose(1, 2)
            state["gk"] = up[:, :, case["q_heads"]:].transpose(1, 2)
    else:
        new, total = _lengths(case)
        page, heads = case["page"], case["heads"] if case["op"] == "cache" else case["k_heads"]
        need = [-(-t // page) for t in total]
        count = sum(need) + 3
        order = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
        table = [[order.pop() for _ in range(c)] + [0] * (max(need) - c) for c in need]
        ints = {"dtype": torch.int32, "device": "cuda"}
        starts = [0]
        for c in new:
            starts.append(starts[-1] + c)
        rows = [0]
        for c in total:
            rows.append(rows[-1] + c)
        state = {"table": torch.tensor(table, **ints), "lens": torch.tensor(total, **ints),
                 "starts": torch.tensor(starts, **ints), "rows": torch.tensor(rows, **ints), "most_new": max(new),
                 "most": max(total), "all_new": starts[-1], "all": rows[-1]}
        state["seq"] = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
        for i, x in enumerate(("k", "v")):
            pages = _normal((count, heads, page, HEAD), seed + 10 + i, "f32")
            if case["pages"] in CODE_MAX:
                state[x + "_pages"], state[x + "_exp"] = _quantise(pages, case["pages"])
            else:
                state[x + "_pages"], state[x + "_exp"] = pages.to(PAGE_TYPES[case["pages"]]), None
            del pages
            if case["op"] == "cache":  # the new rows, out of a projection's (q, k, v) buffer
                both = _normal((starts[-1], 3, heads, HEAD), seed + 20 + i, case["type"])
                state[x] = both[:, 1 + i]
        if case["op"] == "attend":
            state["q"] = _normal((starts[-1], case["q_heads"], HEAD), seed + 30, case["type"])
    state["case"] = dict(case)
    return state


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _rope_own, "cache": _cache_own, "attend": _attend_own}[op](state)
    return {"rope": _rope_plain, "cache": _cache_plain, "attend": _attend_plain}[op](state)


@functools.lru_cache(None)
def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "map-anything_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mapanything.kv_cache import KVBatch, PagedKVCache
    from uniception.models.libs.croco.pos_embed import RoPEAxes

    return RoPEAxes, PagedKVCache, KVBatch


@functools.lru_cache(None)
def _rope_module(sections, layout, spectrum):
    return _package()[0](sections=sections, freq=10000.0, layout=layout, spectrum=spectrum)


def _rope_own(s):
    c = s["case"]
    rope = _rope_module(tuple(s["sections"]), c["layout"], c["spectrum"])
    if not c["grad"]:
        q, k = rope(s["q"], s["positions"], s["k"])
        return {"q": q, "k": k}
    q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
    out_q, out_k = rope(q, s["positions"], k)
    dq, dk = torch.autograd.grad([out_q, out_k], [q, k], [s["gq"], s["gk"]])
    return {"q": out_q.detach(), "k": out_k.detach(), "dq": dq, "dk": dk}


def _pairs(sections, layout, device):
    """Column of u and of v for every pair, axis by axis."""
    u, v, at = [], [], 0
    for n in sections:
        j = torch.arange(n, device=device)
        if layout == "axial":
            u.append(2 * at + j)
            v.append(2 * at + n + j)
        elif layout == "half":
            u.append(at + j)
            v.append(sum(sections) + at + j)
        else:
            u.append(2 * (at + j))
            v.append(2 * (at + j) + 1)
        at += n
    return torch.cat(u), torch.cat(v)


def _turn(x, cos, sin, u, v):
    out = x.float()
    a, b = out[..., u], out[..., v]
    out = out.clone() if out.data_ptr() == x.data_ptr() else out
    out[..., u] = a * cos - b * sin
    out[..., v] = b * cos + a * sin
    return out.to(x.dtype)


def _rope_plain(s):
    c, sections = s["case"], s["sections"]
    u, v = _pairs(sections, c["layout"], s["q"].device)
    axis = torch.repeat_interleave(torch.arange(len(sections), device=u.device), torch.tensor(sections, device=u.device))
    if c["spectrum"] == "axis":
        part = torch.cat([torch.arange(n, dtype=torch.float64, device=u.device) / n for n in sections])
    else:
        part = torch.arange(sum(sections), dtype=torch.float64, device=u.device) / sum(sections)
    angle = s["positions"][..., axis].double() * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=u.device), -part)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = {"q": _turn(s["q"], cos, sin, u, v), "k": _turn(s["k"], cos, sin, u, v)}
    if c["grad"]:
        out["dq"], out["dk"] = _turn(s["gq"], cos, -sin, u, v), _turn(s["gk"], cos, -sin, u, v)
    return out


def _handles(s):
    _, cache, batch = _package()
    return (cache.wrap(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"]),
            batch(s["table"], s["lens"], s["starts"], max_new=s["most_new"], max_kv=s["most"]))


def _cache_own(s):
    cache, batch = _handles(s)
    cache.write(s["k"], s["v"], batch)
    k, v = cache.read(batch, s["rows"], s["all"], dtype=TYPES[s["case"]["type"]])
    return {"k": k, "v": v}


def _cache_plain(s):
    page = s["case"]["page"]
    seq = s["seq"]
    i = torch.arange(s["all_new"], device=seq.device) - s["starts"][seq]
    at = s["lens"][seq] - (s["starts"][seq + 1] - s["starts"][seq]) + i
    where, slot = s["table"][seq, at // page].long(), (at % page).long()
    of = torch.searchsorted(s["rows"], torch.arange(s["all"], device=seq.device, dtype=torch.int32), right=True) - 1
    pos = torch.arange(s["all"], device=seq.device) - s["rows"][of]
    from_page, from_slot = s["table"][of, pos // page].long(), (pos % page).long()
    out = {}
    for x in ("k", "v"):
        pages, exps = s[x + "_pages"], s[x + "_exp"]
        if exps is None:
            pages[where, :, slot] = s[x].to(pages.dtype)
            got = pages[from_page, :, from_slot]
        else:
            codes, power = _quantise(s[x].float(), s["case"]["pages"])
            pages.view(torch.uint8)[where, :, slot] = codes.view(torch.uint8)
            exps[where, :, slot] = power
            got = _values(pages.view(torch.uint8)[from_page, :, from_slot].view(pages.dtype), exps[from_page, :, from_slot])
        out[x] = got.to(TYPES[s["case"]["type"]])
    return out


def _attend_own(s):
    cache, batch = _handles(s)
    out, lse = cache.attend(s["q"], batch, mask_block=s["case"]["block"], return_lse=True)
    return {"out": out, "lse": lse}


def _dense(pages, exps, table):
    """(sequences, heads, places, 64) in fp32 out of the pages."""
    x = pages.view(torch.uint8)[table].view(pages.dtype) if exps is not None else pages[table]
    x = x.float() if exps is None else _values(x, exps[table])
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend_plain(s):
    c = s["case"]
    table, seq = s["table"].long(), s["seq"]
    k, v = _dense(s["k_pages"], s["k_exp"], table), _dense(s["v_pages"], s["v_exp"], table)
    b, heads, places, _ = k.shape
    group = c["q_heads"] // c["k_heads"]
    i = torch.arange(s["all_new"], device=seq.device) - s["starts"][seq]
    q = torch.zeros(b, s["most_new"], c["q_heads"], HEAD, device=k.device)
    q[seq, i] = s["q"].float()
    q = q.view(b, s["most_new"], heads, group, HEAD).permute(0, 2, 1, 3, 4).reshape(b, heads, -1, HEAD)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * 0.125
    new = s["starts"][1:] - s["starts"][:-1]
    at = (s["lens"] - new)[:, None] + torch.arange(s["most_new"], device=k.device)
    end = s["lens"][:, None].expand(-1, s["most_new"])
    if c["block"]:
        end = torch.minimum(end, (at // c["block"] + 1) * c["block"])
    hidden = torch.arange(places, device=k.device) >= end.repeat_interleave(group, 1)[:, None, :, None]
    score.masked_fill_(hidden, float("-inf"))
    most = score.amax(-1, keepdim=True)
    score = score.sub_(most).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score, v) / total
    lse = most + total.log()
    out = out.view(b, heads, s["most_new"], group, HEAD).permute(0, 2, 1, 3, 4).reshape(b, s["most_new"], -1, HEAD)
    lse = lse.view(b, heads, s["most_new"], group).permute(0, 2, 1, 3).reshape(b, s["most_new"], -1)
    return {"out": out[seq, i].to(s["q"].dtype), "lse": lse[seq, i].t().contiguous()}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _rope_exact, "cache": _cache_exact, "attend": _attend_exact}[case["op"]](case, s)


def _rope_exact(case, s):
    """Each pair as a complex number, turned by e^(i p f)."""
    sections, layout = s["sections"], case["layout"]

    def turned(x, sign):
        y = x.double()
        done, at, pairs = y.clone(), 0, sum(sections)
        for a, n in enumerate(sections):
            for j in range(n):
                f = 10000.0 ** (-(j / n if case["spectrum"] == "axis" else (at + j) / pairs))
                angle = sign * s["positions"][:, None, :, a].double() * f
                cu = {"axial": 2 * at + j, "half": at + j, "interleaved": 2 * (at + j)}[layout]
                cv = {"axial": 2 * at + n + j, "half": pairs + at + j, "interleaved": 2 * (at + j) + 1}[layout]
                z = torch.complex(y[..., cu].contiguous(), y[..., cv].contiguous()) * torch.polar(torch.ones_like(angle), angle)
                done[..., cu], done[..., cv] = z.real, z.imag
            at += n
        return done

    out = {"q": turned(s["q"], 1), "k": turned(s["k"], 1)}
    if case["grad"]:
        out["dq"], out["dk"] = turned(s["gq"], -1), turned(s["gk"], -1)
    return out


def _cache_exact(case, s):
    """Sequence by sequence: the old rows as the pages hold them, then the new rows after rounding to the codes."""
    new, total = _lengths(case)
    out = {"k": [], "v": []}
    for x in ("k", "v"):
        done = 0
        for b, (n, t) in enumerate(zip(new, total)):
            ids = s["table"][b, : -(-t // case["page"])].long()
            held = s[x + "_pages"].view(torch.uint8)[ids].view(s[x + "_pages"].dtype).double()
            if s[x + "_exp"] is not None:
                held = held * torch.exp2(s[x + "_exp"][ids].double() - 127)[..., None]
            held = held.transpose(1, 2).flatten(0, 1)[: t - n]
            rows = s[x][done: done + n].double()
            if case["pages"] in CODE_MAX:
                unit = torch.exp2(torch.ceil(torch.log2(rows.abs().amax(-1, keepdim=True) / CODE_MAX[case["pages"]])))
                rows = rows / unit
                if case["pages"] == "int8":
                    rows = rows.round() * unit
                else:  # 3 bits after the leading one, steps of 2^-9 below 2^-6
                    step = torch.exp2(torch.floor(torch.log2(rows.abs().clamp_min(2.0 ** -6))) - 3)
                    rows = (rows / step).round() * step * unit
            else:
                rows = rows.to(PAGE_TYPES[case["pages"]]).double()
            out[x] += [held, rows]
            done += n
        out[x] = torch.cat(out[x])
    return out


def _attend_exact(case, s):
    """One sequence and one head at a time, 4096 queries at most."""
    new, total = _lengths(case)
    group = case["q_heads"] // case["k_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(case["q_heads"], s["all_new"], dtype=torch.float64, device="cuda")
    done = 0
    for b, (n, t) in enumerate(zip(new, total)):
        ids = s["table"][b, : -(-t // case["page"])].long()
        for h in range(case["k_heads"]):
            kv = []
            for x in ("k", "v"):
                held = s[x + "_pages"].view(torch.uint8)[ids, h].view(s[x + "_pages"].dtype).double()
                if s[x + "_exp"] is not None:
                    held = held * torch.exp2(s[x + "_exp"][ids, h].double() - 127)[..., None]
                kv.append(held.flatten(0, 1)[:t])
            for g in range(h * group, (h + 1) * group):
                for r in range(0, n, 4096):
                    m = min(n, r + 4096)
                    score = (s["q"][done + r: done + m, g].double() @ kv[0].t().contiguous()) / 8
                    if case["block"]:
                        p = t - n + torch.arange(r, m, device="cuda")
                        score[torch.arange(t, device="cuda") >= (p[:, None] // case["block"] + 1) * case["block"]] = -math.inf
                    lse[g, done + r: done + m] = torch.logsumexp(score, -1)
                    out[done + r: done + m, g] = torch.softmax(score, -1) @ kv[1]
        done += n
    return {"out": out, "lse": lse}
