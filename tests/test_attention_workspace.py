"""mapa_attention's workspace does not depend on which 16-bit type asks for it first: a buffer kept per stream that an
fp16 call had sized (to nothing) left every later bf16 call on that stream without the split of its last wave, so that a
bf16 forward's roundings depended on what its stream had run before."""

import ctypes

import pytest
import torch


@pytest.mark.parametrize("code,split", [("BF16", True), ("F16", True), ("F32", False)])
def test_workspace_size_by_type(code, split):
    from mapanything import _native as nat

    L = nat.load_library()
    d = nat.AttnDesc(dtype=getattr(nat, code), batch=1, heads=12, seq_q=1370, seq_kv=1370)
    b = nat.AttnDesc(dtype=nat.BF16, batch=1, heads=12, seq_q=1370, seq_kv=1370)
    want = L.mapa_attention_workspace_bytes(ctypes.byref(b)) if split else 0
    assert L.mapa_attention_workspace_bytes(ctypes.byref(d)) == want and (want > 0) == split


@pytest.mark.gpu
def test_bf16_after_fp16_on_a_new_stream():
    from mapanything import _native as nat

    S, H = 700, 12
    C = H * 64
    qkv = torch.randn(S, 3 * C, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")

    def run(dtype):
        x = qkv.to(dtype)
        o = torch.empty(S, C, device="cuda", dtype=dtype)
        nat.attention(x, x[:, C:], x[:, 2 * C:], o, batch=1, heads=H, seq_q=S, seq_kv=S, q_bstride=0, q_rstride=3 * C,
                      k_bstride=0, k_rstride=3 * C, v_bstride=0, v_rstride=3 * C, o_bstride=0, o_rstride=C)
        return o

    outs = []
    kept = dict(nat._AWS)  # (captured graphs of other callers may hold these buffers)
    try:
        for first in (torch.float16, torch.bfloat16):
            nat._AWS.clear()
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                run(first)
                outs.append((run(torch.bfloat16), run(torch.float16)))
            torch.cuda.synchronize()
    finally:
        nat._AWS.clear()
        nat._AWS.update(kept)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
