"""Calls of the language-model operators at their edges, on the CPU: what unseen places hold, what a plain call
keeps, limits that are refused."""
import math

import pytest
import torch

import lm_oracle as O
from tensorflow_k8s_amd.ops import loss as L
from tensorflow_k8s_amd.ops import transformer as TR
from test_lm_ops_cpu import i32, randn


@pytest.mark.parametrize("mask", [
    dict(kv_len=[0, 5]), dict(causal=True, q_start=[-3, 4], Sq=4), dict(causal=True, q_start=[0, 2], Sq=3),
    dict(causal=True, doc_ids=[[4, 4, 4, 1, 1, 4, 4, -1, -1], [-1, 0, 0, 0, 0, 7, 7, 7, 7]]),
    dict(causal=True, prefix_len=[0, 3], kv_len=[7, 2]),
])
@pytest.mark.parametrize("hold", [math.nan, math.inf])
def test_attention_unseen_places_hold_anything(mask, hold):
    """Queries that see nothing and keys that no query sees reach neither the output nor a gradient."""
    kw = dict(mask)
    B, H, Hk, Sk, Sq = 2, 4, 2, 9, kw.pop("Sq", 9)
    ids = i32(kw.pop("doc_ids")) if "doc_ids" in kw else None
    kw = {n: i32(v) if n != "causal" else v for n, v in kw.items()}
    q, k, v = randn(B, Sq, H, 64, seed=1), randn(B, Sk, Hk, 64, seed=2), randn(B, Sk, Hk, 64, seed=3)
    dout = randn(B, Sq, H, 64, seed=4)
    ok, pos = O.visible(B, Sq, Sk, kw.get("causal", False), kw.get("kv_len"), kw.get("q_start"), kw.get("prefix_len"), ids)
    blind, unseen = ~ok.any(2), ~ok.any(1)
    assert blind.any() or unseen.any()
    q[blind], dout[blind], k[unseen], v[unseen] = hold, hold, hold, hold
    sp = TR.AttnSpec(B, H, Sq, Sk, (q.view(B * Sq, -1), 0), (k.view(B * Sk, -1), 0), (v.view(B * Sk, -1), 0), kv_heads=Hk,
                     docs=TR.document_spans(ids) if ids is not None else None, softcap=6.0, **kw)
    out, lse = TR.attention_fwd(sp)
    g = [torch.empty_like(t[0]) for t in (sp.q, sp.k, sp.v)]
    TR.attention_bwd(sp, out, dout.view(B * Sq, -1), lse, *((x, 0) for x in g))
    r = O.attention(q, k, v, ok, pos, sp.scale, 6.0, None, dout)
    O.within(out.view(r["out"].shape), r["out"], r["out_bound"], "out")
    for n, x in zip(("dq", "dk", "dv"), g):
        O.within(x.view(r[n].shape), r[n], r[n + "_bound"], n)
    assert bool((lse.permute(0, 2, 1)[blind] == math.inf).all())


@pytest.mark.parametrize("kw", [dict(softcap=1e-46), dict(softcap=1e39), dict(softcap=1.0, scale=1e-46), dict(softcap=1.0, scale=1e39),
                                dict(softcap=math.nan), dict(softcap=1.0, scale=math.nan)])
def test_attention_refuses_what_float32_does_not_hold(kw):
    """(1e-46 is 0 and 1e39 infinite in float32)"""
    q = randn(16, 128)
    with pytest.raises(ValueError):
        TR.AttnSpec(2, 2, 8, 8, (q, 0), (q, 0), (q, 0), **kw)


def test_plain_3d_buffers_and_types_keep_the_plain_form():
    """Without the new arguments contiguous [B, S, width] buffers and, on the CPU, any type are the plain form: its
    results, its types, its arguments (a negative scale, a kv_len of more than B)."""
    x = randn(2 * 8, 384)
    want = TR.attention_fwd(TR.AttnSpec(2, 2, 8, 8, (x, 0), (x, 128), (x, 256), causal=True, scale=-0.1))
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        for buf in (x.to(dt), x.to(dt).view(2, 8, 384)):
            sp = TR.AttnSpec(2, 2, 8, 8, (buf, 0), (buf, 128), (buf, 256), causal=True, scale=-0.1)
            assert not sp.shaped
            out, lse = TR.attention_fwd(sp)
            assert out.dtype == torch.bfloat16 and torch.equal(out, want[0]) and torch.equal(lse, want[1])
            d = torch.empty_like(buf)
            TR.attention_bwd(sp, out, out, lse, (d, 0), (d, 128), (d, 256))
            assert torch.isfinite(d).all()
    y = x.view(16, 2, 192)[:, 0, :128].contiguous().view(16, 2, 64)  # heads apart: the CPU form takes it
    assert not TR.AttnSpec(2, 2, 8, 8, (y, 0), (y, 0), (y, 0)).shaped
    room = torch.zeros(2, 9, 384, dtype=torch.bfloat16)
    assert TR.AttnSpec(2, 2, 8, 8, (room, 0), (room, 128), (room, 256)).shaped
    assert TR.AttnSpec(2, 2, 8, 8, *((room[:, :8], c) for c in (0, 128, 256))).shaped
    h = x.half()
    sp = TR.AttnSpec(2, 2, 8, 8, (h, 0), (h, 128), (h, 256), kv_heads=2)
    assert sp.shaped and TR.attention_fwd(sp)[0].dtype == torch.float16


@pytest.mark.parametrize("ignore", [2 ** 32 + 5, -2 ** 40 + 7, 2 ** 33])
def test_logprobs_ignore_index_outside_int32(ignore):
    """(modulo 2^32 these are 5, 7 and 0)"""
    x, ids = randn(4, 50, dtype=torch.float32), i32([5, 5, 7, 0])
    w, r = L.token_logprobs(x, ids), L.token_logprobs(x, ids, ignore_index=ignore)
    assert torch.equal(r.logp, w.logp) and r.logp.all()
    g = torch.ones(4)
    assert torch.equal(L.token_logprobs_bwd(x, ids, r, g, ignore_index=ignore), L.token_logprobs_bwd(x, ids, w, g))
