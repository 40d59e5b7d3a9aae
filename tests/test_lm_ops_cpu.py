"""Shaped attention, token log probabilities and the sorted embedding gradient on the CPU: the reference
paths against float64 definitions, gradients against differences, and what the entry points refuse."""
import math

import pytest
import torch

import lm_oracle as O
from tensorflow_k8s_amd.ops import loss as L
from tensorflow_k8s_amd.ops import transformer as TR


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def randn(*shape, seed=0, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def spec(B=2, H=4, Hk=2, D=64, Sq=9, Sk=9, dtype=torch.bfloat16, **kw):
    q, k, v = randn(B * Sq, H * D, seed=1, dtype=dtype), randn(B * Sk, Hk * D, seed=2, dtype=dtype), randn(B * Sk, Hk * D, seed=3, dtype=dtype)
    return TR.AttnSpec(B, H, Sq, Sk, (q, 0), (k, 0), (v, 0), kv_heads=Hk, head_dim=D, **kw)


MASKS = [
    dict(causal=True, softcap=5.0),
    dict(causal=True, prefix_len=[0, 6], slopes=True),
    dict(causal=True, doc_ids=[[4, 4, 4, 1, 1, 4, 4, -1, -1], [-1, 0, 0, 0, 0, 7, 7, 7, 7]]),
    dict(kv_len=[0, 5], slopes=True),
    dict(causal=True, q_start=[-3, 4], Sq=4),
]


@pytest.mark.parametrize("mask", MASKS)
def test_attention_reference(mask):
    kw = dict(mask)
    ids = i32(kw.pop("doc_ids")) if "doc_ids" in kw else None
    Sq, H = kw.pop("Sq", 9), 4
    for n in ("prefix_len", "kv_len", "q_start"):
        if n in kw:
            kw[n] = i32(kw[n])
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.01]) if kw.pop("slopes", False) else None
    sp = spec(Sq=Sq, slopes=slopes, docs=TR.document_spans(ids) if ids is not None else None, **kw)
    out, lse = TR.attention_fwd(sp)
    dout = randn(2 * Sq, H * 64, seed=4)
    dq, dk, dv = (torch.empty_like(t[0]) for t in (sp.q, sp.k, sp.v))
    TR.attention_bwd(sp, out, dout, lse, (dq, 0), (dk, 0), (dv, 0))
    ok, pos = O.visible(2, Sq, 9, kw.get("causal", False), kw.get("kv_len"), kw.get("q_start"), kw.get("prefix_len"), ids)
    r = O.attention(sp.q[0].view(2, Sq, H, 64), sp.k[0].view(2, 9, 2, 64), sp.v[0].view(2, 9, 2, 64), ok, pos, sp.scale,
                    sp.softcap, slopes, dout.view(2, Sq, H, 64))
    O.within(out.view(2, Sq, H, 64), r["out"], r["out_bound"], "out")
    fin = torch.isfinite(r["lse"])
    assert torch.equal(fin, torch.isfinite(lse)) and bool((lse[~fin] == math.inf).all())
    assert torch.allclose(lse[fin].double(), r["lse"][fin], atol=1e-5)
    for n, g in (("dq", dq), ("dk", dk), ("dv", dv)):
        O.within(g.view(r[n].shape), r[n], r[n + "_bound"], n)


def test_attention_oracle_gradient_by_differences():
    """The oracle's gradients (the yardstick of the kernels' tests) against central differences."""
    B, S, H, D = 1, 6, 2, 4
    q, k, v, do = (torch.randn(B, S, H if i in (0, 3) else 1, D, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
                   for i in range(4))
    ids = i32([[0, 0, 0, 0, 2, 2]])
    ok, pos = O.visible(B, S, S, True, doc_ids=ids)
    sl = torch.tensor([0.3, 0.05])

    def f(q, k, v):
        return float((O.attention(q, k, v, ok, pos, 0.5, 1.5, sl)["out"] * do).sum())
    r = O.attention(q, k, v, ok, pos, 0.5, 1.5, sl, do)
    e = 1e-5
    for n, t in (("dq", q), ("dk", k), ("dv", v)):
        for at in [(0, 0, 0, 0), (0, 3, 0, 2), (0, 5, 0, 3)]:
            a, b = t.clone(), t.clone()
            a[at] += e
            b[at] -= e
            args = {"dq": (a, k, v), "dk": (q, a, v), "dv": (q, k, a)}[n], {"dq": (b, k, v), "dk": (q, b, v), "dv": (q, k, b)}[n]
            num = (f(*args[0]) - f(*args[1])) / (2 * e)
            # third-order term e^2 and the cancellation 1e-16 / e, both below 1e-8 here
            assert abs(num - float(r[n][at])) < 1e-7, (n, at)


def test_document_spans():
    ids = i32([[5, 5, 5, 2, 5, -1, -1, 3], [-7, -7, 0, 0, 0, 0, 0, 0]])
    want = i32([[[0, 3]] * 3 + [[3, 4], [4, 5], [0, 0], [0, 0], [7, 8]], [[0, 0]] * 2 + [[2, 8]] * 6])
    assert torch.equal(TR.document_spans(ids), want)
    assert torch.equal(TR.document_spans(i32([[1]])), i32([[[0, 1]]]))


def test_attention_cache_with_room_and_column_views():
    """3-D cache buffers with more rows than Sk and column views equal the tight layout."""
    sp = spec(B=2, Sq=2, Sk=7, causal=True, q_start=i32([5, 3]), softcap=4.0)
    want, _ = TR.attention_fwd(sp)
    kv = torch.zeros(2, 11, 5 * 64, dtype=torch.bfloat16)
    kv[:, :7, 64:192] = sp.k[0].view(2, 7, 128)
    kv[:, :7, 192:] = sp.v[0].view(2, 7, 128)
    sp2 = TR.AttnSpec(2, 4, 2, 7, sp.q, (kv, 64), (kv, 192), causal=True, kv_heads=2, q_start=i32([5, 3]), softcap=4.0)
    got, _ = TR.attention_fwd(sp2)
    assert torch.equal(got, want)


def test_plain_spec_is_unchanged():
    """Without the new arguments a spec is the plain form (its kernels and results)."""
    q = randn(2 * 8, 128)
    assert not TR.AttnSpec(2, 2, 8, 8, (q, 0), (q, 0), (q, 0), causal=True, p_drop=0.1, kv_len=i32([8, 3])).shaped


@pytest.mark.parametrize("kw,err", [
    (dict(D=96), ValueError), (dict(H=4, Hk=3), ValueError), (dict(softcap=-1.0), ValueError),
    (dict(softcap=math.inf), ValueError), (dict(softcap=1.0, scale=0.0), ValueError),
    (dict(prefix_len=i32([1, 2])), ValueError),  # without causal
    (dict(softcap=1.0, kv_len=torch.tensor([1, 2])), ValueError),  # int64
    (dict(softcap=1.0, kv_len=i32([1])), ValueError), (dict(q_start=i32([1, 2, 3])), ValueError),
    (dict(slopes=torch.ones(2)), ValueError), (dict(slopes=torch.ones(4, dtype=torch.float64)), ValueError),
    (dict(docs=i32([[0] * 9] * 2)), ValueError),  # ids, not spans
    (dict(dtype=torch.float32), TypeError), (dict(Sq=0, softcap=1.0), ValueError),
])
def test_attention_refuses(kw, err):
    with pytest.raises(err):
        spec(**kw)


def test_attention_refuses_bad_buffers():
    q = randn(16, 256)
    k = randn(16, 128)
    with pytest.raises(ValueError):  # column out of the buffer
        TR.AttnSpec(2, 4, 8, 8, (q, 8), (k, 0), (k, 0), kv_heads=2, softcap=1.0)
    with pytest.raises(ValueError):  # rows
        TR.AttnSpec(2, 4, 9, 8, (q, 0), (k, 0), (k, 0), kv_heads=2, softcap=1.0)
    sp = TR.AttnSpec(2, 4, 8, 8, (q, 0), (k, 0), (k, 0), kv_heads=2, softcap=1.0)
    out, lse = TR.attention_fwd(sp)
    with pytest.raises(ValueError):  # a gradient buffer without room
        TR.attention_bwd(sp, out, out, lse, (torch.empty_like(q), 0), (torch.empty_like(k), 8), (torch.empty_like(k), 0))
    with pytest.raises(TypeError):
        TR.document_spans(torch.zeros(2, 3))


def logits(T=7, V=50, cols=56, seed=0, dtype=torch.float32):
    return randn(T, cols, seed=seed, dtype=dtype, scale=3.0)


def test_logprobs_reference():
    x = logits()
    x[1, 3:40] = -math.inf
    x[2, :50] = -math.inf
    x[3, 10] = x[3, 20] = x[3, 30] = 50.0  # ties
    ids = i32([0, 3, 4, 20, -100, 50, 49])
    r = L.token_logprobs(x, ids, V=50, top_k=4)
    w = O.logprobs(x, ids, 50, 4)
    assert torch.equal(r.top_ids.long(), w["top_ids"])
    for n in ("logp", "entropy", "lse", "top_logp"):
        assert torch.allclose(getattr(r, n).double(), w[n], atol=2e-5), n
    g = [randn(7, seed=i, dtype=torch.float32) for i in (1, 2)] + [randn(7, 4, seed=3, dtype=torch.float32)]
    d = L.token_logprobs_bwd(x, ids, r, *g, V=50)
    w = O.logprobs(x, ids, 50, 4, *g)
    assert torch.allclose(d[:, :50].double(), w["dlogits"], atol=2e-5) and not d[:, 50:].any()


def test_logprobs_gradient_by_differences():
    x = logits(T=2, V=9, cols=9).double()
    ids = i32([4, 0])
    g1, g2, g3 = torch.tensor([0.7, -0.4]), torch.tensor([0.3, 1.1]), torch.tensor([[0.2, -0.9], [0.5, 0.1]])

    def f(x):
        r = O.logprobs(x, ids, 9, 2)
        return float((r["logp"] * g1).sum() + (r["entropy"] * g2).sum() + (r["top_logp"] * g3).sum())
    d = O.logprobs(x, ids, 9, 2, g1, g2, g3)["dlogits"]
    e = 1e-5
    for t in range(2):
        for c in range(9):
            a, b = x.clone(), x.clone()
            a[t, c] += e
            b[t, c] -= e
            assert abs((f(a) - f(b)) / (2 * e) - float(d[t, c])) < 1e-7


@pytest.mark.parametrize("call,err", [
    (lambda x, i: L.token_logprobs(x, i.long()), ValueError), (lambda x, i: L.token_logprobs(x, i[:3]), ValueError),
    (lambda x, i: L.token_logprobs(x, i, V=0), ValueError), (lambda x, i: L.token_logprobs(x, i, V=57), ValueError),
    (lambda x, i: L.token_logprobs(x, i, top_k=33), ValueError), (lambda x, i: L.token_logprobs(x, i, V=3, top_k=4), ValueError),
    (lambda x, i: L.token_logprobs(x, i, top_k=-1), ValueError), (lambda x, i: L.token_logprobs(x.double(), i), TypeError),
    (lambda x, i: L.token_logprobs(x[0], i), TypeError), (lambda x, i: L.token_logprobs(x.t().contiguous().t(), i), ValueError),
    (lambda x, i: L.token_logprobs_bwd(x, i, L.token_logprobs(x, i), dtop=torch.ones(7, 2)), ValueError),
    (lambda x, i: L.token_logprobs_bwd(x, i, L.token_logprobs(x, i), torch.ones(7).double()), ValueError),
    (lambda x, i: L.token_logprobs_bwd(x, i, L.token_logprobs(x, i), torch.ones(6)), ValueError),
])
def test_logprobs_refuses(call, err):
    with pytest.raises(err):
        call(logits(), i32([0] * 7))


def test_sorted_embedding_reference():
    ids = i32([[3, 0, 3, -1], [9, 3, 10, 0]])
    o = TR.token_order(ids, 10)
    assert o.perm.tolist() == [1, 7, 0, 2, 5, 4, 3, 6] and o.keys.tolist() == [0, 0, 3, 3, 3, 9, 10, 10]
    dy = randn(2, 4, 16)
    want = torch.zeros(10, 16, dtype=torch.float64)
    for t, i in enumerate(ids.reshape(-1).tolist()):
        if 0 <= i < 10:
            want[i] += dy.reshape(8, 16)[t].double() * 4.0
    got = torch.full((10, 16), 7.0)
    TR.embedding_bwd_sorted(o, dy, got, scale=4.0, accumulate=False)
    # three f32 additions of terms below 3 |dy|max scale
    assert torch.allclose(got.double(), want, atol=4 * 2.0 ** -24 * 4 * 3 * float(dy.abs().max()))
    TR.embedding_bwd_sorted(o, dy, got, scale=-4.0)
    assert torch.allclose(got, torch.zeros_like(got), atol=1e-5)


@pytest.mark.parametrize("call,err", [
    (lambda o: TR.token_order(torch.zeros(3, dtype=torch.long), 5), TypeError), (lambda o: TR.token_order(i32([1]), 0), ValueError),
    (lambda o: TR.embedding_bwd_sorted(o, randn(3, 16), torch.zeros(6, 16)), ValueError),
    (lambda o: TR.embedding_bwd_sorted(o, randn(4, 16), torch.zeros(5, 16)), ValueError),
    (lambda o: TR.embedding_bwd_sorted(o, randn(3, 8), torch.zeros(5, 16)), ValueError),
])
def test_sorted_embedding_refuses(call, err):
    with pytest.raises(err):
        call(TR.token_order(i32([1, 2, 3]), 5))
