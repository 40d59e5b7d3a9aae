"""Calls of the language-model operators at their edges: rows that see nothing in a cache divided over blocks, small and
large gradients in half precision, large score caps, lone tokens with odd strides, ids and limits."""
import math

import pytest
import torch

import lm_oracle as O
from tensorflow_k8s_amd.ops import loss as L
from tensorflow_k8s_amd.ops import transformer as TR
from test_lm_ops_gpu import BF, DEV, F32, HF, Case, dev, docs, i32, randn, zipf

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------- few rows over a divided cache

def _ids(S, *rows):
    """Document ids of rows given as runs (id, length), cut or padded (-1) to S."""
    return i32([([d for d, n in row for _ in range(n)] + [-1] * S)[:S] for row in rows])


# every cache is 1024 keys or longer: its keys are divided over blocks
DIVIDED = {
    # the first queries see a whole run, the others stand in the padding or behind the last key
    "padded_tail": lambda: Case(B=2, H=4, Hk=2, Sq=8, Sk=1024, q_start=[996, 1020], doc_ids=_ids(1024, [(0, 1000)], [(0, 1024)])),
    "padded_tail_causal": lambda: Case(B=2, H=4, Hk=2, D=128, Sq=8, Sk=1024, causal=True, q_start=[996, 1020],
                                       doc_ids=_ids(1024, [(0, 1000)], [(3, 1024)])),
    "padded_tail_cap": lambda: Case(B=1, H=2, Hk=1, Sq=8, Sk=1500, causal=True, cap=5.0, q_start=[1196], doc_ids=_ids(1500, [(0, 1200)])),
    "padded_tail_bias_f16": lambda: Case(B=1, H=4, Hk=1, D=128, Sq=5, Sk=2100, dtype=HF, slopes=True, cap=9.0, q_start=[2097],
                                         doc_ids=_ids(2100, [(0, 300), (1, 1800)])),
    "padded_inside": lambda: Case(B=1, H=2, Hk=2, Sq=30, Sk=1600, causal=True, q_start=[1290], doc_ids=_ids(1600, [(0, 1300), (-1, 9), (1, 291)])),
    "before_the_first_key": lambda: Case(B=2, H=4, Hk=2, Sq=6, Sk=1100, causal=True, q_start=[-3, 1090], slopes=True),
    "all_padding": lambda: Case(B=2, H=2, Hk=1, Sq=3, Sk=1030, q_start=[500, 9], doc_ids=_ids(1030, [(-1, 1030)], [(0, 1030)])),
    # shares that lie outside some rows' keys
    "documents": lambda: Case(B=2, H=4, Hk=2, D=128, Sq=8, Sk=2500, causal=True, q_start=[1596, 700],
                              doc_ids=_ids(2500, [(0, 900), (1, 700), (2, 900)], [(0, 704), (1, 1700)])),
    "prefix": lambda: Case(B=3, H=4, Hk=2, Sq=4, Sk=1700, causal=True, q_start=[10, 0, 1696], prefix_len=[1300, 0, 90]),
    "prefix_kv_len": lambda: Case(B=3, H=2, Hk=1, D=128, Sq=4, Sk=1700, causal=True, q_start=[10, 5, 900], prefix_len=[1300, 40, 90], kv_len=[1200, 0, 901]),
    "lengths_both_ways": lambda: Case(B=4, H=8, Hk=2, Sq=3, Sk=1300, kv_len=[0, 1300, 1, 700], slopes=True, cap=20.0),
    "slopes_cap_f16": lambda: Case(B=2, H=4, Hk=4, D=128, Sq=1, Sk=1900, dtype=HF, slopes=True, cap=15.0, kv_len=[1900, 650]),
}


@pytest.mark.parametrize("name", list(DIVIDED))
def test_attention_divided_cache(name):
    c = DIVIDED[name]()
    c.fused = False
    dead_q, dead_k = ~c.ok.any(2), ~c.ok.any(1)
    c.q[dead_q] = math.nan  # rows and keys that no pair uses hold anything
    c.k[dead_k], c.v[dead_k] = math.nan, math.inf
    c.check(grads=False)  # (0 and lse +inf where a row sees nothing)


# ------------------------------------------------------------------------------------- half precision gradients

@pytest.mark.parametrize("scale", [1e4, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("kind", ["long", "long_wide", "long_documents", "first_keys"])
def test_attention_f16_gradients_at_any_scale(kind, cap, scale):
    """f16 gradients of small and large upstream gradients: P (dP - delta) is far below the smallest f16 number, or above
    the largest, where the gradients themselves are not. The relative 2-norm of the error is at most that of two
    roundings, sqrt(2) times that of the exact gradient rounded once (and 6% for the rest)."""
    c = {"long": lambda: Case(B=1, H=2, Hk=1, Sq=2100, causal=True, cap=cap, dtype=HF),
         "long_wide": lambda: Case(B=1, H=1, D=128, Sq=300, Sk=2300, cap=cap, dtype=HF, fused=False),
         "long_documents": lambda: Case(B=1, H=2, Sq=2000, cap=cap, dtype=HF, slopes=0.01, doc_ids=docs(1, 2000, [1500, 400])),
         "first_keys": lambda: Case(B=2, H=2, D=128, Sq=90, causal=True, cap=cap, dtype=HF)}[kind]()
    c.dout = (c.dout.float() * scale).to(HF)
    r, sp = c.oracle(), c.spec()
    out, lse = TR.attention_fwd(sp)
    g = [torch.empty(c.B * S, n * c.D, dtype=HF, device=DEV) for S, n in ((c.Sq, c.H), (c.Sk, c.Hk), (c.Sk, c.Hk))]
    TR.attention_bwd(sp, out, c.dout.reshape(c.B * c.Sq, -1).to(DEV), lse, *((x, 0) for x in g))
    for n, x in zip(("dq", "dk", "dv"), g):
        w = r[n]
        once = (w.to(HF).double() - w).norm()
        assert torch.isfinite(once)
        assert (x.view(w.shape).double().cpu() - w).norm() <= 1.5 * once, n


@pytest.mark.parametrize("kw", [
    dict(B=2, H=2, Sq=130, causal=True, cap=7.0, p_drop=0.2, doc_ids=docs(2, 130, [100, 9])),
    dict(B=1, H=4, Hk=2, D=128, Sq=35, Sk=70, p_drop=0.5, fused=False, slopes=True),
    dict(B=1, H=2, Hk=1, D=128, Sq=300, causal=True, p_drop=0.1),
    dict(B=2, H=4, Hk=2, Sq=3, Sk=90, causal=True, q_start=[87, 30], p_drop=0.3, fused=False),
])
def test_attention_f16_dropout(kw):
    Case(dtype=HF, **kw).check()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kw", [dict(Sq=2, H=4, Hk=2), dict(Sq=1, H=8, Hk=1, D=128, cap=50.0), dict(Sq=70, H=1), dict(Sq=66, H=2, Hk=1, D=128, cap=50.0),
                                dict(Sq=64, H=1, slopes=1e-4)],
                         ids=["few", "few_cap", "tiles", "tiles_cap", "tiles_bias"])
def test_attention_weights_far_below_the_largest(kw, dtype):
    """Each row gives 99% of its weight to one key with V = 0 and shares the rest among 16384: each of them weighs about
    2^-21 of the largest. O is the sum over them: P and O are rounded, sqrt(2) times the error of O rounded once."""
    c = Case(B=1, Sk=16384, dtype=dtype, fused=False, **kw)
    gap = math.log(99 * 16384)
    c.q[..., 0], c.k[..., 0], c.k[:, 300] = 8.0, 0.0, 0.0
    c.k[:, 300, :, 0] = gap * math.sqrt(c.D) / 8.0  # (a cap of 50 takes 0.4 of 14.3 away)
    c.v[:, 300] = 0.0
    r, sp = c.oracle(False), c.spec()
    out, lse = TR.attention_fwd(sp)
    w = r["out"]
    once = (w.to(dtype).double() - w).norm()
    err = (out.view(w.shape).double().cpu() - w).norm()
    print(float(once / w.norm()), float(err / w.norm()), flush=True)
    assert err <= 1.5 * once
    assert float((lse.double().cpu() - r["lse"]).abs().max()) < 2e-5 * 20


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kw", [dict(Sq=3, Sk=300, causal=True, q_start=[297], fused=False), dict(Sq=1, Sk=1500, H=4, D=128, fused=False),
                                dict(Sq=150, causal=True, prefix_len=[0]), dict(Sq=140, H=1, D=128), dict(Sq=100, slopes=1.0)],
                         ids=["few", "few_wide", "tiles", "tiles_wide", "tiles_bias"])
def test_attention_scores_past_float32_integers(kw, dtype):
    """Scores of 1e7 to 1e8, where a float32 step is 1 to 8: a row takes its best key, nothing overflows."""
    c = Case(B=1, dtype=dtype, scale=4000.0, seed=11, **kw)
    c.v = c.v / 4000
    c.check(grads=False)
    c = Case(B=1, dtype=dtype, scale=1500.0, seed=11, **kw)
    c.v = c.v / 1500
    sp = c.spec()
    out, lse = TR.attention_fwd(sp)
    d = [torch.empty_like(t[0]) for t in (sp.q, sp.k, sp.v)]
    TR.attention_bwd(sp, out, c.dout.reshape(out.shape).to(DEV), lse, *((x, t[1]) for x, t in zip(d, (sp.q, sp.k, sp.v))))
    n = [c.H * c.D, c.Hk * c.D, c.Hk * c.D]
    assert all(torch.isfinite(x[:, t[1]:t[1] + w]).all() for x, t, w in zip(d, (sp.q, sp.k, sp.v), n))


# ------------------------------------------------------------------------------------- any score cap

@pytest.mark.parametrize("cap", [1.2e-38, 1e-30, 1e-3, 128.0, 129.0, 512.0, 513.0, 1e4, 1e6, 1e8, 1e30, 2e38])
@pytest.mark.parametrize("kw", [
    dict(B=1, H=2, Hk=1, Sq=150, causal=True),
    dict(B=1, H=2, Hk=1, D=128, Sq=140, causal=True, dtype=HF, slopes=True, doc_ids=docs(1, 140, [60, 29], pad=7)),
    dict(B=2, H=2, Sq=90, Sk=120, kv_len=[120, 40], fused=False, p_drop=0.2),
    dict(B=1, H=1, Sq=100, causal=True, scale=8.0),  # scores of some hundreds: where a cap of 512 still acts
], ids=["causal", "f16_docs_bias", "dropout", "large_scores"])
def test_attention_any_cap(kw, cap):
    """Small and large caps: scores, lse and gradients as exact as without a cap (a large cap leaves the scores alone)."""
    Case(cap=cap, **kw).check()


@pytest.mark.parametrize("cap", [1e-30, 128.0, 129.0, 512.0, 513.0, 1e6, 1e30])
@pytest.mark.parametrize("Sk", [300, 1500])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_attention_any_cap_few_rows(dtype, Sk, cap):
    Case(B=2, H=4, Hk=2, D=128, Sq=2, Sk=Sk, causal=True, kv_len=[Sk, 9], q_start=[Sk - 2, 7], cap=cap, dtype=dtype, fused=False).check(grads=False)


@pytest.mark.parametrize("cap", [30.0, 128.0, 129.0, 512.0, 1e4])
@pytest.mark.parametrize("Sq", [1, 40])
def test_attention_any_cap_lse_near_0(cap, Sq):
    """One key with a score near 0: lse is that score, within 2e-5 (the score's own digits are far below)."""
    for D in (64, 128):
        for seed in range(40):
            Case(B=1, H=2, Sq=Sq, Sk=1, D=D, cap=cap, fused=False, seed=4 * seed, scale=0.3).check(grads=False)


# ------------------------------------------------------------------------------------- strides of lone tokens

def test_attention_lone_tokens_of_any_stride():
    """Sequences of one token: the stride of that dim says nothing, whatever it is (0 in an expanded view)."""
    c = Case(B=3, H=4, Hk=2, Sq=1, Sk=1, cap=3.0, fused=False)
    sp = c.spec()
    k, v = sp.k[0][:1], sp.v[0][:1]
    for shared in (lambda t: t.expand(3, 128), lambda t: t.unsqueeze(0).expand(3, 1, 128),
                   lambda t: torch.as_strided(t, (3, 1, 128), (0, 8, 1))):
        a = TR.AttnSpec(3, 4, 1, 1, sp.q, (shared(k), 0), (shared(v), 0), kv_heads=2, softcap=3.0)
        b = TR.AttnSpec(3, 4, 1, 1, sp.q, (k.repeat(3, 1), 0), (v.repeat(3, 1), 0), kv_heads=2, softcap=3.0)
        res = []
        for s in (a, b):
            out, lse = TR.attention_fwd(s)
            g = [torch.empty(3, n, dtype=BF, device=DEV) for n in (256, 128, 128)]
            TR.attention_bwd(s, out, c.dout.reshape(3, -1).to(DEV), lse, *((x, 0) for x in g))
            res.append([out, lse] + g)
        assert bool(res[1][0].any()) and all(torch.equal(x, y) for x, y in zip(*res))
    one = torch.as_strided(sp.k[0], (1, 1, 128), (128, 8, 1)), torch.as_strided(sp.v[0], (1, 1, 128), (128, 0, 1))
    a = TR.AttnSpec(1, 4, 3, 1, (sp.q[0][:3], 0), (one[0], 0), (one[1], 0), kv_heads=2, softcap=3.0)
    b = TR.AttnSpec(1, 4, 3, 1, (sp.q[0][:3], 0), (k, 0), (v, 0), kv_heads=2, softcap=3.0)
    assert all(torch.equal(x, y) for x, y in zip(TR.attention_fwd(a), TR.attention_fwd(b)))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("slope", [1.0, -1.0])
def test_attention_gradients_under_steep_slopes(slope, dtype):
    """Rows that rest on few keys, near ones or (negative slopes) the farthest: each gradient keeps to two roundings.
    dK and dV: sqrt(2) times the error of the exact gradient rounded once (and 6%). dQ takes delta = dO.out from the
    rounded out that the backward is given, so row i is off by scale e_i sum_j P_ij K_j with e_i = dO_i.(out_i - O_i),
    beside its own rounding: both are known here, their squares add. (With a negative slope all rows rest on the same
    three keys, so the ratio of the two is one draw, not a mean: 1.5 times one rounding does not bound it.)"""
    c = Case(B=1, H=1, D=128, Sq=400, causal=True, dtype=dtype, slopes=slope)
    r, sp = c.oracle(), c.spec()
    out, lse = TR.attention_fwd(sp)
    g = [torch.empty(400, 128, dtype=dtype, device=DEV) for _ in range(3)]
    TR.attention_bwd(sp, out, c.dout.reshape(400, -1).to(DEV), lse, *((x, 0) for x in g))
    Q, K = c.q[0, :, 0].double(), c.k[0, :, 0].double()
    scale = 1 / math.sqrt(128)
    z = (Q @ K.T) * scale - c.slopes[0].double() * (torch.arange(400)[:, None] - torch.arange(400)).abs()
    p = torch.softmax(z.masked_fill(~c.ok[0], -math.inf), 1)
    e = (c.dout[0, :, 0].double() * (out.double().cpu() - r["out"][0, :, 0])).sum(1)
    given = (scale * e[:, None] * (p @ K)).norm()
    for n, x in zip(("dq", "dk", "dv"), g):
        w = r[n]
        once = (w.to(dtype).double() - w).norm()
        err = (x.view(w.shape).double().cpu() - w).norm()
        most = 1.06 * torch.hypot(once, given) if n == "dq" else 1.5 * once
        print(n, float(err / once), float(most / once), flush=True)
        assert err <= most, n


# ------------------------------------------------------------------------------------- gradients in interleaved buffers

def _grads(sp, out, lse, dout, views):
    TR.attention_bwd(sp, out, dout, lse, *((v, 0) for v in views))
    return [v.clone() for v in views]


def test_attention_gradients_in_interleaved_buffers():
    """Gradient views that share memory are refused before a launch, whatever their batch strides; views of one
    buffer that do not share any are written (batches between the tokens, batches any distance apart)."""
    B, S, W = 4, 8, 64
    c = Case(B=B, H=1, Sq=S, cap=3.0, fused=False)
    sp = c.spec()
    out, lse = TR.attention_fwd(sp)
    dout = c.dout.reshape(B * S, W).to(DEV)
    want = _grads(sp, out, lse, dout, [torch.empty(B, S, W, dtype=BF, device=DEV) for _ in range(3)])
    buf = torch.zeros(16384, dtype=BF, device=DEV)
    view = lambda bs, rs, at: torch.as_strided(buf, (B, S, W), (bs, rs, 1), at)  # noqa: E731
    for strides in ([(128, 1024, 0), (192, 1024, 64), (64, 1024, 768)],  # the third batch of dq is the second of dk
                    [(1024, 128, 0), (1032, 128, 64), (1024, 128, 8192)],
                    [(512, 64, 0), (512, 64, 2048), (512, 64, 4032)]):
        with pytest.raises(RuntimeError, match="overlaps"):
            _grads(sp, out, lse, dout, [view(*s) for s in strides])
    assert not buf.any()
    for strides in ([(192, 768, 0), (192, 768, 64), (192, 768, 128)],  # [S, B, 3 W]
                    [(1544, 192, 0), (1544, 192, 64), (1544, 192, 128)],  # [B, S, 3 W], 8 elements between the batches
                    [(64, 1024, 0), (128, 1024, 256), (64, 1024, 704)],
                    [(512, 64, 0), (512, 64, 2048), (512, 64, 4096)]):
        got = _grads(sp, out, lse, dout, [view(*s) for s in strides])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), strides


# ------------------------------------------------------------------------------------- plain calls keep their kernels

def test_attention_plain_3d_buffers_keep_the_plain_kernels():
    """bf16 buffers [B, S, width] of exactly S tokens are the plain form, as 2-D ones are: equal bits, its rules."""
    B, H, S = 2, 2, 40
    x = randn(B * S, 3 * H * 64, seed=3).to(DEV)
    kv_len = i32([40, 7, 1]).to(DEV)  # (the plain form reads the first B)
    res = []
    for buf in (x, x.view(B, S, -1)):
        sp = TR.AttnSpec(B, H, S, S, (buf, 0), (buf, H * 64), (buf, 2 * H * 64), causal=True, kv_len=kv_len)
        assert not sp.shaped
        out, lse = TR.attention_fwd(sp)
        d = torch.empty_like(buf)
        TR.attention_bwd(sp, out, out, lse, (d, 0), (d, H * 64), (d, 2 * H * 64))
        res.append((out, lse, d.view(B * S, -1)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


# ------------------------------------------------------------------------------------- ids and limits

def test_logprobs_ignore_index_outside_int32():
    """An ignore_index that no int32 id can equal ignores nothing."""
    x, ids = randn(4, 50, dtype=F32).to(DEV), i32([5, 5, 7, 0]).to(DEV)
    w = L.token_logprobs(x, ids)
    for ignore in (2 ** 32 + 5, -2 ** 40 + 7, 2 ** 33):
        r = L.token_logprobs(x, ids, ignore_index=ignore)
        assert torch.equal(r.logp, w.logp)
        g = torch.ones(4, device=DEV)
        assert torch.equal(L.token_logprobs_bwd(x, ids, r, g, ignore_index=ignore), L.token_logprobs_bwd(x, ids, w, g))


# (a launch has below 2^32 threads; beyond, their count wraps and no error is reported)

def test_logprobs_of_many_rows():
    T, V = (1 << 24) + 1000, 3
    x = torch.randn(T, V, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(BF)
    ids = torch.randint(0, V, (T,), generator=torch.Generator(DEV).manual_seed(2), device=DEV, dtype=torch.int32)
    g = [torch.randn(T, generator=torch.Generator(DEV).manual_seed(3 + i), device=DEV) for i in range(2)]
    g.append(torch.randn(T, 2, generator=torch.Generator(DEV).manual_seed(5), device=DEV))
    r = L.token_logprobs(x, ids, top_k=2)
    d = L.token_logprobs_bwd(x, ids, r, *g)
    for at in (0, 999, (1 << 23) - 50, (1 << 24) - 50, T - 100):
        s = slice(at, at + 100)
        w = L.token_logprobs(x[s], ids[s], top_k=2)
        for n in ("logp", "entropy", "lse", "norm", "top_logp", "top_ids"):
            assert torch.equal(getattr(r, n)[s], getattr(w, n)), (n, at)
        assert torch.equal(d[s], L.token_logprobs_bwd(x[s], ids[s], w, *(t[s] for t in g))), at
    # every row, against the definition: a few roundings of exponents and logarithms of size 10
    want = torch.log_softmax(x.float(), 1).gather(1, ids.long()[:, None])[:, 0]
    assert float((r.logp - want).abs().max()) < 20 * 2.0 ** -23


def test_document_spans_of_many_rows():
    B = (1 << 22) + 5
    ids = torch.randint(-1, 2, (B, 3), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    assert torch.equal(TR.document_spans(ids.to(DEV)).cpu(), TR.document_spans(ids))


def test_sorted_embedding_of_a_table_of_many_rows():
    V = (1 << 27) + 67
    at = [0, 8, (1 << 25) - 1, 1 << 25, (1 << 25) + 8, 1 << 26, (1 << 27) - 1, V - 4, V - 1]
    dw = torch.full((V, 8), math.nan, device=DEV)
    TR.embedding_bwd_sorted(TR.token_order(i32(at + [-1, V]).to(DEV), V), torch.ones(len(at) + 2, 8, dtype=BF, device=DEV), dw, accumulate=False)
    assert torch.equal(torch.nonzero(dw[:, 3])[:, 0].cpu(), torch.tensor(at))
    assert dw.sum().item() == 8 * len(at)


def test_attention_refuses_grids_past_32_bits():
    e = lambda B, S: torch.empty(1, 1, 64, dtype=BF, device=DEV).expand(B, S, 64)  # noqa: E731
    for B, Sq, Sk in ((9_000_000, 1, 1), (8_000_000, 1, 40), (100_000, 30_000, 1)):
        with pytest.raises(RuntimeError, match="grid too large"):
            TR.attention_fwd(TR.AttnSpec(B, 1, Sq, Sk, (e(B, Sq), 0), (e(B, Sk), 0), (e(B, Sk), 0), softcap=1.0))


# ------------------------------------------------------------------------------------- the operators' neighbours

@pytest.mark.parametrize("T,V,W,scale", [(333, 4099, 512, 22.6), (8192, 3000, 768, 1.0), (20000, 40, 64, 8.0)])
def test_sorted_embedding_agrees_with_the_bucketed_one(T, V, W, scale):
    """Both add the same terms in float32 in an order of their own: n additions each."""
    ids = zipf(T, V).clamp(min=0).to(DEV)
    dy = randn(T, W, seed=2).to(DEV)
    a, b = torch.zeros(V, W, device=DEV), torch.zeros(V, W, device=DEV)
    TR.embedding_bwd_sorted(TR.token_order(ids, V), dy, a, scale=scale)
    TR.embedding_bwd(ids, dy, b, scale=scale)
    n = torch.bincount(ids.long(), minlength=V)[:, None].double().cpu()
    mag = torch.zeros(V, W, dtype=torch.float64).index_add_(0, ids.long().cpu(), dy.double().abs().cpu()) * scale
    O.within(a, b.double().cpu(), 2 * (n + 3) * 2.0 ** -24 * mag, "dword")


# ------------------------------------------------------------------------------------- variants by size

# 449 to 512 blocks of 256 rows at head size 128: the row tiles of 8 waves; beside them, of 4
ROWS = {
    "causal": lambda: Case(B=1, H=32, Hk=4, D=128, Sq=3700, Sk=150, causal=True, q_start=[-3600], cap=6.0, fused=False),
    "full_f16": lambda: Case(B=2, H=16, Hk=2, D=128, Sq=3584 + 130, Sk=97, dtype=HF, kv_len=[97, 40], poison=math.nan, fused=False),
    "bias": lambda: Case(B=1, H=32, Hk=2, D=128, Sq=4000, Sk=90, causal=True, slopes=True, q_start=[-3950], fused=False),
    "prefix": lambda: Case(B=1, H=30, Hk=15, D=128, Sq=3840, Sk=200, causal=True, prefix_len=[70], q_start=[-3700], fused=False),
    "bias_cap": lambda: Case(B=1, H=32, Hk=2, D=128, Sq=3700, Sk=90, causal=True, slopes=True, cap=9.0, q_start=[-3650], fused=False),
    "more_blocks": lambda: Case(B=1, H=34, Hk=2, D=128, Sq=4000, Sk=64, causal=True, q_start=[-3950], fused=False),
}


@pytest.mark.parametrize("name", list(ROWS))
def test_attention_row_tiles(name):
    ROWS[name]().check()


@pytest.mark.parametrize("T", [180000, 180001])
def test_token_order_tiles(T):
    ids = torch.randint(-3, 33003, (T,), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    a, b = TR.token_order(ids.to(DEV), 33000), TR.token_order(ids, 33000)
    assert torch.equal(a.perm.cpu(), b.perm) and torch.equal(a.keys.cpu(), b.keys)


def test_sorted_embedding_of_a_shared_gradient_row():
    """dy of one row for all tokens (the gradient of a mean, an expanded view)."""
    ids = zipf(300, 40).to(DEV)
    row = randn(1, 64, seed=4).to(DEV)
    o, a, b = TR.token_order(ids, 40), torch.zeros(40, 64, device=DEV), torch.zeros(40, 64, device=DEV)
    TR.embedding_bwd_sorted(o, row.expand(300, 64), a, scale=0.5)
    TR.embedding_bwd_sorted(o, row.repeat(300, 1), b, scale=0.5)
    assert bool(a.any()) and torch.equal(a, b)
