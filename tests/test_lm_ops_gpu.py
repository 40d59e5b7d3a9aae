"""Kernels of shaped attention (attn_shaped.hip), token log probabilities (logprobs.hip) and the sorted
embedding gradient (embed_sort.hip) against float64 definitions, within the bounds that their roundings
allow (lm_oracle.py)."""
import math

import pytest
import torch

import lm_oracle as O
from tensorflow_k8s_amd.ops import loss as L
from tensorflow_k8s_amd.ops import transformer as TR

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def randn(*shape, seed=0, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def dev(t):
    return t.to(DEV) if t is not None else None


# ------------------------------------------------------------------------------------- attention

class Case:
    """Inputs of one attention call on the CPU; poison: what rows that no pair uses hold."""

    def __init__(self, B=1, H=2, Hk=None, D=64, Sq=64, Sk=None, dtype=BF, causal=False, cap=0.0, slopes=False, kv_len=None,
                 q_start=None, prefix_len=None, doc_ids=None, p_drop=0.0, fused=None, poison=None, seed=0, scale=1.0):
        Hk, Sk = Hk or H, Sk or Sq
        self.__dict__.update(B=B, H=H, Hk=Hk, D=D, Sq=Sq, Sk=Sk, dtype=dtype, causal=causal, cap=cap, p_drop=p_drop)
        self.kv_len, self.q_start, self.prefix_len = (i32(x) if x is not None else None for x in (kv_len, q_start, prefix_len))
        self.doc_ids = doc_ids
        self.slopes = torch.tensor([slopes * 2.0 ** -(1 + h % 7) for h in range(H)]) if slopes else None
        self.q, self.k, self.v = (randn(B, S, n, D, seed=seed + i, dtype=dtype, scale=scale)
                                  for i, (S, n) in enumerate(((Sq, H), (Sk, Hk), (Sk, Hk))))
        self.dout = randn(B, Sq, H, D, seed=seed + 3, dtype=dtype)
        self.ok, self.pos = O.visible(B, Sq, Sk, causal, self.kv_len, self.q_start, self.prefix_len, doc_ids)
        if poison is not None:
            dead_k, dead_q = ~self.ok.any(1), ~self.ok.any(2)
            if kv_len is not None or doc_ids is not None:
                # beyond kv_len and in padded tokens (not: keys that causality alone hides)
                pad = torch.zeros_like(dead_k)
                if kv_len is not None:
                    pad |= torch.arange(Sk)[None] >= self.kv_len[:, None]
                if doc_ids is not None:
                    pad |= doc_ids < 0
                self.k[pad & dead_k] = poison
                self.v[pad & dead_k] = poison
            self.q[dead_q] = poison
            self.dout[dead_q] = poison
        self.fused = Sq == Sk if fused is None else fused

    def spec(self):
        B, H, Hk, D, Sq, Sk = self.B, self.H, self.Hk, self.D, self.Sq, self.Sk
        if self.fused:
            buf = torch.cat([t.reshape(B * Sq, -1) for t in (self.q, self.k, self.v)], 1).to(DEV)
            ops = [(buf, 0), (buf, H * D), (buf, (H + Hk) * D)]
        else:
            ops = [(t.reshape(-1, t.shape[2] * D).to(DEV), 0) for t in (self.q, self.k, self.v)]
        docs = TR.document_spans(dev(self.doc_ids)) if self.doc_ids is not None else None
        return TR.AttnSpec(B, H, Sq, Sk, *ops, kv_len=dev(self.kv_len), causal=self.causal, p_drop=self.p_drop, seed=77,
                           kv_heads=Hk, head_dim=D, softcap=self.cap, slopes=dev(self.slopes), docs=docs,
                           prefix_len=dev(self.prefix_len), q_start=dev(self.q_start))

    def oracle(self, grads=True):
        keep = None
        if self.p_drop:
            keep = TR.dropout_keep_mask(77, self.B, self.H, self.Sq, self.Sk, self.p_drop).double() * TR.attn_keep_scale(self.p_drop)
        return O.attention(self.q, self.k, self.v, self.ok, self.pos, 1.0 / math.sqrt(self.D), self.cap, self.slopes,
                           self.dout if grads else None, keep, self.dtype)

    def check(self, grads=True):
        sp = self.spec()
        assert sp.shaped
        out, lse = TR.attention_fwd(sp)
        r = self.oracle(grads)
        O.within(out.view(r["out"].shape), r["out"], r["out_bound"], "out")
        live = torch.isfinite(r["lse"])
        g = lse.cpu()
        assert bool((g[~live] == math.inf).all()), "lse of rows that see nothing"
        # float32 scores of magnitude up to |lse| + the cap's native reciprocal, summed in f32
        assert float((g.double() - r["lse"])[live].abs().max() if live.any() else 0.0) <= 2e-5 * (1 + float(r["lse"][live].abs().max() if live.any() else 0.0))
        if not grads:
            return
        bufs = {id(b): torch.full_like(b, 3.0) for b, _ in (sp.q, sp.k, sp.v)}  # every element is overwritten
        views = [(bufs[id(b)], c) for b, c in (sp.q, sp.k, sp.v)]
        TR.attention_bwd(sp, out, self.dout.reshape(self.B * self.Sq, -1).to(DEV), lse, *views)
        for n, (buf, col), S, heads in (("dq", views[0], self.Sq, self.H), ("dk", views[1], self.Sk, self.Hk), ("dv", views[2], self.Sk, self.Hk)):
            got = buf[:, col:col + heads * self.D].reshape(self.B, S, heads, self.D)
            O.within(got, r[n], r[n + "_bound"], n)


def docs(B, S, runs, pad=0):
    """Rows of runs of the given lengths, repeated; the last `pad` tokens are padding."""
    ids = torch.zeros(B, S, dtype=torch.int32)
    for b in range(B):
        i, d = 0, 0
        while i < S:
            n = runs[(d + b) % len(runs)]
            ids[b, i:i + n] = d
            i, d = i + n, d + 1
    if pad:
        ids[:, S - pad:] = -1
    return ids


ATTN = {
    "one_token": lambda: Case(Sq=1, cap=2.0),
    "two_tokens_causal": lambda: Case(H=4, Hk=2, Sq=2, causal=True),
    "tile_edges": lambda: Case(H=4, Hk=2, Sq=128, causal=True),
    "past_tile": lambda: Case(B=2, H=2, Hk=1, Sq=129, causal=True, cap=8.0),
    "odd_full": lambda: Case(B=2, H=3, Sq=77, Sk=131, slopes=True, fused=False),
    "wide_head": lambda: Case(B=1, H=4, Hk=2, D=128, Sq=200, causal=True, cap=6.0),
    "wide_head_f16": lambda: Case(B=1, H=2, D=128, Sq=97, causal=True, dtype=HF, slopes=True),
    "f16_cap": lambda: Case(B=1, H=2, Sq=150, dtype=HF, cap=4.0),
    "docs": lambda: Case(B=2, H=2, Sq=300, causal=True, doc_ids=docs(2, 300, [50, 64, 1, 13, 128]), poison=math.nan),
    "docs_padded": lambda: Case(B=2, H=2, Hk=1, Sq=260, causal=True, cap=9.0, doc_ids=docs(2, 260, [90, 5, 30], pad=70), poison=math.nan),
    "docs_all_padding": lambda: Case(B=2, H=2, Sq=70, causal=True, doc_ids=docs(2, 70, [7], pad=70), poison=math.inf),
    "docs_both_ways": lambda: Case(B=1, H=2, D=128, Sq=190, doc_ids=docs(1, 190, [33, 70], pad=3), poison=math.nan),
    "docs_prefix_slopes": lambda: Case(B=2, H=4, Hk=2, Sq=140, causal=True, slopes=True, prefix_len=[20, 100], doc_ids=docs(2, 140, [60, 17])),
    "prefix": lambda: Case(B=3, H=2, Sq=180, causal=True, prefix_len=[0, 70, 500]),
    "kv_len":
    lambda: Case(B=4, H=2, Hk=1, Sq=90, Sk=150, kv_len=[0, 1, 64, 150], poison=math.nan, fused=False),
    "kv_len_causal": lambda: Case(B=2, H=2, Hk=1, Sq=130, kv_len=[5, 129], causal=True),
    "late_queries": lambda: Case(B=2, H=4, Hk=1, Sq=5, Sk=400, causal=True, q_start=[395, 100], slopes=True),
    "early_queries": lambda: Case(B=2, H=2, Sq=100, Sk=64, causal=True, q_start=[-60, -200], poison=None),
    "shared_one": lambda: Case(B=1, H=12, Hk=1, Sq=66, causal=True),
    "dropout": lambda: Case(B=2, H=2, Sq=130, causal=True, cap=7.0, p_drop=0.2, doc_ids=docs(2, 130, [100, 9])),
    "dropout_shared": lambda: Case(B=1, H=4, Hk=2, D=128, Sq=35, Sk=70, p_drop=0.5, fused=False),
    "dropout_few": lambda: Case(B=2, H=4, Hk=2, Sq=3, Sk=90, causal=True, q_start=[87, 30], p_drop=0.3, fused=False),
    "slopes_up": lambda: Case(B=2, H=4, Hk=2, Sq=170, causal=True, slopes=-1.0, cap=5.0),
    "late_chunk_shared_docs": lambda: Case(B=2, H=6, Hk=2, D=128, Sq=130, Sk=330, causal=True, q_start=[199, 70],
                                           doc_ids=docs(2, 330, [101, 64])),
    "large_scores": lambda: Case(B=1, H=2, Hk=1, Sq=100, causal=True, scale=8.0),
    "many_heads": lambda: Case(B=2, H=16, Hk=8, Sq=65, causal=True, slopes=True),
    # 512 blocks of 256 rows and more: the row tiles of 8 waves
    "many_wide_heads": lambda: Case(B=2, H=256, Hk=2, D=128, Sq=300, Sk=97, causal=True, q_start=[-190, -40], kv_len=[97, 60],
                                    poison=math.nan, fused=False),
    "many_wide_heads_docs": lambda: Case(B=4, H=128, Hk=4, D=128, Sq=257, causal=True, cap=5.0, slopes=True,
                                         doc_ids=docs(4, 257, [70, 129, 11], pad=9), poison=math.nan),
    "long": lambda: Case(B=1, H=2, Hk=1, Sq=1100, causal=True, doc_ids=docs(1, 1100, [700, 129, 271])),
}


@pytest.mark.parametrize("name", list(ATTN))
def test_attention(name):
    ATTN[name]().check()


DECODE = {
    "one": lambda: Case(Sq=1, Sk=1, H=1, fused=False, cap=3.0),
    "one_key_of_many": lambda: Case(B=2, H=8, Hk=2, Sq=1, Sk=500, kv_len=[1, 0], causal=True, q_start=[0, -1], poison=math.nan, fused=False),
    "odd_cache": lambda: Case(B=1, H=16, Sq=1, Sk=777, slopes=True, causal=True, kv_len=[777], q_start=[776]),
    "ragged": lambda: Case(B=5, H=8, Hk=2, D=128, Sq=1, Sk=1500, causal=True, kv_len=[1500, 7, 64, 65, 1000],
                           q_start=[1499, 6, 63, 64, 999], cap=30.0, poison=math.nan),
    "f16": lambda: Case(B=2, H=4, Hk=4, D=128, Sq=1, Sk=333, dtype=HF, kv_len=[333, 200], slopes=True),
    "three_tokens": lambda: Case(B=2, H=6, Hk=2, Sq=3, Sk=600, causal=True, kv_len=[600, 9], q_start=[597, 6], poison=math.nan),
    "eight_tokens": lambda: Case(B=1, H=32, Hk=4, D=128, Sq=8, Sk=2100, causal=True, q_start=[2092]),
    "long": lambda: Case(B=1, H=8, Hk=1, D=64, Sq=1, Sk=9001, kv_len=[9000], causal=True, q_start=[8999], poison=math.inf),
    "docs_cache": lambda: Case(B=1, H=4, Hk=2, Sq=2, Sk=900, causal=True, q_start=[700], doc_ids=docs(1, 900, [200])),
    "few_heads_many_rows": lambda: Case(B=1, H=2, Hk=1, Sq=40, Sk=3000, causal=True, q_start=[2960]),
}


@pytest.mark.parametrize("name", list(DECODE))
def test_attention_few_queries(name):
    DECODE[name]().check(grads=False)


UNSEEN = {
    "chunk_of_documents": lambda: Case(B=2, H=4, Hk=2, Sq=100, Sk=500, causal=True, q_start=[260, 391], doc_ids=docs(2, 500, [217, 31])),
    "chunk_both_ways": lambda: Case(B=1, H=2, D=128, Sq=70, Sk=400, q_start=[150], doc_ids=docs(1, 400, [99, 75])),
    "chunk_dropout": lambda: Case(B=1, H=2, Sq=90, Sk=300, causal=True, q_start=[203], doc_ids=docs(1, 300, [201]), p_drop=0.25),
    "token_of_documents": lambda: Case(B=2, H=8, Hk=2, Sq=1, Sk=700, causal=True, q_start=[650, 90], doc_ids=docs(2, 700, [333, 77])),
    "window_of_lengths": lambda: Case(B=3, H=2, Sq=40, Sk=260, causal=True, q_start=[0, 17, 200], kv_len=[260, 33, 210]),
}


@pytest.mark.parametrize("name", list(UNSEEN))
def test_attention_unseen_keys_hold_anything(name):
    c = UNSEEN[name]()
    dead = ~c.ok.any(1)
    assert dead.any()
    c.k[dead] = math.nan
    c.v[dead] = math.inf
    c.check()


def test_attention_few_queries_gradients():
    Case(B=2, H=4, Hk=2, Sq=3, Sk=300, causal=True, q_start=[297, 20], cap=5.0).check()


def test_attention_strided_cache():
    """K and V as columns of a cache [B, S', width] with room behind Sk, the room full of NaN."""
    c = Case(B=2, H=4, Hk=2, Sq=1, Sk=200, causal=True, q_start=[199, 50], fused=False, cap=4.0)
    cache = torch.full((2, 333, 5 * 64), math.nan, dtype=BF, device=DEV)
    cache[:, :200, 64:192] = c.k.reshape(2, 200, 128).to(DEV)
    cache[:, :200, 192:] = c.v.reshape(2, 200, 128).to(DEV)
    sp = c.spec()
    want, _ = TR.attention_fwd(sp)
    sp2 = TR.AttnSpec(2, 4, 1, 200, sp.q, (cache, 64), (cache, 192), causal=True, kv_heads=2, q_start=sp.q_start, softcap=4.0)
    got, _ = TR.attention_fwd(sp2)
    assert torch.equal(got, want)


def test_attention_matches_plain_form():
    """The shaped kernels on a plain causal call agree with attention.hip within both kernels' roundings."""
    c = Case(B=2, H=2, Sq=256, causal=True, prefix_len=[0, 0])
    sp = c.spec()
    plain = TR.AttnSpec(2, 2, 256, 256, sp.q, sp.k, sp.v, causal=True)
    assert not plain.shaped
    a, b = TR.attention_fwd(sp), TR.attention_fwd(plain)
    r = c.oracle(False)
    O.within(a[0].view(r["out"].shape), b[0].view(r["out"].shape).double().cpu(), 2 * r["out_bound"], "out")
    assert torch.allclose(a[1], b[1], atol=1e-4)


PRECISE = {
    "short_documents": lambda dt: Case(B=2, H=4, Hk=2, Sq=256, causal=True, dtype=dt, doc_ids=docs(2, 256, [9, 17, 40])),
    "steep_slopes": lambda dt: Case(B=1, H=1, D=128, Sq=400, causal=True, dtype=dt, slopes=1.0),
    "first_keys": lambda dt: Case(B=4, H=4, Sq=100, causal=True, cap=20.0, dtype=dt),
}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("name", list(PRECISE))
def test_attention_gradients_have_two_roundings(name, dtype):
    """Rows that rest on few keys: the relative 2-norm of each gradient's error is at most that of two roundings
    of its type, sqrt(2) times the error of the exact gradient rounded once (and 6% for the rest)."""
    c = PRECISE[name](dtype)
    r, sp = c.oracle(), c.spec()
    out, lse = TR.attention_fwd(sp)
    g = [torch.empty(c.B * S, n * c.D, dtype=dtype, device=DEV) for S, n in ((c.Sq, c.H), (c.Sk, c.Hk), (c.Sk, c.Hk))]
    TR.attention_bwd(sp, out, c.dout.reshape(c.B * c.Sq, -1).to(DEV), lse, *((x, 0) for x in g))
    for n, x in zip(("dq", "dk", "dv"), g):
        w = r[n]
        once = (w.to(dtype).double() - w).norm()
        assert (x.view(w.shape).double().cpu() - w).norm() <= 1.5 * once, n


def test_attention_repeats_bitwise():
    c = Case(B=2, H=4, Hk=2, Sq=200, causal=True, cap=6.0, doc_ids=docs(2, 200, [90, 30]))
    res = []
    for _ in range(2):
        sp = c.spec()
        out, lse = TR.attention_fwd(sp)
        d = torch.empty_like(sp.q[0])
        TR.attention_bwd(sp, out, c.dout.reshape(400, -1).to(DEV), lse, *((d, col) for _, col in (sp.q, sp.k, sp.v)))
        res.append((out, lse, d))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("S", [1, 2, 63, 1000, 1024, 1025, 5000])
def test_document_spans(S):
    g = torch.Generator().manual_seed(S)
    ids = torch.randint(-1, 3, (3, S), generator=g, dtype=torch.int32)
    ids[1] = torch.randint(0, 2, (S,), generator=g, dtype=torch.int32).cumsum(0) // 40  # long runs
    ids[2] = 5
    assert torch.equal(TR.document_spans(ids.to(DEV)).cpu(), TR.document_spans(ids))


# ------------------------------------------------------------------------------------- log probabilities

def check_logprobs(T, V, cols, dtype, k, seed=0, make=None, view=False):
    x = randn(T, cols, seed=seed, dtype=dtype, scale=3.0)
    ids = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int32)
    ids[::5] = -100
    if T > 3:
        ids[3] = V  # out of range
    if make:
        make(x, ids)
    gx = x.to(DEV)
    if view:  # rows inside a wider buffer, off alignment
        buf = torch.full((T, cols + 13), math.nan, dtype=dtype, device=DEV)
        buf[:, 5:5 + cols] = gx
        gx = buf[:, 5:5 + cols]
    r = L.token_logprobs(gx, ids.to(DEV), V=V, top_k=k)
    g = [randn(T, seed=seed + 2, dtype=F32), randn(T, seed=seed + 3, dtype=F32), randn(T, k, seed=seed + 4, dtype=F32) if k else None]
    w = O.logprobs(x, ids, V, k, *g)
    # f32: the exponent of a term at distance d below the maximum is off by d 2^-23, a sum of <= 64 terms a
    # lane and 8 joins by 72 2^-24, and values of magnitude |lse| round by |lse| 2^-24
    for n in ("lse", "logp", "entropy", "top_logp"):
        if n == "top_logp" and not k:
            continue
        got, want = getattr(r, n).double().cpu(), w[n]
        ok = torch.isfinite(want)
        assert torch.equal(got[~ok], want[~ok]), n
        assert bool(((got - want)[ok].abs() <= 1e-5 * (1 + want[ok].abs())).all()), n
    if k:
        assert torch.equal(r.top_ids.cpu().long(), w["top_ids"])
    d = L.token_logprobs_bwd(gx, ids.to(DEV), r, *(dev(t) for t in g), V=V)
    assert d.shape == (T, cols) and d.dtype == dtype
    u = O.U[dtype] if dtype != F32 else 2.0 ** -23
    O.within(d[:, :V], w["dlogits"], u * w["dlogits"].abs() + 3e-5 * w["mag"] + O.TINY[dtype], "dlogits")
    assert not d[:, V:].any()


@pytest.mark.parametrize("T,V,cols,dtype,k", [
    (1, 1, 1, F32, 1), (1, 1, 8, BF, 0), (3, 7, 7, HF, 7), (5, 33, 40, BF, 20), (4, 1000, 1000, F32, 32),
    (9, 2048, 2048, BF, 5), (6, 2049, 2049, BF, 5), (2, 16384, 16384, BF, 20), (3, 16385, 16392, HF, 20), (7, 33708, 33792, BF, 20),
    (4, 33708, 33792, BF, 0), (2, 8193, 8193, F32, 1), (3, 50001, 50001, F32, 32), (2, 131072, 131072, BF, 32), (300, 515, 515, BF, 3),
])
def test_logprobs(T, V, cols, dtype, k):
    check_logprobs(T, V, cols, dtype, k)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_logprobs_unaligned_rows(dtype):
    check_logprobs(5, 4099, 4099, dtype, 6, view=True)


def _ties(x, ids):
    x[0] = 0.0          # one value everywhere
    x[1] = -0.0
    x[1, ::3] = 0.0     # equal to -0
    x[2] = torch.arange(x.shape[1]).float().neg().to(x.dtype) // 64
    x[3] = torch.arange(x.shape[1]).float().to(x.dtype) / 512
    x[4, 100:] = x[4].float().max().to(x.dtype)


def _masked(x, ids):
    x[0, 1:] = -math.inf            # one class left
    x[1] = -math.inf                # none left
    x[2, ::2] = -math.inf
    x[3] = torch.finfo(x.dtype).min  # a mask of the type's lowest value on the whole row
    x[4, 5:] = torch.finfo(x.dtype).min
    ids[:5] = torch.tensor([0, 3, 4, 5, 6], dtype=torch.int32)


@pytest.mark.parametrize("dtype,V", [(BF, 600), (BF, 20000), (F32, 9000), (HF, 3000)])
@pytest.mark.parametrize("make", [_ties, _masked])
def test_logprobs_special_rows(make, dtype, V):
    check_logprobs(6, V, V, dtype, 12, make=make)


def _ones(x, ids):
    x[:] = 1.0


def _rising(x, ids):
    x[:] = torch.arange(x.shape[1]).float() / 65536  # the best are in the last parts, thousands above any early bound


@pytest.mark.parametrize("dtype,make", [(F32, None), (F32, _rising), (BF, _rising), (BF, _ones)])
def test_logprobs_one_row_of_many_parts(dtype, make):
    check_logprobs(1, 300001, 300001, dtype, 32, make=make, seed=5)


def test_logprobs_nan_and_inf_rows():
    x = randn(4, 3000, dtype=F32)
    x[0, 7] = math.nan
    x[1, 2000] = math.inf
    r = L.token_logprobs(x.to(DEV), i32([1, 1, 1, 1]).to(DEV))
    assert torch.isnan(r.entropy[:2]).all() and torch.isfinite(r.entropy[2:]).all() and torch.isfinite(r.logp[2:]).all()


def test_logprobs_no_rows():
    x = torch.empty(0, 50, device=DEV)
    r = L.token_logprobs(x, torch.empty(0, dtype=torch.int32, device=DEV), top_k=2)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 2)
    assert L.token_logprobs_bwd(x, torch.empty(0, dtype=torch.int32, device=DEV), r).shape == (0, 50)


# ------------------------------------------------------------------------------------- embedding gradient

def check_embedding(ids, V, W, dtype, scale, accumulate, seed=0, strided=False):
    T = ids.numel()
    dy = randn(T, W, seed=seed, dtype=dtype)
    o = TR.token_order(ids.to(DEV), V)
    key = torch.where((ids >= 0) & (ids < V), ids, V).reshape(-1)
    want_keys, want_perm = torch.sort(key, stable=True)
    assert torch.equal(o.perm.cpu().long(), want_perm) and torch.equal(o.keys.cpu(), want_keys.to(torch.int32))
    start = randn(V, W, seed=seed + 1, dtype=F32)
    got = start.clone().to(DEV) if accumulate else torch.full((V, W), math.nan, device=DEV)
    g = dy.to(DEV)
    if strided:
        buf = torch.full((T, W + 24), math.nan, dtype=dtype, device=DEV)
        buf[:, 16:16 + W] = g
        g = buf[:, 16:16 + W]
    TR.embedding_bwd_sorted(o, g, got, scale=scale, accumulate=accumulate)
    want = torch.zeros(V + 1, W, dtype=torch.float64).index_add_(0, key.long(), dy.double())[:V] * scale
    mag = torch.zeros(V + 1, W, dtype=torch.float64).index_add_(0, key.long(), dy.double().abs())[:V] * abs(scale)
    n = torch.bincount(key, minlength=V + 1)[:V, None].double()
    if accumulate:
        want, mag = want + start.double(), mag + start.double().abs()
    # n additions, the scaling and the accumulation, each half a step of f32
    O.within(got, want, (n + 3) * 2.0 ** -24 * mag, "dword")
    return o, g, got


def zipf(T, V, seed=0):
    u = torch.rand(T, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
    ids = (torch.exp(u * math.log(V + 1.0)).long() - 1).clamp(0, V - 1)
    ids[::37] = -1
    return ids.to(torch.int32)


@pytest.mark.parametrize("T,V,W,dtype,scale,acc", [
    (1, 1, 8, BF, 1.0, True), (1, 5, 64, F32, 2.0, False), (2, 3, 72, HF, 1.0, False), (31, 4, 128, BF, 1.0, True),
    (33, 100, 200, BF, 5.0, False), (64, 1, 64, BF, 1.0, False), (333, 4099, 512, BF, 22.6, False), (1000, 7, 768, F32, 1.0, True),
    (8192, 3000, 96, BF, 1.0, False), (12288, 900, 64, BF, 1.0, False), (12289, 900, 64, F32, 1.0, True), (16384, 500, 64, HF, 1.0, True), (16385, 500, 64, BF, 1.0, False),
    (20000, 40, 8, BF, 1.0, False), (40000, 131072, 16, BF, 1.0, True), (33000, 2_000_000, 8, F32, 1.0, True),
])
def test_sorted_embedding(T, V, W, dtype, scale, acc):
    check_embedding(zipf(T, V), V, W, dtype, scale, acc)


def test_sorted_embedding_one_token_everywhere():
    check_embedding(torch.full((5000,), 3, dtype=torch.int32), 10, 40, BF, 1.0, False)


def test_sorted_embedding_padding_only_and_strided():
    check_embedding(torch.full((100,), -1, dtype=torch.int32), 10, 64, BF, 1.0, False)
    check_embedding(torch.full((100,), 10, dtype=torch.int32), 10, 64, BF, 1.0, True)
    check_embedding(zipf(500, 90), 90, 64, BF, 3.0, False, strided=True)
    check_embedding(zipf(500, 90), 90, 64, F32, 3.0, True, strided=True)


def test_sorted_embedding_no_tokens():
    o = TR.token_order(torch.empty(0, dtype=torch.int32, device=DEV), 130)
    d = torch.full((130, 64), 5.0, device=DEV)
    TR.embedding_bwd_sorted(o, torch.empty(0, 64, dtype=BF, device=DEV), d)
    assert bool((d == 5.0).all())
    TR.embedding_bwd_sorted(o, torch.empty(0, 64, dtype=BF, device=DEV), d, accumulate=False)
    assert not d.any()


@pytest.mark.parametrize("T", [3000, 30000])
def test_sorted_embedding_repeats_bitwise(T):
    ids = zipf(T, 200)
    (_, g, a), (_, _, b) = (check_embedding(ids, 200, 128, BF, 1.0, False) for _ in range(2))
    assert torch.equal(a, b)


def test_sorted_embedding_order_serves_two_tables():
    ids = zipf(900, 50)
    o, g, a = check_embedding(ids, 50, 64, BF, 1.0, False)
    b = torch.zeros_like(a)
    TR.embedding_bwd_sorted(o, g, b, accumulate=True)
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------- refusals on the GPU

def test_refusals_before_launch():
    q = randn(16, 128).to(DEV)
    ok = dict(softcap=1.0)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        b = randn(16, 132).to(DEV)
        TR.attention_fwd(TR.AttnSpec(2, 2, 8, 8, (b, 0), (b, 0), (b, 0), **ok))
    with pytest.raises(RuntimeError, match="dtype"):
        TR.attention_fwd(TR.AttnSpec(2, 2, 8, 8, (q, 0), (q.half(), 0), (q, 0), **ok))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        TR.attention_fwd(TR.AttnSpec(2, 2, 8, 8, (q, 0), (q.cpu(), 0), (q, 0), **ok))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        TR.attention_fwd(TR.AttnSpec(2, 2, 8, 8, (q, 0), (q, 0), (q, 0), kv_len=i32([1, 2]), **ok))
    with pytest.raises(RuntimeError, match="aligned"):
        b = randn(16 * 128 + 4).to(DEV)[4:].view(16, 128)
        TR.attention_fwd(TR.AttnSpec(2, 2, 8, 8, (b, 0), (q, 0), (q, 0), **ok))
    sp = TR.AttnSpec(2, 2, 8, 8, (q, 0), (q, 0), (q, 0), **ok)
    out, lse = TR.attention_fwd(sp)
    with pytest.raises(RuntimeError, match="overlap"):
        e = torch.empty(1, 8, 128, dtype=BF, device=DEV).expand(2, 8, 128)
        TR.attention_bwd(sp, out, out, lse, (e, 0), (torch.empty_like(q), 0), (torch.empty_like(q), 0))
    e = torch.empty(16, 256, dtype=BF, device=DEV)
    for grads in (((q, 0), (e, 0), (e, 128)), ((e, 0), (e, 64), (torch.empty_like(q), 0)), ((e, 0), (e, 128), (out, 0))):
        with pytest.raises(RuntimeError, match="overlaps"):
            TR.attention_bwd(sp, out, torch.ones_like(out), lse, *grads)
    with pytest.raises(RuntimeError, match="lse"):
        TR.attention_bwd(sp, out, out, lse[:1], *((torch.empty_like(q), 0) for _ in range(3)))
    with pytest.raises(RuntimeError):
        TR.embedding_bwd_sorted(TR.token_order(i32([1]).to(DEV), 4), randn(1, 12).to(DEV), torch.zeros(4, 12, device=DEV))
    with pytest.raises(RuntimeError, match="expected Float|dtype"):
        TR.embedding_bwd_sorted(TR.token_order(i32([1]).to(DEV), 4), randn(1, 16).to(DEV), torch.zeros(4, 16, device=DEV, dtype=BF))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        L.token_logprobs(randn(2, 9).to(DEV), i32([0, 1]))


# ------------------------------------------------------------------------------------- streams, graphs, together

@pytest.mark.parametrize("T,V", [(131072, 70000), (131073, 70000), (300001, 9)])
def test_token_order_of_many_tokens(T, V):
    ids = torch.randint(-3, V + 3, (T,), generator=torch.Generator().manual_seed(T), dtype=torch.int32)
    a, b = TR.token_order(ids.to(DEV), V), TR.token_order(ids, V)
    assert torch.equal(a.perm.cpu(), b.perm) and torch.equal(a.keys.cpu(), b.keys)


def test_refuses_too_many_tokens():
    with pytest.raises(RuntimeError, match="2\\^24"):
        TR.token_order(torch.zeros((1 << 24) + 1, dtype=torch.int32, device=DEV), 5)


# ------------------------------------------------------------------------------------- offsets past 32 bits

def test_attention_offsets_past_32_bits():
    """K and V as columns of tokens 2^22 elements apart, 600 of them: 2.5e9 elements."""
    for Sq in (1, 70):
        c = Case(B=1, H=4, Hk=2, Sq=Sq, Sk=600, causal=True, q_start=[600 - Sq], fused=False, cap=4.0)
        sp = c.spec()
        want, lse = TR.attention_fwd(sp)
        wide = torch.empty(1, 600, 1 << 22, dtype=BF, device=DEV)
        for i, x in enumerate((c.k, c.v)):
            wide[0, :, 128 * i:128 * i + 128] = x[0].reshape(600, 128).to(DEV)
        sp2 = TR.AttnSpec(1, 4, Sq, 600, sp.q, (wide, 0), (wide, 128), causal=True, kv_heads=2, q_start=sp.q_start, softcap=4.0)
        got, lse2 = TR.attention_fwd(sp2)
        assert torch.equal(got, want) and torch.equal(lse, lse2)
        dout = c.dout.reshape(Sq, -1).to(DEV)
        g = [torch.empty(n, w, dtype=BF, device=DEV) for n, w in ((Sq, 256), (600, 128), (600, 128))]
        TR.attention_bwd(sp, want, dout, lse, *((x, 0) for x in g))
        dq2 = torch.empty_like(g[0])
        TR.attention_bwd(sp2, got, dout, lse2, (dq2, 0), (wide, 256), (wide, 384))
        assert torch.equal(dq2, g[0])
        assert torch.equal(wide[0, :, 256:384], g[1]) and torch.equal(wide[0, :, 384:512], g[2])
        del wide


def test_logprobs_offsets_past_32_bits():
    T, V = 66000, 33001
    x = torch.empty(T, V, dtype=BF, device=DEV)
    rows = [0, 1, T - 2, T - 1]  # rows far apart, with the same content at both ends
    part = randn(4, V, seed=3).to(DEV)
    x.zero_()
    x[rows] = part
    ids = torch.zeros(T, dtype=torch.int32, device=DEV)
    few = i32([5, 6, 7, 8]).to(DEV)
    ids[rows] = few
    r, w = L.token_logprobs(x, ids, top_k=4), L.token_logprobs(part, few, top_k=4)
    for n in ("logp", "lse", "entropy", "top_logp"):
        assert torch.allclose(getattr(r, n)[rows], getattr(w, n), rtol=1e-5, atol=1e-5), n
    assert torch.equal(r.top_ids[rows], w.top_ids)
    d = L.token_logprobs_bwd(x, ids, r, dlogp=torch.ones(T, device=DEV))
    dw = L.token_logprobs_bwd(part, few, w, dlogp=torch.ones(4, device=DEV))
    assert torch.allclose(d[rows].float(), dw.float(), rtol=2.0 ** -7, atol=1e-6)


def test_sorted_embedding_offsets_past_32_bits():
    V, W = 270000, 8192
    ids = i32([0, V - 1, 3, V - 1]).to(DEV)
    dy = randn(4, W, seed=1).to(DEV)
    dw = torch.full((V, W), math.nan, device=DEV)
    TR.embedding_bwd_sorted(TR.token_order(ids, V), dy, dw, accumulate=False)
    f = dy.float()
    assert torch.equal(dw[0], f[0]) and torch.equal(dw[3], f[2]) and torch.equal(dw[V - 1], f[1] + f[3])
    assert not dw[1:3].any() and not dw[4:V - 1].any()


def _step(ids, docs_ids, table, wqkv, targets, H, Hk, D):
    """One training step of a single attention block on packed documents, with the operators as a user
    combines them: lookup, shaped attention, logits over the shared table, token log probabilities, and
    back to the table's gradient (dense part + tokens in order)."""
    B, S = docs_ids.shape
    W = table.shape[1]
    x = TR.embedding_fwd(ids, table, scale=math.sqrt(W))
    qkv = (x.float() @ wqkv.float().t()).to(BF)
    sp = TR.AttnSpec(B, H, S, S, (qkv, 0), (qkv, H * D), (qkv, (H + Hk) * D), causal=True, kv_heads=Hk, head_dim=D,
                     softcap=10.0, docs=TR.document_spans(docs_ids))
    o, lse = TR.attention_fwd(sp)
    logits = (o.float() @ table.float().t()).to(BF)
    r = L.token_logprobs(logits, targets)
    n = targets.numel()
    dl = L.token_logprobs_bwd(logits, targets, r, dlogp=torch.full((n,), -1.0 / n, device=ids.device),
                              dentropy=torch.full((n,), -0.01 / n, device=ids.device))
    do = (dl.float() @ table.float()).to(BF)
    dtable = dl.float().t().contiguous() @ o.float()
    dqkv = torch.empty_like(qkv)
    TR.attention_bwd(sp, o, do, lse, (dqkv, 0), (dqkv, H * D), (dqkv, (H + Hk) * D))
    dw = dqkv.float().t().contiguous() @ x.float()
    dx = (dqkv.float() @ wqkv.float()).to(BF)
    TR.embedding_bwd_sorted(TR.token_order(ids, table.shape[0]), dx, dtable, scale=math.sqrt(W))
    return {"logp": r.logp, "entropy": r.entropy, "out": o, "dtable": dtable, "dw": dw, "dqkv": dqkv}


def _step_inputs(seed=0):
    B, S, H, Hk, D, V = 2, 96, 4, 2, 64, 520
    g = torch.Generator().manual_seed(seed)
    d = docs(B, S, [40, 25, 31], pad=9)
    ids = torch.randint(0, V, (B * S,), generator=g, dtype=torch.int32)
    tgt = torch.randint(0, V, (B * S,), generator=g, dtype=torch.int32)
    tgt[d.reshape(-1) < 0] = -100
    return [ids, d, randn(V, H * D, seed=seed + 1, scale=0.06), randn((H + 2 * Hk) * D, H * D, seed=seed + 2, scale=0.06), tgt], (H, Hk, D)


def _relnorm(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).norm() / (b.norm() + 1e-30))


def test_operators_together():
    ins, geo = _step_inputs()
    got, want = _step(*(t.to(DEV) for t in ins), *geo), _step(*ins, *geo)
    for n in got:
        # at most 6 roundings to bf16 lie between the inputs and any result on either side: 6 2^-8
        assert torch.isfinite(got[n]).all() and _relnorm(got[n], want[n]) < 6 * 2.0 ** -8, n


def test_operators_captured_and_replayed():
    """The step in a graph: replays on new inputs equal the eager step bit for bit, also after other eager work."""
    ins, geo = _step_inputs()
    st = [t.to(DEV) for t in ins]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _step(*st, *geo)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = _step(*st, *geo)
    for k in range(4):
        new, _ = _step_inputs(seed=10 * k)
        for a, b in zip(st, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(*(t.to(DEV) for t in new), *geo)
        for n in res:
            assert torch.equal(res[n], want[n]), (k, n)


def test_two_graphs_and_two_streams():
    """Two captured few-query attentions and sorted gradients (both use workspaces) replayed on two streams."""
    cs = [DECODE["ragged"](), DECODE["eight_tokens"]()]
    idss = [zipf(4000, 300, seed=s).to(DEV) for s in (1, 2)]
    dys = [randn(4000, 64, seed=s).to(DEV) for s in (3, 4)]

    def work(i):
        out, lse = TR.attention_fwd(specs[i])
        d = torch.empty(300, 64, device=DEV)
        TR.embedding_bwd_sorted(TR.token_order(idss[i], 300), dys[i], d, accumulate=False)
        return out, lse, d
    specs = [c.spec() for c in cs]
    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(i))
        graphs.append(g)
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
            for t in outs[i]:
                t.zero_()
    # eager, both streams at once
    for _ in range(3):
        res = []
        for i in range(2):
            streams[i].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i]):
                res.append(work(i))
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(res[i], want[i]))
