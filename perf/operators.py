"""Cases of the language-model operators: attention with shaped scores (tanh cap, distance bias,
document and prefix masks, shared key/value heads), log probabilities of given tokens with entropy
and top alternatives, and the embedding gradient by sorted tokens.

A case is a dict of plain values. ``prepare`` makes its inputs on the GPU, ``run`` makes one pass:
in elementary float32 torch operations, or (``own``) through the framework's entry points.
``exact`` is the definition in float64.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------- the cases

def _attn(name, **kw):
    c = {"name": name, "op": "attention", "dtype": "bf16", "B": 1, "H": 16, "Hk": 16, "D": 64, "Sq": 1, "Sk": 1,
         "train": False, "causal": True, "cap": 0.0, "slopes": False, "doc": 0, "prefix": 0, "ragged": False}
    c.update(kw)
    return c


def _logp(name, **kw):
    c = {"name": name, "op": "logprobs", "dtype": "bf16", "T": 1, "V": 2, "ld": 0, "k": 0, "train": False}
    c.update(kw)
    c["ld"] = c["ld"] or c["V"]
    return c


def _emb(name, **kw):
    c = {"name": name, "op": "embedding", "dtype": "bf16", "T": 1, "W": 64, "V": 64, "scale": 1.0}
    c.update(kw)
    return c


def listed():
    return [
        # a small model's training step on short packed rows: several sentences share a row of 256 tokens
        _attn("attn_train_short", B=8, H=8, Hk=8, D=64, Sq=256, Sk=256, doc=96, train=True),
        # pretraining on packed documents, the heads and width of a big encoder-decoder
        _attn("attn_train_packed", B=4, H=16, Hk=16, D=64, Sq=2048, Sk=2048, doc=512, train=True),
        # one long sequence with capped scores and four query heads on each key head
        _attn("attn_train_capped", B=1, H=16, Hk=4, D=128, Sq=8192, Sk=8192, cap=30.0, train=True),
        # scoring of odd-length rows under a prefix mask with a distance bias, in half precision
        _attn("attn_prefix_bias", dtype="f16", B=3, H=12, Hk=12, D=64, Sq=1531, Sk=1531, slopes=True, prefix=400),
        # one new token of one request over a short cache: latency
        _attn("attn_decode_one", B=1, H=16, Hk=16, D=64, Sq=1, Sk=777, slopes=True, ragged=True),
        # one new token of sixteen requests over long ragged caches, eight key heads for 32 query heads
        _attn("attn_decode_long", B=16, H=32, Hk=8, D=128, Sq=1, Sk=16384, cap=50.0, ragged=True),
        # a serving step: eight rows, the chosen token's log probability and 20 alternatives
        _logp("logp_serve", T=8, V=33708, ld=33792, k=20),
        # scoring of an evaluation set over a wide vocabulary in float32 with five alternatives
        _logp("logp_score", dtype="f32", T=1021, V=131072, k=5),
        # a training step on token log probabilities with an entropy term: forward and gradient
        _logp("logp_train", T=8192, V=33708, ld=33792, train=True),
        # the gradient of a small table for a short odd batch
        _emb("emb_short", T=333, W=512, V=4099, scale=math.sqrt(512.0)),
        # the gradient of a padded shared table for one training batch of a big encoder-decoder
        _emb("emb_batch", T=8192, W=1024, V=33792, scale=32.0),
        # a long batch of packed documents over a wide vocabulary
        _emb("emb_long", T=65536, W=768, V=131072),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "logprobs", "embedding"])
    if op == "attention":
        D = rng.choice([64, 128])
        Hk = rng.choice([1, 2, 4, 8, 12])
        G = rng.choice([1, 1, 2, 4])
        c = _attn("", dtype=rng.choice(["bf16", "f16"]), H=Hk * G, Hk=Hk, D=D, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                  slopes=rng.random() < 0.3)
        if rng.random() < 0.4:  # a few new tokens over a cache
            c.update(Sq=rng.choice([1, 1, 1, 3, 8]), Sk=_log(rng, 32, 16384), B=_log(rng, 1, 16), ragged=True)
        else:
            S = _log(rng, 17, 4096)
            most = max(1, 200_000_000 // (Hk * G * S * S))
            c.update(Sq=S, Sk=S, B=_log(rng, 1, min(16, most)), train=rng.random() < 0.7)
            kind = rng.choice(["causal", "doc", "prefix", "full"])
            c.update(causal=kind != "full", doc=max(8, S // rng.choice([2, 4, 8])) if kind == "doc" else 0,
                     prefix=S // 3 + 1 if kind == "prefix" else 0)
        del c["name"]
        return c
    if op == "logprobs":
        V = _log(rng, 200, 131072)
        c = _logp("", dtype=rng.choice(["bf16", "f16", "f32"]), V=V, ld=rng.choice([0, (V + 127) // 128 * 128]),
                  T=_log(rng, 1, min(8192, max(2, 130_000_000 // V))), k=rng.choice([0, 1, 5, 20]), train=rng.random() < 0.5)
    else:
        W = 8 * _log(rng, 8, 128)
        c = _emb("", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), T=_log(rng, 1, 65536), W=W, V=_log(rng, 100, 90000),
                 scale=rng.choice([1.0, math.sqrt(W)]))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------- the inputs

def _documents(B, S, mean, seed):
    """Document ids of packed rows: runs of mean/2 to 3 mean/2 tokens, and a padded tail (-1) of up
    to a sixteenth of the row."""
    rng = random.Random(seed)
    rows = []
    for _ in range(B):
        row, n = [], S - rng.randint(0, S // 16)
        while len(row) < n:
            row += [len(row)] * min(rng.randint(max(1, mean // 2), mean + mean // 2), n - len(row))
        rows.append(row + [-1] * (S - n))
    return rows


def _lengths(B, Sq, Sk, seed):
    """Filled lengths of ragged caches, from half full to full (the first one is full)."""
    rng = random.Random(seed)
    return [Sk] + [rng.randint(max(Sq, Sk // 2), Sk) if Sk > Sq else Sk for _ in range(B - 1)]


def _slopes(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    st = {"case": case}
    if case["op"] == "attention":
        B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
        if Sq == Sk:  # one fused projection: q | k | v columns of each token
            st["q"] = st["k"] = st["v"] = randn(B * Sq, (H + 2 * Hk) * D)
            st["cols"] = (0, H * D, (H + Hk) * D)
        else:  # a projected query and the two caches
            st["q"], st["k"], st["v"] = randn(B * Sq, H * D), randn(B * Sk, Hk * D), randn(B * Sk, Hk * D)
            st["cols"] = (0, 0, 0)
        st["doc_ids"] = ints(_documents(B, Sk, case["doc"], seed)) if case["doc"] else None
        st["kv_len"] = st["q_start"] = st["prefix_len"] = st["slopes"] = None
        if case["ragged"]:
            st["kv_len"] = ints(_lengths(B, Sq, Sk, seed))
            st["q_start"] = st["kv_len"] - Sq
        if case["prefix"]:
            rng = random.Random(seed)
            st["prefix_len"] = ints([rng.randint(0, case["prefix"]) for _ in range(B)])
        if case["slopes"]:
            st["slopes"] = torch.tensor(_slopes(H), dtype=torch.float32, device=DEV)
        if case["train"]:
            st["dout"] = randn(B * Sq, H * D)
    elif case["op"] == "logprobs":
        T, V, ld, k = (case[n] for n in ("T", "V", "ld", "k"))
        st["logits"] = randn(T, ld, scale=2.5)
        st["ids"] = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
        st["ids"][torch.rand(T, generator=g, device=DEV) < 0.03] = -100  # prompt and padding tokens
        if case["train"]:
            st["dlogp"] = randn(T, dtype=torch.float32)
            st["dentropy"] = randn(T, scale=0.01, dtype=torch.float32)
            st["dtop"] = randn(T, k, scale=0.1, dtype=torch.float32) if k else None
    else:
        T, W, V = (case[n] for n in ("T", "W", "V"))
        u = torch.rand(T, generator=g, device=DEV, dtype=torch.float64)  # token ids by Zipf's law
        rank = (torch.exp(u * math.log(V + 1.0)).long() - 1).clamp(0, V - 1)
        st["ids"] = torch.randperm(V, generator=g, device=DEV)[rank].to(torch.int32)
        st["ids"][torch.rand(T, generator=g, device=DEV) < 0.02] = -1  # padding
        st["dy"] = randn(T, W)
        st["dword"] = torch.empty(V, W, dtype=torch.float32, device=DEV)
    return st


# ------------------------------------------------------------------------------------- one pass

def run(st):
    op = st["case"]["op"]
    if own:
        return _own_attention(st) if op == "attention" else _own_logprobs(st) if op == "logprobs" else _own_embedding(st)
    return _plain_attention(st) if op == "attention" else _plain_logprobs(st) if op == "logprobs" else _plain_embedding(st)


def _own_attention(st):
    from tensorflow_k8s_amd.ops import transformer as TR
    c = st["case"]
    docs = TR.document_spans(st["doc_ids"]) if st["doc_ids"] is not None else None
    q, k, v = ((st[n], col) for n, col in zip("qkv", st["cols"]))
    sp = TR.AttnSpec(c["B"], c["H"], c["Sq"], c["Sk"], q, k, v, kv_len=st["kv_len"], causal=c["causal"],
                     kv_heads=c["Hk"], head_dim=c["D"], softcap=c["cap"], slopes=st["slopes"], docs=docs,
                     prefix_len=st["prefix_len"], q_start=st["q_start"])
    out, lse = TR.attention_fwd(sp)
    res = {"out": out, "lse": lse}
    if c["train"]:
        d = torch.empty_like(st["q"])
        TR.attention_bwd(sp, out, st["dout"], lse, *((d, col) for col in st["cols"]))
        res["dqkv"] = d
    return res


def _own_logprobs(st):
    from tensorflow_k8s_amd.ops import loss as L
    c = st["case"]
    r = L.token_logprobs(st["logits"], st["ids"], V=c["V"], top_k=c["k"])
    res = {"logp": r.logp, "entropy": r.entropy}
    if c["k"]:
        res["top_logp"], res["top_ids"] = r.top_logp, r.top_ids
    if c["train"]:
        res["dlogits"] = L.token_logprobs_bwd(st["logits"], st["ids"], r, dlogp=st["dlogp"], dentropy=st["dentropy"],
                                              dtop=st["dtop"], V=c["V"])
    return res


def _own_embedding(st):
    from tensorflow_k8s_amd.ops import transformer as TR
    c = st["case"]
    order = TR.token_order(st["ids"], c["V"])
    TR.embedding_bwd_sorted(order, st["dy"], st["dword"], scale=c["scale"], accumulate=False)
    return {"dword": st["dword"], "order": order.perm}


def _visible(st):
    """Which keys each query sees: bool [B or 1, 1, 1, Sq, Sk], and the positions' distance."""
    c = st["case"]
    B, Sq, Sk = c["B"], c["Sq"], c["Sk"]
    j = torch.arange(Sk, device=DEV)
    p = torch.arange(Sq, device=DEV)[None, :] + (st["q_start"][:, None] if st["q_start"] is not None else 0)
    ok = torch.ones(1, Sq, Sk, dtype=torch.bool, device=DEV)
    if c["causal"]:
        ok = j[None, None, :] <= p[:, :, None]
        if st["prefix_len"] is not None:
            ok = ok | (j[None, None, :] < st["prefix_len"][:, None, None])
    if st["kv_len"] is not None:
        ok = ok & (j[None, None, :] < st["kv_len"][:, None, None])
    if st["doc_ids"] is not None:
        d = st["doc_ids"]
        ok = ok & (d[:, :, None] == d[:, None, :]) & (d[:, :, None] >= 0)
    return ok[:, None, None], (p[:, :, None] - j[None, None, :]).abs()[:, None, None]


def _plain_attention(st):
    c = st["case"]
    B, H, Hk, D, Sq, Sk = (c[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
    G, scale, cap = H // Hk, 1.0 / math.sqrt(D), c["cap"]

    def heads(n, i, S, N):  # [B, Hk, G, S, D]
        x = st[n][:, st["cols"][i]:st["cols"][i] + N * D]
        return x.float().reshape(B, S, Hk, N // Hk, D).permute(0, 2, 3, 1, 4)

    q, k, v = heads("q", 0, Sq, H), heads("k", 1, Sk, Hk), heads("v", 2, Sk, Hk)
    ok, dist = _visible(st)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    if cap:
        t = torch.tanh(s / cap)
        s = cap * t
    if st["slopes"] is not None:
        s = s - st["slopes"].reshape(1, Hk, G, 1, 1) * dist
    s = s.masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    del s
    l = p.sum(-1, keepdim=True)
    p = p / l.masked_fill(l == 0, 1.0)
    o = torch.matmul(p, v)
    lse = torch.where(l > 0, m + torch.log(l), math.inf)
    dt = st["q"].dtype

    def tokens(x, S, N):
        return x.permute(0, 3, 1, 2, 4).reshape(B * S, N * D)

    res = {"out": tokens(o, Sq, H).to(dt), "lse": lse.reshape(B, H, Sq)}
    if c["train"]:
        do = st["dout"].float().reshape(B, Sq, Hk, G, D).permute(0, 2, 3, 1, 4)
        ds = p * (torch.matmul(do, v.transpose(-1, -2).contiguous()) - (do * o).sum(-1, keepdim=True))
        if cap:
            ds = ds * (1.0 - t * t)
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).sum(2, keepdim=True) * scale
        dv = torch.matmul(p.transpose(-1, -2).contiguous(), do).sum(2, keepdim=True)
        res["dqkv"] = torch.cat([tokens(dq, Sq, H), tokens(dk, Sk, Hk), tokens(dv, Sk, Hk)], 1).to(dt)
    return res


def _first_k(x, k):
    """The k largest values of each row and their places, equal values by the lowest place."""
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    return v[:, :k], i[:, :k]


def _plain_logprobs(st):
    c = st["case"]
    T, V, ld, k = (c[n] for n in ("T", "V", "ld", "k"))
    x, ids = st["logits"][:, :V].float(), st["ids"].long()
    ok = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1)[:, None]
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    lp = x - lse
    p = torch.exp(lp)
    ent = -(p * lp).sum(1)
    res = {"logp": torch.where(ok, lp.gather(1, at)[:, 0], 0.0), "entropy": ent}
    if k:
        tv, ti = _first_k(x, k)
        res["top_logp"], res["top_ids"] = tv - lse, ti.to(torch.int32)
    if c["train"]:
        glp = torch.where(ok, st["dlogp"], 0.0)[:, None]
        tot = glp + (st["dtop"].sum(1, keepdim=True) if k else 0.0)
        d = -p * (tot + st["dentropy"][:, None] * (lp + ent[:, None]))
        d.scatter_add_(1, at, glp)
        if k:
            d.scatter_add_(1, ti, st["dtop"])
        res["dlogits"] = torch.cat([d, d.new_zeros(T, ld - V)], 1).to(st["logits"].dtype)
    return res


def _plain_embedding(st):
    c = st["case"]
    T, W, V = (c[n] for n in ("T", "W", "V"))
    ids = st["ids"].long()
    key = torch.where((ids >= 0) & (ids < V), ids, V)
    perm = torch.sort(key, stable=True).indices
    d = torch.zeros(V + 1, W, dtype=torch.float32, device=DEV)
    d.index_add_(0, key, st["dy"].float() * c["scale"])
    return {"dword": d[:V], "order": perm.to(torch.int32)}


# ------------------------------------------------------------------------------------- what it takes

def _pairs(c):
    """Visible (query, key) pairs of one head, over the whole batch, of a typical seed."""
    B, Sq, Sk = c["B"], c["Sq"], c["Sk"]
    if c["ragged"]:
        return sum(n * Sq - (Sq * (Sq - 1) // 2 if c["causal"] else 0) for n in _lengths(B, Sq, Sk, 0))
    if c["doc"]:
        n = 0
        for row in _documents(B, Sk, c["doc"], 0):
            runs = {}
            for d in row:
                if d >= 0:
                    runs[d] = runs.get(d, 0) + 1
            n += sum(r * (r + 1) // 2 if c["causal"] else r * r for r in runs.values())
        return n
    n = Sk * (Sk + 1) // 2 if c["causal"] else Sq * Sk
    return B * (n + (c["prefix"] // 2) * (c["prefix"] // 2) // 2)


def work(case):
    c, e = case, {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if c["op"] == "attention":
        B, H, Hk, D, Sq, Sk = (c[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
        kv = sum(_lengths(B, Sq, Sk, 0)) if c["ragged"] else B * Sk
        b = 2 * B * Sq * H * D * e + 2 * kv * Hk * D * e + 4 * B * H * Sq
        f = 4 * _pairs(c) * H * D
        if c["train"]:  # dout in, the three gradients out; five more products
            b += (2 * B * Sq * H + 2 * B * Sk * Hk) * D * e
            f += 10 * _pairs(c) * H * D
        return {"bytes": b, "flops": f}
    if c["op"] == "logprobs":
        T, V, ld, k = (c[n] for n in ("T", "V", "ld", "k"))
        b, f = T * V * e + T * (12 + 8 * k), 6 * T * V
        if c["train"]:  # the gradient's columns; the logits are already counted
            b += T * ld * e + T * (8 + 4 * k)
            f += 8 * T * V
        return {"bytes": b, "flops": f}
    T, W, V = (c[n] for n in ("T", "W", "V"))
    return {"bytes": T * W * e + 8 * T + 4 * V * W, "flops": 2 * T * W}


# ------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["op"] == "embedding":
        ids, out = st["ids"].long(), torch.zeros(c["V"], c["W"], dtype=torch.float64, device=DEV)
        use = (ids >= 0) & (ids < c["V"])
        out.index_put_((ids[use],), st["dy"][use].double() * c["scale"], accumulate=True)
        return {"dword": out, "order": None}
    if c["op"] == "logprobs":
        return _exact_logprobs(st)
    return _exact_attention(st)


def _exact_logprobs(st):
    c = st["case"]
    V, k, parts = c["V"], c["k"], []
    step = max(1, 200_000_000 // V)
    for r in range(0, c["T"], step):
        x, ids = st["logits"][r:r + step, :V].double(), st["ids"][r:r + step].long()
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        use = ((ids >= 0) & (ids < V)).double()
        hot = torch.zeros_like(x).scatter_(1, ids.clamp(0, V - 1)[:, None], use[:, None])
        ent = torch.special.entr(p).sum(1)
        one = {"logp": (hot * lp).sum(1), "entropy": ent}
        if k:
            top = _first_k(x, k)[1]
            one["top_logp"] = lp.gather(1, top)
        if c["train"]:
            up = hot * st["dlogp"][r:r + step, None].double()
            if k:
                up.scatter_add_(1, top, st["dtop"][r:r + step].double())
            d = up - p * up.sum(1, keepdim=True)
            d -= st["dentropy"][r:r + step, None].double() * p * (lp + ent[:, None])
            one["dlogits"] = torch.nn.functional.pad(d, (0, c["ld"] - V))
        parts.append(one)
    out = {n: torch.cat([o[n] for o in parts]) for n in parts[0]}
    if k:
        out["top_ids"] = None
    return out


def _exact_attention(st):
    c = st["case"]
    B, H, Hk, D, Sq, Sk = (c[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
    G = H // Hk
    ok, dist = _visible(st)
    ok, dist = ok[:, 0, 0].expand(B, Sq, Sk), dist[:, 0, 0].expand(B, Sq, Sk)
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H, Sq), math.inf, dtype=torch.float64, device=DEV)
    grad = torch.zeros(B, Sk, H + 2 * Hk, D, dtype=torch.float64, device=DEV) if c["train"] else None

    def head(n, i, b, S, h):
        x = st[n].reshape(B, S, -1)[b]
        return x[:, st["cols"][i] + h * D:st["cols"][i] + (h + 1) * D].double()

    for b in range(B):
        blind = ~ok[b].any(1)
        for h in range(H):
            q, k, v = head("q", 0, b, Sq, h), head("k", 1, b, Sk, h // G), head("v", 2, b, Sk, h // G)
            z = (q @ k.T.contiguous()) / math.sqrt(D)
            slope = 1.0
            if c["cap"]:
                th = torch.tanh(z / c["cap"])
                z, slope = c["cap"] * th, 1.0 - th * th
            if st["slopes"] is not None:
                z = z - st["slopes"][h].double() * dist[b]
            z = z.masked_fill(~ok[b], -math.inf)
            norm = torch.logsumexp(z, 1)
            p = torch.exp(z - norm.masked_fill(blind, 0.0)[:, None])
            out[b, :, h] = p @ v
            lse[b, h] = norm.masked_fill(blind, math.inf)
            if c["train"]:
                do = st["dout"].reshape(B, Sq, H, D)[b, :, h].double()
                dp = do @ v.T.contiguous()
                dz = p * (dp - (p * dp).sum(1, keepdim=True)) * slope / math.sqrt(D)
                grad[b, :, h] = dz @ k
                grad[b, :, H + h // G] += dz.T.contiguous() @ q
                grad[b, :, H + Hk + h // G] += p.T.contiguous() @ do
    res = {"out": out.reshape(B * Sq, H * D), "lse": lse}
    if c["train"]:
        res["dqkv"] = grad.reshape(B * Sk, (H + 2 * Hk) * D)
    return res
