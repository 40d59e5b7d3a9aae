"""Float64 oracles of the language-model operators, written from their definitions, with bounds on what
the kernels' roundings may add. u(t) is half a step of type t relative to the value; F covers the float32
arithmetic of a score, its exponential and a row sum (|x| 2^-24 per operation on exponents of at most ~100)."""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}  # half the smallest f16 step
F = 2e-5


def visible(B, Sq, Sk, causal=False, kv_len=None, q_start=None, prefix_len=None, doc_ids=None):
    """bool [B, Sq, Sk] and the positions [B, Sq], pair by pair from the rule."""
    ok = torch.zeros(B, Sq, Sk, dtype=torch.bool)
    pos = torch.zeros(B, Sq, dtype=torch.long)
    for b in range(B):
        n = min(int(kv_len[b]), Sk) if kv_len is not None else Sk
        run = None
        if doc_ids is not None:
            ids = doc_ids[b].tolist()
            run = [0] * Sk
            for j in range(1, Sk):
                run[j] = run[j - 1] + (ids[j] != ids[j - 1])
        j = torch.arange(Sk)
        for i in range(Sq):
            p = i + (int(q_start[b]) if q_start is not None else 0)
            pos[b, i] = p
            row = j < n
            if causal:
                row = row & ((j <= p) | (j < (int(prefix_len[b]) if prefix_len is not None else 0)))
            if run is not None:
                if 0 <= p < Sk and ids[p] >= 0:
                    row = row & (torch.tensor(run) == run[p])
                else:
                    row = row & False
            ok[b, i] = row
    return ok, pos


def attention(q, k, v, ok, pos, scale, cap=0.0, slopes=None, dout=None, keep=None, dtype=torch.bfloat16):
    """q [B,Sq,H,D], k, v [B,Sk,Hk,D] -> dict of f64 results and bounds. keep: [B,H,Sq,Sk] dropout factor."""
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    u, tiny = U[dtype], TINY[dtype]
    r = {"out": torch.zeros(B, Sq, H, D, dtype=torch.float64), "lse": torch.full((B, H, Sq), math.inf, dtype=torch.float64)}
    r["out_bound"] = torch.zeros_like(r["out"])
    grads = dout is not None
    if grads:
        for n, ref in (("dq", q), ("dk", k), ("dv", v)):
            r[n] = torch.zeros(ref.shape, dtype=torch.float64)
            r[n + "_bound"] = torch.zeros(ref.shape, dtype=torch.float64)
    for b in range(B):
        m = ok[b]
        live_q, live_k = m.any(1), m.any(0)
        for h in range(H):
            # places that no pair uses may hold anything
            Q = torch.where(live_q[:, None], q[b, :, h].double(), 0.0)
            K = torch.where(live_k[:, None], k[b, :, h * Hk // H].double(), 0.0)
            V = torch.where(live_k[:, None], v[b, :, h * Hk // H].double(), 0.0)
            z = (Q @ K.T) * scale
            der = torch.ones_like(z)
            if cap:
                th = torch.tanh(z / cap)
                z, der = cap * th, 1.0 - th * th
            if slopes is not None:
                z = z - slopes[h].double() * (pos[b][:, None] - torch.arange(Sk)[None, :]).abs()
            z = z.masked_fill(~m, -math.inf)
            lse = torch.logsumexp(z, 1)
            p = torch.where(live_q[:, None], torch.exp(z - torch.where(live_q, lse, 0.0)[:, None]), 0.0)
            kp = keep[b, h].double() if keep is not None else torch.ones_like(p)
            pd = p * kp
            o = pd @ V
            r["out"][b, :, h] = o
            r["lse"][b, h] = torch.where(live_q, lse, math.inf)
            # P rounded for the product, the sum, the output rounded
            # (f16 P relative to its row maximum: a subnormal step of the unnormalised P, over l >= 1)
            r["out_bound"][b, :, h] = (u + F) * (pd @ V.abs()) + u * o.abs() + tiny * (m.double() @ V.abs() + 1)
            if not grads:
                continue
            dO = torch.where(live_q[:, None], dout[b, :, h].double(), 0.0)
            dP = (dO @ V.T) * kp
            delta = (dO * o).sum(1, keepdim=True)
            ds = p * (dP - delta) * der
            mag = p * ((dO.abs() @ V.abs().T) * kp + (dO.abs() * o.abs()).sum(1, keepdim=True))
            # dS rounded; delta from the rounded output; float32 on the terms of the difference
            eds = u * ds.abs() + F * mag + u * p * (dO.abs() * (o.abs() + r["out_bound"][b, :, h])).sum(1, keepdim=True) + tiny * m
            eds = eds + p * (dO.abs() * r["out_bound"][b, :, h]).sum(1, keepdim=True)
            g = h * Hk // H
            r["dq"][b, :, h] = ds @ K * scale
            r["dq_bound"][b, :, h] = eds @ K.abs() * scale + tiny
            r["dk"][b, :, g] += ds.T @ Q * scale
            r["dk_bound"][b, :, g] += eds.T @ Q.abs() * scale + tiny
            r["dv"][b, :, g] += pd.T @ dO
            r["dv_bound"][b, :, g] += (u + F) * (pd.T @ dO.abs()) + tiny * (m.double().T @ dO.abs() + 1)
    if grads:
        for n in ("dq", "dk", "dv"):
            r[n + "_bound"] += u * r[n].abs() + u * r[n + "_bound"]
    return r


def within(got, want, bound, what=""):
    """|got - want| <= bound everywhere; no NaN."""
    d = (got.double().cpu() - want).abs()
    bad = ~(d <= bound + 1e-12)
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        i = tuple(at)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: got {float(got.cpu()[i])}, "
                             f"want {float(want[i])} +- {float(bound[i])}")


def logprobs(x, ids, V, k=0, dlogp=None, dent=None, dtop=None, ignore=-100):
    """f64 results of [T, cols] logits; ids ignored or out of range: logp 0, no dlogp."""
    x = x[:, :V].double()
    T = x.shape[0]
    use = (ids >= 0) & (ids < V) & (ids != ignore)
    at = ids.clamp(0, V - 1).long()
    m = x.amax(1)  # lse alone would lose the log of the sum where |m| is large, in 64 bits too
    dead = m == -math.inf
    ls = torch.where(dead, 0.0, torch.log(torch.exp(x - torch.where(dead, 0.0, m)[:, None]).sum(1)))
    lse = m + ls
    lp = torch.where(dead[:, None], -math.inf, (x - m[:, None]) - ls[:, None])
    p = lp.exp()
    ent = torch.where(p > 0, -p * lp, 0.0).sum(1)
    r = {"lse": lse, "entropy": ent, "logp": torch.where(use, lp[torch.arange(T), at], 0.0)}
    up = torch.zeros_like(x)
    if dlogp is not None:
        up[torch.arange(T), at] += torch.where(use, dlogp.double(), 0.0)
    if k:
        # the k best by (value down, column up)
        r["top_ids"] = torch.tensor([sorted(range(V), key=lambda c, t=t: (-float(x[t, c]), c))[:k] for t in range(T)])
        r["top_logp"] = lp.gather(1, r["top_ids"])
        if dtop is not None:
            up.scatter_add_(1, r["top_ids"], dtop.double())
    tot = up.sum(1, keepdim=True)
    gh = dent.double()[:, None] if dent is not None else 0.0
    fin = torch.where(p > 0, lp, 0.0)
    r["dlogits"] = up - p * (tot + gh * (fin + ent[:, None]))
    g = gh.abs() if dent is not None else 0.0
    r["mag"] = up.abs() + p * (up.abs().sum(1, keepdim=True) + g * (fin.abs() + ent[:, None] + 1.0))
    return r
