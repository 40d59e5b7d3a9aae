"""Fused softmax cross-entropy forward+backward (csrc/kernels/loss.hip); token log probabilities with
entropy and alternatives, and their gradient (csrc/kernels/logprobs.hip)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import lib, on_gpu


def softmax_xent(logits: torch.Tensor, labels: torch.Tensor, smoothing: float = 0.0, ignore_index: int = -100,
                 scale: float = 1.0, want_grad: bool = True, want_correct: bool = False, V: int | None = None):
    """Returns (per-row loss f32 [B], dlogits bf16 [B,ld] = scale*(softmax - target) or None, correct f32 [B] or None).
    V < logits.shape[1]: only the first V columns are classes (vocab padded to a multiple of 128);
    the padding columns of dlogits are zero."""
    B, ld = logits.shape
    V = ld if V is None else V
    if not on_gpu(logits):
        if V < ld:
            loss, d, corr = softmax_xent(logits[:, :V], labels, smoothing, ignore_index, scale, want_grad, want_correct)
            if d is not None:
                dp = torch.zeros(B, ld, dtype=torch.bfloat16)
                dp[:, :V] = d
                d = dp
            return loss, d, corr
        x = logits.float()
        lse = torch.logsumexp(x, dim=1)
        valid = (labels != ignore_index) & (labels >= 0) & (labels < V)
        lab = labels.clamp(0, V - 1).long()
        nll = lse - x.gather(1, lab[:, None])[:, 0]
        smooth = lse - x.mean(1)
        loss = torch.where(valid, (1 - smoothing) * nll + smoothing * smooth, torch.zeros_like(lse))
        d = None
        if want_grad:
            p = torch.softmax(x, dim=1)
            t = torch.full_like(p, smoothing / V)
            t.scatter_add_(1, lab[:, None], torch.full((B, 1), 1 - smoothing))
            d = (scale * (p - t) * valid[:, None]).to(torch.bfloat16)
        corr = ((x.argmax(1) == lab) & valid).float() if want_correct else None
        return loss, d, corr
    loss = torch.empty(B, dtype=torch.float32, device=logits.device)
    # the register kernel writes the padding columns itself; only the streaming kernel needs a zeroed buffer
    full = V == ld or bool(lib().xent_full_row(V, ld))
    d = (torch.empty_like(logits) if full else torch.zeros_like(logits)) if want_grad else None
    corr = torch.empty(B, dtype=torch.float32, device=logits.device) if want_correct else None
    lib().softmax_xent(logits, labels, B, V, ld, smoothing, ignore_index, scale, loss, d, corr)
    return loss, d, corr


class TokenLogprobs(NamedTuple):
    """token_logprobs of [T, V] logits: f32 [T] logp, entropy (nats) and lse; with top_k, f32 top_logp and
    int32 top_ids [T, top_k], most probable first, equal logits by the lower id. norm f32 [T, 2] (largest
    logit and the log of the sum over it) is what the backward reads."""
    logp: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logp: torch.Tensor | None
    top_ids: torch.Tensor | None
    norm: torch.Tensor


TOP_K_MAX = 32


def _logprob_args(logits, ids, V, top_k, ignore_index):
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"token_logprobs: logits must be [T, V] bf16 / f16 / f32, got {logits.dtype} {tuple(logits.shape)}")
    V = logits.shape[1] if V is None else V
    if not 1 <= V <= logits.shape[1]:
        raise ValueError(f"token_logprobs: {V} classes of {logits.shape[1]} columns")
    if not 0 <= top_k <= min(TOP_K_MAX, V):
        raise ValueError(f"token_logprobs: top_k must be in 0..{min(TOP_K_MAX, V)}, got {top_k}")
    if ids.dtype != torch.int32 or ids.numel() != logits.shape[0]:
        raise ValueError(f"token_logprobs: ids must be int32 [{logits.shape[0]}], got {ids.dtype} {tuple(ids.shape)}")
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("token_logprobs: logits need unit stride along the classes")
    # an ignore_index that no int32 id can equal ignores nothing (-1 is outside [0, V) already)
    return V, ids.reshape(-1).contiguous(), ignore_index if -2 ** 31 <= ignore_index < 2 ** 31 else -1


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, V: int | None = None, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of ids[t] (int32) under softmax(logits[t, :V]), with the entropy of that
    distribution and its top_k (0..32) alternatives, in one read of the logits (bf16 / f16 / f32, rows any
    stride apart; columns from V on are padding). ids equal to ignore_index or outside [0, V) have logp 0
    (their entropy and alternatives are computed all the same). -inf logits are classes of probability 0; a
    row of nothing else has logp -inf, entropy 0. NaN or +inf in a row make its results NaN."""
    V, ids, ignore_index = _logprob_args(logits, ids, V, top_k, ignore_index)
    if not on_gpu(logits):
        x = logits[:, :V].float()
        m = x.amax(1, keepdim=True)
        none = m == float("-inf")
        ls = torch.where(none, 0.0, torch.log(torch.exp(x - m.masked_fill(none, 0.0)).sum(1, keepdim=True)))
        lp = torch.where(none, float("-inf"), (x - m) - ls)
        p = torch.exp(lp)
        ent = -torch.where(p > 0, p * lp, p * 0.0).sum(1)
        ok = (ids != ignore_index) & (ids >= 0) & (ids < V)
        logp = torch.where(ok, lp.gather(1, ids.clamp(0, V - 1).long()[:, None])[:, 0], 0.0)
        tl = ti = None
        if top_k:
            ti = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top_k]
            tl, ti = lp.gather(1, ti), ti.to(torch.int32)
        return TokenLogprobs(logp, ent, (m + ls)[:, 0], tl, ti, torch.cat([m, ls], 1))
    logp, ent, lse, norm, tl, ti = lib().logprobs_fwd(logits, ids, V, top_k, ignore_index)
    return TokenLogprobs(logp, ent, lse, tl, ti, norm)


def token_logprobs_bwd(logits: torch.Tensor, ids: torch.Tensor, saved: TokenLogprobs, dlogp: torch.Tensor | None = None,
                       dentropy: torch.Tensor | None = None, dtop: torch.Tensor | None = None, V: int | None = None,
                       ignore_index: int = -100) -> torch.Tensor:
    """Gradient of token_logprobs with respect to the logits, in their type and shape (columns from V on
    are zero): dlogp and dentropy f32 [T], dtop f32 [T, k] (of saved.top_logp), each optional. Ignored ids
    take no dlogp. One read of the logits, one write of the gradient."""
    k = 0
    if dtop is not None:
        if saved.top_ids is None or dtop.shape != saved.top_ids.shape:
            raise ValueError("token_logprobs_bwd: dtop needs the alternatives of token_logprobs(top_k=...), same shape")
        k = dtop.shape[1]
    V, ids, ignore_index = _logprob_args(logits, ids, V, k, ignore_index)
    T, cols = logits.shape
    for n, g, shape in (("dlogp", dlogp, (T,)), ("dentropy", dentropy, (T,)), ("dtop", dtop, (T, k))):
        if g is not None and (g.dtype != torch.float32 or tuple(g.shape) != shape):
            raise ValueError(f"token_logprobs_bwd: {n} must be f32 {list(shape)}, got {g.dtype} {list(g.shape)}")
    if not on_gpu(logits):
        x = logits[:, :V].float()
        m, ls = saved.norm[:, :1], saved.norm[:, 1:]
        lp = torch.where(m == float("-inf"), float("-inf"), (x - m) - ls)
        p = torch.exp(lp)
        ok = (ids != ignore_index) & (ids >= 0) & (ids < V)
        up = torch.zeros_like(x)
        if dlogp is not None:
            up.scatter_add_(1, ids.clamp(0, V - 1).long()[:, None], torch.where(ok, dlogp, 0.0)[:, None])
        if dtop is not None:
            up.scatter_add_(1, saved.top_ids.long(), dtop)
        d = up - p * up.sum(1, keepdim=True)
        if dentropy is not None:
            d = d - dentropy[:, None] * torch.where(p > 0, p * (lp + saved.entropy[:, None]), p * 0.0)
        out = torch.zeros(T, cols, dtype=logits.dtype)
        out[:, :V] = d.to(logits.dtype)
        return out
    c = lambda t: t.contiguous() if t is not None else None  # noqa: E731
    return lib().logprobs_bwd(logits, ids, V, ignore_index, saved.norm, saved.entropy, saved.top_ids if k else None,
                              c(dlogp), c(dentropy), c(dtop) if k else None)
