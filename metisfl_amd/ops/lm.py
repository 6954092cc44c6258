"""Operators of language-model training for models of any width, vocabulary and
type (csrc/kernels/layernorm.hip, token_logprobs.hip): LayerNorm, and the log
probabilities of given tokens with entropy and the likeliest alternatives.
``ops.bert`` holds the fixed-shape bf16 forms that the captured BERT step
runs; these take what a user module brings (float32 / bfloat16 / float16, any
row stride) and return new tensors.

Each operator has explicit ``*_fwd`` / ``*_bwd`` calls for static training
steps, whose results carry no graph, and a differentiable form for eager
modules (:func:`layer_norm`, :func:`token_logprobs`).  Device tensors always
run the HIP kernels; CPU tensors run the same formulas in PyTorch (float32, or
float64 for float64 inputs), which the GPU tests compare against.  Work is
issued on the current stream of the tensors' device and can be captured into a
hipGraph; results repeat bit for bit."""
from __future__ import annotations

from typing import NamedTuple

import torch

from metisfl_amd.ops._native import ops

TOP_MAX = 32


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows][last dimension]."""
    if t.dim() == 0:
        raise ValueError("a tensor with at least one dimension is needed")
    rows = 1
    for n in t.shape[:-1]:
        rows *= n
    return t.reshape(rows, t.shape[-1])


def _wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


# ---- LayerNorm --------------------------------------------------------------------
def _check_norm(x, gamma, beta):
    if x.shape[-1] == 0:
        raise ValueError("x has rows of no elements")
    if beta is not None and gamma is None:
        raise ValueError("beta without gamma")
    for nm, p in (("gamma", gamma), ("beta", beta)):
        if p is not None and tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"{nm} has shape {tuple(p.shape)}, expected ({x.shape[-1]},)")
        if p is not None and p.dtype not in (torch.float32, x.dtype):
            raise RuntimeError(f"{nm} must be float32 or of the input's type, got {p.dtype}")
    if beta is not None and beta.dtype != gamma.dtype:
        raise RuntimeError("gamma and beta must have the same type")


def layer_norm_fwd(x, gamma=None, beta=None, eps: float = 1e-5):
    """``(y, mean, rstd)`` of LayerNorm over the last dimension of ``x``:
    y = (x - mean) * rstd * gamma + beta in x's type, mean and rstd float32,
    one for each row.  ``gamma`` / ``beta`` are float32 or of x's type;
    without ``gamma`` the norm has no weights."""
    if x.is_cuda:
        return ops().layer_norm_fwd(x, gamma, beta, eps)
    return _layer_norm_fwd_host(x, gamma, beta, eps)


@torch.no_grad()
def _layer_norm_fwd_host(x, gamma, beta, eps):
    _check_norm(x, gamma, beta)
    w = _wide(_rows(x))
    mean = w.mean(1)
    d = w - mean[:, None]
    rstd = torch.rsqrt((d * d).mean(1) + eps)
    y = d * rstd[:, None]
    if gamma is not None:
        y = y * gamma
    if beta is not None:
        y = y + beta
    y = y.to(x.dtype)
    return y.view(x.shape), mean.view(x.shape[:-1]), rstd.view(x.shape[:-1])


def layer_norm_bwd(dy, x, mean, rstd, gamma=None):
    """``(dx, dgamma, dbeta)`` from the forward's input and statistics; the
    weights' gradients in gamma's type, None without ``gamma``.  They are
    sums in a fixed order (no atomics)."""
    if x.is_cuda:
        return ops().layer_norm_bwd(dy, x, mean, rstd, gamma)
    return _layer_norm_bwd_host(dy, x, mean, rstd, gamma)


@torch.no_grad()
def _layer_norm_bwd_host(dy, x, mean, rstd, gamma):
    _check_norm(x, gamma, None)
    if dy.shape != x.shape:
        raise ValueError(f"dy has shape {tuple(dy.shape)}, expected {tuple(x.shape)}")
    rows = x.numel() // x.shape[-1]
    for nm, s in (("mean", mean), ("rstd", rstd)):
        if s.numel() != rows:
            raise RuntimeError(f"{nm} must be contiguous with {rows} elements")
    d = _wide(_rows(dy))
    xh = (_wide(_rows(x)) - mean.reshape(-1, 1)) * rstd.reshape(-1, 1)
    u = d if gamma is None else d * gamma
    dx = rstd.reshape(-1, 1) * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    dx = dx.to(x.dtype).view(x.shape)
    if gamma is None:
        return dx, None, None
    return dx, (d * xh).sum(0).to(gamma.dtype), d.sum(0).to(gamma.dtype)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        y, mean, rstd = layer_norm_fwd(x, gamma, beta, eps)
        ctx.save_for_backward(x, gamma, mean, rstd)
        ctx.has_beta = beta is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, gamma, mean, rstd = ctx.saved_tensors
        dx, dgamma, dbeta = layer_norm_bwd(dy, x, mean, rstd, gamma)
        return dx, dgamma, dbeta if ctx.has_beta else None, None


def layer_norm(x, gamma=None, beta=None, eps: float = 1e-5):
    """Differentiable LayerNorm over the last dimension (first derivatives)."""
    return _LayerNorm.apply(x, gamma, beta, eps)


# ---- log probabilities of given tokens -----------------------------------------------
class TokenLogprobs(NamedTuple):
    """Results for each row of logits.  ``stats`` ([rows, 3]: the largest
    logit, the sum of exp(x - largest), the entropy) is what the backward
    needs."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: torch.Tensor
    top_ids: torch.Tensor
    stats: torch.Tensor


def _check_logits(logits, targets, vocab, top_k=0):
    columns = logits.shape[-1] if logits.dim() else 0
    vocab = columns if vocab is None else int(vocab)
    if not 0 < vocab <= columns:
        raise ValueError(f"vocab must be between 1 and the logits' {columns} columns, got {vocab}")
    if not 0 <= top_k <= min(TOP_MAX, vocab):
        raise ValueError(f"top_k must be between 0 and {TOP_MAX} and at most vocab, got {top_k}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, expected {tuple(logits.shape[:-1])}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}")
    return vocab


def _soft_ref(z):
    """Maximum, sum, and log probabilities of rows; a row of -inf alone has sum 0."""
    top = torch.where(z.isnan(), torch.full_like(z, float("-inf")), z).amax(1, keepdim=True)
    empty = (z == float("-inf")).all(1, keepdim=True)
    d = z - torch.where(empty, torch.zeros_like(top), top)
    e = torch.exp(d)
    return top, e, e.sum(1, keepdim=True), d, empty


def token_logprobs_fwd(logits, targets, top_k: int = 0, vocab: int | None = None) -> TokenLogprobs:
    """Softmax statistics over the first ``vocab`` columns of ``logits``
    ([..., columns]): the log probability of each row's target, the entropy
    (nats), and the ``top_k`` (at most 32) likeliest tokens with their log
    probabilities, largest first, ties to the lowest id.  All float32, ids
    int64.

    A target outside [0, vocab) marks a row without one: its logp is 0.  A
    row of nothing but -inf gives logp and top_logp -inf and entropy 0; NaN
    or +inf in a row makes its results NaN, and NaN ranks lowest among the
    alternatives.  Rows in which more than 1024 logits (256 in short rows) tie for the
    alternatives (a head initialised to zero) are read ``top_k`` times more."""
    if logits.is_cuda:
        return TokenLogprobs(*ops().token_logprobs_fwd(logits, targets, top_k, vocab))
    return _token_logprobs_fwd_host(logits, targets, top_k, vocab)


@torch.no_grad()
def _token_logprobs_fwd_host(logits, targets, top_k, vocab):
    vocab = _check_logits(logits, targets, vocab, top_k)
    lead = logits.shape[:-1]
    z, t = _wide(_rows(logits)[:, :vocab]), targets.reshape(-1).long()
    top, e, s, d, empty = _soft_ref(z)
    logs = torch.log(s)
    has = (t >= 0) & (t < vocab)
    logp = (d.gather(1, t.clamp(0, vocab - 1)[:, None]) - logs)[:, 0]
    logp = torch.where(empty[:, 0], torch.full_like(logp, float("-inf")), logp)
    logp = torch.where(has, logp, torch.zeros_like(logp))
    entropy = torch.where(empty, torch.zeros_like(s), logs - (e * d.clamp(min=-1e4)).sum(1, keepdim=True) / s)[:, 0]
    key = torch.where(z.isnan(), torch.full_like(z, float("-inf")), z)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top_k]
    top_logp = torch.where(empty, torch.full_like(s, float("-inf")), key.gather(1, ids) - top - logs)
    stats = torch.cat([top, s, entropy[:, None]], 1)
    return TokenLogprobs(logp.view(lead), entropy.view(lead), top_logp.view(*lead, top_k), ids.view(*lead, top_k),
                         stats.view(*lead, 3))


def token_logprobs_bwd(logits, targets, stats, d_logp=None, d_entropy=None, d_top=None, top_ids=None,
                       vocab: int | None = None):
    """Gradient of the logits in their type (columns from ``vocab`` on zero)
    from the forward's ``stats`` and the gradients of its results, each float32
    or None; ``d_top`` needs the forward's ``top_ids``."""
    if logits.is_cuda:
        return ops().token_logprobs_bwd(logits, targets, stats, d_logp, d_entropy, d_top, top_ids, vocab)
    return _token_logprobs_bwd_host(logits, targets, stats, d_logp, d_entropy, d_top, top_ids, vocab)


@torch.no_grad()
def _token_logprobs_bwd_host(logits, targets, stats, d_logp, d_entropy, d_top, top_ids, vocab):
    vocab = _check_logits(logits, targets, vocab)
    lead = tuple(logits.shape[:-1])
    if tuple(stats.shape) != lead + (3,):
        raise ValueError(f"stats have shape {tuple(stats.shape)}, expected {lead + (3,)}")
    for nm, v in (("d_logp", d_logp), ("d_entropy", d_entropy)):
        if v is not None and tuple(v.shape) != lead:
            raise ValueError(f"{nm} has shape {tuple(v.shape)}, expected {lead}")
    if d_top is not None and (top_ids is None or d_top.shape != top_ids.shape or tuple(d_top.shape[:-1]) != lead):
        raise ValueError("d_top needs top_ids, both with the rows' shape and one column for each alternative")
    r, t = _rows(logits), targets.reshape(-1)
    n = r.shape[0]
    flat = lambda v: None if v is None else v.reshape(-1)  # noqa: E731
    flat2 = lambda v: None if v is None else v.reshape(n, v.shape[-1])  # noqa: E731
    z, t, stats = _wide(r[:, :vocab]), t.long(), flat2(stats)
    m, s, entropy = stats[:, :1], stats[:, 1:2], stats[:, 2:]
    empty = (m == float("-inf")) & (s == 0)
    d = z - torch.where(empty, torch.zeros_like(m), m)
    p = torch.exp(d) / s
    has = (t >= 0) & (t < vocab)
    dl = torch.zeros(n, 1, dtype=z.dtype)
    if d_logp is not None:
        dl = torch.where(has, flat(d_logp).to(z.dtype), torch.zeros(n, dtype=z.dtype))[:, None]
    w = dl
    if d_top is not None:
        w = w + flat2(d_top).sum(1, keepdim=True)
    if d_entropy is not None:
        w = w + flat(d_entropy)[:, None] * (d.clamp(min=-1e4) - torch.log(s) + entropy)
    g = (-p * w).scatter_add(1, t.clamp(0, vocab - 1)[:, None], dl)
    if d_top is not None:
        g = g.scatter_add(1, flat2(top_ids), flat2(d_top).to(g.dtype))
    g = torch.where(empty, torch.zeros_like(g), g)
    out = torch.zeros(n, r.shape[1], dtype=logits.dtype)
    out[:, :vocab] = g.to(logits.dtype)
    return out.view(logits.shape)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, vocab):
        r = token_logprobs_fwd(logits, targets, top_k, vocab)
        ctx.save_for_backward(logits, targets, r.stats, r.top_ids)
        ctx.vocab, ctx.top_k = vocab, top_k
        ctx.mark_non_differentiable(r.top_ids, r.stats)
        ctx.set_materialize_grads(False)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logp, d_entropy, d_top, _ids, _stats):
        logits, targets, stats, ids = ctx.saved_tensors
        if d_logp is None and d_entropy is None and (d_top is None or ctx.top_k == 0):
            return None, None, None, None
        dx = token_logprobs_bwd(logits, targets, stats, d_logp, d_entropy, d_top if ctx.top_k else None, ids,
                                ctx.vocab)
        return dx, None, None, None


def token_logprobs(logits, targets, top_k: int = 0, vocab: int | None = None) -> TokenLogprobs:
    """Differentiable :func:`token_logprobs_fwd` (first derivatives of
    ``logp``, ``entropy`` and ``top_logp``).  The mean negative log
    likelihood of the rows that have a target is
    ``-r.logp.sum() / has_target.sum()``."""
    return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k, vocab))
