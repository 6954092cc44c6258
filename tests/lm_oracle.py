"""The definitions of the language-model training operators in 64 bits, for
the tests of ops.lm and ops.optim.MultiTensorAdamW."""
import torch


def half_step(t):
    """Largest relative error of one rounding to ``t``."""
    return torch.finfo(t).eps / 2


def layer_norm(x, gamma, beta, eps, dy=None):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    y = xh * w + (0 if beta is None else beta.double())
    out = {"y": y, "mean": mean[..., 0], "rstd": rstd[..., 0], "xh": xh}
    if dy is not None:
        dy = dy.double()
        u = dy * w
        out["dx"] = rstd * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
        lead = tuple(range(x.dim() - 1))
        out["dgamma"], out["dbeta"] = (dy * xh).sum(lead), dy.sum(lead)
        out["dgamma_abs"], out["dbeta_abs"] = (dy * xh).abs().sum(lead), dy.abs().sum(lead)
    return out


def token_logprobs(logits, targets, k, vocab):
    """Rows with at least one finite logit and no NaN / +inf."""
    z = logits[..., :vocab].double()
    lp = torch.log_softmax(z, -1)
    p = lp.exp()
    has = (targets >= 0) & (targets < vocab)
    at = targets.long().clamp(0, vocab - 1)[..., None]
    logp = torch.where(has, lp.gather(-1, at)[..., 0], 0.0)
    entropy = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :k]
    return {"logp": logp, "entropy": entropy, "top_ids": ids, "top_logp": lp.gather(-1, ids), "lp": lp, "has": has}


def token_logprobs_grad(logits, targets, k, vocab, d_logp, d_entropy, d_top):
    o = token_logprobs(logits, targets, k, vocab)
    lp, p, has = o["lp"], o["lp"].exp(), o["has"]
    g = torch.zeros(logits.shape, dtype=torch.float64, device=logits.device)
    z = g[..., :vocab]
    at = targets.long().clamp(0, vocab - 1)[..., None]
    if d_logp is not None:
        d = torch.where(has, d_logp.double(), 0.0)[..., None]
        z -= p * d
        z.scatter_add_(-1, at, d)
    if d_entropy is not None:
        z -= d_entropy.double()[..., None] * p * (torch.where(p > 0, lp, 0.0) + o["entropy"][..., None])
    if d_top is not None:
        z -= p * d_top.double().sum(-1, keepdim=True)
        z.scatter_add_(-1, o["top_ids"], d_top.double())
    return g


def adamw(p, g, m, v, t, lr, b1, b2, eps, wd):
    p, g = p.double(), g.double()
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    return p - lr * (m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + eps) + wd * p), m, v
