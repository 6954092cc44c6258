"""Timed cases of the operators around the matrix products of a language-model
learner's training step: LayerNorm (forward, backward, weight gradients), the
log probability of given tokens with entropy and the likeliest alternatives
(and its gradient), and the AdamW step over many tensors with 32-bit or 8-bit
states.

``listed()`` names the cases, ``draw(rng)`` makes further ones of the same
ranges, ``prepare`` builds what a program holds before the call, ``run`` makes
one pass: with ``own`` through ``metisfl_amd.ops``, without it through
elementary torch operations in 32 bits.  ``exact`` evaluates the operators'
definitions in 64 bits."""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases ------------------------------------------------------------------------
def listed():
    return [
        # one token's hidden state of an answering model: latency alone counts
        dict(name="ln-token", op="layer_norm", rows=1, width=768, gap=0, dtype="fp32", back=False),
        # 128 sequences of 128 tokens through a base encoder's norm, forward and backward
        dict(name="ln-train-768", op="layer_norm", rows=16384, width=768, gap=0, dtype="bf16", back=True),
        # a user module with an odd width, its input a slice of a wider tensor, in half precision
        dict(name="ln-odd-1001", op="layer_norm", rows=4099, width=1001, gap=7, dtype="fp16", back=True),
        # the widest: long batches of a wide model held in 32 bits
        dict(name="ln-wide-5120", op="layer_norm", rows=24576, width=5120, gap=0, dtype="fp32", back=True),
        # the next token of one sequence over a word-piece vocabulary, five alternatives
        dict(name="lp-token", op="token_logprobs", rows=1, vocab=30522, columns=30528, dtype="bf16", top=5,
             back=False, entropy=False),
        # 20 masked positions of 128 sequences: the masked-token loss and its gradient
        dict(name="lp-masked", op="token_logprobs", rows=2560, vocab=30522, columns=30528, dtype="bf16", top=0,
             back=True, entropy=False),
        # scoring an odd number of answers in 32 bits with twenty alternatives each
        dict(name="lp-score-20", op="token_logprobs", rows=509, vocab=50021, columns=50021, dtype="fp32", top=20,
             back=False, entropy=False),
        # the largest: a long batch over a large vocabulary, loss with an entropy term
        dict(name="lp-large", op="token_logprobs", rows=8192, vocab=128000, columns=128000, dtype="bf16", top=4,
             back=True, entropy=True),
        # the dense image classifier of a small learner: six tensors
        dict(name="adamw-small", op="adamw", layout="dense", tensors=6, spread=0, bits=32, param="fp32", grad="fp32",
             mirror=False),
        # a base encoder: about 200 tensors, bf16 gradients and a bf16 copy of the weights
        dict(name="adamw-encoder", op="adamw", layout="encoder", tensors=199, spread=0, bits=32, param="fp32",
             grad="bf16", mirror=True),
        # the same encoder with its states in 8 bits
        dict(name="adamw8-encoder", op="adamw", layout="encoder", tensors=199, spread=0, bits=8, param="fp32",
             grad="bf16", mirror=True),
        # many ragged tensors of a user module in bf16, states in 8 bits
        dict(name="adamw8-ragged", op="adamw", layout="ragged", tensors=83, spread=11, bits=8, param="bf16",
             grad="fp32", mirror=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "token_logprobs", "adamw"])
    if op == "layer_norm":
        width = _log(rng, 16, 8192)
        rows = _log(rng, 1, min(65536, 60_000_000 // width))
        return dict(op=op, rows=rows, width=width, gap=rng.choice([0, 0, 0, 1, 24]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), back=rng.random() < 0.7)
    if op == "token_logprobs":
        vocab = _log(rng, 32, 200_000)
        rows = _log(rng, 1, min(16384, 400_000_000 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, columns=vocab + rng.choice([0, 0, 1, -vocab % 64]),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), top=rng.choice([0, 1, 5, rng.randint(2, 32)]),
                    back=rng.random() < 0.6, entropy=rng.random() < 0.3)
    return dict(op=op, layout="ragged", tensors=_log(rng, 1, 300), spread=rng.randrange(1, 1 << 20),
                bits=rng.choice([32, 8]), param=rng.choice(["fp32", "fp32", "bf16"]),
                grad=rng.choice(["fp32", "bf16", "fp16"]), mirror=False)


def _sizes(case):
    """Element counts of an optimizer case's tensors, and which of them decay."""
    if case["layout"] == "dense":  # 784-128-128-10
        shapes = [(128, 784), (128,), (128, 128), (128,), (10, 128), (10,)]
    elif case["layout"] == "encoder":  # embeddings, twelve layers, masked-token head
        h, f, v = 768, 4 * 768, 30528
        shapes = [(v, h), (512, h), (2, h), (h,), (h,)]
        for _ in range(12):
            shapes += [(3 * h, h), (3 * h,), (h, h), (h,), (h,), (h,), (f, h), (f,), (h, f), (h,), (h,), (h,)]
        shapes += [(h, h), (h,), (h,), (h,), (v,)]
    else:
        r, shapes, left = random.Random(case["spread"]), [], 48_000_000
        for _ in range(case["tensors"]):
            n = min(_log(r, 1, 3_000_000), max(1, left))
            left -= n
            shapes.append((n,) if r.random() < 0.5 else (1, n))
    return [math.prod(s) for s in shapes], [len(s) > 1 for s in shapes]


def work(case):
    if case["op"] == "layer_norm":
        n, e = case["rows"] * case["width"], SIZE[case["dtype"]]
        w = 4 * case["width"]
        b = 2 * n * e + 8 * case["rows"] + 2 * w
        if case["back"]:
            b += 3 * n * e + 8 * case["rows"] + 3 * w
        return {"bytes": b, "flops": n * (22 if case["back"] else 8)}
    if case["op"] == "token_logprobs":
        n, e = case["rows"] * case["vocab"], SIZE[case["dtype"]]
        b = n * e + case["rows"] * (8 + 8 + 12 * case["top"])
        if case["back"]:
            b += n * e + case["rows"] * (case["columns"] * e + 24)
        return {"bytes": b, "flops": n * (12 if case["back"] else 6)}
    n = sum(_sizes(case)[0])
    state = 16 if case["bits"] == 32 else 4 + 4 * 4 / 128
    return {"bytes": n * (2 * SIZE[case["param"]] + SIZE[case["grad"]] + state + (2 if case["mirror"] else 0)),
            "flops": n * 16}


# ---- inputs -----------------------------------------------------------------------
BLOCK = 128  # elements that share a scale of the 8-bit states
HYPER = dict(learning_rate=2e-4, beta1=0.9, beta2=0.999, epsilon=1e-6, weight_decay=0.01)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _prepare_norm(case, g):
    m, h, t = case["rows"], case["width"], TYPES[case["dtype"]]
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    # hidden states: per-column offsets, a few columns much larger than the others
    col = torch.where(torch.rand(h, generator=g, device=DEV) < 0.01, 8.0, 1.0)
    full = torch.empty(m, h + case["gap"], dtype=t, device=DEV)
    full.copy_(r(m, h + case["gap"]))
    x = full[:, :h]
    x.mul_(col.to(t)).add_((0.3 * r(h)).to(t))
    s = dict(case=case, x=x, gamma=1 + 0.1 * r(h), beta=0.1 * r(h), eps=1e-5)
    if case["back"]:
        s["dy"] = (r(m, h) * 0.05).to(t)
    return s


def _prepare_logprobs(case, g):
    n, v, c, t = case["rows"], case["vocab"], case["columns"], TYPES[case["dtype"]]
    logits = torch.empty(n, c, dtype=t, device=DEV)
    logits.normal_(0.0, 2.0, generator=g)
    target = torch.randint(0, v, (n,), generator=g, device=DEV)
    # the model knows most tokens: their logit stands out
    lift = 6.0 + 4.0 * torch.rand(n, 1, generator=g, device=DEV)
    logits.scatter_add_(1, target[:, None], lift.to(t))
    # some positions carry no token (padding)
    target = torch.where(torch.rand(n, generator=g, device=DEV) < (0.05 if n > 1 else 0.0), -1, target)
    s = dict(case=case, logits=logits, target=target)
    if case["back"]:
        s["d_logp"] = -(0.5 + torch.rand(n, generator=g, device=DEV)) / n
        s["d_entropy"] = -0.01 * torch.rand(n, generator=g, device=DEV) / n if case["entropy"] else None
    return s


def _prepare_adamw(case, g):
    sizes, decay = _sizes(case)
    start, at = [], 0
    for n in sizes:
        start.append(at)
        at += -(-n // BLOCK) * BLOCK
    flat = torch.zeros(at, dtype=TYPES[case["param"]], device=DEV)
    live = torch.zeros(at, dtype=torch.bool, device=DEV)
    params = [flat[a:a + n] for a, n in zip(start, sizes)]
    for a, n in zip(start, sizes):
        live[a:a + n] = True
    flat.copy_(0.02 * torch.randn(at, generator=g, device=DEV) * live)
    size = torch.exp(torch.empty(len(sizes), device=DEV).uniform_(-9, -4, generator=g)).tolist()
    grads = [(torch.randn(n, generator=g, device=DEV) * z).to(TYPES[case["grad"]]) for n, z in zip(sizes, size)]
    # moments in the middle of a run: of the gradients' size, spread over magnitudes
    z = torch.cat([torch.full((-(-n // BLOCK) * BLOCK,), y, device=DEV) for n, y in zip(sizes, size)])
    z = z * torch.exp(torch.randn(at, generator=g, device=DEV)) * live
    m, v = 0.2 * z * torch.randn(at, generator=g, device=DEV), z * z
    s = dict(case=case, flat=flat, params=params, grads=grads, sizes=sizes, seed=12345, decay=decay,
             wd=torch.cat([torch.full((-(-n // BLOCK) * BLOCK,), HYPER["weight_decay"] if d else 0.0, device=DEV)
                           for n, d in zip(sizes, decay)]),
             mirror=flat.to(torch.bfloat16) if case["mirror"] else None, start=start,
             step=torch.full((1,), 10, dtype=torch.int32, device=DEV))
    if case["bits"] == 8:  # codes at the nearest value: any state of the format will do here
        for name, val in (("m", m), ("v", v.sqrt())):
            top = val.view(-1, BLOCK).abs().amax(1)
            scale = _power((torch.frexp(top)[1] - 8).clamp(-117, 120))
            code = (val.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
            s[name], s[name + "_scale"] = code, scale
    else:
        s["m"], s["v"] = m, v
    if own:  # the program's own optimizer object, resumed in the middle of its run
        from metisfl_amd.ops.optim import MultiTensorAdamW, OptimizerSpec
        mirrors = [s["mirror"][a:a + n] for a, n in zip(start, sizes)] if case["mirror"] else None
        s["opt"] = MultiTensorAdamW(OptimizerSpec("adam_weight_decay", **HYPER), params, state_bits=case["bits"],
                                    decay=decay, mirrors=mirrors, seed=s["seed"])
        s["opt"].load_state_dict({k: s[k] for k in ("step", "m", "v", "m_scale", "v_scale") if k in s})
    return s


def prepare(case, seed):
    g = _gen(seed)
    return {"layer_norm": _prepare_norm, "token_logprobs": _prepare_logprobs, "adamw": _prepare_adamw}[case["op"]](case, g)


# ---- the plain forms --------------------------------------------------------------
def _norm_plain(s):
    x, gamma, beta = s["x"].float(), s["gamma"], s["beta"]
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + s["eps"])
    xh = xc * rstd
    t = s["x"].dtype
    out = {"y": (xh * gamma + beta).to(t), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if "dy" in s:
        dy = s["dy"].float()
        u = dy * gamma
        dx = rstd * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
        out |= {"dx": dx.to(t), "dgamma": (dy * xh).sum(0), "dbeta": dy.sum(0)}
    return out


def _top_plain(z, k):
    """The k largest of each row, ties to the lowest index: one sortable whole number for each element."""
    b = (z + 0.0).view(torch.int32)
    b = (b ^ ((b >> 31) & 0x7FFFFFFF)).long()
    key = b * (1 << 32) + ((1 << 32) - 1 - torch.arange(z.shape[1], device=z.device))
    key = torch.topk(key, k, dim=1).values
    return (1 << 32) - 1 - (key & 0xFFFFFFFF)


def _logprobs_plain(s):
    case, v = s["case"], s["case"]["vocab"]
    z = s["logits"][:, :v].float()
    top = z.amax(1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    has = (s["target"] >= 0) & (s["target"] < v)
    at = s["target"].clamp(0, v - 1)[:, None]
    logp = torch.where(has, (d.gather(1, at) - log_total)[:, 0], 0.0)
    entropy = (log_total - (e * d).sum(1, keepdim=True) / total)
    out = {"logp": logp, "entropy": entropy[:, 0]}
    if case["top"]:
        ids = _top_plain(z.contiguous(), case["top"])
        out |= {"top_logp": d.gather(1, ids) - log_total, "top_ids": ids}
    if case["back"]:
        dl = torch.where(has, s["d_logp"], 0.0)[:, None]
        p = e / total
        dz = -p * dl
        if s["d_entropy"] is not None:
            dz = dz - s["d_entropy"][:, None] * p * ((d - log_total) + entropy)
        dz.scatter_add_(1, at, dl)
        full = torch.zeros_like(s["logits"])
        full[:, :v] = dz
        out["dlogits"] = full
    return out


def _mix(x):
    """32 mixed bits of a whole number below 2^32 (held in 64 bits)."""
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _power(exp):
    """2 to a whole power between -126 and 127, exactly."""
    return ((exp + 127) << 23).view(torch.float32)


def _unpacked(code, scale):
    return (code.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _packed(x, dither, least):
    """8-bit codes (e4m3) of x and a power of two for each block: the largest lies in [128, 256), what
    lies between two codes goes up with the dither's chance. `least`: nothing above zero becomes zero."""
    top = x.abs().view(-1, BLOCK).amax(1)
    exp = (torch.frexp(top)[1] - 8).clamp(-117, 120)
    exp = torch.where(top > 0, exp, -117)
    y = (x.abs().view(-1, BLOCK) * _power(-exp)[:, None]).view(-1)
    low = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)
    q = (((y + low).view(torch.int32) + (dither << 4).int()) & ~0xFFFFF).view(torch.float32) - low
    if least:
        q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q)
    return torch.copysign(q, x).to(torch.float8_e4m3fn), _power(exp)


def _adamw_plain(s):
    case, h = s["case"], HYPER
    s["step"] += 1
    t = s["step"].double()
    c1 = (1.0 / (1.0 - h["beta1"] ** t)).float()
    c2 = (1.0 / torch.sqrt(1.0 - h["beta2"] ** t)).float()
    g = torch.cat([torch.nn.functional.pad(x.float(), (0, -x.numel() % BLOCK)) for x in s["grads"]])
    small = case["bits"] == 8
    m = _unpacked(s["m"], s["m_scale"]) if small else s["m"]
    v = _unpacked(s["v"], s["v_scale"]) if small else s["v"]
    v = v * v if small else v
    m = m * h["beta1"] + g * (1.0 - h["beta1"])
    v = v * h["beta2"] + (g * (1.0 - h["beta2"])) * g
    r = torch.sqrt(v)
    p = s["flat"].float()
    p = p - ((m * c1) / (r * c2 + h["epsilon"]) + p * s["wd"]) * h["learning_rate"]
    if small or case["param"] == "bf16":
        at = torch.arange(p.numel(), device=p.device)
        key = _mix((s["step"].long() ^ s["seed"]) & 0xFFFFFFFF)
        bits = _mix(((at & 0xFFFFFFFF) ^ key) + (at >> 32) * 0x9E3779B1 & 0xFFFFFFFF)
    if small:
        for name, val, part in (("m", m, bits & 0xFFFF), ("v", r, bits >> 16)):
            code, scale = _packed(val, part, name == "v")
            s[name].copy_(code)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if case["param"] == "bf16":
        more = _mix(bits) >> 16
        p = ((p.view(torch.int32) + more.int()) & ~0xFFFF).view(torch.float32)
    s["flat"].copy_(p)
    out = {"params": s["flat"], "m": s["m"], "v": s["v"]}
    if small:
        out |= {"m_scale": s["m_scale"], "v_scale": s["v_scale"]}
    if s["mirror"] is not None:
        s["mirror"].copy_(p.to(torch.bfloat16))
        out["mirror"] = s["mirror"]
    return out


# ---- one pass -----------------------------------------------------------------------
def _norm_own(s):
    from metisfl_amd.ops import lm
    y, mean, rstd = lm.layer_norm_fwd(s["x"], s["gamma"], s["beta"], s["eps"])
    out = {"y": y, "mean": mean, "rstd": rstd}
    if "dy" in s:
        dx, dgamma, dbeta = lm.layer_norm_bwd(s["dy"], s["x"], mean, rstd, s["gamma"])
        out |= {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    return out


def _logprobs_own(s):
    from metisfl_amd.ops import lm
    case = s["case"]
    r = lm.token_logprobs_fwd(s["logits"], s["target"], top_k=case["top"], vocab=case["vocab"])
    out = {"logp": r.logp, "entropy": r.entropy}
    if case["top"]:
        out |= {"top_logp": r.top_logp, "top_ids": r.top_ids}
    if case["back"]:
        out["dlogits"] = lm.token_logprobs_bwd(s["logits"], s["target"], r.stats, d_logp=s["d_logp"],
                                               d_entropy=s["d_entropy"], vocab=case["vocab"])
    return out


def _adamw_own(s):
    opt = s["opt"]
    opt.step(s["grads"])
    out = {"params": s["flat"], "m": opt.m, "v": opt.v}
    if s["case"]["bits"] == 8:
        out |= {"m_scale": opt.m_scale, "v_scale": opt.v_scale}
    if s["mirror"] is not None:
        out["mirror"] = s["mirror"]
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _norm_own, "token_logprobs": _logprobs_own, "adamw": _adamw_own}[op](state)
    return {"layer_norm": _norm_plain, "token_logprobs": _logprobs_plain, "adamw": _adamw_plain}[op](state)


# ---- the definitions in 64 bits -------------------------------------------------------
def _norm_exact(s):
    x, w = s["x"].double(), s["gamma"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    inv = (var + s["eps"]).rsqrt()
    n = (x - mean) * inv
    out = {"y": n * w + s["beta"].double(), "mean": mean.squeeze(1), "rstd": inv.squeeze(1)}
    if "dy" in s:
        dy = s["dy"].double()
        dn = dy * w
        h = x.shape[1]
        out["dx"] = inv / h * (h * dn - dn.sum(1, keepdim=True) - n * (dn * n).sum(1, keepdim=True))
        out["dgamma"], out["dbeta"] = torch.einsum("ij,ij->j", dy, n), dy.sum(0)
    return out


def _logprobs_exact(s):
    case, v, k = s["case"], s["case"]["vocab"], s["case"]["top"]
    rows, out = s["logits"].shape[0], {"logp": [], "entropy": []}
    if k:
        out |= {"top_logp": [], "top_ids": None}
    if case["back"]:
        out["dlogits"] = []
    for a in range(0, rows, 1024):
        part = slice(a, a + 1024)
        lp = torch.log_softmax(s["logits"][part, :v].double(), 1)
        p, target = lp.exp(), s["target"][part]
        has = ((target >= 0) & (target < v)).double()
        at = target.clamp(0, v - 1).unsqueeze(1)
        h = -(p * lp).sum(1)
        out["logp"].append(lp.gather(1, at).squeeze(1) * has)
        out["entropy"].append(h)
        if k:
            out["top_logp"].append(lp.topk(k, 1).values)
        if case["back"]:
            dl = s["d_logp"][part].double() * has
            dz = torch.zeros(lp.shape[0], case["columns"], dtype=torch.float64, device=lp.device)
            dz[:, :v] -= p * dl.unsqueeze(1)
            if s["d_entropy"] is not None:
                dz[:, :v] -= p * (lp + h.unsqueeze(1)) * s["d_entropy"][part].double().unsqueeze(1)
            dz[torch.arange(lp.shape[0], device=lp.device), at.squeeze(1)] += dl
            out["dlogits"].append(dz)
    return {n: torch.cat(x) if x is not None else None for n, x in out.items()}


def _bits_exact(a):
    """The mixing of a whole number's 32 bits, by remainders."""
    a = a * 2654435761 % 4294967296
    a = a ^ torch.div(a, 32768, rounding_mode="floor")
    a = a * 1779033703 % 4294967296
    return a ^ torch.div(a, 65536, rounding_mode="floor")


def _code_exact(x, chance, least):
    """Codes of the 8-bit format: whole steps of an eighth of the binade, the rest up by chance."""
    b = x.reshape(-1, BLOCK)
    power = torch.floor(torch.log2(b.abs().amax(1).clamp_min(1e-300))) - 7
    y = (b / torch.exp2(power.clamp(-117, 120)).unsqueeze(1)).reshape(-1)
    size = y.abs()
    unit = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))) - 3)
    code = torch.floor(size / unit + chance) * unit
    if least:
        code = torch.where(size > 0, torch.maximum(code, torch.full_like(code, 2.0 ** -9)), code)
    return code * torch.sign(y)


def _adamw_exact(s):
    case, lr, b1, b2 = s["case"], HYPER["learning_rate"], HYPER["beta1"], HYPER["beta2"]
    t = int(s["step"]) + 1
    n = s["flat"].numel()
    g = torch.zeros(n, dtype=torch.float64, device=DEV)
    for a, x in zip(s["start"], s["grads"]):
        g[a:a + x.numel()] = x.double()
    if case["bits"] == 8:
        m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (s["v"].double() * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = s["flat"].double()
    p = p - lr * (m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + HYPER["epsilon"]) + s["wd"].double() * p)
    out = {"params": p}
    key = _bits_exact(torch.tensor([t ^ s["seed"]], device=DEV))
    if case["bits"] == 8 or case["param"] == "bf16":
        bits = _bits_exact(torch.arange(n, device=DEV) ^ key)
    if case["param"] == "bf16":  # between two bf16 values: up by chance
        unit = torch.exp2(torch.floor(torch.log2(p.abs().clamp_min(1e-30))) - 7)
        more = torch.div(_bits_exact(bits), 65536, rounding_mode="floor").double() / 65536
        out["params"] = torch.floor(p.abs() / unit + more) * unit * torch.sign(p)
    if case["bits"] == 8:
        out["m"] = _code_exact(m, (bits % 65536).double() / 65536, False)
        out["v"] = _code_exact(v.sqrt(), torch.div(bits, 65536, rounding_mode="floor").double() / 65536, True)
        # a power of two that turns on the last bit of the block's largest: no value in between to be near to
        out |= {"m_scale": None, "v_scale": None}
    else:
        out |= {"m": m, "v": v}
    if s["mirror"] is not None:
        out["mirror"] = p
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _norm_exact, "token_logprobs": _logprobs_exact, "adamw": _adamw_exact}[case["op"]](s)
