"""Fused flat-buffer optimizers (K3/K4/K5).

One launch updates EVERY trainable variable of a learner: the fp32 master
weights, the optimizer slots and the bf16 compute copy.  The optimizer kinds
and their hyper-parameters mirror ``OptimizerConfig`` of the reference
(metisfl/proto/model.proto:116-151, applied in
metisfl/models/keras/keras_model_ops.py:245-283):

* ``vanilla_sgd``      p -= lr * (g + l2*p + l1*sign(p))
* ``momentum_sgd``     v = mu*v - lr*g ; p += v            (Keras form)
* ``fed_prox``         p -= lr * (g + mu*(p - p_community))
* ``adam``             bias-corrected Adam (Keras default eps 1e-7)
* ``adam_weight_decay`` Adam + decoupled weight decay

:class:`MultiTensorAdamW` is the Adam / AdamW step over a user module's own
tensors (any sizes and types, no flat buffer), with states in 32 or 8 bits.

FedProx note: the reference's Keras FedProx keeps its ``vstar`` slot at zero
(fed_prox.py:44-60); here the anchor is the community
model received for the round, which is the algorithm's intended semantics.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from metisfl_amd.ops._native import ops

OPT_SGD, OPT_MOMENTUM, OPT_FEDPROX, OPT_ADAM, OPT_ADAMW = range(5)
_KIND = {
    "vanilla_sgd": OPT_SGD,
    "momentum_sgd": OPT_MOMENTUM,
    "fed_prox": OPT_FEDPROX,
    "adam": OPT_ADAM,
    "adam_weight_decay": OPT_ADAMW,
}


@dataclass
class OptimizerSpec:
    kind: str = "vanilla_sgd"
    learning_rate: float = 0.01
    l1: float = 0.0
    l2: float = 0.0
    momentum: float = 0.0
    proximal_term: float = 0.0
    beta1: float = 0.9
    beta2: float = 0.999
    epsilon: float = 1e-7
    weight_decay: float = 0.0
    extra: dict = field(default_factory=dict)

    @property
    def mode(self) -> int:
        return _KIND[self.kind]

    @property
    def needs_m(self) -> bool:
        return self.mode in (OPT_MOMENTUM, OPT_ADAM, OPT_ADAMW)

    @property
    def needs_v(self) -> bool:
        return self.mode in (OPT_ADAM, OPT_ADAMW)

    @property
    def needs_anchor(self) -> bool:
        return self.mode == OPT_FEDPROX

    @classmethod
    def from_proto(cls, pb) -> "OptimizerSpec":
        """Build from a ``metisfl.OptimizerConfig`` message."""
        which = pb.WhichOneof("config")
        if which is None:
            raise ValueError("OptimizerConfig has no optimizer set")
        c = getattr(pb, which)
        if which == "vanilla_sgd":
            return cls(which, c.learning_rate, l1=c.L1_reg, l2=c.L2_reg)
        if which == "momentum_sgd":
            return cls(which, c.learning_rate, momentum=c.momentum_factor)
        if which == "fed_prox":
            return cls(which, c.learning_rate, proximal_term=c.proximal_term)
        if which == "adam":
            return cls(which, c.learning_rate, beta1=c.beta_1 or 0.9, beta2=c.beta_2 or 0.999,
                       epsilon=c.epsilon or 1e-7)
        if which == "adam_weight_decay":
            return cls(which, c.learning_rate, weight_decay=c.weight_decay)
        raise ValueError(f"unsupported optimizer {which}")


def fused_step(spec: OptimizerSpec, p: torch.Tensor, g: torch.Tensor,
               m: torch.Tensor | None = None, v: torch.Tensor | None = None,
               anchor: torch.Tensor | None = None, p16: torch.Tensor | None = None,
               lr_scale: torch.Tensor | None = None, step: torch.Tensor | None = None,
               zero_grad: bool = False, zero_region: torch.Tensor | None = None,
               tick: bool = False) -> None:
    """Apply one optimizer step in place over flat buffers.  ``zero_grad``
    writes 0 back into ``g`` once consumed and ``zero_region`` (e.g. the
    BatchNorm accumulators) is cleared by the same launch, so the next step's
    atomic accumulations start from zero without a memset node.
    ``tick``: also increment ``step`` once, after the optimizer has read it
    (inside the same launch for the modes that never read it)."""
    if p.is_cuda:
        ops().fused_optimizer(spec.mode, p, g, m, v, anchor, p16, spec.learning_rate, spec.l1,
                              spec.l2, spec.momentum, spec.proximal_term, spec.beta1, spec.beta2,
                              spec.epsilon, spec.weight_decay, lr_scale, step, zero_grad,
                              zero_region, tick)
        return
    _reference_step(spec, p, g, m, v, anchor, p16, lr_scale, step)
    if zero_grad:
        g.zero_()
    if zero_region is not None:
        zero_region.zero_()
    if tick:
        step.add_(1)


class OptRange:
    """One fused optimizer step over a range of the flat model (views of the
    master, gradient, slots, anchor and weight mirror): the unit an
    optimizer tail carries (conv32.h OptTail -- the range's update rides in a
    later layer's paired backward launch).  ``run()`` is the stand-alone
    launch (fallback paths)."""

    def __init__(self, spec: OptimizerSpec, p, g, m=None, v=None, anchor=None, mirror=None,
                 lr_scale=None, step=None, zero_grad: bool = True):
        self.spec, self.p, self.g, self.m, self.v = spec, p, g, m, v
        self.anchor, self.mirror, self.lr_scale, self.step, self.zero_grad = anchor, mirror, lr_scale, step, zero_grad

    @property
    def numel(self) -> int:
        return int(self.p.numel())

    def hyper(self) -> list[float]:
        s = self.spec
        return [s.learning_rate, s.l1, s.l2, s.momentum, s.proximal_term, s.beta1, s.beta2, s.epsilon,
                s.weight_decay]

    def binding_args(self) -> tuple:
        """The trailing optimizer-tail arguments of conv32_backward_pair."""
        return (self.p, self.g, self.m, self.v, self.anchor, self.mirror, self.lr_scale, self.step,
                self.spec.mode, self.hyper(), self.zero_grad)

    def run(self) -> None:
        fused_step(self.spec, self.p, self.g, self.m, self.v, self.anchor, self.mirror, self.lr_scale, self.step,
                   zero_grad=self.zero_grad)


STATE_BLOCK = 128  # elements that share a scale of MultiTensorAdamW's 8-bit states


class MultiTensorAdamW:
    """Adam / AdamW over a list of tensors, the whole step in one launch (up to a
    million elements) or two, and one more for each further 384 tensors
    (csrc/kernels/multi_adamw.hip).

    ``params``: contiguous float32 or bfloat16 tensors on one device, updated
    in place, no two of them sharing memory; they and their mirrors keep storage,
    size and type for the optimizer's life (a step refuses one that was moved,
    cut or cast).  ``decay``: which of them take ``spec.weight_decay`` (default:
    all).  A step goes by the values that ``spec`` has then.  ``mirrors``: a
    bfloat16 copy of each parameter (or None) that the step refreshes.
    ``lr_scale``: a float32 device tensor of one element that the step
    multiplies the learning rate with.

    The states are flat buffers, each tensor's segment padded to a multiple of
    128 elements: ``m`` and ``v`` float32 (``state_bits=32``), or
    (``state_bits=8``, a quarter of the memory) float8_e4m3fn codes of m and
    of sqrt(v), whose values are codes times ``m_scale`` / ``v_scale``, one
    power of two for each 128 elements.  What lies between two codes is
    rounded up with the chance of its distance, drawn from a mix of ``seed``,
    step and place: equal seeds give equal results.  bfloat16 parameters are
    rounded the same way.  ``step_count`` is an int32 device tensor.  The
    tensors may be written in place; putting another in an attribute's place is
    refused.

    :meth:`step` can be captured into a hipGraph with the gradients of the
    captured backward; the graph keeps the spec's values (``lr_scale`` is read
    by every replay) and points into the optimizer's states and tables: keep the
    optimizer as long as the graph is replayed."""

    def __init__(self, spec: OptimizerSpec, params, *, state_bits: int = 32, decay=None, mirrors=None,
                 lr_scale: torch.Tensor | None = None, seed: int = 0):
        _adam_decay(spec)
        if state_bits not in (32, 8):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        self.spec, self.params, self.state_bits, self.seed = spec, tuple(params), state_bits, int(seed) & 0xFFFFFFFF
        if not self.params:
            raise ValueError("no parameters")
        n = len(self.params)
        decay = [True] * n if decay is None else [bool(d) for d in decay]
        self.mirrors = (None,) * n if mirrors is None else tuple(mirrors)
        if len(decay) != n or len(self.mirrors) != n:
            raise ValueError(f"decay and mirrors must have one entry for each of the {n} parameters")
        dev = self.params[0].device
        for p, q in zip(self.params, self.mirrors):
            if p.dtype not in (torch.float32, torch.bfloat16) or not p.is_contiguous() or p.device != dev:
                raise ValueError("parameters must be contiguous float32 or bfloat16 tensors on one device")
            if q is not None and (q.dtype != torch.bfloat16 or not q.is_contiguous() or q.device != dev
                                  or q.numel() != p.numel()):
                raise ValueError("a mirror must be a contiguous bfloat16 tensor of its parameter's size and device")
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                       for t in self.params + self.mirrors if t is not None and t.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("parameters and mirrors must not share memory (list a tied weight once)")
        self.decay = tuple(decay)
        offsets, total = [], 0
        for p in self.params:
            offsets.append(total)
            total += -(-p.numel() // STATE_BLOCK) * STATE_BLOCK
        self.offsets = tuple(offsets)
        zeros = lambda k, t: torch.zeros(k, dtype=t, device=dev)  # noqa: E731
        st = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.m, self.v = zeros(total, st), zeros(total, st)
        self.m_scale, self.v_scale = (zeros(total // STATE_BLOCK, torch.float32) if state_bits == 8 else None
                                      for _ in range(2))
        self.step_count = zeros(1, torch.int32)
        self.lr_scale = lr_scale
        if dev.type != "cuda" and lr_scale is not None and (
                lr_scale.dtype != torch.float32 or lr_scale.numel() != 1 or lr_scale.device != dev):
            raise ValueError("lr_scale must be a float32 tensor of one element on the parameters' device")
        self._plan = None
        self._held = [_storage_of(t) for t in self.params + self.mirrors]
        if dev.type == "cuda":
            self._plan = ops().AdamPlan(self.params, self.mirrors, self.decay, self.m, self.v,
                                        self.m_scale, self.v_scale, self.step_count, lr_scale, self.offsets)

    # what the device tables point to: values may change in place, another object would not be seen
    _KEPT = frozenset(("params", "mirrors", "decay", "state_bits", "offsets", "m", "v", "m_scale", "v_scale",
                       "step_count", "lr_scale"))

    def __setattr__(self, name, value):
        if name in self._KEPT and value is not self.__dict__.get(name, value):
            raise AttributeError(f"{name} is kept for the optimizer's life: change its values in place")
        super().__setattr__(name, value)

    @torch.no_grad()
    def step(self, grads=None) -> None:
        """One update.  ``grads``: one contiguous float32 / bfloat16 / float16
        tensor for each parameter (default: their ``.grad``); a parameter whose
        gradient is None stays as it is, its states too."""
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        s = self.spec
        wd = _adam_decay(s)
        if self._plan is not None:
            self._plan.step(grads, s.learning_rate, s.beta1, s.beta2, s.epsilon, wd, self.seed)
        else:
            self._reference(grads, wd)

    # -- states ------------------------------------------------------------------------
    def state_dict(self) -> dict:
        """The states' tensors (not copies); see :meth:`load_state_dict`."""
        d = {"step": self.step_count, "m": self.m, "v": self.v}
        if self.state_bits == 8:
            d |= {"m_scale": self.m_scale, "v_scale": self.v_scale}
        return d

    @torch.no_grad()
    def load_state_dict(self, state: dict) -> None:
        """Copies the states of an optimizer over tensors of the same sizes,
        in the same number of bits."""
        own = self.state_dict()
        if set(state) != set(own):
            raise ValueError(f"states {sorted(state)}, expected {sorted(own)}")
        for k, t in own.items():
            if state[k].dtype != t.dtype or state[k].shape != t.shape:
                raise ValueError(f"state {k} is {state[k].dtype} {tuple(state[k].shape)}, "
                                 f"expected {t.dtype} {tuple(t.shape)}")
        for k, t in own.items():
            t.copy_(state[k])

    # -- the same step on the CPU ------------------------------------------------------
    def _reference(self, grads, wd) -> None:
        if len(grads) != len(self.params):
            raise ValueError(f"got {len(grads)} gradients for {len(self.params)} parameters")
        n = len(self.params)
        for i, (p, q, g) in enumerate(zip(self.params, self.mirrors, grads)):
            for what, t, held in (("parameter", p, self._held[i]), ("mirror", q, self._held[n + i])):
                if _storage_of(t) != held:
                    raise ValueError(f"{what} {i} has another storage, size or type than at construction")
            if g is None:
                continue
            if g.dtype not in (torch.float32, torch.bfloat16, torch.float16) or not g.is_contiguous() \
                    or g.numel() != p.numel() or g.device != p.device:
                raise ValueError("a gradient must be contiguous with its parameter's size and device")
        s, f = self.spec, torch.float32
        self.step_count += 1
        t = int(self.step_count)
        c1 = torch.tensor(1.0 / (1.0 - s.beta1 ** t), dtype=f)
        c2 = torch.tensor(1.0 / (1.0 - s.beta2 ** t) ** 0.5, dtype=f)
        lr = torch.tensor(s.learning_rate, dtype=f)
        if self.lr_scale is not None:
            lr = lr * self.lr_scale.reshape(())
        key = _mix32(torch.tensor([(t ^ self.seed) & 0xFFFFFFFF]))
        for i, (p, g) in enumerate(zip(self.params, grads)):
            if g is None or p.numel() == 0:
                continue
            n = p.numel()
            a = self.offsets[i]
            b = a + -(-n // STATE_BLOCK) * STATE_BLOCK
            pad = lambda x: torch.nn.functional.pad(x.reshape(-1).to(f), (0, b - a - n))  # noqa: E731,B023
            at = torch.arange(a, b)
            bits = _mix32((((at & 0xFFFFFFFF) ^ key) + (at >> 32) * 0x9E3779B1) & 0xFFFFFFFF)
            g, w = pad(g), pad(p.detach())
            if self.state_bits == 8:
                blocks = slice(a // STATE_BLOCK, b // STATE_BLOCK)
                m = _decode(self.m[a:b], self.m_scale[blocks])
                v = _decode(self.v[a:b], self.v_scale[blocks]) ** 2
            else:
                m, v = self.m[a:b], self.v[a:b]
            m = m * s.beta1 + g * (1.0 - s.beta1)
            v = v * s.beta2 + (g * (1.0 - s.beta2)) * g
            r = v.double().sqrt().float()  # correctly rounded, as the kernel's (torch's fp32 one on the CPU is not)
            w = w - ((m * c1) / (r * c2 + s.epsilon) + w * (wd if self.decay[i] else 0.0)) * lr
            if self.state_bits == 8:
                self.m[a:b], self.m_scale[blocks] = _encode(m, bits & 0xFFFF, False)
                self.v[a:b], self.v_scale[blocks] = _encode(r, bits >> 16, True)
            else:
                self.m[a:b], self.v[a:b] = m, v
            if p.dtype == torch.bfloat16:
                up = (w.view(torch.int32) + (_mix32(bits) >> 16).int()) & ~0xFFFF
                w = torch.where(w.isfinite(), up.view(f), w)
            w = w[:n]
            p.copy_(w.view(p.shape))
            if self.mirrors[i] is not None:
                self.mirrors[i].copy_(w.view(self.mirrors[i].shape))


def _adam_decay(spec: OptimizerSpec) -> float:
    """The decoupled weight decay of a spec that MultiTensorAdamW takes."""
    mode = spec.mode
    if mode not in (OPT_ADAM, OPT_ADAMW):
        raise ValueError(f"MultiTensorAdamW needs adam or adam_weight_decay, got {spec.kind}")
    if not (0 <= spec.beta1 < 1 and 0 <= spec.beta2 < 1):
        raise ValueError(f"beta1 and beta2 must be at least 0 and below 1, got {spec.beta1} and {spec.beta2}")
    return spec.weight_decay if mode == OPT_ADAMW else 0.0


def _storage_of(t: torch.Tensor | None):
    """What a tensor's place, size and type are told by."""
    return None if t is None else (t.data_ptr(), t.numel(), t.dtype, t.is_contiguous())


def _mix32(x: torch.Tensor) -> torch.Tensor:
    """32 mixed bits of whole numbers below 2^32 (int64 tensors)."""
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _decode(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return (code.float().view(-1, STATE_BLOCK) * scale[:, None]).view(-1)


def _encode(x: torch.Tensor, dither: torch.Tensor, least: bool):
    """e4m3 codes and scales (2^E, the block's largest finite value in [128, 256)
    codes) of x; ``dither`` of 2^16: the chance to go up.  ``least``: values
    above 0 stay above it."""
    size = x.abs()
    top = torch.where(size.isfinite(), size, torch.zeros_like(size)).view(-1, STATE_BLOCK).amax(1)
    e = torch.where(top > 0, (torch.frexp(top)[1] - 8).clamp(min=-117), torch.tensor(-117, dtype=torch.int32))
    power = lambda k: ((k + 127) << 23).to(torch.int32).view(torch.float32)  # noqa: E731
    y = (size.view(-1, STATE_BLOCK) * power(-e)[:, None]).view(-1)
    low = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)
    q = (((y + low).view(torch.int32) + (dither << 4).int()) & ~0xFFFFF).view(torch.float32) - low
    if least:
        q = torch.where(y > 0, q.clamp(min=2.0 ** -9), q)
    q = torch.where(y < 512, q, torch.full_like(q, float("nan")))
    return torch.copysign(q, x).to(torch.float8_e4m3fn), power(e)


NO_OPT_TAIL = (None, None, None, None, None, None, None, None, 0, [0.0] * 9, False)


@torch.no_grad()
def _reference_step(spec, p, g, m, v, anchor, p16, lr_scale, step):
    lr = spec.learning_rate * (float(lr_scale[0]) if lr_scale is not None else 1.0)
    mode = spec.mode
    if mode == OPT_SGD:
        gr = g + spec.l2 * p
        if spec.l1:
            gr = gr + spec.l1 * torch.sign(p)
        p.sub_(lr * gr)
    elif mode == OPT_MOMENTUM:
        m.mul_(spec.momentum).sub_(lr * g)
        p.add_(m)
    elif mode == OPT_FEDPROX:
        p.sub_(lr * (g + spec.proximal_term * (p - anchor)))
    else:
        t = float(int(step[0]) + 1) if step is not None else 1.0
        m.mul_(spec.beta1).add_((1 - spec.beta1) * g)
        v.mul_(spec.beta2).add_((1 - spec.beta2) * g * g)
        mh = m / (1 - spec.beta1 ** t)
        vh = v / (1 - spec.beta2 ** t)
        upd = mh / (vh.sqrt() + spec.epsilon)
        if mode == OPT_ADAMW:
            upd = upd + spec.weight_decay * p
        p.sub_(lr * upd)
    if p16 is not None:
        p16.copy_(p.to(torch.bfloat16))


def split_pack(x: torch.Tensor, y: torch.Tensor) -> None:
    """y (int32) = packed (hi << 16 | lo) bf16 split of the fp32 x."""
    if x.is_cuda:
        ops().split_pack_f32(x, y)
        return
    hi = x.to(torch.bfloat16)
    lo = (x - hi.float()).to(torch.bfloat16)
    h = hi.view(torch.int16).to(torch.int32) & 0xFFFF
    lw = lo.view(torch.int16).to(torch.int32) & 0xFFFF
    y.copy_((h << 16) | lw)


def cast_bf16(x: torch.Tensor, y: torch.Tensor) -> None:
    if x.is_cuda:
        ops().cast_f32_bf16(x, y)
    else:
        y.copy_(x.to(torch.bfloat16))


def scale_(x: torch.Tensor, w: float, wdev: torch.Tensor | None = None) -> None:
    if x.is_cuda:
        ops().scale_f32(x, float(w), wdev)
    else:
        x.mul_(float(wdev[0]) if wdev is not None else float(w))


def tick(step: torch.Tensor, inc: int = 1) -> None:
    if step.is_cuda:
        ops().tick(step, inc)
    else:
        step.add_(inc)
