"""Muon for LoRA factors: momentum updates orthogonalised by Newton-Schulz steps, one launch for a layer's factors.

    orthogonalize(x)                      the Newton-Schulz polynomial of each [m, n] matrix of x [..., m, n]
    muon_step(params, grads, buffers, lr) one update of many tensors, in place
    Muon(params, lr)                      the same as a torch optimizer

The reference trains its factors with AdamW (scripts/train.py) and has no counterpart. The short side of every matrix is
at most 64, the width of a LoRA block of the fused layer; ExpertsLoRA's [k, r, H] parameters are k matrices each.
"""
import ctypes
import functools

import torch

from . import _lib

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 16
MAX_SHORT_SIDE = 64
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_ADJUST = {"original": 0, "match_rms_adamw": 1}


@functools.lru_cache(maxsize=16)
def _triples(steps, coefficients):
    return (ctypes.c_double * (3 * steps))(*[float(v) for t in coefficients for v in t])


def _coefficients(who, steps, coefficients):
    """Host array of 3 * steps doubles: one (a, b, c) for every step, or a triple of its own for each."""
    if not 1 <= steps <= MAX_STEPS:
        raise _lib.SmelbError(f"{who}: {steps} steps (1..{MAX_STEPS})")
    c = tuple(coefficients)
    if len(c) == 3 and not hasattr(c[0], "__len__"):
        c = (c,) * steps
    if len(c) != steps or any(not hasattr(t, "__len__") or len(t) != 3 for t in c):
        raise _lib.SmelbError(f"{who}: coefficients are three numbers, or three for each of the {steps} steps")
    return _triples(steps, tuple(map(tuple, c)))


def _matrices(who, t, what):
    """(batch, rows, cols) of a checked CUDA tensor [..., m, n]."""
    if not t.is_cuda:
        raise _lib.SmelbError(f"{who}: smelb runs on CUDA tensors only ({what} is on {t.device})")
    if t.dim() < 2 or t.dtype not in _DTYPES:
        raise _lib.SmelbError(f"{who}: {what} must be fp32 or bf16 matrices [..., m, n] (got {t.dtype} {tuple(t.shape)})")
    m, n = t.shape[-2:]
    if not 1 <= min(m, n) <= MAX_SHORT_SIDE:
        raise _lib.SmelbError(f"{who}: {what}: the short side of {m} x {n} must be 1..{MAX_SHORT_SIDE}")
    return t.numel() // (m * n), m, n


def orthogonalize(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The Newton-Schulz polynomial of each matrix of x [..., m, n] (fp32 or bf16, min(m, n) <= 64): x / (|x|_F + eps), then
    `steps` (1..16) times X <- a X + b (X X^T) X + c (X X^T)^2 X on the short side. coefficients is (a, b, c), or one triple
    for each step. With the default ones the singular values end near 1. Returns a new tensor of x's shape and type; all
    sums and products are fp64, the result is rounded once. Steps that would let the rounding of fp64 grow into the result
    (the product of the a^2 but the last above 2^26: the default ones from the ninth on) are taken in pairs of doubles, which
    is much slower.

    A matrix of zeros gives zeros; one with an infinity or NaN gives NaN and leaves the others alone. There is no
    gradient: x must not require one unless gradients are off."""
    if torch.is_grad_enabled() and x.requires_grad:
        raise _lib.SmelbError("orthogonalize: there is no backward; call it under torch.no_grad()")
    batch, m, n = _matrices("orthogonalize", x, "x")
    if not eps > 0:
        raise _lib.SmelbError("orthogonalize: eps must be positive")
    steps = int(steps)
    c = _coefficients("orthogonalize", steps, coefficients)
    x = x.contiguous()
    out = torch.empty_like(x)
    if batch:
        nb = _lib.load().smelb_orthogonalize_workspace_bytes(batch, m, n)
        ws = torch.empty(nb, dtype=torch.uint8, device=x.device) if nb > 0 else None
        _lib.call_on(x.device, "smelb_orthogonalize", x.data_ptr(), _DTYPES[x.dtype], batch, m, n, steps, c,
                     float(eps), out.data_ptr(), _lib.ptr(ws), nb, _lib.stream_of(x.device))
    return out


def muon_step(params, grads, buffers, lr, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="original", steps=5,
              coefficients=COEFFICIENTS, eps=1e-7):
    """One Muon update of the tensors params[i] with the gradients grads[i] and momentum buffers buffers[i], in place:

        m <- momentum m + (1 - momentum) g;  u = momentum m + (1 - momentum) g (nesterov) or m
        p <- p (1 - lr weight_decay) - lr f orthogonalize(u)

    for every [m, n] matrix of a tensor, f = sqrt(max(1, m / n)) ("original") or 0.2 sqrt(max(m, n)) ("match_rms_adamw").
    params: contiguous fp32 or bf16 [..., m, n], min(m, n) <= 64, all of one type and device; grads alike; buffers: contiguous
    fp32 of the params' shapes. A param or buffer that shares memory with another tensor is refused. One kernel launch takes
    up to 48 tensors whose short sides round up to the same multiple of 8 (short sides above 32, and very long matrices, take
    three)."""
    who = "muon_step"
    params, grads, buffers = list(params), list(grads), list(buffers)
    if not len(params) == len(grads) == len(buffers):
        raise _lib.SmelbError(f"{who}: {len(params)} params, {len(grads)} grads, {len(buffers)} buffers")
    if adjust not in _ADJUST:
        raise _lib.SmelbError(f"{who}: adjust must be one of {sorted(_ADJUST)}")
    if not eps > 0:
        raise _lib.SmelbError(f"{who}: eps must be positive")
    steps = int(steps)
    c = _coefficients(who, steps, coefficients)
    if not params:
        return
    dev, dtype = params[0].device, params[0].dtype
    if not params[0].is_cuda or dtype not in _DTYPES:
        _matrices(who, params[0], "params[0]")  # says which it is
    on, fp32, most = dev.index, torch.float32, MAX_SHORT_SIDE
    rows, keep = [], []
    for i, (p, g, m) in enumerate(zip(params, grads, buffers)):
        shape = p.shape
        if not (p.dtype is dtype and g.dtype is dtype and m.dtype is fp32 and g.shape == shape == m.shape and
                p.get_device() == g.get_device() == m.get_device() == on and len(shape) >= 2 and
                p.is_contiguous() and m.is_contiguous()):
            _refuse(who, i, p, g, m, dtype, dev)
        a, b = shape[-2], shape[-1]
        if not (a > 0 and b > 0 and (a <= most or b <= most)):
            _refuse(who, i, p, g, m, dtype, dev)
        if not g.is_contiguous():
            g = g.contiguous()
            keep.append(g)
        rows += (p.data_ptr(), g.data_ptr(), m.data_ptr(), p.numel() // (a * b), a, b)
    written = [q for q in rows[0::6] + rows[2::6] if q]
    once = set(written)
    if len(once) < len(written) or not once.isdisjoint(rows[1::6]):
        raise _lib.SmelbError(f"{who}: a tensor is given twice")
    # the fields of a MuonTensor are eight bytes each: an array of integers is an array of them
    table = (ctypes.c_int64 * len(rows))(*rows)
    nb = _lib.load().smelb_muon_workspace_bytes(table, len(params))
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb > 0 else None
    _lib.call_on(dev, "smelb_muon_step", table, len(params), _DTYPES[dtype], float(lr), float(momentum),
                 1 if nesterov else 0, float(weight_decay), _ADJUST[adjust], steps, c, float(eps), _lib.ptr(ws), nb,
                 _lib.stream_of(dev))
    # as torch's in-place operations do
    torch.autograd.graph.increment_version([t for t in params + buffers if not t.is_inference()])


def _refuse(who, i, p, g, m, dtype, dev):
    """Says what is wrong with tensor i of a step."""
    _matrices(who, p, f"params[{i}]")
    if p.dtype != dtype or p.device != dev:
        raise _lib.SmelbError(f"{who}: params[{i}] is {p.dtype} on {p.device}, params[0] {dtype} on {dev}")
    if g.dtype != dtype or g.device != dev or g.shape != p.shape:
        raise _lib.SmelbError(f"{who}: grads[{i}] is {g.dtype} {tuple(g.shape)} on {g.device}, its parameter {dtype} "
                              f"{tuple(p.shape)} on {dev}")
    if m.dtype != torch.float32 or m.device != dev or m.shape != p.shape:
        raise _lib.SmelbError(f"{who}: buffers[{i}] must be fp32 {tuple(p.shape)} on {dev} (got {m.dtype} "
                              f"{tuple(m.shape)} on {m.device})")
    raise _lib.SmelbError(f"{who}: params[{i}] and buffers[{i}] must be contiguous (they are updated in place)")


class Muon(torch.optim.Optimizer):
    """muon_step as a torch optimizer over parameters [..., m, n] with min(m, n) <= 64 (the factors of ExpertsLoRA and
    MLPLoRA). State per parameter: momentum_buffer, fp32 of the parameter's shape. A parameter without a gradient is
    left alone. lr may change between steps (a scheduler's); a captured step keeps the lr it was captured with. The step
    that makes a parameter's state cannot be captured."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="original", steps=5,
                 coefficients=COEFFICIENTS, eps=1e-7):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f"Muon: lr={lr} momentum={momentum} weight_decay={weight_decay}")
        if adjust not in _ADJUST:
            raise ValueError(f"Muon: adjust must be one of {sorted(_ADJUST)}")
        if not eps > 0:
            raise ValueError("Muon: eps must be positive")
        _coefficients("Muon", steps, coefficients)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      adjust=adjust, steps=steps, coefficients=coefficients, eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2 or not 1 <= min(p.shape[-2:]) <= MAX_SHORT_SIDE:
                    raise ValueError(f"Muon: parameter of shape {tuple(p.shape)}: the last two dimensions need a short side "
                                     f"of 1..{MAX_SHORT_SIDE}")

    def load_state_dict(self, state_dict):
        """As torch's, with the buffers of bf16 parameters kept in fp32."""
        super().load_state_dict(state_dict)
        mine = [p for group in self.param_groups for p in group["params"]]
        theirs = [i for group in state_dict["param_groups"] for i in group["params"]]
        for p, i in zip(mine, theirs):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None:
                self.state[p]["momentum_buffer"] = m.to(device=p.device, dtype=torch.float32, copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_kind = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():  # each replay would fill it with zeros again
                        raise _lib.SmelbError("Muon: take a step before one is captured (it makes the momentum buffers)")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32,
                                                                memory_format=torch.contiguous_format)
                by_kind.setdefault((p.device, p.dtype), []).append((p, p.grad, state["momentum_buffer"]))
            for tensors in by_kind.values():
                muon_step(*zip(*tensors), lr=group["lr"], momentum=group["momentum"], nesterov=group["nesterov"],
                          weight_decay=group["weight_decay"], adjust=group["adjust"], steps=group["steps"],
                          coefficients=group["coefficients"], eps=group["eps"])
        return loss
