"""The router's balance loss and usage statistics and the orthogonalised (Muon) update of LoRA factors: cases, inputs, plain
forms and the values in 64 bits.

`own` false: elementary torch operations. `own` true: the calls a user makes of smelb (balance_loss, expert_usage, orthogonalize,
muon_step).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)  # the quintic Newton-Schulz polynomial
STEPS, EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
AUX = 0.01  # weight of the balance loss in a training step: the gradient that reaches it


def _smelb():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "smel-ft_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import smelb
    return smelb


def listed():
    return [
        # the balance loss on a handful of tokens: a debugging step, where the calls themselves are the time
        {"name": "balance_few", "op": "balance", "T": 7, "E": 32, "K": 4, "S": 0, "mask": False},
        # one training micro-batch of the 256-expert layer as one pool of tokens
        {"name": "balance_microbatch", "op": "balance", "T": 4096, "E": 256, "K": 8, "S": 0, "mask": False},
        # a packed batch of ragged sequences with padding inside and rows behind the last one, 128 experts
        {"name": "balance_packed", "op": "balance", "T": 8189, "E": 128, "K": 8, "S": 37, "mask": True},
        # the routing of a whole optimizer step at once, per sequence
        {"name": "balance_step", "op": "balance", "T": 131072, "E": 256, "K": 8, "S": 32, "mask": True},
        # the statistics callback of one micro-batch
        {"name": "usage_microbatch", "op": "usage", "T": 4096, "E": 256, "K": 8, "topv": "bf16", "mask": False},
        # the statistics of a calibration pass with padded rows, fp32 weights and an odd number of tokens
        {"name": "usage_pass", "op": "usage", "T": 65537, "E": 128, "K": 8, "topv": "fp32", "mask": True},
        # the A factors of 12 selected experts at rank 16
        {"name": "ortho_factors", "op": "ortho", "B": 12, "m": 16, "n": 2048, "dtype": "fp32"},
        # tall B factors in bf16 at an odd length and a rank between the powers of two
        {"name": "ortho_tall_bf16", "op": "ortho", "B": 29, "m": 703, "n": 24, "dtype": "bf16"},
        # many wide-rank factors
        {"name": "ortho_rank64", "op": "ortho", "B": 192, "m": 64, "n": 2048, "dtype": "fp32"},
        # the update of one dense MLP's six factors
        {"name": "muon_mlp", "op": "muon", "layers": 1, "k": 0, "r": 16, "H": 2048, "I": 512},
        # the update of one layer: 12 selected experts and the shared expert
        {"name": "muon_layer", "op": "muon", "layers": 1, "k": 12, "r": 16, "H": 2048, "I": 512},
        # the update of two layers with half of their experts selected
        {"name": "muon_block", "op": "muon", "layers": 2, "k": 128, "r": 16, "H": 2048, "I": 512},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("balance", "usage", "ortho", "muon"))
    if op in ("balance", "usage"):
        E = rng.choice((8, 32, 60, 64, 128, 256, 512, _log(rng, 4, 512)))
        T = _log(rng, 1, 131072 * 256 // max(E, 256))
        K = rng.randint(1, min(E, 16))
        mask = rng.random() < 0.5
        if op == "balance":
            return {"op": op, "T": T, "E": E, "K": K, "S": 0 if rng.random() < 0.4 else _log(rng, 1, 300), "mask": mask}
        return {"op": op, "T": T, "E": E, "K": K, "topv": rng.choice(("bf16", "fp32")), "mask": mask}
    if op == "ortho":
        d = rng.choice((8, 16, 32, 64, rng.randint(1, 64)))
        n = _log(rng, d, 16384)
        B = _log(rng, 1, max(1, min(4096, 192 * 64 * 64 * 2048 // (d * max(d, 16) * n))))
        m, n = (d, n) if rng.random() < 0.5 else (n, d)
        return {"op": op, "B": B, "m": m, "n": n, "dtype": rng.choice(("fp32", "bf16"))}
    r = rng.choice((8, 16, 32, 64, rng.randint(1, 64)))
    H, I = _log(rng, 64, 2816), _log(rng, 32, 704)
    k = rng.randint(0, 2) if rng.random() < 0.3 else _log(rng, 1, max(1, min(128, 128 * 16 * 16 // (r * max(r, 16)))))
    return {"op": op, "layers": rng.randint(1, 2), "k": k, "r": r, "H": H, "I": I}


# ------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _routing(c, g):
    """Router probabilities with a skewed popularity of the experts (a few hot ones, a long tail), the K largest of each row and
    their renormalised weights."""
    T, E, K = c["T"], c["E"], c["K"]
    hot = -0.5 * torch.log(1.0 + torch.randperm(E, generator=g, device="cuda").float())
    probs = torch.softmax(torch.randn(T, E, generator=g, device="cuda") * 1.2 + hot, -1)
    v, topi = torch.topk(probs, K, dim=-1)
    return probs, v / v.sum(-1, keepdim=True), topi


def _gradients(B, m, n, g):
    """Gradients of LoRA factors: a product over a few to many tokens, so of full or low rank, with a decaying spectrum; every
    seventh matrix is zero (an expert without tokens) and every fifth has rank one (one token)."""
    d = min(m, n)
    scale = 10.0 ** (-0.1 * torch.arange(d, device="cuda", dtype=torch.float32))
    a = torch.randn(B, m, d, generator=g, device="cuda") * scale
    b = torch.randn(B, d, n, generator=g, device="cuda")
    keep = torch.ones(B, d, 1, device="cuda")
    keep[4::5, 1:] = 0.0
    keep[6::7] = 0.0
    return torch.bmm(a, b * keep) * 1e-3


def _factor_shapes(c):
    r, H, I, k = c["r"], c["H"], c["I"], c["k"]
    one = [(r, H), (I, r), (r, H), (I, r), (r, I), (H, r)]
    layer = ([(k, *s) for s in one] if k else []) + one
    return layer * c["layers"]


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] in ("balance", "usage"):
        probs, topv, topi = _routing(c, g)
        s = {"case": c, "probs": probs, "topi": topi, "mask": None}
        if c["mask"]:
            s["mask"] = torch.rand(c["T"], generator=g, device="cuda") < 0.9
        if c["op"] == "usage":
            s["topv"] = topv.to(torch.bfloat16) if c["topv"] == "bf16" else topv
            return s
        s["cu"] = None
        if c["S"]:
            # S sequences of random lengths, empty ones among them, and a few rows behind the last one
            cuts = torch.randint(0, c["T"] + 1, (c["S"],), generator=g, device="cuda").sort().values
            s["cu"] = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), cuts)).to(torch.int32)
        s["probs"].requires_grad_(True)
        s["go"] = torch.full((), AUX, device="cuda")
        return s
    if c["op"] == "ortho":
        x = _gradients(c["B"], c["m"], c["n"], g)
        return {"case": c, "x": x.to(torch.bfloat16) if c["dtype"] == "bf16" else x}
    params, grads, bufs = [], [], []
    for shape in _factor_shapes(c):
        m, n = shape[-2:]
        B = shape[0] if len(shape) == 3 else 1
        params.append(torch.randn(shape, generator=g, device="cuda") * 0.02)
        grads.append(_gradients(B, m, n, g).view(shape))
        bufs.append(_gradients(B, m, n, g).view(shape))
    return {"case": c, "p": params, "g": grads, "m": bufs}


# ------------------------------------------------------------------------------------------------------- plain forms
def _sequence_of(T, cu):
    """Sequence of each row (-1 behind the last one)."""
    t = torch.arange(T, device=cu.device)
    s = torch.searchsorted(cu[1:].long().contiguous(), t, right=True)
    return torch.where(s < cu.numel() - 1, s, -1)


def _plain_balance(probs, topi, mask, cu, go):
    T, E = probs.shape
    K = topi.shape[1]
    S = 1 if cu is None else cu.numel() - 1
    seq = torch.zeros(T, dtype=torch.int64, device=probs.device) if cu is None else _sequence_of(T, cu)
    valid = seq >= 0 if mask is None else (seq >= 0) & mask
    at = torch.where(valid, seq, S)  # row S takes what does not count
    n = torch.zeros(S + 1, dtype=torch.float64, device=probs.device).index_add_(0, at, torch.ones_like(at, dtype=torch.float64))[:S]
    counts = torch.zeros(S + 1, E, dtype=torch.int64, device=probs.device)
    counts.view(-1).index_add_(0, (at[:, None] * E + topi).view(-1), torch.ones_like(topi).view(-1))
    mass = torch.zeros(S + 1, E, device=probs.device).index_add_(0, at, probs)[:S]
    counts = counts[:S]
    some = (n > 0).sum().clamp(min=1)
    f = torch.where(n > 0, E / (K * n * n), 0.0)[:, None] * counts / some
    loss = (f * mass).sum().float()
    rows = torch.cat((f, torch.zeros(1, E, dtype=f.dtype, device=f.device))) * go
    return loss, counts if cu is not None else counts[0], rows.float()[at]


def _plain_usage(probs, topv, topi, mask):
    T, E = probs.shape
    valid = torch.ones(T, dtype=torch.bool, device=probs.device) if mask is None else mask
    e = torch.where(valid[:, None], topi, E).view(-1)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=probs.device).index_add_(0, e, torch.ones_like(e))[:E]
    weight = torch.zeros(E + 1, dtype=torch.float64, device=probs.device).index_add_(0, e, topv.double().view(-1))[:E]
    mass = torch.where(valid[:, None], probs, 0.0).sum(0)
    return counts, mass, weight.float()


def _plain_ortho(x):
    """In 64 bits: in 32 the small singular values, which the steps grow by up to 485, come out up to 6e-5 off."""
    tall = x.shape[-2] > x.shape[-1]
    X = x.double().mT if tall else x.double()
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    a, b, c = COEF
    for _ in range(STEPS):
        G = X @ X.mT
        X = a * X + (b * G + c * (G @ G)) @ X
    return X.mT if tall else X


def _plain_muon(p, g, m):
    m.copy_(MOMENTUM * m + (1 - MOMENTUM) * g)
    u = (1 - MOMENTUM) * g + MOMENTUM * m
    adj = math.sqrt(max(1.0, p.shape[-2] / p.shape[-1]))
    p.copy_(p.double() * (1 - LR * DECAY) - LR * adj * _plain_ortho(u))


def run(state):
    c = state["case"]
    if c["op"] == "balance":
        if own:
            loss, counts = _smelb().balance_loss(state["probs"], state["topi"], mask=state["mask"], cu_seqlens=state["cu"])
            dprobs, = torch.autograd.grad(loss, state["probs"], state["go"])
        else:
            loss, counts, dprobs = _plain_balance(state["probs"].detach(), state["topi"], state["mask"], state["cu"], state["go"])
        return {"loss": loss, "counts": counts, "dprobs": dprobs}
    if c["op"] == "usage":
        f = _smelb().expert_usage if own else _plain_usage
        counts, mass, weight = f(state["probs"], state["topv"], state["topi"], state["mask"])
        return {"counts": counts, "prob_mass": mass, "weight_mass": weight}
    if c["op"] == "ortho":
        return _smelb().orthogonalize(state["x"], steps=STEPS, coefficients=COEF, eps=EPS) if own else _plain_ortho(state["x"]).to(state["x"].dtype)
    if own:
        _smelb().muon_step(state["p"], state["g"], state["m"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY, steps=STEPS,
                           coefficients=COEF, eps=EPS)
    else:
        for p, g, m in zip(state["p"], state["g"], state["m"]):
            _plain_muon(p, g, m)
    return {"p": state["p"], "m": state["m"]}


# -------------------------------------------------------------------------------------------------- 64 bits, and work
def _exact_ortho(x):
    """The polynomial on the singular values."""
    U, s, Vt = np.linalg.svd(x, full_matrices=False)
    t = s / (np.sqrt((s * s).sum(-1, keepdims=True)) + EPS)
    a, b, c = COEF
    for _ in range(STEPS):
        t = a * t + b * t ** 3 + c * t ** 5
    return U @ (t[..., None] * Vt)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] in ("balance", "usage"):
        probs, topi = s["probs"].detach().cpu().numpy().astype(np.float64), s["topi"].cpu().numpy()
        T, E, K = c["T"], c["E"], c["K"]
        valid = np.ones(T, bool) if s["mask"] is None else s["mask"].cpu().numpy()
        if c["op"] == "usage":
            w = s["topv"].cpu().float().numpy().astype(np.float64)
            return {"counts": None, "prob_mass": probs[valid].sum(0),
                    "weight_mass": np.bincount(topi[valid].reshape(-1), weights=w[valid].reshape(-1), minlength=E)}
        cu = [0, T] if s["cu"] is None else s["cu"].cpu().tolist()
        loss, grad, some = 0.0, np.zeros((T, E)), 0
        for t0, t1 in zip(cu[:-1], cu[1:]):
            rows = np.nonzero(valid[t0:t1])[0] + t0
            if not rows.size:
                continue
            some += 1
            f = np.bincount(topi[rows].reshape(-1), minlength=E) / (K * rows.size)  # share of the choices
            loss += E * float((f * probs[rows].mean(0)).sum())
            grad[rows] = E * f / rows.size
        some = max(some, 1)
        return {"loss": loss / some, "counts": None, "dprobs": grad * (np.float64(np.float32(AUX)) / some)}
    if c["op"] == "ortho":
        return _exact_ortho(s["x"].double().cpu().numpy())
    out = {"p": [], "m": []}
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        p, g, m = (t.double().cpu().numpy() for t in (p, g, m))
        m = MOMENTUM * m + (1 - MOMENTUM) * g
        u = (1 - MOMENTUM) * g + MOMENTUM * m
        out["m"].append(m)
        out["p"].append(p * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, p.shape[-2] / p.shape[-1])) * _exact_ortho(u))
    return out


def _ortho_flops(B, m, n):
    d, L = min(m, n), max(m, n)
    return B * (d * (d + 1) * L + 2 * d * d * L + (4 * STEPS - 3) * 2 * d ** 3)


def work(case):
    c = case
    if c["op"] in ("balance", "usage"):
        T, E, K = c["T"], c["E"], c["K"]
        b = T * E * 4 + T * K * 8 + (T if c["mask"] else 0)
        if c["op"] == "usage":
            return {"bytes": b + T * K * (2 if c["topv"] == "bf16" else 4) + E * 16, "flops": T * E + T * K}
        S = max(c["S"], 1)
        return {"bytes": b + T * E * 4 + S * E * 8 + (S + 1) * 4, "flops": 2 * T * E + T * K}
    if c["op"] == "ortho":
        return {"bytes": 2 * c["B"] * c["m"] * c["n"] * (4 if c["dtype"] == "fp32" else 2), "flops": _ortho_flops(c["B"], c["m"], c["n"])}
    b = f = 0
    for shape in _factor_shapes(c):
        B = shape[0] if len(shape) == 3 else 1
        b += 20 * B * shape[-2] * shape[-1]
        f += _ortho_flops(B, shape[-2], shape[-1])
    return {"bytes": b, "flops": f}
