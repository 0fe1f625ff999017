"""Losses and statistics of the routing tables that route / route_gemma4 return and moe_forward hands to its stats
callback: the balance loss with its gradient, and the per-expert usage that selects the experts to train.

    balance_loss(probs, topi, mask, cu_seqlens)   (loss, counts); differentiable w.r.t. probs
    expert_usage(probs, topv, topi, mask)         (counts, prob_mass, weight_mass)

The reference computes such tables in the consumer of its stats callback (smel/moe.py:258-259) and has no balance loss.
In a training step:

    aux = []
    out = smelb.moe_forward(x, W, ex, top_k, lora, stats=lambda p, v, i: aux.append(smelb.balance_loss(p, i)[0]))
    (task_loss(out) + 0.01 * aux[0]).backward()

probs is differentiable there, so the loss reaches x through the layer's own router backward. The router's weight is frozen
and gets no gradient: the loss trains what lies below the layer. moe_block_gemma4 and moe_forward_ep take the same callback (with
moe_forward_ep each rank's loss is of its own tokens). LayerMajorRunner calls it in its forward alone, which keeps no graph: there
the loss and the usage are figures to watch.
"""
import torch

from . import _lib


def _tables(who, probs, topi, mask):
    """Checked routing tables: (probs with unit column stride, its row pitch, topi, mask as bytes)."""
    ps, ts = probs.shape, topi.shape
    ok = (probs.is_cuda and topi.is_cuda and probs.dtype is torch.float32 and topi.dtype is torch.int64 and
          len(ps) == 2 and len(ts) == 2 and ts[0] == ps[0] and 1 <= ps[1] <= 512 and 1 <= ts[1] <= 32 and
          probs.get_device() == topi.get_device())
    if mask is not None:
        ok = (ok and mask.is_cuda and mask.get_device() == probs.get_device() and mask.shape == ps[:1] and
              (mask.dtype is torch.bool or mask.dtype is torch.uint8))
    if not ok:
        _refuse(who, probs, topi, mask)
    if not probs.is_contiguous() and (probs.stride(1) != 1 or (probs.stride(0) < ps[1] and ps[0] > 1)):
        probs = probs.contiguous()
    return probs, probs.stride(0), topi.contiguous(), None if mask is None else mask.contiguous()


def _refuse(who, probs, topi, mask):
    """Says what is wrong with the tables."""
    for name, t in (("probs", probs), ("topi", topi), ("mask", mask)):
        if t is None and name == "mask":
            continue
        if not t.is_cuda:
            raise _lib.SmelbError(f"{who}: smelb runs on CUDA tensors only ({name} is on {t.device})")
        if t.device != probs.device:
            raise _lib.SmelbError(f"{who}: {name} on {t.device}, probs on {probs.device}")
    if probs.dtype != torch.float32 or probs.dim() != 2:
        raise _lib.SmelbError(f"{who}: probs must be fp32 [T, E] (got {probs.dtype} {tuple(probs.shape)})")
    T, E = probs.shape
    if topi.dtype != torch.int64 or topi.dim() != 2 or topi.shape[0] != T:
        raise _lib.SmelbError(f"{who}: topi must be int64 [{T}, K] (got {topi.dtype} {tuple(topi.shape)})")
    if not 1 <= E <= 512 or not 1 <= topi.shape[1] <= 32:
        raise _lib.SmelbError(f"{who}: E={E} (1..512) and K={topi.shape[1]} (1..32)")
    raise _lib.SmelbError(f"{who}: mask must be bool or uint8 [{T}] (got {mask.dtype} {tuple(mask.shape)})")


def _loss(p, ld, topi, mask, cu, counts):
    """The loss and its gradient's rows; fills counts."""
    dev = p.device
    T, E = p.shape
    S = 1 if cu is None else cu.numel() - 1
    loss = torch.empty((), dtype=torch.float32, device=dev)
    coef = torch.empty(S * E + 1, dtype=torch.float32, device=dev)
    nb = _lib.load().smelb_balance_workspace_bytes(T, E, S, 0)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _lib.call_on(dev, "smelb_balance_loss_fwd", p.data_ptr(), ld, topi.data_ptr(), _lib.ptr(mask), _lib.ptr(cu), S, T, E,
                 topi.shape[1], loss.data_ptr(), counts.data_ptr(), coef.data_ptr(), ws.data_ptr(), nb,
                 _lib.stream_of(dev))
    return loss, coef, (S, T, E)


class _BalanceLossFn(torch.autograd.Function):
    """The loss alone, of probs and the checked tables as one object: autograd's time on the host grows with the inputs and
    outputs it sees."""

    @staticmethod
    def forward(ctx, probs, tables):
        loss, ctx.coef, ctx.sizes = _loss(*tables)
        mask, cu = tables[3:5]
        ctx.given = mask is not None or cu is not None
        if ctx.given:
            ctx.save_for_backward(mask, cu)
        return loss

    @staticmethod
    def backward(ctx, go):
        if torch.is_grad_enabled():  # create_graph: the gradient depends on go, which this call would hide
            raise _lib.SmelbError("balance_loss: there is no second derivative")
        mask, cu = ctx.saved_tensors if ctx.given else (None, None)
        S, T, E = ctx.sizes
        coef = ctx.coef
        dev = coef.device
        if go.dtype != torch.float32 or go.device != dev:
            go = go.to(device=dev, dtype=torch.float32)
        d = torch.empty(T, E, dtype=torch.float32, device=dev)
        _lib.call_on(dev, "smelb_balance_loss_bwd", coef.data_ptr(), go.data_ptr(), _lib.ptr(mask), _lib.ptr(cu), S, T, E,
                     d.data_ptr(), _lib.stream_of(dev))
        return d, None


def balance_loss(probs, topi, mask=None, cu_seqlens=None):
    """(loss fp32 0-dim, counts int64) of the routing probs fp32 [T, E] and topi int64 [T, K].

    Per sequence s with n_s rows kept by `mask` (bool or uint8 [T], None: all), counts c[s, e] of their choices and sums
    P[s, e] of their probs:  loss = mean over the sequences with n_s > 0 of  E / (K n_s^2) sum_e c[s, e] P[s, e],
    which is 1 for uniform probabilities; the loss is 0 when no row is kept. cu_seqlens (int32 [S + 1], not decreasing, on
    the device) gives sequence s the rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 (empty ones allowed) and counts the
    shape [S, E]; without it all rows are one sequence and counts has the shape [E]. Rows outside every sequence and rows
    that the mask drops may hold anything and get a zero gradient.

    Differentiable w.r.t. probs, with the counts as constants; the same inputs give the same bits. Choices outside [0, E)
    are not counted and recorded in the status word (read_status)."""
    p, ld, topi, mask = _tables("balance_loss", probs, topi, mask)
    cu, shape = cu_seqlens, p.shape[1:]
    if cu is not None:
        if not cu.is_cuda or cu.device != p.device:
            raise _lib.SmelbError(f"balance_loss: cu_seqlens on {cu.device}, probs on {p.device}")
        if cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 2:
            raise _lib.SmelbError(f"balance_loss: cu_seqlens must be int32 [sequences + 1] (got {cu.dtype} "
                                  f"{tuple(cu.shape)})")
        cu = cu.contiguous()
        shape = (cu.numel() - 1, p.shape[1])
    counts = torch.empty(shape, dtype=torch.int64, device=p.device)
    tables = (p, ld, topi, mask, cu, counts)
    loss = _BalanceLossFn.apply(probs, tables) if probs.requires_grad else _loss(*tables)[0]
    return loss, counts


def expert_usage(probs, topv, topi, mask=None):
    """(counts int64 [E], prob_mass fp32 [E], weight_mass fp32 [E]) over the rows that `mask` keeps: how often each expert
    was chosen, the sum of its probabilities and the sum of its routing weights. probs fp32 [T, E], topv bf16 or fp32
    [T, K], topi int64 [T, K], as a stats callback gets them. No gradient; the same inputs give the same bits."""
    p, ld, i, mask = _tables("expert_usage", probs.detach() if probs.requires_grad else probs, topi, mask)
    dev = p.device
    if topv.dtype not in (torch.bfloat16, torch.float32) or topv.shape != i.shape or topv.device != dev:
        raise _lib.SmelbError(f"expert_usage: topv must be bf16 or fp32 {tuple(i.shape)} on {dev} (got {topv.dtype} "
                              f"{tuple(topv.shape)} on {topv.device})")
    topv = topv.detach().contiguous() if topv.requires_grad else topv.contiguous()
    T, E = p.shape
    counts = torch.empty(E, dtype=torch.int64, device=dev)
    prob_mass = torch.empty(E, dtype=torch.float32, device=dev)
    weight_mass = torch.empty(E, dtype=torch.float32, device=dev)
    nb = _lib.load().smelb_balance_workspace_bytes(T, E, 1, 1)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _lib.call_on(dev, "smelb_expert_usage", p.data_ptr(), ld, topv.data_ptr(), 1 if topv.dtype == torch.float32 else 0,
                 i.data_ptr(), _lib.ptr(mask), T, E, i.shape[1], counts.data_ptr(), prob_mass.data_ptr(),
                 weight_mass.data_ptr(), ws.data_ptr(), nb, _lib.stream_of(dev))
    return counts, prob_mass, weight_mass
