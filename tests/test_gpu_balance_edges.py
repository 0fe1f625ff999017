"""Where the routing losses can go wrong besides their formulas. Bounds as in test_gpu_balance.py unless stated."""
import copy

import pytest
import torch

from oracle import moe_oracle as O
from test_gpu_balance import check, routing
from test_gpu_gemma import _gemma_inputs, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need CUDA"
    return torch.device("cuda:0")


@pytest.mark.parametrize("E,K", [(512, 32), (33, 32), (64, 1)])
def test_counts_of_short_runs_every_time(dev, E, K):
    """Runs of 1 to 31 rows whose choices name few experts over and over: each warp's table starts at zero."""
    import smelb
    T = 20000
    probs, topi, _, g = routing(dev, T, E, K, E, repeat=True)
    topi %= 7
    ends = torch.randint(1, 32, (2000,), generator=g, device=dev).cumsum(0)
    cu = torch.cat((ends.new_zeros(1), ends[ends < T])).to(torch.int32)
    loss, counts, d = check(dev, probs, topi, None, cu)
    for _ in range(30):
        again = smelb.balance_loss(probs, topi, None, cu)
        assert torch.equal(again[0], loss) and torch.equal(again[1], counts)


def balance(probs, topi, E):
    """The loss of all rows as one sequence, differentiable, in the type of probs."""
    f = torch.bincount(topi.reshape(-1), minlength=E).to(probs.dtype) / topi.numel()
    return E * (f * probs.mean(0)).sum()


def test_through_the_gemma_block(dev, golden):
    """moe_block_gemma4 with the loss from its stats callback: loss and dh against the oracle in 64 bits with the same choices."""
    import smelb
    d = golden("gemma_block.pt")
    c = d["cfg"]
    ex, lora, W = _gemma_inputs(d, dev)
    h = d["h"].bfloat16().to(dev).requires_grad_(True)
    xm = d["xm"].bfloat16().to(dev)
    gy = d["gy"].bfloat16().to(dev)
    rec = {}

    def stats(p, v, i):
        rec["loss"], rec["counts"] = smelb.balance_loss(p, i)
        rec["usage"] = smelb.expert_usage(p, v, i)
        rec["i"], rec["v"] = i.cpu(), v.detach().cpu()

    out = smelb.moe_block_gemma4(h, xm, W, ex, c["K"], c["eps"], c["act"], lora, stats=stats)
    weight = 30.0
    ((out.float() * gy.float()).sum() + weight * rec["loss"]).backward()
    E, dt = rec["counts"].numel(), torch.float64
    w = torch.zeros(E, dtype=dt).index_add_(0, rec["i"].reshape(-1), rec["v"].double().reshape(-1))
    assert torch.equal(rec["counts"], rec["usage"][0])
    assert bool(((rec["usage"][2].double().cpu() - w).abs() <= (128 * c["K"] + 17) * 2.0 ** -24 * w).all())
    s = c["alpha"] / c["r"]
    h64 = h.detach().cpu().to(dt).requires_grad_(True)
    W64 = {k: v.cpu().to(dt) for k, v in W.items()}
    sel = c["sel"]
    ref, probs, _, _ = O.moe_block_gemma4(
        h64, xm.cpu().to(dt), W64, O.dequant_int4(d["gu_q"], d["gu_scale"], d["gu_zero"], dt),
        O.dequant_int4(d["dn_q"], d["dn_scale"], d["dn_zero"], dt), c["K"], c["eps"], sel, d["gu"][sel].bfloat16().to(dt),
        d["dn"][sel].bfloat16().to(dt), {**{k: v.to(dt) for k, v in d["lora_ex"].items()}, "scale": s},
        {**{k: v.to(dt) for k, v in d["lora_sh"].items()}, "scale": s}, c["act"], rec["i"])
    aux = balance(probs, rec["i"], E)
    assert abs(rec["loss"].item() - aux.item()) <= 2.0 ** -7 * aux.item()  # bf16 logits
    ((ref * gy.cpu().to(dt)).sum() + weight * aux).backward()
    close(h.grad, h64.grad, "dh")
    assert smelb.read_status() == 0


def test_through_the_expert_parallel_layer(dev):
    """One rank of moe_forward_ep and moe_forward on the same tokens: the same loss, and dx with it within the layers' bound."""
    import smelb
    from smelb import ep
    from smelb.synth import qwen_layer
    K = 4
    L = qwen_layer(T=700, H=512, E=32, K=K, I=256, S=256, n_sel=4, r=16, seed=3, device=dev)
    W, ex, x = L["W"], L["ex"], L["x"]
    lora = [L["lora"], copy.deepcopy(L["lora"])]
    gy = torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(5), device=dev).bfloat16()
    shard = ep.shard_layer(ex, lora[1], 0, 1)
    comm = ep.EPGroup(cap=x.shape[0], H=x.shape[1], K=K)
    try:
        got = []
        for layer in (lambda t, s: smelb.moe_forward(t, W, ex, K, lora[0], s),
                      lambda t, s: ep.moe_forward_ep(t, W, shard, K, comm, s)):
            rec = []
            xl = x.detach().clone().requires_grad_(True)
            out = layer(xl, lambda p, v, i: rec.append((*smelb.balance_loss(p, i), i)))
            ((out.float() * gy.float()).sum() + 100.0 * rec[0][0]).backward()
            got.append((*rec[0], xl.grad))
        (loss, counts, topi, dx), (loss_ep, counts_ep, topi_ep, dx_ep) = got
        same = bool((topi == topi_ep).all())
        assert same and torch.equal(counts, counts_ep)
        assert abs(loss.item() - loss_ep.item()) <= 2 * 129 * 2.0 ** -24 * loss.item()
        close(dx_ep, dx, "dx")
        assert smelb.read_status() == 0
    finally:
        torch.cuda.synchronize()
        comm.close()


def test_in_the_layer_major_runner(dev):
    """The runner's callback hands out tables without a graph: figures of every layer and micro-batch, and a training step as
    without them."""
    import smelb
    from smelb.runner import LayerMajorRunner
    from smelb.synth import qwen_layer
    K = 4
    layers = {l: qwen_layer(T=64, H=512, E=32, K=K, I=256, S=256, n_sel=4, r=16, seed=l, device=dev) for l in (0, 1)}
    hs = [layers[0]["x"].detach().clone(), layers[1]["x"].detach()[:33].clone()]
    runner = LayerMajorRunner({l: (v["W"], v["ex"]) for l, v in layers.items()}, [0, 1], top_k=K)
    seen = {}

    def stats(l, m, p, v, i):
        seen[l, m] = (*smelb.balance_loss(p, i), smelb.expert_usage(p, v, i)[0])

    out, ckpt = runner.forward([h.clone() for h in hs], keep_ckpt=True, stats_cb=stats)
    plain_out, _ = runner.forward([h.clone() for h in hs])
    assert all(torch.equal(a, b) for a, b in zip(out, plain_out)) and set(seen) == {(l, m) for l in (0, 1) for m in (0, 1)}
    for (l, m), (loss, counts, again) in seen.items():
        assert not loss.requires_grad and torch.equal(counts, again) and counts.sum().item() == hs[m].shape[0] * K
        assert 0.0 < loss.item() <= 32.0  # E at most: every choice and all probability on one expert
    grads = runner.backward(ckpt, [torch.ones_like(o) for o in out])
    assert all(g.shape == h.shape and bool(g.isfinite().all()) for g, h in zip(grads, hs))
