"""smelb.balance_loss and smelb.expert_usage on the GPU against a plain implementation in 64 bits.

Tolerances. The terms of every sum are not negative, so a sum of n terms added one after the other in fp32 is off by at
most n 2^-24 relative. A tile sums at most 128 rows in fp32 (an expert's routing weights: at most 128 K terms when a row
names one expert K times) and the rest is added in 64 bits; with the final rounding that is (128 + 1) 2^-24 for prob_mass
and the loss, (128 K + 17) 2^-24 for weight_mass (16 per-warp tables are added). The gradient is the product of three
values rounded once each with two roundings of its own: 5 * 2^-24."""
import pytest
import torch

from oracle import moe_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need CUDA"
    return torch.device("cuda:0")


def plain(probs, topi, mask=None, cu=None):
    """(loss, counts [S, E], d loss / d probs) in 64 bits on the CPU."""
    probs, topi = probs.detach().double().cpu(), topi.cpu()
    T, E = probs.shape
    K = topi.shape[1]
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu().bool()
    cu = [0, T] if cu is None else cu.cpu().tolist()
    S = len(cu) - 1
    counts, grad, losses = torch.zeros(S, E, dtype=torch.int64), torch.zeros(T, E, dtype=torch.float64), []
    for s in range(S):
        rows = torch.arange(cu[s], cu[s + 1])[keep[cu[s]:cu[s + 1]]]
        n = rows.numel()
        if n == 0:
            continue
        e = topi[rows].reshape(-1)
        counts[s] = torch.bincount(e[(e >= 0) & (e < E)], minlength=E)
        f = E * counts[s].double() / (K * n * n)
        losses.append((f * probs[rows].sum(0)).sum())
        grad[rows] = f
    some = max(len(losses), 1)
    return sum(losses, torch.zeros((), dtype=torch.float64)) / some, counts, grad / some


def routing(dev, T, E, K, seed, repeat=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    probs = torch.softmax(torch.randn(T, E, generator=g, device=dev) * 1.5, -1)
    topi = torch.randint(0, E, (T, K), generator=g, device=dev) if repeat else probs.topk(K, -1).indices
    topv = torch.rand(T, K, generator=g, device=dev)
    return probs, topi, topv, g


def check(dev, probs, topi, mask=None, cu=None, go=0.37):
    import smelb
    p = probs.detach().requires_grad_(True)
    loss, counts = smelb.balance_loss(p, topi, mask, cu)
    assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == torch.int64
    d, = torch.autograd.grad(loss, p, torch.tensor(go, device=dev))
    rl, rc, rd = plain(probs, topi, mask, cu)
    assert torch.equal(counts.cpu(), rc if cu is not None else rc[0])
    assert abs(loss.double().cpu() - rl) <= 129 * U * abs(rl)
    rd = rd * torch.tensor(go, dtype=torch.float32).double()
    assert d.shape == probs.shape and bool(((d.double().cpu() - rd).abs() <= 5 * U * rd).all())
    return loss, counts, d


SIZES = [(1, 1, 1), (1, 512, 32), (2, 3, 2), (17, 7, 3), (16, 32, 4), (129, 130, 8), (1000, 64, 8), (333, 511, 5),
         (4096, 256, 8), (9473, 128, 8), (80001, 60, 4)]


@pytest.mark.parametrize("T,E,K", SIZES)
@pytest.mark.parametrize("masked", [False, True])
def test_balance_loss_one_sequence(dev, T, E, K, masked):
    probs, topi, _, g = routing(dev, T, E, K, T + E)
    mask = (torch.rand(T, generator=g, device=dev) < 0.8) if masked else None
    check(dev, probs, topi, mask)


@pytest.mark.parametrize("T,E,K,cu", [
    (64, 32, 4, [0, 64]),
    (64, 32, 4, [0, 0, 0, 1, 17, 17, 40, 64, 64]),     # empty sequences, lengths of one
    (700, 128, 8, [5, 30, 31, 500, 650]),              # rows before the first and behind the last sequence
    (40000, 256, 8, [0, 1, 39000, 39100, 39998]),      # one long sequence over many tiles
    (33, 7, 2, list(range(34))),                       # every row a sequence
    (3000, 512, 8, sorted((i * 37) % 2990 for i in range(400))),   # a few rows each
    (6000, 33, 3, [7] + list(range(10, 5000, 31)) + [5990]),        # runs just below a warp's, then a long one
    (5000, 128, 8, list(range(0, 5000, 33)) + [5000]),              # and just above
    (24, 60, 1, sorted((i * 7) % 25 for i in range(258))),          # more sequences than rows
    (2000, 64, 8, [0] * 700 + [1000] * 900 + [2000]),  # more sequences than a block has threads, most empty
])
@pytest.mark.parametrize("masked", [False, True])
def test_balance_loss_packed(dev, T, E, K, cu, masked):
    probs, topi, _, g = routing(dev, T, E, K, T)
    mask = (torch.rand(T, generator=g, device=dev) < 0.7).to(torch.uint8) if masked else None
    check(dev, probs, topi, mask, torch.tensor(cu, dtype=torch.int32, device=dev))


def test_balance_loss_nothing_kept(dev):
    """No kept row at all, a whole sequence masked away, and no rows: loss and gradient 0 there."""
    import smelb
    probs, topi, _, _ = routing(dev, 100, 32, 4, 1)
    none = torch.zeros(100, dtype=torch.bool, device=dev)
    loss, counts, d = check(dev, probs, topi, none)
    assert loss.item() == 0 and counts.sum().item() == 0 and not d.any()
    part = none.clone()
    part[60:] = True
    check(dev, probs, topi, part, torch.tensor([0, 50, 100], dtype=torch.int32, device=dev))
    loss, counts = smelb.balance_loss(probs[:0], topi[:0])
    assert loss.item() == 0 and counts.sum().item() == 0
    loss, counts = smelb.balance_loss(probs[:0], topi[:0], None, torch.zeros(4, dtype=torch.int32, device=dev))
    assert loss.item() == 0 and counts.shape == (3, 32) and not counts.any()
    p = probs[:0].detach().requires_grad_(True)
    smelb.balance_loss(p, topi[:0])[0].backward()
    assert p.grad.shape == (0, 32)
    c, m, w = smelb.expert_usage(probs[:0], probs[:0, :4], topi[:0])
    assert not c.any() and not m.any() and not w.any()


def test_masked_and_outside_rows_are_not_read(dev):
    """Rows the mask drops and rows outside every sequence hold NaN, infinities and indices far out of range."""
    import smelb
    probs, topi, topv, g = routing(dev, 300, 60, 4, 2)
    mask = torch.rand(300, generator=g, device=dev) < 0.6
    cu = torch.tensor([3, 100, 290], dtype=torch.int32, device=dev)
    t = torch.arange(300, device=dev)
    dead = ~mask | (t < 3) | (t >= 290)
    bad_p, bad_i, bad_v = probs.clone(), topi.clone(), topv.clone()
    bad_p[dead] = torch.tensor([float("nan"), float("inf"), -float("inf")], device=dev).repeat(20)
    bad_i[dead] = 1 << 40
    smelb.read_status()
    a = check(dev, probs, topi, mask, cu)
    b = check(dev, bad_p, bad_i, mask, cu)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    bad_v[~mask], bad_p, bad_i = float("nan"), probs.clone(), topi.clone()
    bad_p[~mask], bad_i[~mask] = float("nan"), -7
    u, v = smelb.expert_usage(probs, topv, topi, mask), smelb.expert_usage(bad_p, bad_v, bad_i, mask)
    assert all(torch.equal(x, y) for x, y in zip(u, v))
    assert smelb.read_status() == 0


def test_indices_out_of_range_are_recorded_and_not_counted(dev):
    import smelb
    probs, topi, topv, _ = routing(dev, 50, 32, 4, 3)
    topi[7, 1], topi[9, 0] = -1, 32
    smelb.read_status()
    check(dev, probs, topi)
    assert smelb.read_status() == 7
    c, _, w = smelb.expert_usage(probs, topv, topi)
    assert c.sum().item() == 198 and smelb.read_status() == 7
    keep = (topi >= 0) & (topi < 32)
    assert abs(w.double().sum() - topv[keep].double().sum()).item() < 1e-3


@pytest.mark.parametrize("T,E,K", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("masked", [False, True])
def test_expert_usage(dev, T, E, K, dtype, masked):
    """Choices may name one expert more than once (`repeat`)."""
    import smelb
    for repeat in (False, True):
        probs, topi, topv, g = routing(dev, T, E, K, T + K, repeat)
        topv = topv.to(dtype)
        mask = (torch.rand(T, generator=g, device=dev) < 0.8) if masked else None
        counts, mass, weight = smelb.expert_usage(probs, topv, topi, mask)
        keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu()
        e = topi.cpu()[keep].reshape(-1)
        assert torch.equal(counts.cpu(), torch.bincount(e, minlength=E))
        rm = probs.cpu().double()[keep].sum(0)
        rw = torch.zeros(E, dtype=torch.float64).index_add_(0, e, topv.cpu().double()[keep].reshape(-1))
        assert bool(((mass.cpu().double() - rm).abs() <= 129 * U * rm).all())
        assert bool(((weight.cpu().double() - rw).abs() <= (128 * K + 17) * U * rw).all())
        again = smelb.expert_usage(probs, topv, topi, mask)
        assert all(torch.equal(x, y) for x, y in zip((counts, mass, weight), again))


def test_strides_and_alignment(dev):
    """A column slice of a wider table, a table that does not start on 16 bytes, a row taken over and over and a
    transposed one give what their copies give."""
    import smelb
    wide, topi, topv, _ = routing(dev, 500, 72, 4, 4)
    topi = topi % 64
    slices = [wide[:, 8:72], wide[:, 3:67], wide.reshape(-1)[1:1 + 64 * 500].view(500, 64), wide[:1, :64].expand(500, 64),
              wide[:64, :64].t().contiguous().t().repeat(8, 1)[:500], wide[::2, :64].repeat(2, 1)]
    for p in slices:
        a = check(dev, p, topi)
        b = check(dev, p.contiguous().clone(), topi)
        assert abs(a[0] - b[0]) <= 129 * U * b[0] and torch.equal(a[2], b[2])
        m = smelb.expert_usage(p, topv, topi)[1]
        r = p.double().sum(0)
        assert bool(((m.double() - r).abs() <= 129 * U * r).all())
    t = wide[:64, :64].t()  # unit stride along the rows
    check(dev, t, topi[:64])
    check(dev, wide[:, :64], topi.t().contiguous().t())


def test_same_bits_and_other_streams(dev):
    """Equal inputs give equal bits, also on another stream with the default one busy."""
    import smelb
    probs, topi, _, _ = routing(dev, 20000, 256, 8, 5)
    cu = torch.tensor([0, 5000, 5001, 20000], dtype=torch.int32, device=dev)
    ref = check(dev, probs, topi, None, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p = probs.detach().requires_grad_(True)
        loss, counts = smelb.balance_loss(p, topi, None, cu)
        d, = torch.autograd.grad(loss, p, torch.tensor(0.37, device=dev))
    side.synchronize()
    assert torch.equal(loss, ref[0]) and torch.equal(counts, ref[1]) and torch.equal(d, ref[2])


def test_captured_twice_and_replayed(dev):
    """Two graphs of the same call, replayed in turn and on two streams at once, on inputs that change between."""
    import smelb
    probs, topi, topv, _ = routing(dev, 3000, 128, 8, 6)
    mask = torch.ones(3000, dtype=torch.bool, device=dev)
    p = probs.clone().requires_grad_(True)

    def step():
        loss, counts = smelb.balance_loss(p, topi, mask)
        d, = torch.autograd.grad(loss, p)
        return (loss, counts, d, *smelb.expert_usage(p.detach(), topv, topi, mask))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        probs2, topi2, _, _ = routing(dev, 3000, 128, 8, 60 + k)
        with torch.no_grad():
            p.copy_(probs2)
        topi.copy_(topi2)
        mask[k * 100:k * 100 + 50] = False
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_gradient_against_differences(dev):
    """The loss is linear in probs while the choices stay: a difference of two losses is the gradient's product with
    the step."""
    import smelb
    probs, topi, _, g = routing(dev, 257, 32, 4, 7)
    cu = torch.tensor([0, 100, 257], dtype=torch.int32, device=dev)
    p = probs.clone().requires_grad_(True)
    d, = torch.autograd.grad(smelb.balance_loss(p, topi, None, cu)[0], p)
    step = torch.rand(257, 32, generator=g, device=dev)
    a, b = smelb.balance_loss(probs + step, topi, None, cu)[0], smelb.balance_loss(probs, topi, None, cu)[0]
    want = (d.double() * step.double()).sum()
    assert abs((a.double() - b.double()) - want) <= 2 * 131 * U * (a.double() + b.double())


def test_no_second_derivative(dev):
    import smelb
    probs, topi, _, _ = routing(dev, 20, 8, 2, 8)
    p = probs.clone().requires_grad_(True)
    loss = smelb.balance_loss(p, topi)[0]
    with pytest.raises(smelb.SmelbError, match="second derivative"):
        torch.autograd.grad(loss, p, create_graph=True)


def test_through_the_layer(dev, golden):
    """moe_forward with the loss taken in its stats callback, as a training step uses it: dx and the usage against the
    oracle in 64 bits with the same choices, and a no-loss step as before."""
    import smelb
    d = golden("moe_c1.pt")
    c = d["cfg"]
    bank = smelb.Int4Experts({"q": d["gu_q"].to(dev), "scale": d["gu_scale"].to(dev), "zero": d["gu_zero"].to(dev)},
                             {"q": d["dn_q"].to(dev), "scale": d["dn_scale"].to(dev), "zero": d["dn_zero"].to(dev)})
    ex = smelb.LayerExperts(bank)
    W = {k: v.bfloat16().to(dev) for k, v in d["W"].items()}
    E, weight = c["E"], 40.0
    x = d["x"].bfloat16().to(dev).requires_grad_(True)
    mask = torch.arange(x.shape[0], device=dev) % 5 != 0
    rec = {}

    def stats(p, v, i):
        rec["loss"], rec["counts"] = smelb.balance_loss(p, i, mask)
        rec["usage"] = smelb.expert_usage(p, v, i, mask)
        rec["i"] = i

    out = smelb.moe_forward(x, W, ex, c["K"], None, stats=stats)
    gy = d["gy"].bfloat16().to(dev)
    (out.float() * gy.float()).sum().add(weight * rec["loss"]).backward()
    assert torch.equal(rec["counts"], rec["usage"][0])
    x64 = x.detach().cpu().double().requires_grad_(True)
    gu = O.dequant_int4(d["gu_q"], d["gu_scale"], d["gu_zero"]).double()
    dn = O.dequant_int4(d["dn_q"], d["dn_scale"], d["dn_zero"]).double()
    W64 = {k: v.cpu().double() for k, v in W.items()}
    topi = rec["i"].cpu()
    ref, _, _, _ = O.moe_layer(x64, W64, gu, dn, c["K"], topi=topi)
    probs = torch.softmax(torch.nn.functional.linear(x64, W64["mlp.gate.weight"]), -1)
    keep = mask.cpu()
    f = torch.bincount(topi[keep].reshape(-1), minlength=E).double() / (c["K"] * keep.sum())
    aux = E * (f * probs[keep].mean(0)).sum()
    assert abs(rec["loss"].item() - aux.item()) <= 2.0 ** -7 * aux.item()  # bf16 logits
    ((ref * gy.cpu().double()).sum() + weight * aux).backward()
    e, cs = O.rel_err(x.grad.float().cpu(), x64.grad), O.cosine(x.grad.float().cpu(), x64.grad)
    assert e < 2e-2 and cs > 0.9999, (e, cs)
    assert smelb.read_status() == 0
