"""smelb.orthogonalize, muon_step and Muon on the GPU against the polynomial on the singular values in 64 bits.

Tolerances. The Gram matrix, the products of the short side and the product with x are fp64, whose errors (grown by at
most 1e5) stay below 1e-9 of the result; it is rounded once, 2^-24 |o| (bf16: 2^-8 |o|)."""
import math

import numpy as np
import pytest
import torch

from oracle import moe_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
COEF = (3.4445, -4.7750, 2.0315)
NAMES = ("A_gate", "B_gate", "A_up", "B_up", "A_down", "B_down")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need CUDA"
    return torch.device("cuda:0")


def exact(x, steps=5, coef=COEF, eps=1e-7):
    """The polynomial of each matrix in 64 bits."""
    x = x.detach().double().cpu().numpy()
    if x.shape[-2] > x.shape[-1]:
        return exact(torch.from_numpy(np.swapaxes(x, -1, -2).copy()), steps, coef, eps).mT
    Uf, s, Vt = np.linalg.svd(x, full_matrices=False)
    n = np.sqrt((s * s).sum(-1, keepdims=True)) + eps
    t = s / n
    cs = [coef] * steps if np.ndim(coef) == 1 else coef
    for a, b, c in cs:
        t = t * (a + b * t ** 2 + c * t ** 4)
    return torch.from_numpy(Uf @ (t[..., None] * Vt))


def matrices(dev, shape, kind, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    m, n = shape[-2:]
    d = min(m, n)
    k = {"full": d, "rank1": 1, "rank3": min(3, d), "decay": d}[kind]
    a = torch.randn(*shape[:-2], m, k, generator=g, device=dev)
    if kind == "decay":
        a = a * 10.0 ** (-0.25 * torch.arange(k, device=dev))
    return a @ torch.randn(*shape[:-2], k, n, generator=g, device=dev) if kind != "full" else torch.randn(*shape, generator=g, device=dev)


def check(out, x, **k):
    ref = exact(x, **k)
    o = out.detach().double().cpu()
    assert out.shape == x.shape and out.dtype == x.dtype
    err = (o - ref).abs()
    rms = ref.pow(2).mean((-1, -2), keepdim=True).sqrt()
    tol = U * ref.abs() + 1e-9 * rms
    if x.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    assert bool((err <= tol).all()), f"{tuple(x.shape)}: {(err / tol.clamp(min=1e-300)).max().item():.2f} of the bound"


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 5), (8, 8), (8, 9), (16, 16), (16, 2048), (2048, 16), (512, 16), (24, 703), (703, 24),
          (33, 100), (100, 31), (48, 513), (64, 64), (64, 65), (64, 2048), (2051, 64), (57, 1000), (5, 20001), (20001, 3),
          (16, 40000), (40000, 12), (64, 6003), (1, 30000), (8, 55296), (24, 15001), (15872, 20), (32, 12000), (10495, 30),
          (16, 26112), (60001, 8)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orthogonalize(dev, m, n, dtype):
    """Full, low and decaying rank and a matrix of zeros, side by side in one batch."""
    import smelb
    x = torch.stack([matrices(dev, (m, n), kind, m + n) for kind in ("full", "rank1", "rank3", "decay")] +
                    [torch.zeros(m, n, device=dev)]).to(dtype)
    out = smelb.orthogonalize(x)
    check(out, x)
    assert not out[-1].any()
    assert torch.equal(out, smelb.orthogonalize(x))


@pytest.mark.parametrize("batch,m,n", [(1, 16, 2048), (300, 16, 512), (700, 512, 16), (150, 64, 300), (0, 16, 64), (1000, 2, 3),
                                       (4100, 33, 34), (5000, 8, 16)])
def test_orthogonalize_batches(dev, batch, m, n):
    import smelb
    x = matrices(dev, (batch, m, n), "full", batch)
    out = smelb.orthogonalize(x)
    if batch:
        check(out, x)
    assert out.shape == x.shape
    y = smelb.orthogonalize(x.reshape(batch, 1, m, n))
    assert torch.equal(y.reshape(out.shape), out)


@pytest.mark.parametrize("scale", [1e-44, 1e-30, 1e-8, 1.0, 1e30])
def test_orthogonalize_scales(dev, scale):
    """Squares that fp32 cannot hold, denormals, and norms near and below eps."""
    import smelb
    for shape in ((2, 16, 300), (2, 300, 16), (1, 64, 64)):
        x = matrices(dev, shape, "full", 5) * scale
        check(smelb.orthogonalize(x), x)
        check(smelb.orthogonalize(x, eps=1e-30), x, eps=1e-30)


@pytest.mark.parametrize("steps,coef", [(1, COEF), (3, (1.5, -0.5, 0.0)), (10, COEF), (16, (1.875, -1.25, 0.375)),
                                        (2, ((4.0, -6.0, 3.0), (1.875, -1.25, 0.375)))])
def test_orthogonalize_polynomials(dev, steps, coef):
    import smelb
    for shape in ((3, 16, 257), (2, 257, 40)):
        x = matrices(dev, shape, "full", steps)
        check(smelb.orthogonalize(x, steps=steps, coefficients=coef), x, steps=steps, coef=coef)


def test_a_converging_polynomial_gives_orthonormal_rows(dev):
    import smelb
    x = matrices(dev, (4, 16, 512), "full", 1)
    o = smelb.orthogonalize(x, steps=16, coefficients=(1.875, -1.25, 0.375)).double()
    assert (o @ o.mT - torch.eye(16, device=dev, dtype=torch.float64)).abs().max() < 1e-5


def test_values_that_are_not_numbers_stay_in_their_matrix(dev):
    import smelb
    x = matrices(dev, (6, 16, 100), "full", 2)
    want = smelb.orthogonalize(x)
    x[1, 3, 7], x[4, 0, 99] = float("nan"), float("inf")
    out = smelb.orthogonalize(x)
    assert out[1].isnan().all() and out[4].isnan().all()
    for i in (0, 2, 3, 5):
        assert torch.equal(out[i], want[i])


def test_strides_alignment_and_aliasing(dev):
    import smelb
    base = matrices(dev, (4, 40, 300), "full", 3)
    for x in (base[:, :16], base[:, ::3, 1:258], base[:, :16].mT, base[::2, 5:9, ::7], base.reshape(-1)[1:1 + 3 * 16 * 200].view(3, 16, 200),
              base[:1, :8].expand(5, 8, 300)):
        assert torch.equal(smelb.orthogonalize(x), smelb.orthogonalize(x.contiguous().clone()))
        check(smelb.orthogonalize(x), x)
    for dt in (torch.bfloat16, torch.float32):
        y = base.to(dt).reshape(-1)[3:3 + 2 * 7 * 129].view(2, 129, 7)
        check(smelb.orthogonalize(y), y)


def emulate(p, g, m_in, m_out, mu, nesterov):
    """The update u that the step orthogonalises, from its own new buffer, in its fp32 operations; and the buffer's."""
    mu32, omu32 = torch.tensor(mu, dtype=torch.float32).double(), torch.tensor(1.0 - mu, dtype=torch.float32)
    og = (omu32 * g.float().cpu()).double()
    m = (mu32 * m_in.cpu().double() + og).float()
    u = (mu32 * m_out.cpu().double() + og).float() if nesterov else m_out.cpu()
    return u, m


def check_step(before, params, grads, bufs, lr, mu=0.95, nesterov=True, wd=0.0, adjust="original", **k):
    for (p0, m0), p, g, m in zip(before, params, grads, bufs):
        u, m_want = emulate(p0, g, m0, m, mu, nesterov)
        assert bool(((m.cpu() - m_want).abs() <= 2 * U * m_want.abs()).all())
        if p.numel() == 0:
            continue
        ref = exact(u, **k)
        rms = ref.pow(2).mean((-1, -2), keepdim=True).sqrt()
        otol = U * ref.abs() + 1e-9 * rms
        rows, cols = p.shape[-2:]
        f = lr * (math.sqrt(max(1.0, rows / cols)) if adjust == "original" else 0.2 * math.sqrt(max(rows, cols)))
        kept = p0.cpu().double() * (1 - lr * wd)
        want = kept - f * ref
        # decay and step rounded once each, their products and the sum
        tol = U * (2 * kept.abs() + f * ref.abs() + want.abs()) * 1.001 + f * otol
        if p.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (want.abs() + tol)
        err = (p.cpu().double() - want).abs()
        assert bool((err <= tol).all()), f"{tuple(p.shape)}: {(err / tol.clamp(min=1e-300)).max().item():.2f} of the bound"


def tensors(dev, shapes, seed, dtype=torch.float32):
    g = torch.Generator(device=dev).manual_seed(seed)
    params = [(torch.randn(s, generator=g, device=dev) * 0.02).to(dtype) for s in shapes]
    kinds = ("full", "rank1", "rank3", "decay")
    grads = [(matrices(dev, s, kinds[i % 4], seed + i) * 1e-3).to(dtype) for i, s in enumerate(shapes)]
    bufs = [matrices(dev, s, kinds[(i + 1) % 4], seed + 100 + i) * 1e-3 for i, s in enumerate(shapes)]
    return params, grads, bufs


LAYER = [(3, 16, 512), (3, 128, 16), (3, 16, 512), (3, 128, 16), (3, 16, 128), (3, 512, 16), (16, 512), (96, 16), (16, 512),
         (96, 16), (16, 96), (512, 16)]


@pytest.mark.parametrize("options", [dict(), dict(nesterov=False), dict(wd=0.1), dict(adjust="match_rms_adamw", mu=0.0),
                                     dict(steps=3, coef=(1.5, -0.5, 0.0))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_muon_step(dev, options, dtype):
    import smelb
    shapes = LAYER + [(8, 33), (33, 8), (2, 2, 24, 40), (64, 130), (0, 16, 64), (1, 1), (45, 77)]
    params, grads, bufs = tensors(dev, shapes, 7, dtype)
    before = [(p.clone(), m.clone()) for p, m in zip(params, bufs)]
    o = dict(options)
    smelb.muon_step(params, grads, bufs, lr=0.02, momentum=o.get("mu", 0.95), nesterov=o.get("nesterov", True),
                    weight_decay=o.get("wd", 0.0), adjust=o.get("adjust", "original"), steps=o.get("steps", 5),
                    coefficients=o.get("coef", COEF))
    check_step(before, params, grads, bufs, 0.02, **o)


@pytest.mark.parametrize("shapes", [
    [(301, 16, 2048), (333, 16, 512), (7, 1000, 16), (1, 16, 30), (50, 513, 12)],
    [(101, 32, 2816), (51, 352, 32), (3, 32, 353), (1, 25, 25), (90, 25, 705)],
    [(150, 8, 4096), (1, 2000, 8), (5, 7, 600), (601, 8, 8)],
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_muon_step_long_and_short_matrices(dev, shapes, dtype):
    """Enough matrices that short ones share a cluster: batches that do not fill their last one, one to eight blocks for a
    matrix."""
    import smelb
    params, grads, bufs = tensors(dev, shapes, 5, dtype)
    before = [(p.clone(), m.clone()) for p, m in zip(params, bufs)]
    smelb.muon_step(params, grads, bufs, lr=0.02, weight_decay=0.1)
    check_step(before, params, grads, bufs, 0.02, wd=0.1)


def test_muon_step_many_tensors(dev):
    """More tensors than one launch takes, and long ones that a block reads twice."""
    import smelb
    shapes = [(16, 64 + i) if i % 2 else (64 + i, 16) for i in range(150)] + [(16, 40000), (30001, 9), (64, 5000)]
    params, grads, bufs = tensors(dev, shapes, 11)
    before = [(p.clone(), m.clone()) for p, m in zip(params, bufs)]
    smelb.muon_step(params, grads, bufs, lr=0.1, weight_decay=0.01)
    check_step(before, params, grads, bufs, 0.1, wd=0.01)
    smelb.muon_step([], [], [], lr=0.1)


def test_unaligned_and_noncontiguous_gradients(dev):
    import smelb
    g = torch.Generator(device=dev).manual_seed(3)
    flat = torch.randn(3, 3 * 16 * 200 + 8, generator=g, device=dev)
    for o in (1, 2, 4):
        p, m = flat[0][o:o + 9600].clone().view(3, 16, 200), flat[2][o:o + 9600].view(3, 16, 200).clone()
        q = torch.empty(9601, device=dev)[1:].view(3, 16, 200).copy_(p)
        n = torch.empty(9601, device=dev)[1:].view(3, 16, 200).copy_(m)
        grad = flat[1][o:o + 9600].view(3, 16, 200)
        smelb.muon_step([p], [grad.contiguous().clone()], [m], lr=0.1)
        smelb.muon_step([q], [grad], [n], lr=0.1)
        assert torch.equal(p, q) and torch.equal(m, n)
        smelb.muon_step([p], [grad.mT.contiguous().mT], [m], lr=0.1)
        smelb.muon_step([q], [grad], [n], lr=0.1)
        assert torch.equal(p, q) and torch.equal(m, n)


def test_a_backward_over_changed_parameters_is_refused(dev):
    """The step changes params in place, and autograd notices as after any in-place operation."""
    import smelb
    p = torch.randn(16, 64, device=dev, requires_grad=True)
    y = (p * p).sum()
    smelb.muon_step([p], [torch.randn(16, 64, device=dev)], [torch.zeros(16, 64, device=dev)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_streams_and_graphs(dev):
    """On another stream, captured twice and replayed at once: each replay moves its own tensors one step."""
    import smelb
    sets = [tensors(dev, LAYER, 20 + i) for i in range(2)]
    ref = [[[t.clone() for t in ts] for ts in s] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        smelb.muon_step(*sets[0], lr=0.1)
    side.synchronize()
    smelb.muon_step(*ref[0], lr=0.1)
    graphs = []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            smelb.muon_step(*s, lr=0.1)
            o = smelb.orthogonalize(s[1][0])
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for r in ref:
            smelb.muon_step(*r, lr=0.1)
        for s, r in zip(sets, ref):
            for a, b in zip(s, r):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(o, smelb.orthogonalize(sets[1][1][0]))


def test_optimizer(dev):
    """Muon over parameter groups: the steps of muon_step, the state's round trip (bf16 parameters too), a scheduler's lr,
    parameters without a gradient left alone."""
    import smelb
    for dtype in (torch.float32, torch.bfloat16):
        params, grads, bufs = tensors(dev, LAYER, 31, dtype)
        ps = [torch.nn.Parameter(p.clone()) for p in params]
        idle = torch.nn.Parameter(torch.ones(16, 8, device=dev, dtype=dtype))
        opt = smelb.Muon([{"params": ps[:5]}, {"params": ps[5:] + [idle], "weight_decay": 0.1}], lr=0.05)
        bufs = [torch.zeros_like(m) for m in bufs]
        for k in range(3):
            for group in opt.param_groups:
                group["lr"] = 0.05 / (k + 1)
            for p, g in zip(ps, grads):
                p.grad = g * (k + 1)
            assert opt.step(lambda: 3.0) == 3.0
            smelb.muon_step(params[:5], [g * (k + 1) for g in grads[:5]], bufs[:5], lr=0.05 / (k + 1))
            smelb.muon_step(params[5:], [g * (k + 1) for g in grads[5:]], bufs[5:], lr=0.05 / (k + 1), weight_decay=0.1)
            assert all(torch.equal(a, b) for a, b in zip(ps, params))
            if k == 1:
                new = smelb.Muon([{"params": ps[:5]}, {"params": ps[5:] + [idle], "weight_decay": 0.1}], lr=0.05)
                new.load_state_dict(opt.state_dict())
                opt = new
        assert bool((idle == 1).all()) and idle not in opt.state
        assert all(opt.state[p]["momentum_buffer"].dtype == torch.float32 and
                   torch.equal(opt.state[p]["momentum_buffer"], m) for p, m in zip(ps, bufs))


def test_a_training_step_of_the_layer(dev, golden):
    """The operators as a training step uses them: moe_forward, the balance loss from its stats callback, backward, and
    Muon over the layer's LoRA factors. Each factor moves by the orthogonalised update of its own gradient."""
    import smelb
    d = golden("moe_c1.pt")
    c = d["cfg"]
    sel = c["sel"]
    bank = smelb.Int4Experts({"q": d["gu_q"].to(dev), "scale": d["gu_scale"].to(dev), "zero": d["gu_zero"].to(dev)},
                             {"q": d["dn_q"].to(dev), "scale": d["dn_scale"].to(dev), "zero": d["dn_zero"].to(dev)})
    ex = smelb.LayerExperts(bank, sel, d["gu"][sel].bfloat16().to(dev), d["dn"][sel].bfloat16().to(dev))
    W = {k: v.bfloat16().to(dev) for k, v in d["W"].items()}
    lora = smelb.LayerLoRA(smelb.ExpertsLoRA(sel, c["H"], c["I"], c["r"], c["alpha"]),
                           smelb.MLPLoRA(c["H"], c["S"], c["r"], c["alpha"])).to(dev)
    opt = smelb.Muon(lora.parameters(), lr=0.02, weight_decay=0.01)
    x = d["x"].bfloat16().to(dev)
    gy = d["gy"].bfloat16().to(dev)
    for _ in range(3):
        aux = []
        out = smelb.moe_forward(x.clone().requires_grad_(True), W, ex, c["K"], lora,
                                stats=lambda p, v, i: aux.append(smelb.balance_loss(p, i)[0]))
        opt.zero_grad()
        ((out.float() * gy.float()).mean() + 0.01 * aux[0]).backward()
        ps = [p for p in lora.parameters()]
        before = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone() if p in opt.state else torch.zeros_like(p))
                  for p in ps]
        opt.step()
        check_step(before, [p.detach() for p in ps], [p.grad for p in ps], [opt.state[p]["momentum_buffer"] for p in ps],
                   0.02, wd=0.01)
    assert smelb.read_status() == 0


def test_status_and_oracle_agree_on_the_iteration(dev):
    """The polynomial on the singular values is the iteration itself: the plain products in 64 bits."""
    x = matrices(dev, (3, 16, 100), "decay", 4).double().cpu()
    X = x / (x.pow(2).sum((-1, -2), keepdim=True).sqrt() + 1e-7)
    a, b, c = COEF
    for _ in range(5):
        G = X @ X.mT
        X = a * X + (b * G + c * G @ G) @ X
    assert O.rel_err(exact(x), X) < 1e-9
