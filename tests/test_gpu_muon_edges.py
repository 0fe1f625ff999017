"""Where the orthogonalised updates can go wrong besides their formulas: order within a block, host threads, polynomials that
grow, small eps, overlapping tensors, captured optimizer steps. Bounds as in test_gpu_muon.py unless stated."""
import math
import threading
from fractions import Fraction

import numpy as np
import pytest
import torch

from test_gpu_muon import COEF, U, check, check_step, matrices, tensors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need CUDA"
    return torch.device("cuda:0")


@pytest.mark.parametrize("shape", [(3000, 8, 64), (3000, 5, 40), (3000, 16, 64), (3000, 11, 33), (40, 16, 9000), (40, 8, 9000)])
def test_many_blocks_side_by_side_give_the_same_bits(dev, shape):
    """Blocks of up to 16 rows with all SMs full: each matrix gets one scale for all of its rows, every time."""
    import smelb
    x = matrices(dev, shape, "full", 9)
    first = smelb.orthogonalize(x)
    check(first[::37], x[::37])
    for _ in range(20):
        assert torch.equal(smelb.orthogonalize(x), first)


@pytest.mark.parametrize("rows", [24, 40])
def test_host_threads_with_other_sizes(dev, rows):
    """Threads that launch the same kernels with more and with less shared memory, each on its own stream: none is refused."""
    import smelb
    xs = [matrices(dev, (1, rows, n), "full", n) for n in (40, 500, 2000, 4000)]
    want = [smelb.orthogonalize(x) for x in xs]
    torch.cuda.synchronize()
    failed = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    out = smelb.orthogonalize(xs[k])
                torch.cuda.current_stream().synchronize()
                assert torch.equal(out, want[k])
        except Exception as e:  # noqa: BLE001
            failed.append((k, e))

    threads = [threading.Thread(target=work, args=(k % 4,)) for k in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def truth(x, steps, coef=COEF, eps=1e-7, bits=260):
    """The iteration on x in whole numbers of 2^-bits: what 64 bits cannot hold once small singular values have grown."""
    if x.dim() > 2:
        return torch.stack([truth(m, steps, coef, eps, bits) for m in x])
    if x.shape[0] > x.shape[1]:
        return truth(x.mT, steps, coef, eps, bits).mT
    fix = lambda v: int(Fraction(float(v)) * (1 << bits))  # noqa: E731
    X = np.array([[fix(v) for v in row] for row in x.double().cpu().tolist()], dtype=object)
    n = math.isqrt(int((X * X).sum())) + fix(eps)
    X = (X << bits) // n
    for a, b, c in [coef] * steps if np.ndim(coef) == 1 else coef:
        G = X @ X.T >> bits
        S = fix(b) * G + (fix(c) * (G @ G >> bits)) >> bits
        S[np.diag_indices(len(S))] += fix(a)
        X = S @ X >> bits
    return torch.tensor([[float(Fraction(int(v), 1 << bits)) for v in row] for row in X], dtype=torch.float64)


def check_grown(out, x, steps, coef=COEF):
    """One rounding of the result, 1e-9 for the sums, and 2^-53 * 2^26 for a rounding of G that has grown as far as the kernels in
    single doubles let it (the result's singular values are at most 1.3)."""
    ref = truth(x, steps, coef)
    rms = ref.pow(2).mean((-1, -2), keepdim=True).sqrt()
    tol = U * ref.abs() + 1e-9 * rms + 2.0 ** -27
    if x.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{tuple(x.shape)}, {steps} steps: {(err / tol).max().item():.2f} of the bound"


@pytest.mark.parametrize("steps", [7, 8, 10, 12, 14, 16])
@pytest.mark.parametrize("m,n", [(16, 96), (96, 16), (5, 40), (1, 9), (24, 60), (33, 70), (100, 64), (3, 4200)])
def test_many_steps_on_matrices_of_low_rank(dev, m, n, steps):
    """Singular values near zero, as gradients of few tokens have, grow by 3.4 a step: to one after 16 of fp32's rounding."""
    import smelb
    for dtype in (torch.float32, torch.bfloat16):
        kinds = ("rank1", "rank3", "decay") if m * n < 3000 else ("rank1",)
        x = torch.stack([matrices(dev, (m, n), kind, steps + m) for kind in kinds] + [torch.zeros(m, n, device=dev)]).to(dtype)
        out = smelb.orthogonalize(x, steps=steps)
        check_grown(out, x, steps)
        assert not out[-1].any() and torch.equal(out, smelb.orthogonalize(x, steps=steps))


def test_growth_is_what_counts(dev):
    """Triples of their own for each step, large ones first, and many steps that grow little."""
    import smelb
    coef = ((8.28721, -23.5959, 17.30039), (4.10706, -2.94785, 0.54484), (3.94869, -2.90890, 0.55182), (3.31842, -2.48849, 0.51005),
            (2.30065, -1.66890, 0.41888), (1.89130, -1.26800, 0.37680), (1.875, -1.25, 0.375), (1.875, -1.25, 0.375),
            (1.875, -1.25, 0.375), (1.875, -1.25, 0.375))
    for shape in ((2, 16, 60), (2, 40, 50)):
        for kind in ("rank1", "decay"):
            x = matrices(dev, shape, kind, 3)
            for steps in (8, 10):
                check_grown(smelb.orthogonalize(x, steps=steps, coefficients=coef[:steps]), x, steps, coef[:steps])
            check_grown(smelb.orthogonalize(x, steps=16, coefficients=(1.875, -1.25, 0.375)), x, 16, (1.875, -1.25, 0.375))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_step_of_many_steps(dev, dtype, nesterov):
    """Full-rank updates, which the 64-bit singular values still settle, of every size class in one step."""
    import smelb
    shapes = [(3, 16, 128), (3, 128, 16), (1, 1), (8, 8), (2, 600, 24), (40, 90), (64, 64), (2, 7, 5000), (0, 16, 32), (1, 30)]
    params, grads, bufs = tensors(dev, shapes, 13, dtype)
    grads, bufs = [torch.randn_like(g) * 1e-3 for g in grads], [torch.randn_like(m) * 1e-3 for m in bufs]
    before = [(p.clone(), m.clone()) for p, m in zip(params, bufs)]
    smelb.muon_step(params, grads, bufs, lr=0.02, nesterov=nesterov, weight_decay=0.1, steps=12)
    check_step(before, params, grads, bufs, 0.02, nesterov=nesterov, wd=0.1, steps=12)


def test_many_steps_strides_values_and_aliasing(dev):
    import smelb
    base = matrices(dev, (4, 40, 300), "full", 3)
    for x in (base[:, :16], base[:, ::3, 1:258], base[:, :16].mT, base.reshape(-1)[1:1 + 3 * 16 * 200].view(3, 16, 200)):
        assert torch.equal(smelb.orthogonalize(x, steps=10), smelb.orthogonalize(x.contiguous().clone(), steps=10))
        check(smelb.orthogonalize(x, steps=10), x, steps=10)
    x = matrices(dev, (6, 16, 100), "full", 2)
    want = smelb.orthogonalize(x, steps=10)
    x[1, 3, 7], x[4, 0, 99] = float("nan"), float("inf")
    out = smelb.orthogonalize(x, steps=10)
    assert out[1].isnan().all() and out[4].isnan().all()
    assert all(torch.equal(out[i], want[i]) for i in (0, 2, 3, 5))
    for scale in (1e-44, 1e-8, 1e30):
        y = matrices(dev, (2, 16, 60), "full", 5) * scale
        check(smelb.orthogonalize(y, steps=9), y, steps=9)


@pytest.mark.parametrize("eps", [1e-80, 1e-300])
def test_zeros_stay_zeros_with_any_eps(dev, eps):
    """1 / eps^4 is past fp64 here; matrices of fp32's smallest numbers are orthogonalised as any other."""
    import smelb
    for m, n in ((4, 9), (8, 40), (16, 300), (30, 24), (100, 40), (64, 2048), (16, 5000)):
        for steps in (5, 10):
            x = matrices(dev, (4, m, n), "full", m)
            x[1], x[2] = 0.0, x[2] * 1e-43
            out = smelb.orthogonalize(x, eps=eps, steps=steps)
            assert not out[1].any()
            check(out[::2], x[::2], eps=eps, steps=steps)
    p = [torch.ones(3, 16, 64, device=dev), torch.ones(2, 64, 40, device=dev)]
    zeros = [torch.zeros_like(t) for t in p]
    smelb.muon_step(p, zeros, [z.clone() for z in zeros], lr=0.1, eps=eps)
    assert all(bool((t == 1).all()) for t in p)


@pytest.mark.parametrize("shape", [(3000, 16, 96), (3000, 96, 13), (600, 30, 200), (300, 64, 240), (40, 16, 5000)])
def test_bf16_results_are_rounded_once(dev, shape):
    """Next to the middle between two bf16 numbers a rounding to fp32 on the way would decide wrongly: none may be more than
    half a step off (but for 1e-9, what the sums in 64 bits may be off)."""
    import smelb
    x = matrices(dev, shape, "full", 8).bfloat16()
    X = x.double() if shape[1] <= shape[2] else x.double().mT  # the iteration itself, on the device for its size
    X = X / (X.square().sum((-1, -2), keepdim=True).sqrt() + 1e-7)
    a, b, c = COEF
    for _ in range(5):
        G = X @ X.mT
        X = a * X + (b * G + c * G @ G) @ X
    ref = X if shape[1] <= shape[2] else X.mT
    out = smelb.orthogonalize(x).double()
    step = torch.exp2(torch.floor(torch.log2(ref.abs())) - 7)  # bf16 keeps seven bits behind the first
    err = (out - ref).abs()
    assert ref.numel() > 3e6 and bool((err <= step / 2 + 1e-9 * step).all()), (err / step).max().item()


def test_captured_optimizer_steps_keep_their_momentum(dev):
    """A captured first step would make new buffers of zeros at each replay: it is refused, and after one step in the open the
    replays are the steps."""
    import smelb
    params, grads, _ = tensors(dev, [(3, 16, 128), (96, 16), (64, 40)], 17)
    ps, qs = ([torch.nn.Parameter(p.clone()) for p in params] for _ in range(2))
    opt, ref = smelb.Muon(ps, lr=0.05), smelb.Muon(qs, lr=0.05)
    for p, q, g in zip(ps, qs, grads):
        p.grad, q.grad = g.clone(), g.clone()
    with pytest.raises(smelb.SmelbError, match="take a step before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    ref.step()
    for _ in range(3):
        graph.replay()
        ref.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert all(torch.equal(opt.state[p]["momentum_buffer"], ref.state[q]["momentum_buffer"]) for p, q in zip(ps, qs))


def test_bf16_results_below_the_normal_numbers(dev):
    """Multiples of 2^-133 are bf16's numbers there."""
    import smelb
    x = torch.randn(2000, 1, 60, generator=torch.Generator(device=dev).manual_seed(4), device=dev).bfloat16()
    x[:, 0, 1:] *= torch.exp2(torch.randint(-134, -120, (2000, 59), device=dev).float()).bfloat16()
    X = x.double()
    t = X.square().sum((-1, -2), keepdim=True).sqrt()
    s = t / (t + 1e-7)
    a, b, c = COEF
    r = s.clone()
    for _ in range(5):
        r = r * (a + b * r ** 2 + c * r ** 4)
    ref = X / t * r
    step = torch.exp2(torch.floor(torch.log2(ref.abs())).clamp(min=-126) - 7)
    err = (smelb.orthogonalize(x).double() - ref).abs()
    assert bool((err[ref != 0] <= (step / 2 * (1 + 1e-9))[ref != 0]).all()) and bool((err[ref == 0] == 0).all())
