"""What smelb.orthogonalize, muon_step, Muon and their C entry points refuse before any launch (no GPU needed)."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    import smelb
    t = torch.zeros(4, 16, 32)
    with pytest.raises(smelb.SmelbError, match="CUDA tensors only"):
        smelb.orthogonalize(t)
    with pytest.raises(smelb.SmelbError, match="CUDA tensors only"):
        smelb.muon_step([t], [t], [t], lr=0.1)


class _Fake:
    def __init__(self, shape, dtype=torch.float32, device="cuda:0", at=1 << 20):
        self.at = at
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, torch.device(device), True
        self.requires_grad = False

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return self.shape[-1] != 99

    def data_ptr(self):
        return self.at

    def get_device(self):
        return self.device.index


@pytest.mark.parametrize("t,text", [(_Fake((16,)), "matrices"), (_Fake((16, 32), torch.float16), "matrices"),
                                    (_Fake((65, 65)), "short side"), (_Fake((2, 0, 4)), "short side"),
                                    (_Fake((4, 128, 100)), "short side")])
def test_bad_matrices(t, text):
    import smelb
    with pytest.raises(smelb.SmelbError, match=text):
        smelb.orthogonalize(t)


def test_bad_options():
    import smelb
    ok = _Fake((2, 16, 32))
    for k, text in (({"steps": 0}, "steps"), ({"steps": 17}, "steps"), ({"coefficients": (1.0, 2.0)}, "coefficients"),
                    ({"coefficients": ((1, 2, 3), (1, 2, 3))}, "coefficients"), ({"eps": 0.0}, "eps"),
                    ({"eps": float("nan")}, "eps")):
        with pytest.raises(smelb.SmelbError, match=text):
            smelb.orthogonalize(ok, **k)
        with pytest.raises(smelb.SmelbError, match=text):
            smelb.muon_step([ok], [ok], [ok], lr=0.1, **k)
    grad = torch.zeros(4, 4, requires_grad=True)
    with pytest.raises(smelb.SmelbError, match="no backward"):
        smelb.orthogonalize(grad)


def test_tensors_that_do_not_fit_together():
    import smelb
    ok = _Fake((2, 16, 32))
    for p, g, m, text in (([ok], [], [ok], "0 grads"), ([ok], [_Fake((2, 32, 16))], [ok], "grads"),
                          ([ok], [_Fake((2, 16, 32), torch.bfloat16)], [ok], "grads"),
                          ([ok], [ok], [_Fake((2, 16, 32), torch.bfloat16)], "buffers"),
                          ([ok], [ok], [_Fake((2, 16, 32), device="cuda:1")], "buffers"),
                          ([ok, _Fake((2, 16, 32), torch.bfloat16)], [ok, ok], [ok, ok], "params"),
                          ([_Fake((16, 99))], [_Fake((16, 99))], [_Fake((16, 99))], "contiguous")):
        with pytest.raises(smelb.SmelbError, match=text):
            smelb.muon_step(p, g, m, lr=0.1)
    a, b, c = (_Fake((2, 16, 32), at=k << 20) for k in (1, 2, 3))
    for p, g, m in (([a], [b], [a]), ([a, a], [b, b], [c, _Fake((2, 16, 32), at=5 << 20)]), ([a], [a], [b]),
                    ([a], [c], [c]), ([a, b], [c, c], [_Fake((2, 16, 32), at=7 << 20)] * 2)):
        with pytest.raises(smelb.SmelbError, match="twice"):
            smelb.muon_step(p, g, m, lr=0.1)
    with pytest.raises(smelb.SmelbError, match="adjust"):
        smelb.muon_step([ok], [ok], [ok], lr=0.1, adjust="rms")


def test_optimizer_arguments():
    import smelb
    ok = torch.nn.Parameter(torch.zeros(4, 16, 512))
    for bad in (torch.zeros(16), torch.zeros(100, 65), torch.zeros(0, 4)):
        with pytest.raises(ValueError, match="short side"):
            smelb.Muon([ok, torch.nn.Parameter(bad)])
    for k in ({"lr": -1.0}, {"momentum": 1.0}, {"weight_decay": -0.1}, {"adjust": "x"}, {"eps": 0.0}):
        with pytest.raises(ValueError):
            smelb.Muon([ok], **k)
    with pytest.raises(smelb.SmelbError, match="steps"):
        smelb.Muon([ok], steps=40)
    assert smelb.Muon([ok]).step() is None  # nothing has a gradient


def test_c_entry_points_check_their_arguments():
    from smelb import _lib
    lib = _lib.load()
    fake = 1 << 20  # never dereferenced: a check fails first
    coef = (ctypes.c_double * 15)(*([1.0, 0.0, 0.0] * 5))
    o = lambda **k: lib.smelb_orthogonalize(*{**dict(x=fake, dtype=0, batch=1, m=16, n=32, steps=5, coef=coef,  # noqa: E731
                                                     eps=1e-7, out=fake, ws=None, nb=0, st=None),
                                                **k}.values())
    for k, rc, text in (({"x": None}, -6, "null"), ({"out": None}, -6, "null"), ({"dtype": 2}, -2, "dtype"),
                        ({"m": 0}, -1, "short side"), ({"m": 65, "n": 65}, -1, "short side"), ({"batch": -1}, -1, "-1 x"),
                        ({"n": 1 << 24}, -1, "short side"), ({"steps": 0}, -6, "steps"), ({"steps": 17}, -6, "steps"),
                        ({"coef": None}, -6, "steps"), ({"eps": 0.0}, -6, "eps"), ({"eps": float("nan")}, -6, "eps")):
        assert o(**k) == rc and text in _lib.last_error(), (k, _lib.last_error())
    assert o(batch=0, x=None, out=None) == 0
    assert o(m=64, n=2048) == -3 and "workspace" in _lib.last_error()
    assert o(m=64, n=2048, ws=fake + 8, nb=1 << 30) == -6 and "aligned" in _lib.last_error()
    t = (_lib.MuonTensor * 2)()
    t[0].p = t[0].g = t[0].m = fake
    t[0].batch, t[0].rows, t[0].cols = 1, 16, 32
    t[1].p = t[1].g = fake
    t[1].batch, t[1].rows, t[1].cols = 1, 16, 32
    step = lambda n=2, adjust=0: lib.smelb_muon_step(t, n, 0, 0.1, 0.9, 1, 0.0, adjust, 5, coef, 1e-7, None, 0,  # noqa: E731
                                                   None)
    assert step() == -6 and "null" in _lib.last_error()  # checked for every tensor before the first launch
    assert step(adjust=2) == -6 and step(n=-1) == -6 and step(n=0) == 0


def test_workspace_sizes():
    """Short sides up to 32 need none unless they are longer than eight blocks hold; the rest a partial Gram matrix for each
    block and the polynomial's matrix. The largest launch of a call decides."""
    from smelb import _lib
    lib = _lib.load()
    ws = lib.smelb_orthogonalize_workspace_bytes
    assert ws(12, 16, 2048) == 0 and ws(12, 2048, 16) == 0 and ws(5, 32, 4096) == 0 and ws(0, 64, 2048) == 0
    assert ws(5, 32, 4097) > 0 and ws(1, 16, 4097) > 0 and ws(1, 33, 40) > 0
    assert ws(1000, 64, 2048) >= 1000 * (36 + 64) * 64 * 8 and ws(1, 64, 1 << 20) >= 32 * 36 * 64 * 8
    assert ws(1 << 20, 64, 64) == ws(4096, 64, 64)  # rounds of 4096 matrices
    assert ws(1, 65, 65) == -1 and ws(-1, 16, 16) == -1
    t = (_lib.MuonTensor * 2)()
    for i, (b, m, n) in enumerate(((3, 64, 500), (7, 2000, 48))):
        t[i].batch, t[i].rows, t[i].cols = b, m, n
    assert lib.smelb_muon_workspace_bytes(t, 2) == max(ws(3, 64, 500), ws(7, 2000, 48))
    assert lib.smelb_muon_workspace_bytes(t, 0) == 0 and lib.smelb_muon_workspace_bytes(None, 0) == 0


def test_overlapping_tensors_are_refused():
    """A tensor that is written may share memory with no other one, whole or in part; gradients may with each other."""
    from smelb import _lib
    lib = _lib.load()
    coef = (ctypes.c_double * 15)(*([1.0, 0.0, 0.0] * 5))
    size, at = 16 * 32 * 4, 1 << 20  # the addresses are never used: a check fails first

    def step(*tensors, dtype=0):
        t = (_lib.MuonTensor * len(tensors))()
        for i, (p, g, m, batch) in enumerate(tensors):
            t[i].p, t[i].g, t[i].m, t[i].batch, t[i].rows, t[i].cols = at + p, at + g, at + m, batch, 16, 32
        # the last check before the launches wants a 256-byte aligned workspace: -6 with this text is "no overlap found"
        rc = lib.smelb_muon_step(t, len(tensors), dtype, 0.1, 0.9, 1, 0.0, 0, 5, coef, 1e-7, 8, 0, None)
        return rc, _lib.last_error()

    fine = (-6, "aligned")
    for tensors, dtype, want in (
            (((0, size, 2 * size, 1),), 0, fine),
            (((0, size, 2 * size, 1), (3 * size, size, 4 * size, 1)), 0, fine),             # one gradient for two
            (((0, size, 2 * size, 1), (3 * size, size + 64, 4 * size, 1)), 0, (-6, "share")),   # it reaches into a buffer
            (((0, size // 2, size, 1),), 1, fine),                                            # bf16: half the bytes
            (((0, size // 2, size, 1),), 0, (-6, "share")),
            (((4, size + 4, size, 1),), 0, (-6, "share")),
            (((0, size, 2 * size, 2),), 0, (-6, "share")),                                    # a longer batch
            (((0, 9 * size, 2 * size, 2), (4 * size, 5 * size, size - 4, 1)), 0, (-6, "share")),
            (((0, 0, 0, 0), (0, size, 2 * size, 1)), 0, fine),                                # an empty one anywhere
            (((10 * size, 0, 20 * size, 8), (9 * size, 30 * size, 17 * size - 4, 1)), 0, (-6, "share"))):
        rc, text = step(*tensors, dtype=dtype)
        assert rc == want[0] and want[1] in text, (tensors, rc, text)
    o = lambda x, out: lib.smelb_orthogonalize(at + x, 0, 1, 16, 32, 5, coef, 1e-7, at + out, 8, 0, None)  # noqa: E731
    for x, out, text in ((0, 0, "aligned"), (0, size, "aligned"), (0, 4, "share"), (size - 4, 0, "share")):
        assert o(x, out) == -6 and text in _lib.last_error(), (x, out)
