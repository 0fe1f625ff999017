"""What smelb.balance_loss / expert_usage and their C entry points refuse, checked before any launch (no GPU needed)."""
import pytest
import torch


def test_cpu_tensors_are_refused():
    import smelb
    p, i = torch.rand(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(smelb.SmelbError, match="CUDA tensors only"):
        smelb.balance_loss(p, i)
    with pytest.raises(smelb.SmelbError, match="CUDA tensors only"):
        smelb.expert_usage(p, torch.rand(4, 2), i)


class _Fake:
    """A stand-in with the attributes that the checks read."""

    def __init__(self, shape, dtype, device="cuda:0"):
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, torch.device(device), True

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return self.device.index


@pytest.mark.parametrize("probs,topi,mask,text", [
    (((4, 8), torch.bfloat16), ((4, 2), torch.int64), None, "fp32"),
    (((4, 8, 1), torch.float32), ((4, 2), torch.int64), None, "fp32"),
    (((4, 8), torch.float32), ((4, 2), torch.int32), None, "int64"),
    (((4, 8), torch.float32), ((5, 2), torch.int64), None, "int64"),
    (((4, 513), torch.float32), ((4, 2), torch.int64), None, "E=513"),
    (((4, 8), torch.float32), ((4, 33), torch.int64), None, "K=33"),
    (((4, 8), torch.float32), ((4, 0), torch.int64), None, "K=0"),
    (((4, 8), torch.float32), ((4, 2), torch.int64), ((4,), torch.float32), "mask"),
    (((4, 8), torch.float32), ((4, 2), torch.int64), ((5,), torch.bool), "mask"),
    (((4, 8), torch.float32), ((4, 2), torch.int64), ((4,), torch.bool, "cuda:1"), "cuda:1"),
])
def test_bad_tables_are_refused(probs, topi, mask, text):
    from smelb import SmelbError
    from smelb.balance import _tables
    with pytest.raises(SmelbError, match=text):
        _tables("balance_loss", _Fake(*probs), _Fake(*topi), None if mask is None else _Fake(*mask))


def test_c_entry_points_check_their_arguments():
    from smelb import _lib
    lib = _lib.load()
    fake = 1 << 20  # never dereferenced: a check fails first
    fwd = lambda **k: lib.smelb_balance_loss_fwd(*{**dict(  # noqa: E731
        probs=fake, ld=8, topi=fake, mask=None, cu=None, S=1, T=4, E=8, K=2, loss=fake, counts=fake, coef=fake, ws=fake,
        nb=1 << 30, st=None), **k}.values())
    for k, rc, text in (({"probs": None}, -6, "null pointer"), ({"loss": None}, -6, "null pointer"),
                        ({"T": -1}, -1, "T=-1"), ({"T": 1 << 31}, -1, "T="), ({"E": 513}, -1, "E=513"),
                        ({"K": 33}, -1, "K=33"), ({"S": 0}, -1, "sequences=0"), ({"S": 2}, -6, "without cu_seqlens"),
                        ({"ld": 7}, -1, "row pitch 7"), ({"nb": 16}, -3, "workspace"), ({"ws": fake + 8}, -6, "aligned")):
        assert fwd(**k) == rc and text in _lib.last_error(), (k, _lib.last_error())
    assert lib.smelb_balance_loss_bwd(None, fake, None, None, 1, 4, 8, fake, None) == -6
    assert lib.smelb_balance_loss_bwd(fake, fake, None, None, 3, 4, 8, fake, None) == -6
    assert lib.smelb_balance_loss_bwd(fake, fake, None, None, 1, 0, 8, None, None) == 0
    assert lib.smelb_expert_usage(fake, 8, None, 0, fake, None, 4, 8, 2, fake, fake, fake, fake, 1 << 30, None) == -6
    assert lib.smelb_expert_usage(fake, 8, fake, 0, fake, None, 4, 600, 2, fake, fake, fake, fake, 1 << 30, None) == -1
    assert lib.smelb_expert_usage(fake, 8, fake, 0, fake, None, 4, 8, 2, fake, fake, fake, fake, 8, None) == -3


def test_workspace_holds_a_record_for_every_meeting_of_a_tile_and_a_sequence():
    """Tile b and sequence s use record b + s; the workspace has a record for the last of both, at any lengths."""
    from smelb import _lib
    ws = _lib.load().smelb_balance_workspace_bytes
    for T, E, S in ((0, 8, 1), (1, 8, 1), (4096, 256, 1), (4096, 256, 300), (1 << 22, 512, 7)):
        rows = min(128, max(16, ((T + 591) // 592 + 15) // 16 * 16))
        tiles = -(-T // rows)
        assert ws(T, E, S, 0) >= (tiles + S) * (8 * E + 4) + S * 12
        assert ws(T, E, 1, 1) >= (tiles + 1) * (12 * E + 4)
    assert ws(-1, 8, 1, 0) == 0 and ws(4, 0, 1, 0) == 0
