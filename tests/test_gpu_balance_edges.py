"""Where the routing losses can go wrong besides their formulas. Bounds as in test_gpu_balance.py unless stated."""
import pytest
import torch

from test_gpu_balance import check, routing

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
