"""Where the orthogonalised updates can go wrong besides their formulas: order within a block, host threads, polynomials that
grow, small eps, overlapping tensors, captured optimizer steps. Bounds as in test_gpu_muon.py unless stated."""
import threading

import pytest
import torch

from test_gpu_muon import check, matrices

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
