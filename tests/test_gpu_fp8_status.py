"""What fp8.synchronize reports: an in-kernel wait that ran out, once, whoever
asks and whatever else is synchronised meanwhile."""
import threading

import pytest
import torch

from witchcraft_b200 import fp8
from witchcraft_b200._lib import lib

pytestmark = pytest.mark.gpu

TIMEOUT = -5


def run_out(stream):
    assert lib().wc_selftest_fp8_timeout(1_000_000, stream.cuda_stream) == 0


def test_a_wait_that_ran_out_is_raised_once():
    fp8.synchronize()
    run_out(torch.cuda.current_stream())
    with pytest.raises(fp8.WcError, match="timed out"):
        fp8.synchronize()
    fp8.synchronize()
    x = torch.ones(4, 256, device="cuda")
    a, sa = fp8.quantize(x)               # and the context works on
    w, sw = fp8.quantize_weight(x)
    assert (fp8.matmul(a, sa, w, sw, torch.float32) - 256).abs().max() < 1e-2


def test_each_wait_is_reported_exactly_once():
    """Two threads synchronise two streams while one of these has waits that run
    out, each of them over before the next begins."""
    fp8.synchronize()
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    device = torch.cuda.current_device()
    stop, seen = threading.Event(), []

    def watch():
        torch.cuda.set_device(device)
        while not stop.is_set():
            seen.append(lib().wc_fp8_sync(other.cuda_stream))

    t = threading.Thread(target=watch)
    t.start()
    own = []
    for _ in range(200):
        run_out(mine)
        own.append(lib().wc_fp8_sync(mine.cuda_stream))
    stop.set()
    t.join()
    assert set(own) | set(seen) <= {0, TIMEOUT}
    assert own.count(TIMEOUT) + seen.count(TIMEOUT) == 200


@pytest.mark.parametrize("limit", [0, 10 ** 11])
def test_selftest_refuses(limit):
    assert lib().wc_selftest_fp8_timeout(limit, None) == -1
