"""Products enqueued from several host threads, each on a stream of its own."""
import threading

import pytest
import torch

from test_gpu_fp8 import operands
from witchcraft_b200 import fp8

pytestmark = pytest.mark.gpu


def test_same_bits_from_every_thread():
    jobs = []
    for m, k, n in [(1, 768, 768), (32, 768, 2304), (300, 2048, 768), (4000, 768, 2304)]:
        a, sa, (gate, up) = operands(m, k, n, mats=2)
        jobs.append(lambda a=a, sa=sa, gate=gate, up=up: (
            fp8.matmul(a, sa, *gate, torch.float32), *fp8.gated_matmul(a, sa, *gate, *up)))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    device, failed = torch.cuda.current_device(), []

    def work():
        try:
            torch.cuda.set_device(device)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = [job() for job in jobs]
                    fp8.synchronize()
                    for g, w in zip(got, want):
                        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(g, w))
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
