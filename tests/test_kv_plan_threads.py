"""vvb_kv_plan_dev from two host threads at once, with shared memory of different sizes:
neither call may change what the other one launches with."""
import threading

import numpy as np
import pytest

import _paged
from test_kv_plan import Device, build

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_rows", [(4096, 3000), (40000, 40000)])
def test_two_threads_plan_different_numbers_of_sequences(max_rows):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import vvb200 as vv
    torch.cuda.set_device(0)
    sides, errors = [], []
    for n, m in zip((8192, 3000), max_rows):
        new, lens, table, stack, count, n_pages = build(np.random.default_rng(n), n, 3, "mixed", m)
        d = Device(new, lens, table, stack, count, n_pages, m)
        sides.append((d, d.args(vv), _paged.plan(new, lens, table, stack, count, m), torch.cuda.Stream()))
    torch.cuda.synchronize()
    begin = threading.Barrier(2)

    def work(d, args, want, stream):
        torch.cuda.set_device(0)
        begin.wait()
        for _ in range(1500):
            r = vv.vvb_kv_plan_dev(args, stream)
            if r != 0:
                errors.append((d.n, r))
                return
        stream.synchronize()

    threads = [threading.Thread(target=work, args=s) for s in sides]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for d, _, want, _ in sides:                        # the same inputs every time: the same outputs
        d.compare(want)
