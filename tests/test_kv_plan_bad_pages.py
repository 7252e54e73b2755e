"""vvb_kv_plan_dev with entries, in a table or on the stack, that are no page of the pool:
their rows get slot -1, whatever the number would be after the shift by the page's size."""
import numpy as np
import pytest

from test_kv_plan import Device

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BAD = [-1, -7, 40, 1 << 25, (1 << 26) + 3, -(1 << 26) + 3, 2 ** 31 - 1, -(2 ** 31)]


@pytest.mark.parametrize("max_rows", [600, 5000, 40000])
def test_rows_on_no_page_of_the_pool_have_no_slot(max_rows):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import vvb200 as vv
    torch.cuda.set_device(0)
    n, n_pages = len(BAD) + 1, 40
    # sequence b: ten positions on a bad page of its own, seventy new tokens: fifty-four there, sixteen on a new page
    table = np.full((n, 2), -1)
    table[:-1, 0], table[-1, 0] = BAD, 11
    lens, new = np.full(n, 10), np.full(n, 70)
    stack = np.concatenate([np.arange(12, 12 + 10), [(1 << 26) + 5, 3], np.full(30, -9)])
    d = Device(new, lens, table, stack, 12, n_pages, max_rows)
    assert vv.vvb_kv_plan_dev(d.args(vv)) == 0
    torch.cuda.synchronize()
    slots, pos = d.slots[:max_rows].tolist(), d.positions[:max_rows].tolist()
    rows = min(70 * n, max_rows)
    fresh = [3, (1 << 26) + 5, 21, 20, 19, 18, 17, 16, 15]
    for b in range(n):
        if 70 * (b + 1) > max_rows:
            continue
        page = [table[b, 0], fresh[b]]
        for r in range(70):
            p = 10 + r
            want = int(page[p // 64]) * 64 + p % 64 if 0 <= page[p // 64] < n_pages else -1
            assert (slots[70 * b + r], pos[70 * b + r]) == (want, p), (b, r)
    assert all(s == -1 for s in slots[rows:])
