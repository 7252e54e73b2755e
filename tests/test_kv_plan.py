"""vvb_kv_plan_dev: block tables, slot map and positions from request lengths,
against the definition worked out sequence by sequence in Python integers
(tests/_paged.py). Every output is a whole number and has to be equal."""
import numpy as np
import pytest

import _paged

P = 0x1000                                            # a fake address: never dereferenced


def fake(vv, **kw):
    a = dict(new_tokens=P, lens=P, lens_out=P, block_table=P, free_pages=P, free_count=P, free_count_out=P, row_start=P,
             slot_map=P, positions=P, status=P, n_seqs=4, table_stride=8, n_pages=32, max_rows=16)
    a.update(kw)
    return vv.make_kv_plan(*a.values())


@pytest.fixture(scope="module")
def lib():
    import vvb200
    return vvb200


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("kw,want", [
    (dict(new_tokens=None), "VV_ERR_NULL_PTR"), (dict(lens=None), "VV_ERR_NULL_PTR"), (dict(lens_out=None), "VV_ERR_NULL_PTR"),
    (dict(block_table=None), "VV_ERR_NULL_PTR"), (dict(free_pages=None), "VV_ERR_NULL_PTR"), (dict(free_count=None), "VV_ERR_NULL_PTR"),
    (dict(free_count_out=None), "VV_ERR_NULL_PTR"), (dict(row_start=None), "VV_ERR_NULL_PTR"), (dict(slot_map=None), "VV_ERR_NULL_PTR"),
    (dict(positions=None), "VV_ERR_NULL_PTR"), (dict(n_seqs=-1), "VV_ERR_INVALID_ARG"), (dict(table_stride=0), "VV_ERR_INVALID_ARG"),
    (dict(n_pages=-1), "VV_ERR_INVALID_ARG"), (dict(max_rows=-1), "VV_ERR_INVALID_ARG"), (dict(table_stride=1 << 25), "VV_ERR_OVERFLOW"),
    (dict(n_pages=1 << 25), "VV_ERR_OVERFLOW"), (dict(n_seqs=8193), "VV_ERR_UNSUPPORTED"), (dict(status=P + 2), "VV_ERR_INVALID_ARG"),
    (dict(lens=P + 1), "VV_ERR_INVALID_ARG"), (dict(n_seqs=0), "VV_OK"), (dict(n_seqs=0, status=None, max_rows=0, slot_map=None), "VV_OK"),
])
def test_plan_refusals(lib, kw, want):
    assert lib.vvb_kv_plan_dev(fake(lib, **kw), stream=0) == getattr(lib, want)


def test_plan_null_argument_block(lib):
    assert lib._lib.vvb_kv_plan_dev(None, None) == lib.VV_ERR_NULL_PTR


def test_plan_reference_by_hand():
    """The Python definition on a case small enough to write down."""
    table = np.full((4, 3), -1)
    table[0, :2] = [7, 3]                             # 70 positions
    table[2, 0] = 5                                   # 10 positions, released
    got = _paged.plan([2, 65, -1, 0], [70, 0, 10, 0], table, [9, 8], 2, 70)
    assert got["pushed"] == [9, 8, 5] and got["count"] == 1 and got["status"] == [0, 0, 0, 0]
    assert got["table"][1].tolist() == [5, 8, -1] and got["lens"] == [72, 65, 0, 0] and got["start"] == [0, 2, 67, 67, 67]
    assert got["slots"][:4] == [3 * 64 + 6, 3 * 64 + 7, 320, 321] and got["slots"][66:] == [8 * 64, -1, -1, -1]
    assert got["positions"][:3] == [70, 71, 0] and got["positions"][66:] == [64, -1, -1, -1]


# ------------------------------------------------------------------ GPU
torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def vv(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return lib


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def requests(rng, n, stride, kind, max_rows):
    lens = rng.integers(0, stride * 64 // 2 + 1, n)
    if kind == "step":
        new = np.ones(n, np.int64)
    elif kind == "mixed":
        new = rng.choice([-1, 0, 1, 1, 1, 63, 64, 65, 200], n)
        lens[rng.random(n) < 0.2] = 0
    elif kind in ("scarce", "pages"):                 # more is asked for than there is: rows and tables, or pages, run out
        new = rng.choice([-5, 0, 1, 64, 128, 129, stride * 64], n)
    else:
        new = rng.integers(0, max(1, 2 * max_rows // n) + 1, n)
    return new, lens


def build(rng, n, stride, kind, max_rows):
    new, lens = requests(rng, n, stride, kind, max_rows)
    pages = -(-lens // 64)
    held = int(pages.sum())
    need = int((-(-(lens + np.maximum(new, 0)) // 64) - pages).sum())
    n_pages = held + (need // 3 if kind == "scarce" else need // 25 if kind == "pages" else need + 4)
    order = rng.permutation(n_pages)
    table = np.full((n, stride), -7)
    table[np.arange(stride)[None, :] < pages[:, None]] = order[:held]
    stack = np.full(max(n_pages, 1), -9)
    stack[: n_pages - held] = order[held:]
    return new, lens, table, stack, n_pages - held, n_pages


class Device:
    def __init__(self, new, lens, table, stack, count, n_pages, max_rows, in_place=False, status=True, offset=0):
        n = len(new)
        self.new, self.lens, self.table, self.stack, self.count = ints(new), ints(lens), ints(table), ints(stack), ints([count])
        self.lens_out = self.lens if in_place else torch.full_like(self.lens, -3)
        self.count_out = self.count if in_place else torch.full_like(self.count, -3)
        self.start = torch.full((n + 1,), -3, dtype=torch.int32, device="cuda")
        self.rows = torch.full((2, max_rows + 8 + offset), -5, dtype=torch.int32, device="cuda")
        self.slots, self.positions = self.rows[0, offset:], self.rows[1, offset:]
        self.status = torch.full((n,), -3, dtype=torch.int32, device="cuda") if status else None
        self.n, self.n_pages, self.max_rows = n, n_pages, max_rows

    def args(self, vv):
        return vv.make_kv_plan(self.new, self.lens, self.lens_out, self.table, self.stack, self.count, self.count_out, self.start,
                               self.slots, self.positions, self.status, self.n, self.table.shape[1], self.n_pages, self.max_rows)

    def compare(self, want):
        torch.cuda.synchronize()
        assert self.lens_out.tolist() == list(want["lens"]) and self.start.tolist() == want["start"]
        assert self.count_out.item() == want["count"]
        if self.status is not None:
            assert self.status.tolist() == want["status"]
        assert np.array_equal(self.table.cpu().numpy(), want["table"])
        assert self.stack.tolist()[: len(want["pushed"])] == want["pushed"]
        m = self.max_rows
        assert self.slots[:m].tolist() == want["slots"] and self.positions[:m].tolist() == want["positions"]
        assert bool((self.slots[m:] == -5).all()) and bool((self.positions[m:] == -5).all())


@gpu
@pytest.mark.parametrize("n,stride,kind,max_rows", [
    (1, 1, "step", 1), (1, 4, "step", 0), (16, 64, "step", 16), (16, 64, "step", 21), (3, 7, "mixed", 700),
    (255, 33, "mixed", 9000), (1025, 12, "mixed", 50000), (64, 9, "scarce", 4000), (700, 20, "scarce", 30000), (64, 9, "pages", 20000), (300, 4, "pages", 40000), (33, 5, "pages", 4096),
    (9, 300, "rows", 4096), (9, 300, "rows", 4097), (2000, 64, "rows", 131072), (8192, 3, "mixed", 200001), (8192, 2, "step", 8192),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_equals_the_definition(vv, n, stride, kind, max_rows, in_place):
    rng = np.random.default_rng(n * 7 + stride + max_rows)
    new, lens, table, stack, count, n_pages = build(rng, n, stride, kind, max_rows)
    want = _paged.plan(new, lens, table, stack, count, max_rows)
    if kind in ("scarce", "pages"):
        assert set(want["status"]) == ({0, 2, 3} if kind == "scarce" else {0, 1, 2})
    d = Device(new, lens, table, stack, count, n_pages, max_rows, in_place, status=not in_place, offset=1 if in_place else 0)
    n0 = vv.launch_count()
    assert vv.vvb_kv_plan_dev(d.args(vv)) == 0 and vv.launch_count() - n0 == 1
    d.compare(want)
    if not in_place:                                  # the same inputs again: the same outputs
        assert vv.vvb_kv_plan_dev(d.args(vv)) == 0
        d.compare(want)


@gpu
def test_plan_values_out_of_range(vv):
    """Lengths below zero count as zero, a stack height beyond the pool is cut, row sums stop at INT_MAX, a length
    beyond the table is refused and its pages are not counted twice."""
    big = 2 ** 31 - 1
    new, lens = np.array([3, big, big, 1, -1]), np.array([-50, 0, 5, 9999, 9999])
    table = np.arange(5 * 4).reshape(5, 4) + 40
    want = _paged.plan(new, lens, table, np.arange(6), 6, 10)
    d = Device(new, lens, table, np.concatenate([np.arange(6), np.full(20, -9)]), 10 ** 9, 6, 10)
    # height cut to the pool's 6 pages: the released ones find no room
    assert vv.vvb_kv_plan_dev(d.args(vv)) == 0
    torch.cuda.synchronize()
    assert d.start.tolist() == [0, 3, big, big, big, big] == want["start"]
    assert d.status.tolist() == [0, 2, 2, 2, 0] == want["status"]
    assert d.lens_out.tolist() == [3, 0, 5, 9999, 0] and d.count_out.item() == 5
    assert d.table[0].tolist() == [5, 41, 42, 43] and d.stack[6:].tolist() == [-9] * 20
    assert d.slots[:10].tolist() == [320, 321, 322] + [-1] * 7


@gpu
def test_plan_replayed_from_a_graph_follows_the_lengths(vv):
    """A decode loop: in place, captured once, replayed until a sequence's table is full; between replays a sequence
    ends and another one enters through the device array of new tokens."""
    rng = np.random.default_rng(5)
    n, stride, max_rows = 6, 3, 40
    lens, table = np.array([0, 60, 100, 63, 128, 190]), np.full((n, stride), -7)
    pages = -(-lens // 64)
    order = rng.permutation(30)
    table[np.arange(stride)[None, :] < pages[:, None]] = order[: pages.sum()]
    stack = np.concatenate([order[pages.sum():], np.full(pages.sum(), -9)])
    count = 30 - int(pages.sum())
    d = Device(np.ones(n), lens, table, stack, count, 30, max_rows, in_place=True)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    a = d.args(vv)
    with torch.cuda.graph(g, stream=s):
        assert vv.vvb_kv_plan_dev(a, s) == 0
    free = list(stack[:count])
    for step, new in enumerate([[1] * 6, [1, 1, -1, 1, 1, 1], [1, 1, 30, 1, 0, 1], [0, -1, 2, 1, 1, 1], [1, 5, 1, -1, -1, 1]]):
        d.new.copy_(ints(new))
        want = _paged.plan(new, lens, table, np.array(free), len(free), max_rows)
        g.replay()
        torch.cuda.synchronize()
        d.compare(want)
        lens, table, free = np.array(want["lens"]), want["table"], want["pushed"][: want["count"]]
        if step == 4:
            assert want["status"][5] == 2             # 190 + 2 positions fill its three pages


@gpu
def test_plan_cluster_replayed_from_a_graph(vv):
    """The forms for long row lists (8 and 16 CTAs), captured and replayed with other lengths."""
    rng = np.random.default_rng(8)
    for n, stride, max_rows in ((300, 40, 20000), (900, 40, 80000)):
        new, lens, table, stack, count, n_pages = build(rng, n, stride, "rows", max_rows)
        d = Device(new, lens, table, stack, count, n_pages, max_rows)
        keep = [t.clone() for t in (d.new, d.lens, d.table, d.stack, d.count)]
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        a = d.args(vv)
        with torch.cuda.graph(g, stream=s):
            assert vv.vvb_kv_plan_dev(a, s) == 0
        for change in (np.zeros(n, np.int64), rng.integers(-2, 3, n)):
            for t, k in zip((d.new, d.lens, d.table, d.stack, d.count), keep):
                t.copy_(k)
            tokens = np.where(change < -1, -1, np.maximum(new - np.maximum(change, 0), 0))
            d.new.copy_(ints(tokens))
            want = _paged.plan(tokens, lens, table, stack, count, max_rows)
            g.replay()
            torch.cuda.synchronize()
            d.compare(want)
