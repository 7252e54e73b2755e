"""vvb_attn_decode_dev: attention of one new token per sequence over the cache,
against softmax attention in float64 over the decoded cache (tests/_paged.py,
where the tolerances are derived)."""
import numpy as np
import pytest

import _paged
from _paged import E4M3, E5M2, FP16, PAGE, TQ1_5, TQ2, TQ3, TQ4

P = 0x1000


@pytest.fixture(scope="module")
def lib():
    import vvb200
    return vvb200


def fake(vv, **kw):
    a = dict(q=P, out=P, k_store=P, v_store=P, lens=P, n_seqs=3, n_q_heads=28, n_kv_heads=4, head_dim=128, n_slots=640)
    k = dict(block_table=P, table_stride=8, scratch=P, scratch_bytes=1 << 40)
    for name, v in kw.items():
        (a if name in a else k)[name] = v
    return vv.make_attn_decode(*a.values(), **k)


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), "VV_ERR_NULL_PTR"), (dict(out=None), "VV_ERR_NULL_PTR"), (dict(k_store=None), "VV_ERR_NULL_PTR"),
    (dict(v_store=None), "VV_ERR_NULL_PTR"), (dict(lens=None), "VV_ERR_NULL_PTR"), (dict(scratch=None), "VV_ERR_NULL_PTR"),
    (dict(n_seqs=-1), "VV_ERR_INVALID_ARG"), (dict(n_q_heads=0), "VV_ERR_INVALID_ARG"), (dict(n_kv_heads=0), "VV_ERR_INVALID_ARG"),
    (dict(n_q_heads=27), "VV_ERR_INVALID_ARG"), (dict(n_slots=-1), "VV_ERR_INVALID_ARG"), (dict(table_stride=0), "VV_ERR_INVALID_ARG"),
    (dict(scale=float("nan")), "VV_ERR_INVALID_ARG"), (dict(scale=float("inf")), "VV_ERR_INVALID_ARG"),
    (dict(head_dim=96), "VV_ERR_UNSUPPORTED"), (dict(head_dim=0), "VV_ERR_INVALID_ARG"), (dict(kv_format=7), "VV_ERR_UNSUPPORTED"),
    (dict(kv_format=-1), "VV_ERR_UNSUPPORTED"), (dict(kv_format=TQ4), "VV_ERR_NULL_PTR"),
    (dict(kv_format=TQ4, head_dim=64, k_meta=P, v_meta=P), "VV_ERR_UNSUPPORTED"), (dict(kv_format=TQ4, k_meta=P + 2, v_meta=P), "VV_ERR_UNSUPPORTED"),
    (dict(q=P + 8), "VV_ERR_UNSUPPORTED"), (dict(k_store=P + 4), "VV_ERR_UNSUPPORTED"), (dict(scratch=P + 8), "VV_ERR_UNSUPPORTED"),
    (dict(lens=P + 2), "VV_ERR_INVALID_ARG"), (dict(block_table=P + 2), "VV_ERR_INVALID_ARG"), (dict(lse=P + 1), "VV_ERR_INVALID_ARG"),
    (dict(n_q_heads=8192), "VV_ERR_UNSUPPORTED"), (dict(table_stride=1 << 25), "VV_ERR_OVERFLOW"), (dict(n_seqs=8193), "VV_ERR_UNSUPPORTED"), (dict(scratch_bytes=0), "VV_ERR_INVALID_ARG"),
    (dict(n_seqs=0), "VV_OK"),
])
def test_attn_refusals(lib, kw, want):
    assert lib.vvb_attn_decode_dev(fake(lib, **kw), stream=0) == getattr(lib, want)
    assert lib._lib.vvb_attn_decode_dev(None, None) == lib.VV_ERR_NULL_PTR


def test_attn_scratch_size(lib):
    n = lib.vvb_attn_decode_scratch_bytes(64, 28, 4, 128)
    assert 0 < n <= 64 << 20
    assert lib.vvb_attn_decode_scratch_bytes(0, 28, 4, 128) == 0 and lib.vvb_attn_decode_scratch_bytes(3, 27, 4, 128) == 0


def test_decoding_by_hand():
    """The test's own reading of the stored codes, against the oracle's restatement of the reference."""
    import oracle
    R = oracle.restated()
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 128)).astype(np.float16)
    for fmt in (TQ4, TQ3, TQ2, TQ1_5):
        store, meta = R.kv_store_tq(x, None, fmt)
        got = _paged.decode(store.reshape(3, 2, -1), meta, fmt, 128)
        for r in range(3):
            for h in range(2):
                assert np.allclose(got[r, h], R.kv_load_tq(store.reshape(3, 2, -1)[r, h], meta[r, h], fmt), rtol=1e-6)


# ------------------------------------------------------------------ GPU
torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def vv(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return lib


class Case:
    """A cache in some format, its sequences, and the call's other arrays (scratch filled with NaN bytes)."""

    def __init__(self, vv, lens, nq, nkv, hd, fmt, paged=True, seed=0, qscale=1.5, dist="normal", poison=True, slack=1):
        rng = np.random.default_rng(seed)
        self.vv, self.lens, self.nq, self.nkv, self.hd, self.fmt, self.paged = vv, np.array(lens), nq, nkv, hd, fmt, paged
        n = len(lens)
        if paged:
            pages = -(-self.lens // PAGE)
            self.stride = int(max(pages.max(), 1)) + slack
            n_pages = int(pages.sum()) + 3
            order = rng.permutation(n_pages)
            self.table = np.full((n, self.stride), -1, np.int32)
            self.table[np.arange(self.stride)[None, :] < pages[:, None]] = order[: pages.sum()]
            self.rows = n_pages * PAGE
        else:
            self.stride, self.table = int(max(self.lens.max(), 1)) + slack, None
            self.rows = n * self.stride
        tq = fmt >= TQ4
        vb = _paged.vec_bytes(fmt, hd)
        kv, metas = [], []
        for _ in range(2):
            if tq:
                kv.append(rng.integers(0, 256, (self.rows, nkv, vb), dtype=np.uint8))
                metas.append((np.abs(1 + 0.3 * rng.standard_normal((self.rows, nkv))) + 0.02).astype(np.float16))
            else:
                x = rng.standard_normal((self.rows, nkv, hd)).astype(np.float32)
                if dist == "wide":
                    x *= np.exp(2 * rng.standard_normal((self.rows, nkv, 1))).astype(np.float32)
                t = torch.from_numpy(x)
                t = t.half() if fmt == FP16 else t.clamp(-400, 400).to(torch.float8_e4m3fn if fmt == E4M3 else torch.float8_e5m2)
                kv.append(t.contiguous().view(torch.uint8).numpy().reshape(self.rows, nkv, vb).copy())
        self.kv, self.metas = kv, metas
        live = np.zeros(self.rows, bool)
        for b in range(n):
            live[self.slots(b)] = True
        if poison:                                     # what no key lies in holds NaN and infinities
            for x in kv:
                x[~live] = 0x7F if fmt == E4M3 else 0x7E if fmt == FP16 else 0xFF
            for i, m in enumerate(metas):
                m[~live] = [np.nan, np.inf][i]
        self.q = (qscale * rng.standard_normal((n, nq, hd))).astype(np.float16)

    def slots(self, b):
        j = np.arange(self.lens[b])
        return self.table[b, j // PAGE].astype(np.int64) * PAGE + j % PAGE if self.paged else b * self.stride + j

    def upload(self, len_add=0, lse=True, scale=None):
        d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.dk, self.dv = d(self.kv[0]), d(self.kv[1])
        self.dm = [d(m) for m in self.metas] or [None, None]
        self.dq, self.dlens = d(self.q), d((self.lens - len_add).astype(np.int32))
        self.dtable = d(self.table) if self.paged else None
        n = len(self.lens)
        guard = torch.full((n + 2, self.nq, self.hd), 5.0, dtype=torch.float16, device="cuda")
        self.guard, self.dout = guard, guard[1:-1]
        self.dlse = torch.full((n, self.nq), 5.0, device="cuda") if lse else None
        size = self.vv.vvb_attn_decode_scratch_bytes(n, self.nq, self.nkv, self.hd)
        self.scratch = torch.full((size + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        self.scale = self.hd ** -0.5 if scale is None else scale
        self.args = self.vv.make_attn_decode(self.dq, self.dout, self.dk, self.dv, self.dlens, n, self.nq, self.nkv, self.hd, self.rows,
                                             block_table=self.dtable, table_stride=self.stride, len_add=len_add, kv_format=self.fmt,
                                             k_meta=self.dm[0], v_meta=self.dm[1], lse=self.dlse, scratch=self.scratch, scratch_bytes=size,
                                             scale=scale)
        return self

    def run(self, stream=None):
        assert self.vv.vvb_attn_decode_dev(self.args, stream) == 0
        torch.cuda.synchronize()
        assert bool((self.scratch[-16:] == 0xFF).all()) and bool((self.guard[0] == 5).all()) and bool((self.guard[-1] == 5).all())
        return self.dout.cpu().numpy(), None if self.dlse is None else self.dlse.cpu().numpy()

    def check(self, out, lse):
        for b in range(len(self.lens)):
            s = self.slots(b)
            k, v = (_paged.decode(x[s], self.metas[i][s] if self.metas else None, self.fmt, self.hd) for i, x in enumerate(self.kv))
            want, wlse, absout, worst = _paged.attention(self.q[b].astype(np.float64), k, v, self.scale)
            tol, tol_lse = _paged.tolerances(want, absout, worst, wlse, len(s), self.hd, self.fmt)
            err = np.abs(out[b].astype(np.float64) - want)
            assert (err <= tol).all(), (b, len(s), float((err / tol).max()))
            if len(s) == 0:
                assert not out[b].any() and (lse is None or np.isneginf(lse[b]).all())
            elif lse is not None:
                el = np.abs(lse[b].astype(np.float64) - wlse)
                assert (el <= tol_lse).all(), (b, len(s), float((el / tol_lse).max()))


RAGGED = [1, 0, 63, 64, 65, 17, 127, 128, 129, 700, 2, 0, 1000, 15, 16, 31, 33]


@gpu
@pytest.mark.parametrize("fmt", range(7))
@pytest.mark.parametrize("paged", [True, False])
def test_attn_ragged_batch(vv, fmt, paged):
    c = Case(vv, RAGGED, 28, 4, 128, fmt, paged, seed=fmt).upload()
    n0 = vv.launch_count()
    out, lse = c.run()
    assert 1 <= vv.launch_count() - n0 <= 2
    c.check(out, lse)


@gpu
@pytest.mark.parametrize("nq,nkv,hd", [(1, 1, 128), (12, 2, 128), (12, 12, 64), (9, 3, 64), (8, 1, 128), (16, 2, 256), (40, 8, 128), (16, 1, 128),
                                       (24, 2, 64), (17, 1, 256), (20, 1, 128), (33, 1, 64), (15, 5, 256)])
@pytest.mark.parametrize("fmt", [FP16, E4M3, E5M2])
def test_attn_head_layouts(vv, nq, nkv, hd, fmt):
    c = Case(vv, [200, 1, 77, 0, 513], nq, nkv, hd, fmt, seed=nq).upload()
    c.check(*c.run())


@gpu
@pytest.mark.parametrize("nq,nkv", [(1, 1), (20, 2), (16, 1), (3, 3), (33, 1)])
@pytest.mark.parametrize("fmt", [TQ4, TQ3, TQ2, TQ1_5])
def test_attn_rotated_formats_head_layouts(vv, nq, nkv, fmt):
    c = Case(vv, [200, 1, 77, 0, 513], nq, nkv, 128, fmt, seed=nq, paged=nkv != 3).upload()
    c.check(*c.run())


@gpu
@pytest.mark.parametrize("lens,fmt,paged", [([1], FP16, True), ([14449], FP16, False), ([40000, 3], FP16, True), ([60000], E4M3, True),
                                            ([9000] * 5, TQ4, True), ([3000, 1, 2999] * 9, E5M2, True), ([70] * 300, FP16, True),
                                            ([1] * 1000, FP16, True), ([5] * 700, TQ2, True), ([20000], TQ1_5, False), ([64] * 148, TQ3, True)])
def test_attn_long_and_many(vv, lens, fmt, paged):
    c = Case(vv, lens, 28 if len(lens) < 200 else 8, 4, 128, fmt, paged, seed=len(lens)).upload()
    c.check(*c.run())


# by the blocks a table has room for and the number of sequences the work is cut differently: whole sequences to
# warps or to CTAs, or cut between CTAs with their pieces found by item or by CTA: sequences, blocks, blocks of the
# rotated formats
BLOCK = {FP16: 64, E4M3: 128, E5M2: 128, TQ4: 384, TQ3: 256, TQ2: 256, TQ1_5: 256}
WAYS = {"warps": (250, 1, 1), "warps_edge": (222, 3, 2), "warps_many": (445, 5, 2), "ctas_few": (2, 8, 4), "ctas": (30, 10, 5), "ctas_many": (150, 4, 4),
        "ctas_most": (97, 16, 7), "cut_few": (5, 9, 5), "cut_nine": (9, 39, 7), "cut": (20, 12, 6), "cut_many": (112, 17, 9)}


@gpu
@pytest.mark.parametrize("fmt", range(7))
@pytest.mark.parametrize("way", WAYS)
def test_attn_every_way_of_cutting_the_work(vv, way, fmt):
    n, top = WAYS[way][0], WAYS[way][2 if fmt >= TQ4 else 1] * BLOCK[fmt]
    top -= n % 7
    rng = np.random.default_rng(n + fmt)
    lens = np.where(rng.random(n) < 0.1, 0, np.exp(rng.uniform(0, np.log(top + 1), n))).astype(np.int64)
    lens[rng.integers(n)] = top
    c = Case(vv, lens, 16, 4, 128, fmt, seed=n, slack=0).upload()
    n0 = vv.launch_count()
    out, lse = c.run()
    assert vv.launch_count() - n0 == (2 if way.startswith("cut") else 1)
    c.check(out, lse)
    again = c.run()
    assert np.array_equal(again[0], out) and np.array_equal(again[1], lse)


@gpu
def test_attn_nothing_but_empty_sequences(vv):
    for n, room in ((1, 1), (5, 40), (1000, 1)):
        c = Case(vv, [0] * n, 28, 4, 128, FP16, seed=n, slack=room).upload()
        c.check(*c.run())


@gpu
def test_attn_as_many_sequences_as_a_call_takes(vv):
    lens = np.arange(8192) % 4
    c = Case(vv, lens, 2, 1, 64, FP16, seed=30).upload()
    c.check(*c.run())
    c = Case(vv, np.where(np.arange(8192) == 5000, 700, lens), 1, 1, 64, E4M3, seed=31).upload()
    c.check(*c.run())


@gpu
@pytest.mark.parametrize("lens", [[0], [1, 0, 63, 64, 65, 128, 5, 700], [20000, 3, 0, 9000], [40] * 30 + [0, 2000] + [16] * 70])
def test_attn_tables_for_more_than_32_bits_of_cut_line(vv, lens):
    """Tables wide enough that the line of blocks, were they full, passes what is cut in 32 bits: the same parts."""
    width = -(-(1 << 25) // (4 * len(lens)) // 64)      # over 2^21 groups of 16 keys
    c = Case(vv, lens, 28, 4, 128, FP16, seed=33)
    wide = np.full((len(lens), max(width, c.table.shape[1])), -1, np.int32)
    wide[:, :c.table.shape[1]] = c.table
    outs = []
    for table in (c.table, wide):
        c.table, c.stride = table, table.shape[1]
        c.upload()
        o, l = c.run()
        c.check(o, l)
        outs.append((o, l))
    if max(lens) > 700:                                 # both are cut, into the same parts
        assert np.array_equal(outs[0][0].view(np.uint16), outs[1][0].view(np.uint16)) and np.array_equal(outs[0][1], outs[1][1])


@gpu
@pytest.mark.parametrize("lens", [[900, 0, 5, 70], [0, 0, 64, 9000], [1100, 5, 0, 3000] * 5])
def test_attn_scratch_of_zeros_or_of_another_call(vv, lens):
    c = Case(vv, lens, 28, 4, 128, FP16, seed=34).upload()
    want = c.run()
    c.check(*want)
    for other in (None, [3000] * 20, [7000, 3], [0, 40]):
        c.scratch[:-16].zero_()
        if other is not None:
            x = Case(vv, other, 28, 4, 128, FP16, seed=35).upload()
            x.args.scratch = c.args.scratch
            x.run()
        got = c.run()
        assert np.array_equal(got[0].view(np.uint16), want[0].view(np.uint16)) and np.array_equal(got[1], want[1])


@gpu
def test_attn_cut_work_captured_in_a_graph(vv):
    """Many items, cut between CTAs: an ordinary launch followed by a dependent one, replayed behind other kernels."""
    c = Case(vv, [1100, 5, 0, 3000] * 5, 28, 4, 128, E4M3, seed=32, poison=False).upload()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    src = c.dq.clone()
    with torch.cuda.graph(g, stream=s):
        c.dq.copy_(src)
        for _ in range(3):
            assert vv.vvb_attn_decode_dev(c.args, s) == 0
    for lens in (c.lens, c.lens // 2, c.lens):
        c.dlens.copy_(torch.from_numpy(lens.astype(np.int32)))
        c.dq.zero_(), c.dout.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        c.lens = lens
        c.check(c.dout.cpu().numpy(), c.dlse.cpu().numpy())


@gpu
def test_attn_contiguous_cache_shorter_than_its_sequences_claim(vv):
    """Lengths beyond the rows that the cache has: cut there, nothing beyond is read."""
    c = Case(vv, [300, 200], 4, 2, 128, FP16, paged=False, seed=21, slack=0).upload()
    c.dlens.copy_(torch.tensor([2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32))
    c.args.n_slots = 500                                # the second sequence's stretch ends after 200
    out, lse = c.run()
    c.check(out, lse)


@gpu
def test_attn_values_of_wide_range(vv):
    """Keys and values over several orders of magnitude, sharp and flat softmax, other scales, without lse."""
    for scale, qscale in ((None, 1.0), (0.5, 1.0), (1e-3, 1.0), (0.0, 1.0), (-0.1, 2.0), (1.0, 4.0)):
        c = Case(vv, [500, 3, 64, 1200], 28, 4, 128, FP16, seed=3, dist="wide", qscale=qscale).upload(scale=scale, lse=scale != 0.5)
        c.check(*c.run())


@gpu
@pytest.mark.parametrize("sigma", [6e-6, 3e-3, 300.0])
@pytest.mark.parametrize("fmt", [TQ4, TQ1_5])
def test_attn_rotated_formats_with_small_and_large_rms(vv, sigma, fmt):
    """The RMS of V spans FP16's range, from one key to the next as well: weights times RMS must keep their digits."""
    c = Case(vv, [300, 2, 90], 28, 4, 128, fmt, seed=4)
    rng = np.random.default_rng(1)
    m = (sigma * np.exp(1.5 * rng.standard_normal(c.metas[1].shape))).astype(np.float16)
    c.metas[1][:] = np.where(np.isinf(c.metas[1]), c.metas[1], np.minimum(m, 6e4))
    c.upload()
    c.check(*c.run())


@gpu
def test_attn_one_key_far_above_the_rest_wherever_it_lies(vv):
    for at in (0, 15, 16, 63, 64, 500, 998):
        c = Case(vv, [999], 28, 4, 128, FP16, seed=at)
        k = c.kv[0].view(np.float16).reshape(c.rows, 4, 128)
        k[c.slots(0)[at]] = np.sign(c.q[0].reshape(4, 7, 128)[:, 3]) * 6.0
        c.upload()
        c.check(*c.run())


@gpu
def test_attn_tail_of_tiny_weights(vv):
    """A hundred thousand keys at e^-17 of the largest: together they are 0.4 % of the result, each is below FP16's
    normal range."""
    n = 100_000
    c = Case(vv, [n], 1, 1, 128, FP16, seed=8)
    s = c.slots(0)
    k, v = (x.view(np.float16).reshape(c.rows, 128) for x in c.kv)
    k[s] = 0
    v[s] = 1000.0
    k[s[77], 0], v[s[77]] = 17.0 * 11.3125, 1.0
    c.q[:] = 0
    c.q[0, 0, 0] = 1.0
    c.upload()
    c.check(*c.run())


@gpu
@pytest.mark.parametrize("depth", [26.0, 50.0, 200.0])
def test_attn_weights_too_small_to_matter_do_not_add_up(vv, depth):
    """A hundred thousand keys far below the largest, with values near FP16's largest."""
    n = 100_000
    c = Case(vv, [n], 1, 1, 128, FP16, seed=9)
    s = c.slots(0)
    k, v = (x.view(np.float16).reshape(c.rows, 128) for x in c.kv)
    k[s] = 0
    v[s] = 60000.0
    k[s[n // 3], 0], v[s[n // 3]] = depth * 11.3125, 1.0
    c.q[:] = 0
    c.q[0, 0, 0] = 1.0
    c.upload()
    c.check(*c.run())


@gpu
def test_attn_infinite_values(vv):
    """An infinity in V stays one where its key has weight, with any sign of the values around it."""
    c = Case(vv, [90, 300], 8, 2, 128, FP16, seed=22)
    v = c.kv[1].view(np.float16).reshape(c.rows, 2, 128)
    s = c.slots(1)
    v[s[::7], 0, 5] = np.inf
    v[s[::11], 1, 100] = -np.inf
    c.upload()
    out, lse = c.run()
    assert np.isposinf(out[1, :4, 5]).all() and np.isneginf(out[1, 4:, 100]).all() and np.isfinite(out).sum() == out.size - 8
    v[s[::7], 0, 5], v[s[::11], 1, 100] = 0.0, 0.0
    out[1, :4, 5], out[1, 4:, 100] = 0.0, 0.0
    for h, d in [(h, 5) for h in range(4)] + [(h, 100) for h in range(4, 8)]:
        kk, vw = (_paged.decode(x[s], None, FP16, 128) for x in c.kv)
        out[1, h, d] = _paged.attention(c.q[1].astype(np.float64), kk, vw, c.scale)[0][h, d]
    c.check(out, lse)


@gpu
def test_attn_infinite_scores(vv):
    """A key whose score is -inf has no weight; where every key's is, the row is empty: zeros and -inf. +inf and NaN
    in a live key give NaN, and only in the heads and sequences that see it."""
    c = Case(vv, [100, 100, 100, 50], 8, 2, 128, FP16, seed=2)
    k = c.kv[0].view(np.float16).reshape(c.rows, 2, 128)
    c.q[:, :, 0] = np.abs(c.q[:, :, 0]) + np.float16(0.5)
    s = [c.slots(b) for b in range(4)]
    k[s[0][40], 0, 0] = -np.inf
    k[s[1], 1, 0] = -np.inf
    k[s[2][99], 1, 0] = np.inf
    c.upload()
    out, lse = c.run()
    assert np.isnan(out[2, 4:]).all() and np.isnan(lse[2, 4:]).all() and np.isfinite(out[2, :4]).all()
    assert not out[1, 4:].any() and np.isneginf(lse[1, 4:]).all()
    k[s[0][40], 0, 0] = -60000.0                        # as good as -inf for the float64 check
    k[s[1], 1, 0], k[s[2][99], 1, 0] = 0.0, 0.0
    # (those two rows apart)
    keep_out, keep_lse = out.copy(), lse.copy()
    c.upload()
    again, alse = c.run()
    keep_out[1, 4:], keep_out[2, 4:], keep_lse[1, 4:], keep_lse[2, 4:] = again[1, 4:], again[2, 4:], alse[1, 4:], alse[2, 4:]
    c.check(keep_out, keep_lse)


@gpu
def test_attn_pages_outside_the_cache_are_left_out(vv):
    """Entries of the table that name no page of the cache: their keys are masked, wherever they lie."""
    c = Case(vv, [300, 64, 700, 129], 28, 4, 128, FP16, seed=6)
    n_pages = c.rows // PAGE
    whole = c.table.copy()
    c.table[0, 1], c.table[1, 0], c.table[2, 10], c.table[3, 0], c.table[3, 2] = -1, n_pages, 2 ** 31 - 1, -(2 ** 31), n_pages + 5
    c.upload()
    out, lse = c.run()
    for b in range(4):
        j = np.arange(c.lens[b])
        ok = (c.table[b, j // PAGE] >= 0) & (c.table[b, j // PAGE] < n_pages)
        s = (whole[b, j // PAGE].astype(np.int64) * PAGE + j % PAGE)[ok]
        k, v = (_paged.decode(x[s], None, FP16, 128) for x in c.kv)
        want, wlse, absout, worst = _paged.attention(c.q[b].astype(np.float64), k, v, c.scale)
        tol, tol_lse = _paged.tolerances(want, absout, worst, wlse, len(s), 128, FP16)
        assert (np.abs(out[b] - want) <= tol).all()
        assert np.isneginf(lse[b]).all() if len(s) == 0 else (np.abs(lse[b] - wlse) <= tol_lse).all()


@gpu
def test_attn_lengths_beyond_the_table_are_cut(vv):
    c = Case(vv, [128, 100, 64], 4, 2, 128, FP16, seed=9, slack=0).upload()
    out, lse = c.run()
    c.check(out, lse)
    c.dlens.copy_(torch.tensor([10 ** 9, 100, -5], dtype=torch.int32))
    out2, lse2 = c.run()
    assert np.array_equal(out2[:2], out[:2]) and not out2[2].any() and np.isneginf(lse2[2]).all()
    c.dlens.copy_(torch.tensor([2 ** 31 - 1, 100, -(2 ** 31)], dtype=torch.int32))
    for add in (2 ** 31 - 1, -(2 ** 31)):
        c.args.len_add = add
        got, _ = c.run()
        if add > 0:                                    # the third: 2^31 - 1 - 2^31 = -1 keys; the second is cut to the table's 128
            assert np.array_equal(got[0], out[0]) and not got[2].any()
        else:
            assert not got.any()


@gpu
def test_attn_same_bits_again_in_place_and_on_other_streams(vv):
    c = Case(vv, [3000, 77, 0, 512, 9000], 28, 4, 128, FP16, seed=11).upload()
    d = Case(vv, [100] * 40, 28, 4, 128, E4M3, seed=12).upload()
    out, lse = c.run()
    dout, dlse = d.run()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):                                # two calls at once, each with its own scratch
        assert vv.vvb_attn_decode_dev(c.args, s1) == 0 and vv.vvb_attn_decode_dev(d.args, s2) == 0
    torch.cuda.synchronize()
    assert np.array_equal(c.dout.cpu().numpy(), out) and np.array_equal(c.dlse.cpu().numpy(), lse)
    assert np.array_equal(d.dout.cpu().numpy(), dout) and np.array_equal(d.dlse.cpu().numpy(), dlse)
    c.args.out = c.dq.data_ptr()
    assert vv.vvb_attn_decode_dev(c.args) == 0
    assert np.array_equal(c.dq.cpu().numpy(), out)


@gpu
def test_attn_graph_follows_lengths_and_two_graphs_share_a_scratch(vv):
    """Captured once, replayed while the lengths grow and shrink on the device; a second graph with the same scratch
    replayed in between."""
    top = [700, 2000, 64, 10]
    c = Case(vv, top, 28, 4, 128, FP16, seed=13, poison=False).upload()
    d = Case(vv, [50, 900], 12, 2, 128, TQ4, seed=14).upload()
    d.scratch = c.scratch
    d.args.scratch = c.scratch.data_ptr()
    s = torch.cuda.Stream()
    graphs = []
    for x in (c, d):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            assert vv.vvb_attn_decode_dev(x.args, s) == 0
        graphs.append(g)
    for lens in ([1, 1, 1, 1], top, [699, 1999, 63, 9], [0, 0, 0, 0], [64, 65, 0, 10], [0, 2000, 0, 0]):
        c.dlens.copy_(torch.tensor(lens, dtype=torch.int32))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        c.lens = np.array(lens)
        c.check(c.dout.cpu().numpy(), c.dlse.cpu().numpy())
        d.check(d.dout.cpu().numpy(), d.dlse.cpu().numpy())


@gpu
def test_attn_device_position_of_a_contiguous_cache(vv):
    """len_add = 1 with the position of the newest token, as the decode step holds it."""
    c = Case(vv, [1, 400, 65], 12, 2, 128, FP16, paged=False, seed=15).upload(len_add=1)
    c.check(*c.run())


@gpu
def test_attn_odd_cache_of_a_rotated_format(vv):
    """An odd number of RMS values: the last one has no neighbour in its 32-bit word."""
    c = Case(vv, [333], 7, 1, 128, TQ4, paged=False, seed=16, slack=0).upload()
    assert c.rows * c.nkv % 2 == 1
    c.check(*c.run())


@gpu
@pytest.mark.parametrize("fmt", [FP16, E4M3])
def test_attn_rows_whose_offset_passes_32_bits(vv, fmt):
    nq, nkv, hd = 28, 4, 128
    vb = _paged.vec_bytes(fmt, hd)
    n_pages = (1 << 32) // (PAGE * nkv * vb) + 9
    c = Case(vv, [650, 130], nq, nkv, hd, fmt, seed=17)
    small = c.rows // PAGE
    c.upload()
    k, v = (torch.empty(n_pages * PAGE, nkv, vb, dtype=torch.uint8, device="cuda") for _ in range(2))
    where = np.arange(small) + (n_pages - small)        # the same pages at the far end
    k[-c.rows:], v[-c.rows:] = c.dk, c.dv
    c.dtable.copy_(torch.from_numpy(np.where(c.table >= 0, where[c.table], -1).astype(np.int32)))
    c.args.k_store, c.args.v_store, c.args.n_slots = k.data_ptr(), v.data_ptr(), n_pages * PAGE
    c.check(*c.run())
