"""vvb_attn_decode_dev: an infinity in V has its sign in the result however small its key's
weight is, since a finite score has a weight above zero; everything else stays as float64
has it. One key has a score `depth` above the others', the infinity lies under one of
those. Formats whose V can be infinite: FP16, E5M2, and the rotated ones through the RMS."""
import numpy as np
import pytest

import _paged
from _paged import E5M2, FP16, TQ1_5, TQ2, TQ3, TQ4
from test_attn_decode import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEPTHS = [0.0, 10.0, 14.0, 16.0, 20.0, 24.0, 32.0, 48.0, 96.0, 192.0, 1024.0]      # E5M2 has them all


@pytest.fixture(scope="module")
def vv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import vvb200
    torch.cuda.set_device(0)
    return vvb200


def _numbers(c, fmt, which):
    """Writes x (float) into the K (0) or V (1) rows s."""
    flat = c.kv[which].reshape(c.rows, c.nkv, -1)
    dt = torch.float16 if fmt == FP16 else torch.float8_e5m2

    def put(s, x):
        flat[s] = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(dt).view(torch.uint8).numpy().reshape(*np.shape(x)[:-1], -1)
    return put


# (keys, where the largest score lies, where the infinities lie): one warp's step, one CTA, cut between CTAs
PLACES = [(16, 3, (9,)), (16, 9, (3,)), (60, 40, (5, 59)), (700, 1, (699,)), (700, 690, (2,)), (9000, 4500, (0, 8999)), (9000, 8000, (100,))]


@pytest.mark.parametrize("n,top,at", PLACES)
@pytest.mark.parametrize("fmt", [FP16, E5M2])
@pytest.mark.parametrize("nq,hd", [(4, 128), (20, 64), (3, 256)])
def test_an_infinity_under_any_weight(vv, n, top, at, fmt, nq, hd):
    for depth in DEPTHS:
        c = Case(vv, [n, 33], nq, 1, hd, fmt, seed=n)
        s = c.slots(0)
        k = np.zeros((n, 1, hd))
        k[top, 0, 0] = depth
        _numbers(c, fmt, 0)(s, k)
        v = _paged.decode(c.kv[1][s], None, fmt, hd)
        finite = v.copy()
        for i, j in enumerate(at):
            v[j, 0, 5 + i], v[j, 0, hd - 1 - i] = np.inf, -np.inf
        v[at[0], 0, 17] = np.nan
        if len(at) > 1:                                # infinities of both signs in one sum
            v[at[0], 0, 30], v[at[1], 0, 30] = np.inf, -np.inf
        _numbers(c, fmt, 1)(s, v)
        c.q[0] = 0
        c.q[0, :, 0] = np.where(np.arange(nq) % 2 == 0, 1.0, -1.0)       # odd heads: all the weight on the others
        out, lse = c.upload(scale=1.0).run()
        for i in range(len(at)):
            assert np.isposinf(out[0, :, 5 + i]).all() and np.isneginf(out[0, :, hd - 1 - i]).all(), depth
        odd = [5 + i for i in range(len(at))] + [hd - 1 - i for i in range(len(at))] + [17] + ([30] if len(at) > 1 else [])
        assert np.isnan(out[0, :, 17]).all() and (len(at) == 1 or np.isnan(out[0, :, 30]).all())
        # the rest, with the infinities out of the way
        _numbers(c, fmt, 1)(s, finite)
        want = _paged.attention(c.q[0].astype(np.float64), _paged.decode(c.kv[0][s], None, fmt, hd), finite, 1.0)[0]
        out[0][:, odd] = want[:, odd].astype(np.float16)
        c.check(out, lse)


@pytest.mark.parametrize("n,top,at", PLACES)
@pytest.mark.parametrize("fmt", [TQ4, TQ3, TQ2, TQ1_5])
def test_an_infinite_rms_under_any_weight(vv, n, top, at, fmt):
    at = at[:1]
    for depth in DEPTHS:
        c = Case(vv, [n, 33], 3, 1, 128, fmt, seed=n)
        s = c.slots(0)
        c.kv[0][s] = c.kv[0][s[0]]                     # the same codes: scores go by the RMS
        levels = _paged.decode(c.kv[0][s[:1]], np.ones((1, 1), np.float16), fmt, 128)[0, 0]
        c.q[0] = np.sign(levels)
        c.q[0, 1] *= -1
        unit = float(np.abs(levels).sum())
        c.metas[0][s] = 0
        c.metas[0][s[top]] = depth / unit
        c.metas[1][s[list(at)]] = np.inf
        want = np.sign(_paged.decode(c.kv[1][s], np.ones((n, 1), np.float16), fmt, 128)[at[0], 0]) * np.inf
        out, lse = c.upload(scale=1.0).run()
        assert np.array_equal(out[0].astype(np.float64), np.broadcast_to(want, (3, 128))), depth
        c.metas[1][s[list(at)]] = 0
        out[0] = c.upload(scale=1.0).run()[0][0]
        c.check(out, lse)


@pytest.mark.parametrize("fmt", [FP16, E5M2])
def test_a_new_maximum_far_above_an_infinite_sum(vv, fmt):
    """Scores that climb by hundreds from key to key: what was summed is scaled down again and again."""
    c = Case(vv, [600], 4, 1, 128, fmt, seed=1)
    s = c.slots(0)
    k = np.zeros((600, 1, 128))
    k[:, 0, 0] = 2.0 ** np.clip(np.arange(600) // 40, 0, 14)
    _numbers(c, fmt, 0)(s, k)
    v = _paged.decode(c.kv[1][s], None, fmt, 128)
    v[0, 0, 7] = np.inf
    _numbers(c, fmt, 1)(s, v)
    c.q[:] = 0
    c.q[0, :, 0] = 1.0
    out, _ = c.upload(scale=1.0).run()
    assert np.isposinf(out[0, :, 7]).all() and np.isfinite(np.delete(out[0], 7, axis=1)).all()


@pytest.mark.parametrize("lens", [[40, 0, 50, 0, 0, 30] * 60, [70, 0, 900, 0, 1200] * 8])
def test_empty_sequences_among_infinite_ones_in_place(vv, lens):
    """out is q, and the queries of sequences without keys hold the bits that a conversion makes of a NaN: zeros there."""
    c = Case(vv, lens, 4, 1, 128, FP16, seed=5)
    flat = c.kv[1].view(np.float16).reshape(c.rows, 1, 128)
    k = c.kv[0].view(np.float16).reshape(c.rows, 1, 128)
    c.q[:, :, 1:], c.q[:, :, 0] = 0, 1
    for b, n in enumerate(lens):
        if n == 0:
            c.q[b] = np.uint16(0x7fff).view(np.float16)
            continue
        s = c.slots(b)
        k[s], k[s[n // 2], 0, 0] = 0, 30.0             # the infinity weighs e^-30 of the largest
        flat[s[0], 0, 3] = -np.inf
    c.upload(scale=1.0)
    c.args.out = c.dq.data_ptr()
    assert vv.vvb_attn_decode_dev(c.args) == 0
    torch.cuda.synchronize()
    out = c.dq.cpu().numpy()
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any()
        else:
            assert np.isneginf(out[b, :, 3]).all() and np.isfinite(np.delete(out[b], 3, axis=1)).all()
