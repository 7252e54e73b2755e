"""vvb_attn_decode_dev: every way of cutting the work for heads of 64 and 256, groups above
eight and one query head to a cache head, against float64 (tests/_paged.py)."""
import numpy as np
import pytest

from _paged import E4M3, E5M2, FP16, TQ1_5, TQ2, TQ3, TQ4
from test_attn_decode import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import vvb200
    torch.cuda.set_device(0)
    return vvb200


# positions of a block: four warps of 16 keys, 32 where a row is under 256 bytes, 64 where it is under 64
SHAPES = [(FP16, 3, 1, 256, 64), (E4M3, 3, 1, 256, 64), (E5M2, 4, 2, 256, 64), (FP16, 2, 2, 64, 128), (E5M2, 3, 3, 64, 128), (FP16, 20, 1, 64, 128),
          (FP16, 16, 1, 128, 64), (E4M3, 11, 1, 128, 128), (TQ4, 9, 1, 128, 384), (TQ3, 16, 1, 128, 256), (TQ2, 12, 1, 128, 256),
          (TQ1_5, 16, 1, 128, 256), (TQ3, 3, 3, 128, 256)]


@pytest.mark.parametrize("n,blocks", [(1, 1), (1, 3), (2, 30), (40, 2), (40, 12), (130, 20), (500, 4), (900, 1), (950, 2), (1000, 3), (1800, 4)])
@pytest.mark.parametrize("fmt,nq,nkv,hd,block", SHAPES)
def test_attn_ways_of_other_heads(vv, fmt, nq, nkv, hd, block, n, blocks):
    if n * blocks * block * nkv > 800_000:
        n = max(1, 800_000 // (blocks * block * nkv))
    rng = np.random.default_rng(n + fmt + hd)
    top = blocks * block
    lens = np.where(rng.random(n) < 0.1, 0, np.exp(rng.uniform(0, np.log(top + 1), n))).astype(np.int64)
    lens[rng.integers(n)] = top
    c = Case(vv, lens, nq, nkv, hd, fmt, seed=n, slack=0).upload()
    out, lse = c.run()
    pick = np.unique(np.concatenate([rng.integers(0, n, 60), [0, n - 1, int(np.argmax(lens))]]))      # checked in float64
    for b in pick:
        d = Case.__new__(Case)
        d.__dict__ = dict(c.__dict__)
        d.lens, d.q = lens[b:b + 1], c.q[b:b + 1]
        d.slots = lambda _, b=b: c.slots(b)
        d.check(out[b:b + 1], lse[b:b + 1])
    again = c.run()
    assert np.array_equal(again[0].view(np.uint16), out.view(np.uint16)) and np.array_equal(again[1], lse)


# sequences, blocks, whether one kernel does it: at the limits between the ways and past them, four cache heads
EDGES = [(2, 8, True), (2, 9, False), (16, 10, True), (16, 11, False), (24, 14, True), (24, 15, False), (47, 14, True), (48, 16, True), (48, 17, False),
         (148, 2, True), (148, 3, True), (222, 3, True), (222, 4, True), (444, 5, True), (444, 6, True), (1332, 8, True), (1332, 9, True)]


@pytest.mark.parametrize("n,blocks,one", EDGES)
@pytest.mark.parametrize("fmt", [FP16, E5M2])
def test_attn_at_the_limits_of_the_ways(vv, fmt, n, blocks, one):
    rng = np.random.default_rng(n + blocks)
    top = blocks * (64 if fmt == FP16 else 128)
    lens = np.where(rng.random(n) < 0.2, 0, np.exp(rng.uniform(0, np.log(min(top, 300) + 1), n))).astype(np.int64)
    lens[rng.integers(n)] = top
    c = Case(vv, lens, 8, 4, 128, fmt, seed=n, slack=0).upload()
    n0 = vv.launch_count()
    out, lse = c.run()
    assert vv.launch_count() - n0 == (1 if one else 2)
    c.check(out, lse)


@pytest.mark.parametrize("n,blocks,one", [(2, 4, True), (2, 5, False), (16, 5, True), (16, 6, False), (24, 7, True), (24, 8, False), (60, 8, True), (60, 9, False), (148, 1, True), (300, 3, True), (444, 5, True), (444, 6, True)])
@pytest.mark.parametrize("fmt,block", [(TQ4, 384), (TQ3, 256), (TQ1_5, 256)])
def test_attn_at_the_limits_of_the_ways_of_rotated_formats(vv, fmt, block, n, blocks, one):
    rng = np.random.default_rng(n + blocks)
    lens = np.where(rng.random(n) < 0.2, 0, np.exp(rng.uniform(0, np.log(300), n))).astype(np.int64)
    lens[rng.integers(n)] = blocks * block
    c = Case(vv, lens, 8, 4, 128, fmt, seed=n, slack=0).upload()
    n0 = vv.launch_count()
    out, lse = c.run()
    assert vv.launch_count() - n0 == (1 if one else 2)
    c.check(out, lse)
