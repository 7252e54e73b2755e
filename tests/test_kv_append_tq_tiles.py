"""Appends in the rotated formats of long prompts with few heads, where a CTA takes several
row slots of several rows each: its rotated K has to fit the staging buffer whatever the
heads, or K would not be stored at all. Codes and RMS values have to be those of calls of
64 rows, which take one row a slot (and are pinned to the oracle elsewhere)."""
import numpy as np
import pytest

import _paged

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
HD, PIECE = 128, 64
SHAPES = [(8, 8, 2000), (8, 8, 4000), (4, 4, 4000), (3, 3, 5000), (6, 3, 5000), (5, 5, 4000), (10, 5, 4000), (6, 6, 3000), (7, 7, 3000),
          (1, 1, 8200), (2, 2, 7300), (16, 16, 1500), (32, 32, 1000), (28, 4, 2500)]


@pytest.fixture(scope="module")
def vv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import vvb200
    torch.cuda.set_device(0)
    return vvb200


@pytest.mark.parametrize("nq,nkv,rows", SHAPES)
@pytest.mark.parametrize("fmt", [_paged.TQ4, _paged.TQ3, _paged.TQ2, _paged.TQ1_5])
def test_long_appends_store_every_key(vv, nq, nkv, rows, fmt):
    g = torch.Generator(device="cuda").manual_seed(rows + nq + fmt)
    half = lambda *s: torch.randn(s, generator=g, device="cuda").half()  # noqa: E731
    q, k, v, ref = half(rows, nq, HD), half(rows, nkv, HD), half(rows, nkv, HD), half(nkv * HD)
    cache = lambda: [torch.full((rows, nkv, _paged.vec_bytes(fmt, HD)), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2)] + \
        [torch.full((rows, nkv), -7.0, dtype=torch.float16, device="cuda") for _ in range(2)]  # noqa: E731
    want, one, many = cache(), cache(), cache()
    wq = q.clone()
    for i in range(0, rows, PIECE):
        j = min(i + PIECE, rows)
        assert vv.vvb_kv_append_dev(wq[i:j], k[i:j].clone(), v[i:j], want[0], want[1], j - i, nq, nkv, HD, k_ref=ref, position_offset=i,
                                    cache_offset=i, kv_format=fmt, k_meta=want[2], v_meta=want[3]) == 0
    oq = q.clone()
    assert vv.vvb_kv_append_dev(oq, k.clone(), v, one[0], one[1], rows, nq, nkv, HD, k_ref=ref, kv_format=fmt, k_meta=one[2], v_meta=one[3]) == 0
    # the ragged form: rows in another order, every ninth without a slot
    order = torch.from_numpy(np.random.default_rng(rows).permutation(rows).astype(np.int32)).cuda()
    slots = torch.where(torch.arange(rows, device="cuda") % 9 == 4, -1, order)
    mq = torch.full_like(q, 9.0)
    at = order.long()
    a = vv.make_kv_append_slots(q[at].contiguous(), mq, k[at].contiguous(), v[at].contiguous(), many[0], many[1], slots, order, rows, nq, nkv, HD,
                                rows, k_ref=ref, kv_format=fmt, k_meta=many[2], v_meta=many[3])
    assert vv.vvb_kv_append_slots_dev(a) == 0
    torch.cuda.synchronize()
    assert bool((want[2] > 0).all()) and torch.equal(oq, wq)
    for x, y in zip(one, want):
        assert torch.equal(x, y)
    live = slots >= 0
    assert torch.equal(mq[live], wq[at][live]) and bool((mq[~live] == 9.0).all())
    stored = torch.zeros(rows, dtype=torch.bool, device="cuda")
    stored[order[live].long()] = True
    for x, y, fresh in zip(many, want, cache()):
        assert torch.equal(x[stored], y[stored]) and torch.equal(x[~stored], fresh[~stored])
