"""vvb_kv_append_slots_dev: the rows of a ragged batch into their slots. The bytes
have to be those of vvb_kv_append_dev called once per sequence with that sequence's
page table (itself pinned to the oracle and the reference elsewhere)."""
import numpy as np
import pytest

import _paged

P = 0x1000


@pytest.fixture(scope="module")
def lib():
    import vvb200
    return vvb200


def fake(vv, **kw):
    a = dict(q=P, q_out=P, k=P, v=P, k_store=P, v_store=P, slot_map=P, positions=P, rows=4, n_q_heads=28, n_kv_heads=4, head_dim=128,
             n_slots=640)
    kws = {k: kw.pop(k) for k in list(kw) if k not in a}
    a.update(kw)
    return vv.make_kv_append_slots(*a.values(), **kws)


@pytest.mark.parametrize("kw,want", [
    (dict(q=None), "VV_ERR_NULL_PTR"), (dict(q_out=None), "VV_ERR_NULL_PTR"), (dict(k=None), "VV_ERR_NULL_PTR"), (dict(v=None), "VV_ERR_NULL_PTR"),
    (dict(k_store=None), "VV_ERR_NULL_PTR"), (dict(v_store=None), "VV_ERR_NULL_PTR"), (dict(slot_map=None), "VV_ERR_NULL_PTR"),
    (dict(positions=None), "VV_ERR_NULL_PTR"), (dict(rows=-1), "VV_ERR_INVALID_ARG"), (dict(n_q_heads=0), "VV_ERR_INVALID_ARG"),
    (dict(n_kv_heads=0), "VV_ERR_INVALID_ARG"), (dict(head_dim=0), "VV_ERR_INVALID_ARG"), (dict(n_slots=-1), "VV_ERR_INVALID_ARG"),
    (dict(slot_map=P + 2), "VV_ERR_INVALID_ARG"), (dict(positions=P + 1), "VV_ERR_INVALID_ARG"),
    (dict(kv_format=7), "VV_ERR_UNSUPPORTED"), (dict(kv_format=-1), "VV_ERR_UNSUPPORTED"), (dict(kv_format=3), "VV_ERR_NULL_PTR"),
    (dict(kv_format=3, k_meta=P, v_meta=P, head_dim=64), "VV_ERR_UNSUPPORTED"), (dict(head_dim=24), "VV_ERR_UNSUPPORTED"),
    (dict(head_dim=1024), "VV_ERR_UNSUPPORTED"), (dict(q=P + 2), "VV_ERR_UNSUPPORTED"), (dict(q_out=P + 8), "VV_ERR_UNSUPPORTED"),
    (dict(q_bias=P + 2), "VV_ERR_UNSUPPORTED"), (dict(rows=0), "VV_OK"),
])
def test_append_slots_refusals(lib, kw, want):
    assert lib.vvb_kv_append_slots_dev(fake(lib, **kw), stream=0) == getattr(lib, want)
    assert lib._lib.vvb_kv_append_slots_dev(None, None) == lib.VV_ERR_NULL_PTR


torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def vv(lib):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.set_device(0)
    return lib


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def same(a, b):
    return bool((a.contiguous().view(torch.uint8) == b.contiguous().view(torch.uint8)).all())


SHAPES = [([1], [0], 28, 4, 128), ([1] * 16, list(range(0, 16 * 97, 97)), 28, 4, 128), ([5, 0, 64, 1, 130], [60, 9, 0, 127, 1], 28, 4, 128),
          ([700, 3], [13, 9000], 12, 2, 128), ([33, 70], [0, 5], 40, 8, 128), ([9, 20], [63, 64], 3, 3, 64), ([37], [2], 16, 2, 256)]


@gpu
@pytest.mark.parametrize("count,cached,nq,nkv,hd", SHAPES)
@pytest.mark.parametrize("fmt", range(7))
def test_append_slots_equals_one_call_per_sequence(vv, count, cached, nq, nkv, hd, fmt):
    if fmt >= _paged.TQ4 and hd != 128:
        pytest.skip("the rotated formats have 128-wide heads")
    rng = np.random.default_rng(sum(count) + 10 * fmt + nq)
    count, cached = np.array(count), np.array(cached)
    pad, rows = 3, int(count.sum()) + 3
    pages = -(-(count + cached) // 64)
    n_pages = int(pages.sum()) + 2
    order = rng.permutation(n_pages)
    table = np.zeros((len(count), pages.max()), np.int32)
    table[np.arange(pages.max())[None, :] < pages[:, None]] = order[: pages.sum()]
    seq = np.repeat(np.arange(len(count)), count)
    start = np.cumsum(count) - count
    pos = cached[seq] + np.arange(len(seq)) - start[seq]
    slots = table[seq, pos // 64] * 64 + pos % 64
    slots, pos = np.concatenate([slots, [-1, n_pages * 64, 2 ** 31 - 1]]).astype(np.int32), np.concatenate([pos, [-1, 7, 10 ** 9]]).astype(np.int32)
    f16 = lambda *s: dev(rng.standard_normal(s).astype(np.float16))  # noqa: E731
    q, k, v = f16(rows, nq, hd), f16(rows, nkv, hd), f16(rows, nkv, hd)
    bias = {"q_bias": f16(nq * hd), "k_bias": f16(nkv * hd), "v_bias": f16(nkv * hd)} if fmt != _paged.E5M2 else {}
    ref = {"k_ref": f16(nkv * hd)} if fmt in (_paged.E4M3, _paged.TQ4) else {}
    vb, tq = _paged.vec_bytes(fmt, hd), fmt >= _paged.TQ4
    new_cache = lambda: [torch.full((n_pages * 64, nkv, vb), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2)] + \
        [torch.full((n_pages * 64, nkv), 7.0, dtype=torch.float16, device="cuda") if tq else None for _ in range(2)]  # noqa: E731
    got, want = new_cache(), new_cache()
    keep = [t.clone() for t in (q, k, v)]
    out = torch.full_like(q, 9.0)
    n0 = vv.launch_count()
    a = vv.make_kv_append_slots(q, out, k, v, got[0], got[1], dev(slots), dev(pos), rows, nq, nkv, hd, n_pages * 64, kv_format=fmt,
                                k_meta=got[2], v_meta=got[3], **bias, **ref)
    assert vv.vvb_kv_append_slots_dev(a) == 0 and vv.launch_count() - n0 == 1
    assert all(same(x, y) for x, y in zip((q, k, v), keep))                     # the inputs are only read
    wq = q.clone()
    for b in range(len(count)):
        if count[b]:
            i, j = int(start[b]), int(start[b] + count[b])
            assert vv.vvb_kv_append_dev(wq[i:j], k[i:j].clone(), v[i:j], want[0], want[1], int(count[b]), nq, nkv, hd, kv_format=fmt,
                                        k_meta=want[2], v_meta=want[3], page_table=dev(table[b]), position_offset=int(cached[b]),
                                        cache_offset=int(cached[b]), **bias, **ref) == 0
    torch.cuda.synchronize()
    assert same(out[:-pad], wq[:-pad]) and bool((out[-pad:] == 9.0).all())      # rows without a slot are left alone
    for x, y in zip(got, want):
        assert x is None or same(x, y)
    # in place
    a = vv.make_kv_append_slots(q, q, k, v, got[0], got[1], dev(slots), dev(pos), rows, nq, nkv, hd, n_pages * 64, kv_format=fmt,
                                k_meta=got[2], v_meta=got[3], **bias, **ref)
    assert vv.vvb_kv_append_slots_dev(a) == 0
    torch.cuda.synchronize()
    assert same(q[:-pad], out[:-pad]) and same(q[-pad:], keep[0][-pad:])


@gpu
def test_append_slots_far_rows_of_a_large_cache(vv):
    """Cache rows whose byte offset passes 32 bits, and positions far out."""
    nq, nkv, hd, rows = 4, 4, 128, 5
    n_slots = (1 << 32) // (nkv * hd * 2) + 192
    k_store = torch.empty(n_slots, nkv, hd, dtype=torch.float16, device="cuda")
    v_store = torch.empty_like(k_store)
    slots = np.array([n_slots - 1, 3, n_slots - 130, n_slots, 64], np.int32)
    pos = np.array([100000, 0, 65536, 3, 77], np.int32)
    q, k, v = (torch.randn(rows, n, hd, device="cuda").half() for n in (nq, nkv, nkv))
    out = torch.zeros_like(q)
    k_store[:256].zero_(), k_store[-256:].zero_()
    assert vv.vvb_kv_append_slots_dev(vv.make_kv_append_slots(q, out, k, v, k_store, v_store, dev(slots), dev(pos), rows, nq, nkv, hd, n_slots)) == 0
    for r in (0, 1, 2, 4):
        one = q[r:r + 1].clone(), k[r:r + 1].clone()
        assert vv.vvb_rope_qk_dev(one[0], one[1], 1, nq, nkv, hd, int(pos[r]), None, 1e6) == 0
        torch.cuda.synchronize()
        s = int(slots[r])
        assert same(out[r:r + 1], one[0]) and same(k_store[s:s + 1], one[1]) and same(v_store[s:s + 1], v[r:r + 1])
    assert not out[3].any() and int((k_store[-256:].abs().sum((1, 2)) > 0).sum()) == 2 and int((k_store[:256].abs().sum((1, 2)) > 0).sum()) == 2
