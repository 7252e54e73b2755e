"""The serving operators together, as a decode loop uses them: plan, append, (rotate,)
attention(, un-rotate) over a pool of pages, captured in one graph and replayed while
dialogues enter, grow and end. After every step the plan is compared with the
definition, the cache rows with one append call per sequence, and the attention with
float64 over the stored bytes."""
import numpy as np
import pytest

import _paged

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def vv():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import vvb200
    torch.cuda.set_device(0)
    return vvb200


def ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


STEPS = [[70, 1, 0, 200], [1, 1, 64, 1], [1, 62, 1, 1], [1, 1, 1, -1], [1, -1, 1, 130], [1, 5, 0, 1], [400, 0, 0, 0], [1, 1, 1, 1]]


@pytest.mark.parametrize("fmt", [_paged.FP16, _paged.E4M3, _paged.TQ4])
def test_decode_loop_over_the_paged_cache(vv, fmt):
    n, nq, nkv, hd, stride, n_pages, rows = 4, 28, 4, 128, 6, 14, 288
    tq, vb = fmt >= _paged.TQ4, _paged.vec_bytes(fmt, hd)
    g = torch.Generator(device="cuda").manual_seed(fmt)
    half = lambda *s: torch.randn(s, generator=g, device="cuda").half()  # noqa: E731
    new, lens, count = ints([0] * n), ints([0] * n), ints([n_pages])
    table, stack = ints(np.full((n, stride), -1)), ints(np.arange(n_pages)[::-1])
    start, slots, positions, status = ints([0] * (n + 1)), ints([0] * rows), ints([0] * rows), ints([0] * n)
    q, k, v = (torch.zeros(rows, h, hd, dtype=torch.float16, device="cuda") for h in (nq, nkv, nkv))
    bias = [half(h * hd) for h in (nq, nkv, nkv)]
    k_store, v_store = (torch.zeros(n_pages * 64, nkv, vb, dtype=torch.uint8, device="cuda") for _ in range(2))
    metas = [torch.zeros(n_pages * 64, nkv, dtype=torch.float16, device="cuda") if tq else None for _ in range(2)]
    out, lse = torch.zeros(n, nq, hd, dtype=torch.float16, device="cuda"), torch.zeros(n, nq, device="cuda")
    size = vv.vvb_attn_decode_scratch_bytes(n, nq, nkv, hd)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    plan = vv.make_kv_plan(new, lens, lens, table, stack, count, count, start, slots, positions, status, n, stride, n_pages, rows)
    append = vv.make_kv_append_slots(q, q, k, v, k_store, v_store, slots, positions, rows, nq, nkv, hd, n_pages * 64, q_bias=bias[0],
                                     k_bias=bias[1], v_bias=bias[2], kv_format=fmt, k_meta=metas[0], v_meta=metas[1])
    newest = torch.zeros(n, nq, hd, dtype=torch.float16, device="cuda")      # the last row of each sequence
    attn = vv.make_attn_decode(newest, out, k_store, v_store, lens, n, nq, nkv, hd, n_pages * 64, block_table=table, table_stride=stride,
                               kv_format=fmt, k_meta=metas[0], v_meta=metas[1], lse=lse, scratch=scratch, scratch_bytes=size)
    rotated = torch.zeros_like(newest)

    def step(stream):
        vv.check(vv.vvb_kv_plan_dev(plan, stream))
        vv.check(vv.vvb_kv_append_slots_dev(append, stream))
        newest.copy_(q[(start[1:].long() - 1).clamp(0, rows - 1)])
        if tq:
            vv.check(vv.vvb_kv_rotate_dev(newest, nq, hd, n, stream))
        vv.check(vv.vvb_attn_decode_dev(attn, stream))
        rotated.copy_(out)
        if tq:
            vv.check(vv.vvb_kv_unrotate_dev(out, nq, hd, n, stream))

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(stream)
    h_lens, h_table, free = np.zeros(n, np.int64), np.full((n, stride), -1), list(np.arange(n_pages)[::-1])
    want_cache = [t.clone() if t is not None else None for t in (k_store, v_store, *metas)]
    for tokens in STEPS:
        new.copy_(ints(tokens))
        for t in (q, k, v):
            t.copy_(half(*t.shape))
        was = [t.clone() for t in (q, k, v)]
        want = _paged.plan(tokens, h_lens, h_table, np.array(free), len(free), rows)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == want["status"] and lens.tolist() == list(want["lens"]) and slots.tolist() == want["slots"]
        assert count.item() == want["count"] and np.array_equal(table.cpu().numpy(), want["table"])
        assert positions.tolist() == want["positions"]
        for b in range(n):                             # the cache, one call per sequence
            i, j = want["start"][b], want["start"][b + 1]
            if j > i and want["status"][b] == 0:
                at = want["lens"][b] - (j - i)
                assert vv.vvb_kv_append_dev(was[0][i:j], was[1][i:j], was[2][i:j], want_cache[0], want_cache[1], j - i, nq, nkv, hd,
                                            q_bias=bias[0], k_bias=bias[1], v_bias=bias[2], page_table=ints(want["table"][b]),
                                            position_offset=at, cache_offset=at, kv_format=fmt, k_meta=want_cache[2],
                                            v_meta=want_cache[3]) == 0
        torch.cuda.synchronize()
        for x, y in zip((k_store, v_store, *metas), want_cache):
            assert x is None or torch.equal(x, y)
        assert torch.equal(q, was[0])
        kv = [t.cpu().numpy() for t in (k_store, v_store)]
        ms = [t.cpu().numpy() if t is not None else None for t in metas]
        got, glse, gq = rotated.cpu().numpy(), lse.cpu().numpy(), newest.cpu().numpy()
        for b in range(n):
            p = np.arange(want["lens"][b])
            s = want["table"][b, p // 64].astype(np.int64) * 64 + p % 64
            kk, vw = (_paged.decode(x[s], m[s] if tq else None, fmt, hd) for x, m in zip(kv, ms))
            o, l, absout, worst = _paged.attention(gq[b].astype(np.float64), kk, vw, hd ** -0.5)
            tol, tol_lse = _paged.tolerances(o, absout, worst, l, len(s), hd, fmt)
            assert (np.abs(got[b] - o) <= tol).all()
            assert np.isneginf(glse[b]).all() if len(s) == 0 else (np.abs(glse[b] - l) <= tol_lse).all()
        h_lens, h_table, free = np.array(want["lens"]), want["table"], want["pushed"][: want["count"]]
