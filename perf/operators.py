"""The serving operators over the paged KV cache, with their plain forms: the step plan
(block tables, slot map and positions from request lengths), the batched bias + RoPE +
cache append through the slot map, and the attention of one new token per sequence over
the cache. ``own`` selects the library's kernels; otherwise `run` computes the same in
elementary torch operations."""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64
FP16, E4M3, E5M2, TQ4 = 0, 1, 2, 3
THETA = 1e6
LEVELS = [0.127960, 0.386970, 0.654379, 0.938657, 1.251845, 1.613787, 2.065280, 2.725112]   # 4-bit code book, upper half
F8 = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}


def listed():
    return [
        # plan: sixteen running dialogues, one token each -- every decode step begins with it
        {"name": "plan_step_16", "op": "plan", "seqs": 16, "table": 256, "rows": 16, "kind": "step", "lens": 1},
        # plan: a server's mixed batch: prompts entering, dialogues running, slots idle or ending
        {"name": "plan_mixed_256", "op": "plan", "seqs": 256, "table": 512, "rows": 16384, "kind": "mixed", "lens": 2},
        # plan: a full admission wave, more rows than a chunk of any one prompt
        {"name": "plan_mixed_2000", "op": "plan", "seqs": 2000, "table": 512, "rows": 131072, "kind": "mixed", "lens": 3},
        # append: the decode step of sixteen dialogues, 7B heads
        {"name": "append_step_16_fp16", "op": "append", "rows": 16, "pad": 0, "seqs": 16, "nq": 28, "nkv": 4, "hd": 128,
         "fmt": FP16, "bias": True, "lens": 4},
        # append: a ragged chunk of prompts into an FP8 cache, the batch padded to its capacity
        {"name": "append_ragged_2500_e4m3", "op": "append", "rows": 2500, "pad": 60, "seqs": 9, "nq": 28, "nkv": 4, "hd": 128,
         "fmt": E4M3, "bias": True, "lens": 5},
        # append: the long prompt of the benchmark, split over four sequences
        {"name": "append_14449_fp16", "op": "append", "rows": 14449, "pad": 0, "seqs": 4, "nq": 28, "nkv": 4, "hd": 128,
         "fmt": FP16, "bias": False, "lens": 6},
        # attention: one dialogue, a few hundred positions: latency
        {"name": "attn_1x300_fp16", "op": "attn", "seqs": 1, "longest": 300, "spread": "full", "nq": 28, "nkv": 4, "hd": 128,
         "fmt": FP16, "paged": True, "lse": False, "lens": 7},
        # attention: one dialogue over the benchmark's long prompt, contiguous cache, length from the device position
        {"name": "attn_1x14449_fp16", "op": "attn", "seqs": 1, "longest": 14449, "spread": "full", "nq": 28, "nkv": 4, "hd": 128,
         "fmt": FP16, "paged": False, "lse": False, "lens": 8},
        # attention: a server's ragged batch, some slots empty, log-sum-exp asked for
        {"name": "attn_96_ragged_fp16", "op": "attn", "seqs": 96, "longest": 16384, "spread": "log", "nq": 28, "nkv": 4, "hd": 128,
         "fmt": FP16, "paged": True, "lse": True, "lens": 9},
        # attention: long dialogues in the FP8 cache
        {"name": "attn_48_long_e4m3", "op": "attn", "seqs": 48, "longest": 8200, "spread": "half", "nq": 28, "nkv": 4, "hd": 128,
         "fmt": E4M3, "paged": True, "lse": False, "lens": 10},
        # attention: the same in the 4-bit cache
        {"name": "attn_48_long_tq4", "op": "attn", "seqs": 48, "longest": 8200, "spread": "half", "nq": 28, "nkv": 4, "hd": 128,
         "fmt": TQ4, "paged": True, "lse": False, "lens": 11},
        # attention: many short sequences, one query head to a cache head, 64-wide heads
        {"name": "attn_200_short_e5m2", "op": "attn", "seqs": 200, "longest": 500, "spread": "log", "nq": 12, "nkv": 12, "hd": 64,
         "fmt": E5M2, "paged": True, "lse": False, "lens": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn"])
    lens = rng.randrange(1000, 1 << 30)
    if op == "plan":
        kind = rng.choice(["step", "mixed"])
        seqs = _log(rng, 1, 2000)
        rows = seqs if kind == "step" else _log(rng, max(2 * seqs, 64), max(131072 * seqs // 2000, 8 * seqs, 4096))
        return {"op": op, "seqs": seqs, "table": rng.choice([130, 256, 512]), "rows": rows, "kind": kind, "lens": lens}
    nq, nkv, hd = rng.choice([(28, 4, 128), (28, 4, 128), (12, 2, 128), (40, 8, 128), (16, 16, 64), (9, 3, 64), (16, 2, 256)])
    if op == "append":
        rows = _log(rng, 1, 14449 * 4096 // max(4096, (nq + 2 * nkv) * hd))
        return {"op": op, "rows": rows, "pad": rng.choice([0, 0, rows // 9]), "seqs": rng.randint(1, min(rows, 40)), "nq": nq, "nkv": nkv,
                "hd": hd, "fmt": rng.choice([FP16, E4M3, E5M2]), "bias": rng.random() < 0.5, "lens": lens}
    seqs = _log(rng, 1, 96)
    longest = _log(rng, 1, min(16384, 78_000_000 // (seqs * nkv * hd)))
    fmt = rng.choice([FP16, E4M3, E5M2, TQ4] if hd == 128 else [FP16, E4M3, E5M2])
    return {"op": op, "seqs": seqs, "longest": longest, "spread": rng.choice(["full", "half", "log"]), "nq": nq, "nkv": nkv, "hd": hd,
            "fmt": fmt, "paged": seqs > 1 or rng.random() < 0.5, "lse": False, "lens": lens}


# ------------------------------------------------------------------------ what a case's requests are
def _plan_requests(c):
    """(cached positions, new tokens) of every sequence: by the case alone."""
    r, n = np.random.RandomState(c["lens"] % (1 << 31)), c["seqs"]
    cap = c["table"] * PAGE
    lens = np.exp(r.uniform(0, math.log(cap // 2), n)).astype(np.int64)
    new = np.ones(n, np.int64)
    if c["kind"] == "mixed":
        what = r.rand(n)
        new[what < 0.15] = 0                        # idle
        new[what < 0.05] = -1                       # ending
        enter = what > 0.6                          # a prompt, or a chunk of one
        share = r.exponential(1.0, n) * enter
        left = max(0, c["rows"] - n)
        new[enter] = 1 + np.floor(0.9 * left * share / max(share.sum(), 1e-9)).astype(np.int64)[enter]
        new = np.minimum(new, cap // 2)
        lens[enter & (r.rand(n) < 0.7)] = 0
    return lens, new


def _pages(lens):
    return -(-np.maximum(lens, 0) // PAGE)


def _append_requests(c):
    """(positions already cached, rows) of every sequence."""
    r, n, rows = np.random.RandomState(c["lens"] % (1 << 31)), c["seqs"], c["rows"] - c["pad"]
    cuts = np.sort(r.choice(np.arange(1, rows), n - 1, replace=False)) if n > 1 and rows > 1 and n <= rows else np.zeros(0, np.int64)
    count = np.diff(np.concatenate([[0], cuts, [rows]])).astype(np.int64)
    return r.randint(0, 9000, len(count)).astype(np.int64), count


def _attn_lens(c):
    r, n, top = np.random.RandomState(c["lens"] % (1 << 31)), c["seqs"], c["longest"]
    if c["spread"] == "full":
        lens = np.full(n, top, np.int64)
    elif c["spread"] == "half":
        lens = r.randint(top // 2, top + 1, n).astype(np.int64)
    else:
        lens = np.exp(r.uniform(0, math.log(top + 1), n)).astype(np.int64)
        lens[r.rand(n) < 0.03] = 0                  # slots without a request
    lens[0] = top
    return lens


def _row_bytes(c):
    """Bytes of one cached position, K and V, with what is kept beside the codes."""
    n = 2 * c["nkv"]
    return n * (64 + 2) if c["fmt"] == TQ4 else n * c["hd"] * (2 if c["fmt"] == FP16 else 1)


def work(case):
    c = case
    if c["op"] == "plan":
        lens, new = _plan_requests(c)
        live = np.maximum(new, 0)
        # lengths and counts in; lengths, starts, status, pages and rows out
        moved = 8 * c["seqs"] + 12 * c["seqs"] + 8 * c["rows"] + 8 * int((_pages(lens + live) - _pages(lens)).sum()) + 8 * int(_pages(lens[new < 0]).sum())
        return {"bytes": float(moved), "flops": 0.0}
    if c["op"] == "append":
        rows = c["rows"] - c["pad"]
        return {"bytes": float(rows * (2 * c["nq"] * c["hd"] * 2 + 2 * c["nkv"] * c["hd"] * 2 + _row_bytes(c)) + 8 * c["rows"]),
                "flops": float(rows * (c["nq"] + c["nkv"]) * c["hd"] * 3)}
    lens = _attn_lens(c)
    total = int(lens.sum())
    return {"bytes": float(total * _row_bytes(c) + c["seqs"] * (4 * c["nq"] * c["hd"] + 4) + (4 * c["seqs"] * c["nq"] if c["lse"] else 0)),
            "flops": float(4 * total * c["nq"] * c["hd"])}


# ------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _tables(lens, width, seed, spare=3):
    """Block table [n, width] of random pages of one pool (-1 where there is none) and the pool's pages."""
    pages = _pages(lens)
    total = int(pages.sum()) + spare
    order = np.random.RandomState(seed % (1 << 31)).permutation(total)
    table = np.full((len(lens), max(1, width)), -1, np.int64)
    table[np.arange(table.shape[1])[None, :] < pages[:, None]] = order[: int(pages.sum())]
    return table, total, order[int(pages.sum()):]


def _cache(c, rows, g):
    """K and V rows of the cache's format: (k, v, k_meta, v_meta)."""
    shape = (rows, c["nkv"], c["hd"])
    got = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
        if c["fmt"] == FP16:
            got.append((x, None))
        elif c["fmt"] in F8:
            got.append((x.to(F8[c["fmt"]]).view(torch.uint8), None))
        else:
            cuts = torch.tensor([0.5 * (a + b) for a, b in zip(LEVELS, LEVELS[1:])], device="cuda")
            code = torch.bucketize(x.float().abs(), cuts).to(torch.uint8)
            code = torch.where(x < 0, 7 - code, 8 + code)
            sigma = (1.0 + 0.2 * torch.randn(shape[:2], generator=g, device="cuda")).abs().add_(0.05).half()
            got.append(((code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), sigma))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = {"case": c}
    if c["op"] == "plan":
        lens, new = _plan_requests(c)
        after = np.where(new < 0, 0, lens + np.maximum(new, 0))
        need = int((_pages(lens + np.maximum(new, 0)) - _pages(lens)).sum())
        table, n_pages, free = _tables(lens, c["table"], seed, spare=need + 5)
        stack = np.full(n_pages, -1, np.int64)
        stack[: len(free)] = free
        s.update(lens=_ints(lens), new=_ints(new), table=_ints(table), stack=_ints(stack), count=_ints([len(free)]), n_pages=n_pages,
                 lens_out=_ints(after * 0), count_out=_ints([0]), start=_ints(np.zeros(c["seqs"] + 1)), slots=_ints(np.zeros(c["rows"])),
                 positions=_ints(np.zeros(c["rows"])), status=_ints(np.zeros(c["seqs"])))
        s["table_out"], s["stack_out"] = s["table"], s["stack"]
    elif c["op"] == "append":
        cached, count = _append_requests(c)
        table, n_pages, _ = _tables(cached + count, int(_pages(cached + count).max()), seed)
        seq = np.repeat(np.arange(len(count)), count)
        pos = cached[seq] + np.arange(len(seq)) - (np.cumsum(count) - count)[seq]
        slots = table[seq, pos // PAGE] * PAGE + pos % PAGE
        rows, width, kvw = c["rows"], c["nq"] * c["hd"], c["nkv"] * c["hd"]
        half = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)  # noqa: E731
        s.update(q=half(rows, c["nq"], c["hd"]), k=half(rows, c["nkv"], c["hd"]), v=half(rows, c["nkv"], c["hd"]),
                 slots=_ints(np.concatenate([slots, np.full(rows - len(slots), -1)])),
                 positions=_ints(np.concatenate([pos, np.full(rows - len(pos), -1)])), n_slots=n_pages * PAGE)
        s["q_out"] = torch.zeros_like(s["q"])
        dt = torch.float16 if c["fmt"] == FP16 else torch.uint8
        s["k_cache"], s["v_cache"] = (torch.zeros(n_pages * PAGE, c["nkv"], c["hd"], device="cuda", dtype=dt) for _ in range(2))
        s["bias"] = [half(w) if c["bias"] else None for w in (width, kvw, kvw)]
        freq = [np.float32(math.pow(THETA, float(np.float32(-2.0 * i) / np.float32(c["hd"])))) for i in range(c["hd"] // 2)]
        s["freq"] = torch.tensor(np.array(freq, np.float32), device="cuda")
    else:
        lens = _attn_lens(c)
        if c["paged"]:
            width = int(_pages(lens).max()) + 2      # the table has room to grow
            table, n_pages, _ = _tables(lens, width, seed)
            rows = n_pages * PAGE
            s["table"], s["width"] = _ints(table), width
        else:
            rows = s["width"] = int(lens.max()) + 51
            s["table"] = None
        s["k"], s["v"], s["k_meta"], s["v_meta"] = _cache(c, rows, g)
        s["q"] = 1.5 * torch.randn(c["seqs"], c["nq"], c["hd"], generator=g, device="cuda", dtype=torch.float16)
        s["out"] = torch.zeros_like(s["q"])
        s["lse"] = torch.zeros(c["seqs"], c["nq"], device="cuda") if c["lse"] else None
        s["rows"] = rows
        s["lens"] = _ints(lens if c["paged"] else lens - 1)      # contiguous: the device position of the newest token
        s["longest"] = int(lens.max())
        s["add"] = 0 if c["paged"] else 1
    if own:
        _handle(s)
    return s


def _handle(s):
    """The argument block that a user's program fills once and launches every step."""
    root = os.path.join(os.getcwd(), "vibevoice.c_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import vvb200 as vv
    c = s["case"]
    s["vv"], s["stream"] = vv, torch.cuda.current_stream().cuda_stream
    if c["op"] == "plan":
        s["args"] = vv.make_kv_plan(s["new"], s["lens"], s["lens_out"], s["table"], s["stack"], s["count"], s["count_out"], s["start"],
                                    s["slots"], s["positions"], s["status"], c["seqs"], c["table"], s["n_pages"], c["rows"])
        s["call"] = vv.vvb_kv_plan_dev
    elif c["op"] == "append":
        bq, bk, bv = s["bias"]
        s["args"] = vv.make_kv_append_slots(s["q"], s["q_out"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                                            c["rows"], c["nq"], c["nkv"], c["hd"], s["n_slots"], q_bias=bq, k_bias=bk, v_bias=bv,
                                            theta=THETA, kv_format=c["fmt"])
        s["call"] = vv.vvb_kv_append_slots_dev
    else:
        size = vv.vvb_attn_decode_scratch_bytes(c["seqs"], c["nq"], c["nkv"], c["hd"])
        s["scratch"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
        s["args"] = vv.make_attn_decode(s["q"], s["out"], s["k"], s["v"], s["lens"], c["seqs"], c["nq"], c["nkv"], c["hd"], s["rows"],
                                        block_table=s["table"], table_stride=s["width"], len_add=s["add"], kv_format=c["fmt"],
                                        k_meta=s["k_meta"], v_meta=s["v_meta"], lse=s["lse"], scratch=s["scratch"], scratch_bytes=size)
        s["call"] = vv.vvb_attn_decode_dev


# ------------------------------------------------------------------------ one pass
def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        s["vv"].check(s["call"](s["args"], s["stream"]))
        if op == "plan":
            return _plan_outputs(s)
        if op == "append":
            return _append_outputs(s)
        return {"out": s["out"], "lse": s["lse"]}
    return {"plan": _plan, "append": _append, "attn": _attn}[op](s)


def _plan_outputs(s):
    return {k: s[k] for k in ("lens_out", "table_out", "stack_out", "count_out", "start", "slots", "positions", "status")}


def _plan(s):
    c = s["case"]
    n, width, dev = c["seqs"], c["table"], "cuda"
    lens, new, table = s["lens"].long(), s["new"].long(), s["table"].long()
    ends = new < 0
    add = new.clamp(min=0)
    have = (lens + PAGE - 1) // PAGE
    start = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), add.cumsum(0)])
    full = ~ends & (lens + add > width * PAGE)
    no_rows = ~ends & ~full & (start[1:] > c["rows"])
    need = torch.where(ends | full | no_rows, 0, (lens + add + PAGE - 1) // PAGE - have)
    # released pages go onto the stack in order
    freed = torch.where(ends, have, 0)
    at = s["count"].long() + (freed.cumsum(0) - freed)[:, None] + torch.arange(width, device=dev)[None, :]
    at = torch.where(torch.arange(width, device=dev)[None, :] < freed[:, None], at, s["n_pages"])
    stack = torch.cat([s["stack"].long(), torch.zeros(1, dtype=torch.long, device=dev)]).scatter(0, at.reshape(-1), table.reshape(-1))
    avail = s["count"].long() + freed.sum()
    upto = need.cumsum(0)
    no_pages = (need > 0) & (upto > avail)
    ok = ~(ends | full | no_rows | no_pages)
    taken = torch.where(ok & (need > 0), upto, 0).max()
    # admitted sequences take pages from the top
    blk = torch.arange(width, device=dev)[None, :] - have[:, None]
    fresh = ok[:, None] & (blk >= 0) & (blk < need[:, None])
    top = (avail - 1 - (upto - need)[:, None] - blk).clamp(0, s["n_pages"])
    table = torch.where(fresh, stack[top], table)
    row = torch.arange(c["rows"], device=dev)
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True).clamp(max=n - 1)
    live = (row < start[-1]) & ok[seq]
    pos = torch.where(live, lens[seq] + row - start[seq], 0)
    slot = table[seq, pos // PAGE] * PAGE + pos % PAGE
    out = {"lens_out": torch.where(ends, 0, torch.where(ok, lens + add, lens)), "table_out": table, "stack_out": stack[:-1],
           "count_out": (avail - taken).reshape(1), "start": start, "slots": torch.where(live, slot, -1),
           "positions": torch.where(live, pos, -1), "status": full * 2 + no_rows * 3 + no_pages * 1}
    return {k: v.to(torch.int32) for k, v in out.items()}


def _append_outputs(s):
    c = s["case"]
    k, v = s["k_cache"], s["v_cache"]
    if c["fmt"] in F8:
        k, v = k.view(F8[c["fmt"]]), v.view(F8[c["fmt"]])
    return {"q": s["q_out"], "k_cache": k, "v_cache": v}


def _encode(x, fmt):
    """FP16 values to the cache's format: FP8 rounds to nearest even and saturates; below the smallest normal it rounds half up."""
    if fmt == FP16:
        return x
    low, step, most = (2.0 ** -6, 2.0 ** -9, 448.0) if fmt == E4M3 else (2.0 ** -14, 2.0 ** -16, 57344.0)
    x = x.float()
    small = torch.floor(x.abs() / step + 0.5) * step * torch.sign(x)
    return torch.where(x.abs() < low, small, x.clamp(-most, most)).to(F8[fmt]).view(torch.uint8)


def _append(s):
    c = s["case"]
    live = s["slots"] >= 0
    slots = torch.where(live, s["slots"], s["n_slots"]).long()
    angle = (s["positions"].float()[:, None] * s["freq"][None, :]).double()
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def biased(x, b):
        return x if b is None else (x.float() + b.float().view(1, *x.shape[1:])).half()

    def turned(x):
        lo, hi = x.float().chunk(2, dim=-1)
        return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], dim=-1).half()

    bq, bk, bv = s["bias"]
    s["q_out"].copy_(torch.where(live[:, None, None], turned(biased(s["q"], bq)), s["q_out"]))
    for name, x in (("k_cache", turned(biased(s["k"], bk))), ("v_cache", biased(s["v"], bv))):
        room = torch.cat([s[name], s[name][:1]])
        room[slots] = _encode(x, c["fmt"])
        s[name].copy_(room[:-1])
    return _append_outputs(s)


def _values(rows, meta, fmt):
    """Cache rows as 32-bit values."""
    if fmt == FP16:
        return rows.float()
    if fmt in F8:
        return rows.view(F8[fmt]).float()
    book = torch.tensor([-x for x in reversed(LEVELS)] + LEVELS, device=rows.device)
    code = torch.stack([rows & 15, rows >> 4], dim=-1).flatten(-2).long()
    return book[code] * meta.float()[..., None]


def _attn(s):
    c = s["case"]
    n, nkv, hd = c["seqs"], c["nkv"], c["hd"]
    lens = s["lens"].long() + s["add"]
    at = torch.arange(s["longest"], device="cuda")
    live = at[None, :] < lens[:, None]
    if c["paged"]:
        slot = s["table"].long()[:, at // PAGE] * PAGE + (at % PAGE)[None, :]
    else:
        slot = at[None, :].expand(n, -1)
    slot = torch.where(live, slot, 0)
    k = _values(s["k"][slot], s["k_meta"][slot] if c["fmt"] == TQ4 else None, c["fmt"])
    q = s["q"].float().view(n, nkv, c["nq"] // nkv, hd)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(hd))
    del k
    score = score.masked_fill(~live[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = _values(s["v"][slot], s["v_meta"][slot] if c["fmt"] == TQ4 else None, c["fmt"])
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / total.clamp(min=1e-37)
    lse = torch.where(total > 0, top + total.clamp(min=1e-37).log(), -math.inf)
    return {"out": out.reshape(n, c["nq"], hd).half(), "lse": lse.reshape(n, c["nq"]) if c["lse"] else None}


# ------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None                                  # whole numbers only
    s = prepare(case, seed)
    if c["op"] == "append":
        # the definition: the bias sum and the rotated value are FP16 values, the angle is the 32-bit product
        rows = int((s["slots"] >= 0).sum())
        to16 = lambda x: x.half().double()  # noqa: E731
        angle = (s["positions"][:rows].to(torch.float32).unsqueeze(1) * s["freq"].unsqueeze(0)).to(torch.float64).unsqueeze(1)
        got = {}
        for name, x, b, rotate in (("q", s["q"], s["bias"][0], True), ("k_cache", s["k"], s["bias"][1], True), ("v_cache", s["v"], s["bias"][2], False)):
            x = x[:rows].double()
            if b is not None:
                x = to16(x + b.double().reshape(1, x.shape[1], x.shape[2]))
            if rotate:
                z = torch.view_as_complex(torch.stack(x.split(c["hd"] // 2, dim=2), dim=-1))
                z = z * torch.polar(torch.ones_like(angle), angle)
                x = torch.cat([z.real, z.imag], dim=2)
            if name == "q":
                got[name] = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
                got[name][:rows] = x
                continue
            whole = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
            if c["fmt"] == FP16:
                whole[s["slots"][:rows].long()] = x
            else:
                x = to16(x)
                bits, least = (3, -6) if c["fmt"] == E4M3 else (2, -14)
                powers = torch.tensor([2.0 ** e for e in range(-32, 32)], dtype=torch.float64, device="cuda")
                ulp = powers[(torch.frexp(x)[1].long() - 1).clamp(min=least) - bits + 32]
                near = torch.where(x.abs() < 2.0 ** least, torch.floor(x.abs() / ulp + 0.5), torch.round(x.abs() / ulp)) * ulp
                whole[s["slots"][:rows].long()] = torch.copysign(near.clamp(max=448.0 if bits == 3 else 57344.0), x)
            got[name] = whole
        return got
    lens = _attn_lens(c)
    n, group = c["seqs"], c["nq"] // c["nkv"]
    out = torch.zeros(n, c["nq"], c["hd"], dtype=torch.float64, device="cuda")
    lse = torch.full((n, c["nq"]), -math.inf, dtype=torch.float64, device="cuda")
    codes = torch.tensor([-v for v in LEVELS[::-1]] + LEVELS, dtype=torch.float64, device="cuda")
    for b in range(n):
        top = int(lens[b])
        if top == 0:
            continue
        if c["paged"]:
            pages = s["table"][b, : -(-top // PAGE)].long()
            rows = (pages[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:top]
        else:
            rows = torch.arange(top, device="cuda")
        kv = []
        for x, m in ((s["k"], s["k_meta"]), (s["v"], s["v_meta"])):
            x = x[rows]
            if c["fmt"] == TQ4:
                x = codes[torch.cat([(x & 15)[..., None], (x >> 4)[..., None]], dim=-1).reshape(top, c["nkv"], c["hd"]).int()] * m[rows].double()[..., None]
            elif c["fmt"] != FP16:
                x = x.view(F8[c["fmt"]]).to(torch.float32)
            kv.append(x.double().repeat_interleave(group, dim=1))
        z = torch.einsum("hd,lhd->hl", s["q"][b].double(), kv[0]) / math.sqrt(c["hd"])
        out[b] = torch.einsum("hl,lhd->hd", torch.softmax(z, dim=1), kv[1])
        lse[b] = torch.logsumexp(z, dim=1)
    return {"out": out, "lse": lse if c["lse"] else None}
