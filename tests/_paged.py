"""Plain statements of the serving operators over the paged cache, for the tests:
the step plan in Python integers, cache decoding and attention in float64."""
import numpy as np

PAGE = 64
FP16, E4M3, E5M2, TQ4, TQ3, TQ2, TQ1_5 = range(7)
TQ_BYTES = {TQ4: 64, TQ3: 48, TQ2: 32, TQ1_5: 24}
_HALF = {TQ4: [0.127960, 0.386970, 0.654379, 0.938657, 1.251845, 1.613787, 2.065280, 2.725112],
         TQ3: [0.244756, 0.755588, 1.343258, 2.150300], TQ2: [0.452456, 1.511418]}
LEVELS = {f: np.array([-x for x in reversed(h)] + h) for f, h in _HALF.items()}
PAIRS = np.array([-1.500251, +0.674678, -1.127883, -0.787015, -0.283251, +0.390133, -0.103102, +1.624620,
                  +0.100120, -1.618563, +0.286482, -0.379555, +1.134227, +0.790368, +1.496572, -0.666578]).reshape(8, 2)


def plan(new, lens, table, stack, count, max_rows):
    """The definition, one sequence after the other. Returns a dict of new arrays."""
    n, stride = table.shape
    lens_out, table, stack = list(lens), table.copy(), list(stack[:count])
    pages = lambda x: -(-max(int(x), 0) // PAGE)  # noqa: E731
    for b in range(n):
        if new[b] < 0:
            stack += [int(x) for x in table[b, :min(pages(lens[b]), stride)]]
    pushed = list(stack)
    start, status, slots, positions = [0], [0] * n, [-1] * max_rows, [-1] * max_rows
    asked, height = 0, len(stack)
    for b in range(n):
        length, add = max(int(lens[b]), 0), max(int(new[b]), 0)
        first = start[-1]
        start.append(min(first + add, 2 ** 31 - 1))
        if new[b] < 0:
            lens_out[b] = 0
            continue
        if length + add > stride * PAGE:
            status[b] = 2
            continue
        if add and first + add > max_rows:
            status[b] = 3
            continue
        need = pages(length + add) - pages(length)
        asked += need
        if need and asked > height:
            status[b] = 1
            continue
        for k in range(need):
            table[b, pages(length) + k] = stack.pop()
        for r in range(add):
            p = length + r
            positions[first + r] = p
            slots[first + r] = int(table[b, p // PAGE]) * PAGE + p % PAGE
        lens_out[b] = length + add
    return {"lens": lens_out, "table": table, "pushed": pushed, "count": len(stack), "start": start, "status": status,
            "slots": slots, "positions": positions}


def vec_bytes(fmt, hd):
    return TQ_BYTES.get(fmt, 2 * hd if fmt == FP16 else hd)


def decode(store, meta, fmt, hd):
    """Stored bytes [..., vec_bytes] (uint8) and RMS values to float64 [..., hd]."""
    import torch
    if fmt == FP16:
        return store.view(np.float16).astype(np.float64)
    if fmt in (E4M3, E5M2):
        dt = torch.float8_e4m3fn if fmt == E4M3 else torch.float8_e5m2
        return torch.from_numpy(np.ascontiguousarray(store)).view(dt).float().numpy().astype(np.float64)
    width = {TQ4: 4, TQ3: 3, TQ2: 2, TQ1_5: 3}[fmt]
    bits = np.unpackbits(store, axis=-1, bitorder="little").astype(np.int64)
    code = (bits.reshape(*store.shape[:-1], 8 * store.shape[-1] // width, width) << np.arange(width)).sum(-1)
    x = PAIRS[code].reshape(*store.shape[:-1], hd) if fmt == TQ1_5 else LEVELS[fmt][code]
    return x * meta.astype(np.float64)[..., None]


def attention(q, k, v, scale):
    """q [nq, hd], k and v [n, nkv, hd] in float64 -> out [nq, hd], lse [nq], and what the tolerance needs."""
    nq, hd = q.shape
    n, nkv = k.shape[:2]
    if n == 0:
        return np.zeros((nq, hd)), np.full(nq, -np.inf), np.zeros((nq, hd)), np.zeros(nq)
    g = nq // nkv
    kk, vv = np.repeat(k, g, axis=1), np.repeat(v, g, axis=1)
    s = scale * np.einsum("hd,nhd->hn", q, kk)
    worst = abs(scale) * np.einsum("hd,nhd->hn", np.abs(q), np.abs(kk)).max(1)      # sum |q k| of the largest key
    m = s.max(1, keepdims=True)
    p = np.exp(s - m)
    z = p.sum(1, keepdims=True)
    return np.einsum("hn,nhd->hd", p / z, vv), (m + np.log(z))[:, 0], np.einsum("hn,nhd->hd", p / z, np.abs(vv)), worst


def tolerances(out, absout, worst, lse, n, hd, fmt):
    """(of out, of lse), derived before any run.
    A score: hd products summed in FP32 (hd * 2^-24 of sum |q k|), the factor scale and its change to base 2
    (2^-23 of it), and for the rotated formats levels kept as FP16 values after a common factor: within 9.0e-5 of
    the level for 4 bits (2 and 3 bits less), 1.6e-4 for 1.5 bits. e^x: the score's rounding as an absolute error
    of the exponent, plus 2^-21 for the exponential itself. A weight is kept to 2^-21 (a pair of FP16 values).
    The sums over n keys in FP32: sqrt(n) + 16 roundings of 2^-24 (blocks, then joined), taken as n * 2^-24 when
    n is small. Output: half an FP16 step, 2^-11, or half the smallest subnormal, 2^-25."""
    lev = 0.0 if fmt <= E5M2 else 1.6e-4 if fmt == TQ1_5 else 9.0e-5
    ds = worst * (hd * 2.0 ** -24 + 2.0 ** -23 + lev) + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2.0 ** -22
    sums = min(n, 16 + np.sqrt(n)) * 2.0 ** -24
    rel = np.expm1(2 * ds) + 2.0 ** -20 + lev + 2 * sums
    tol_out = np.abs(out) * 2.0 ** -11 + 2.0 ** -25 + absout * rel[:, None] * (1 + 2.0 ** -11)
    tol_lse = ds + 2.0 ** -20 + sums + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2.0 ** -22
    return tol_out, tol_lse
