"""CPU restatement (numpy) of the 4-bit key/value cache, of appending to it and of attention over it: test infrastructure only.

The layout is written out index by index; quantization follows the operator's definition in float32 one rounding at a time, attention
its formula in float64 with what a bound on the kernels' error needs beside it."""
import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0] + [-v for v in (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)])


def k_place(D, d):
    """(word, nibble) of dimension d of a token's keys."""
    s, kk, n = d // 32, d % 32 // 8, d % 8
    return kk * (D // 32) + s, n


def v_place(D, d):
    """(word, nibble) of dimension d of a token's values."""
    H, W = D // 16, D // 8
    i, rest = d // 16, d % 16
    return rest % W, i + H * (rest // W)


def new_cache(pages, heads, page, D, group, fill=0):
    """Empty cache tensors; unused places hold `fill` codes and NaN scales."""
    kc = np.full((pages, heads, page, D // 8), fill, np.int32)
    vc = np.full((pages, heads, page // 4, D // 8, 4), fill, np.int32)
    sc = np.full((pages, heads, D // group, page), np.nan, np.float16)
    return [kc, vc, sc, sc.copy()]


def encode(y):
    """4-bit codes of float32 y, to nearest, ties to the even code."""
    a = np.abs(y)
    edges = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
    with np.errstate(invalid="ignore"):
        code = sum((a >= e if up else a > e).astype(np.int64) for e, up in edges)
    return code + 8 * np.signbit(y)


def quantize(x, group):
    """(codes, scales) of float32 x [..., D]; a group that fits fp16 has a scale of 10912 at most, whose largest code does."""
    g = x.astype(np.float32).reshape(*x.shape[:-1], -1, group)
    with np.errstate(over="ignore"):
        top = np.abs(g).max(-1)
        scales = (top / np.float32(6.0)).astype(np.float16)
    scales = np.where(top <= 65504, np.minimum(scales, np.float16(10912)), scales)
    s = scales.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(s > 0, g / s, np.float32(0))
    return encode(y).reshape(x.shape), scales


def put(cache, page, head, off, k_codes, k_scales, v_codes, v_scales):
    """Codes [D] and scales [D/group] of one token and head at their place."""
    kc, vc, ks, vs = cache
    D = len(k_codes)
    for c, codes, place in ((kc, k_codes, k_place), (vc, v_codes, v_place)):
        words = np.zeros(D // 8, np.uint32)
        for d in range(D):
            w, n = place(D, d)
            words[w] |= np.uint32(int(codes[d]) << (4 * n))
        if c is kc:
            c[page, head, off] = words.view(np.int32)
        else:
            c[page, head, off // 4, :, off % 4] = words.view(np.int32)
    ks[page, head, :, off], vs[page, head, :, off] = k_scales, v_scales


def get(cache, pages, head, offs):
    """(k, v) float64 [n, D] of n tokens of one head."""
    kc, vc, ks, vs = cache
    D = kc.shape[-1] * 8
    group, pages, offs = D // ks.shape[2], np.asarray(pages, np.int64), np.asarray(offs, np.int64)
    out = []
    for words, place, sc in ((kc[pages, head, offs], k_place, ks), (vc[pages, head, offs // 4, :, offs % 4], v_place, vs)):
        at = np.array([place(D, d) for d in range(D)])
        codes = (words.astype(np.int64)[:, at[:, 0]] >> (4 * at[:, 1])) & 15
        with np.errstate(invalid="ignore"):
            out.append(VALUES[codes] * np.repeat(sc[pages, head][np.arange(len(pages)), :, offs].astype(np.float64), group, axis=-1))
    return out


def rotate(x, cs, interleaved):
    """float32 x [H, D], its first 2 * len(cs) dimensions turned by cs float32 [rot/2, 2], one rounding at a time."""
    half = len(cs)
    c, s = cs[:, 0], cs[:, 1]
    out = x.copy()
    i, j = (np.arange(0, 2 * half, 2), np.arange(1, 2 * half, 2)) if interleaved else (np.arange(half), np.arange(half, 2 * half))
    a, b = x[:, i], x[:, j]
    out[:, i] = a * c - b * s
    out[:, j] = b * c + a * s
    return out


def places(table, lengths, starts, rows, pages, page):
    """For every row: (sequence, position, page or -1, offset), sequence -1 for a row of none."""
    B, width = table.shape
    if starts is None:
        starts = np.arange(B + 1) * (rows // B)
    out = []
    for t in range(rows):
        b = next((i for i in range(B) if starts[i] <= t < starts[i + 1]), -1)
        if b < 0:
            out.append((-1, 0, -1, 0))
            continue
        pos = int(lengths[b]) - int(starts[b + 1]) + t
        pg = int(table[b, pos // page]) if 0 <= pos < width * page else -1
        out.append((b, pos, pg if 0 <= pg < pages else -1, pos % page))
    return out


def attention(q, cache, table, lengths, starts, scale, rounded=False):
    """(out, tol) float64 [T, Hq, D] for float16 q: the formula, and how far a kernel may be off that forms scores and sums in float32, rounds the weights
    (times 2^10 and the value's scale) to fp16 once and the output once; `rounded`: that also rounds every key and value, code * scale, to fp16 once
    (the weights then without the value's scale).  Rows of no sequence: NaN.

    Terms of tol: half a step of the output, 2^-11 |o| (2^-25 where it is subnormal); half a step of every weight, 2^-11 sum p |v|, or 2^-25 * 6 in units of
    2^10 for subnormal ones (fewer where scales above 32 raise the maximum); twice (numerator and denominator) the relative error of a weight, exp of a score that is off by (D + 8) float32 half steps of
    sum |q k| and whose product with scale and difference to the maximum (at most 2 max |s|) round, and two steps of the exponential; the sums over L keys, of at most
    L / 32 + 64 additions one after the other.  `rounded`: a score is off by 2^-11 sum |q k| more (2^-25 sum |q| for subnormal keys, 2^-22 where
    eighths of them are rounded: blocks of up to 128 rows whose last one sees more than 1024 keys), the values by 2^-11 sum p |v|
    and 2^-25."""
    pages, heads, page = cache[0].shape[:3]
    T, Hq, D = q.shape
    share, u = Hq // heads, 2.0 ** -24
    out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    where = places(table, lengths, starts, T, pages, page)
    for b in sorted({w[0] for w in where if w[0] >= 0}):
        n = min(int(lengths[b]), table.shape[1] * page)
        ids = [(int(table[b, j // page]), j % page, j) for j in range(max(n, 0))]
        ids = [(p, o, j) for p, o, j in ids if 0 <= p < pages]
        pos = np.array([j for _, _, j in ids], np.int64)
        for h in range(heads):
            ks, vs = get(cache, [p for p, _, _ in ids], h, [o for _, o, _ in ids])
            big = max(1.0, float(np.nanmax(np.where(np.isfinite(vs), np.abs(vs), 0), initial=0.0)) / 6 / 32)
            for t in (i for i, w in enumerate(where) if w[0] == b):
                seen = np.nonzero(pos <= where[t][1])[0]
                for qh in range(h * share, (h + 1) * share):
                    if len(seen) == 0:
                        out[t, qh], tol[t, qh] = 0.0, 0.0
                        continue
                    k, v = ks[seen], vs[seen]
                    x = q[t, qh].astype(np.float64)
                    s = scale * (k @ x)
                    mag = scale * (np.abs(k) @ np.abs(x)).max()
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    o, pv = p @ v, p @ np.abs(v)
                    eps = mag * (D + 8) * u + 4 * np.abs(s).max() * u + 4 * u
                    more, unit = 0.0, 6 * big
                    if rounded:
                        eps += mag * 2.0 ** -11 + scale * np.abs(x).sum() * 2.0 ** (-22 if len(seen) > 1024 - 128 else -25)
                        more, unit = 2.0 ** -11 * pv + 2.0 ** -25, max(unit, np.abs(v).max())
                    L = len(seen)
                    out[t, qh] = o
                    tol[t, qh] = (2.0 ** -11 * np.abs(o) + 2.0 ** -25 + (2.0 ** -11 + np.expm1(2 * eps) + (L / 32 + 64) * 2 * u) * pv + L * unit * 2.0 ** -35 + more)
    return out, tol
