"""CPU restatement of the paged 8-bit cache (include/exl_amd.h: exl_paged_slots, exl_paged_append, exl_paged_attention) in numpy and 64 bits,
one row and one page at a time -- test infrastructure only."""
import numpy as np

TOP = {"fp8": 448.0, "int8": 127.0}
EXP = {"fp8": (-15, 7), "int8": (-24, 9)}


def slots(past, new, held, table, ring, counters, block, max_len, max_new, rows, row_stride=0):
    """In place on the numpy arrays held, table, ring, counters; returns (starts, slots, positions)."""
    n, blocks = len(past), len(ring)
    starts, out, positions = np.zeros(n + 1, np.int32), np.full(rows, -1, np.int32), np.zeros(rows, np.int32)
    free = [int(ring[(counters[0] + i) % blocks]) for i in range(counters[1])]
    back, missing, taken, at = [], 0, 0, 0
    for b in range(n):
        start = min(b * row_stride, rows) if row_stride else at
        take = max(0, min(int(new[b]), max_new, rows - start, row_stride if row_stride else rows))
        starts[b] = start
        if new[b] < 0:
            back += [int(x) for x in table[b, :held[b]]]
            table[b, :held[b]] = -1
            held[b] = 0
            continue
        want = max(0, -(-min(int(past[b]) + take, max_len) // block) - int(held[b]))
        if (new[b] > 0 or held[b] > 0) and past[b] > int(held[b]) * block:         # earlier tokens found no block: the row gets none behind them
            missing += want
            want = 0
        for _ in range(want):
            if taken < len(free):
                table[b, held[b]] = free[taken]
                held[b] += 1
                taken += 1
            else:
                missing += 1
        for i in range(take):
            pos = int(past[b]) + i
            positions[start + i] = pos
            if pos < max_len and pos // block < held[b] and 0 <= table[b, pos // block] < blocks:
                out[start + i] = table[b, pos // block] * block + pos % block
        at = start + take
    starts[n] = min(n * row_stride, rows) if row_stride else at
    for i, x in enumerate(back):
        ring[(counters[0] + counters[1] + i) % blocks] = x
    counters[:] = [(counters[0] + taken) % blocks, counters[1] - taken + len(back), missing, 0]
    return starts, out, positions


def nearest(x, code):
    """The code's value nearest to each x (ties to even, saturating); NaN stays NaN (int8: 0)."""
    x = np.asarray(x, np.float64)
    nan = np.isnan(x)
    y = np.clip(np.where(nan, 0.0, x), -TOP[code], TOP[code])
    if code == "int8":
        return np.rint(y)
    step = np.ldexp(1.0, np.maximum(np.frexp(y)[1] - 1, -6) - 3)
    return np.where(nan, np.nan, np.rint(y / step) * step)


def exponent(amax, code):
    lo, hi = EXP[code]
    return next(e for e in range(lo, hi + 1) if e == hi or amax <= TOP[code] * 2.0 ** e)


def rotate(x, sin, cos, positions):
    """x [tokens, heads, hd], tables [positions, hd]"""
    half = x.shape[-1] // 2
    s, c = (np.asarray(t, np.float64)[positions][:, None, :] for t in (sin, cos))
    return x * c + np.concatenate((-x[..., half:], x[..., :half]), -1) * s


def append(k, v, slot, key_codes, value_codes, key_scales, value_scales, code, positions=None, sin=None, cos=None):
    """k, v [rows, kv_heads, hd]; codes as numbers: key_codes [blocks, kvh, block, hd16], value_codes [blocks, kvh, hd16, block]; in place."""
    blocks, _, block, hd16 = key_codes.shape
    hd = k.shape[-1]
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    if sin is not None:
        k = rotate(k, sin, cos, np.clip(positions, 0, len(sin) - 1))
    cap = TOP[code] * 2.0 ** EXP[code][1]
    t = 0
    while t < len(slot):
        if slot[t] < 0 or slot[t] // block >= blocks:
            t += 1
            continue
        page, off, n = slot[t] // block, slot[t] % block, 1
        while t + n < len(slot) and off + n < block and slot[t + n] == slot[t] + n:
            n += 1
        for x, codes, scales in ((k, key_codes, key_scales), (v, value_codes.swapaxes(2, 3), value_scales)):
            for h in range(codes.shape[1]):
                new = np.clip(x[t:t + n, h], -cap, cap)
                e = exponent(np.max(np.abs(np.where(np.isnan(new), 0.0, new))), code)
                if off:
                    old = int(np.frexp(scales[page, h])[1]) - 1
                    if e > old:
                        codes[page, h, :off] = nearest(codes[page, h, :off] * 2.0 ** (old - e), code)
                    e = max(e, old)
                scales[page, h] = 2.0 ** e
                codes[page, h, off:off + n, :hd] = nearest(new * 2.0 ** -e, code)
                codes[page, h, off:off + n, hd:] = 0
        t += n


def attention(q, starts, past, new, table, key_codes, value_codes, key_scales, value_scales, max_new, scale=None, sin=None, cos=None, sharp=None):
    """q [rows, heads, hd]; returns (out, bound): the rows that belong to no row of the batch are NaN in both.

    bound: how far a kernel may be off that rounds q after the rotation (2^-11 of each element, if there is one), the weights p (2^-11 of each,
    2^-25 where they are subnormal) and the result (2^-11) to fp16 and sums n terms in fp32: with a = sum p |v| / sum p and d = scale * sum |q k|
    (what the scores' terms add up to)
        |delta s| <= u = d * 2^-11 (rotated) + d * hd * 2^-24 + 2^-21 * (1 + |s|)   (products, sums and exp2's argument in fp32)
        |delta o| <= a * (2 u + 2 * 2^-11 + keys * 2^-23) + keys * 2^-25 * max |v| / sum p + (2^-11 |o| + 2^-25)

    sharp = b: the bound of a kernel that rotates q in fp32 (2^-24 of both products), holds it to b bits (2^-b of each element, 2^-24 at least: the last
    place of an fp16 rest, of a halved query; not rotated: exact) and the weights in fp16 relative to 2^7 or more at the largest (so that a
    subnormal one is off by 2^-32 of it), each key with its own error
        u_j = scale * sum |k_j| * (2^-b |q'| + 2^-24 (|q cos| + |q sin|) + 2^-24) + d_j * 2 hd * 2^-24 + 2^-21 * (1 + |s_j| + max |s|)
        |delta o| <= (sum p_j u_j |v_j - o| + sum (2^-11 p_j + 2^-32) |v_j|) / sum p + a * keys * 2^-24 + 2^-11 |o| + 2^-25
    (a weight's rounding counts in the numerator alone; keys * 2^-25 each for the numerator's sum and the denominator's, of which a lane adds a
    quarter at most; first order: u_j is well below 1)"""
    rows, heads, hd = q.shape
    blocks, kvh, block, _ = key_codes.shape
    out = np.full((rows, heads, hd), np.nan)
    bound = np.full((rows, heads, hd), np.nan)
    scale = hd ** -0.5 if not scale else scale
    for b in range(len(past)):
        n = max(0, min(int(new[b]), max_new, rows - int(starts[b])))
        keys = min(int(past[b]) + n, table.shape[1] * block)
        j = np.arange(keys)
        page = table[b][j // block] if keys else np.zeros(0, np.int64)
        there = (page >= 0) & (page < blocks)
        page = np.where(there, page, 0)
        for i in range(n):
            t = starts[b] + i
            x = np.asarray(q[t], np.float64)
            if sin is not None:
                at = np.array([min(int(past[b]) + i, len(sin) - 1)])
                size = rotate(np.abs(x)[None], np.abs(sin), np.abs(cos), at)[0]
                half = hd // 2
                size[:, :half] += 2 * np.abs(x[:, half:]) * np.abs(np.asarray(sin, np.float64)[at[0], :half])      # |q cos| + |q sin|
                x = rotate(x[None], sin, cos, at)[0]
            seen = there & (j <= past[b] + i)
            for h in range(heads):
                g = h * kvh // heads
                k = key_codes[page, g, j % block][seen][:, :hd] * key_scales[page, g][seen][:, None]
                v = value_codes[page, g, :, j % block][seen][:, :hd] * value_scales[page, g][seen][:, None]
                if len(k) == 0:
                    out[t, h] = bound[t, h] = 0.0
                    continue
                s = scale * (k @ x[h])
                d = scale * (np.abs(k) @ np.abs(x[h]))
                if sharp:
                    p, top = np.exp(s - s.max()), np.abs(s).max()
                    o, n, av = p @ v / p.sum(), len(k), np.abs(v)
                    u = d * hd * 2.0 ** -23 + 2.0 ** -21 * (1 + np.abs(s) + top)
                    if sin is not None:
                        u += scale * (np.abs(k) @ (2.0 ** -sharp * np.abs(x[h]) + 2.0 ** -24 * size[h] + 2.0 ** -24))
                    out[t, h] = o
                    bound[t, h] = (((p * u) @ np.abs(v - o) + (2.0 ** -11 * p + 2.0 ** -32) @ av) / p.sum() + (p @ av / p.sum()) * n * 2.0 ** -24
                                   + 2.0 ** -11 * np.abs(o) + 2.0 ** -25)
                    continue
                u = d.max() * (2.0 ** -11 * (sin is not None) + hd * 2.0 ** -24) + 2.0 ** -21 * (1 + np.abs(s).max())
                p = np.exp(s - s.max())
                out[t, h] = p @ v / p.sum()
                a = p @ np.abs(v) / p.sum()
                bound[t, h] = (a * (2 * u + 2 * 2.0 ** -11 + len(k) * 2.0 ** -23) + len(k) * 2.0 ** -25 * np.abs(v).max() / p.sum()
                               + 2.0 ** -11 * np.abs(out[t, h]) + 2.0 ** -25)
    return out, bound
