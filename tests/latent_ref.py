"""Latent attention plainly in float64 (numpy): appends, products a head, the absorbed and the expanded form."""
import numpy as np


def kept_row(slot, pos, *, keys, table=None, kept_pages=0, page=16):
    """The kept row of a position."""
    return slot * keys + pos if table is None else int(table[slot * kept_pages + pos // page]) * page + pos % page


def turned(x, angles, halves):
    """x [..., rope] rotated by angles [..., rope / 2, 2], and the size of each pair (|a| + |b|)."""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    out, size = np.empty_like(x), np.empty_like(x)
    first, second = (slice(0, half), slice(half, None)) if halves else (slice(0, None, 2), slice(1, None, 2))
    a, b = x[..., first], x[..., second]
    c, s = np.asarray(angles, np.float64)[..., 0], np.asarray(angles, np.float64)[..., 1]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return out, size


def normed(x, gain, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gain, np.float64)


def attend(q, kept, slots, positions, *, rank, scale, back=None, **where):
    """(out, sum of w |v|, the largest error unit of a row's scores: sum |q| |row| |scale|) of each row and head; kept
    rows that a row does not see are not looked at."""
    q = np.asarray(q, np.float64)
    out, size = (np.zeros((*q.shape[:2], rank)) for _ in range(2))
    spread = np.zeros(q.shape[:2])
    for r, (slot, pos) in enumerate(zip(slots, positions)):
        lo = 0 if back is None else max(0, int(pos) - back)
        rows = np.array([kept_row(int(slot), j, **where) for j in range(lo, int(pos) + 1)])
        k = np.asarray(kept[rows], np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            x = q[r] @ k.T * scale
            w = np.exp(x - x.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[r] = w @ k[:, :rank]
            size[r] = w @ np.abs(k[:, :rank])
            spread[r] = (np.abs(q[r]) @ np.abs(k).T).max(-1) * abs(scale)
    return out, size, spread


def flash(q, k, v, r, *, scale, first, key_first, back=None):
    """The same of whole sequences; None where no sequence has the row."""
    q, k, v, r = (np.asarray(x, np.float64) for x in (q, k, v, r))
    heads, nope = k.shape[1:]
    out, size = (np.full((*q.shape[:2], v.shape[-1]), np.nan) for _ in range(2))
    spread = np.zeros(q.shape[:2])
    for a, b, ka, kb in zip(first[:-1], first[1:], key_first[:-1], key_first[1:]):
        for i in range(a, b):
            pos = (kb - ka) - (b - a) + i - a
            lo = 0 if back is None else max(0, pos - back)
            if pos < 0:
                out[i] = size[i] = 0
                continue
            for h in range(heads):
                rows = np.concatenate([k[ka + lo:ka + pos + 1, h], r[ka + lo:ka + pos + 1]], -1)
                with np.errstate(invalid="ignore", over="ignore"):
                    x = rows @ q[i, h] * scale
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    vv = v[ka + lo:ka + pos + 1, h]
                    out[i, h], size[i, h] = w @ vv, w @ np.abs(vv)
                    spread[i, h] = (np.abs(rows) @ np.abs(q[i, h])).max() * abs(scale)
    return out, size, spread


def bound(out, size, spread, steps, weight):
    """How far an output may be off. A score's products are exact and `steps` accumulating ones round at 2^-21 each, so a
    score is off by spread * steps * 2^-21 at most; a weight by twice that (its own and the sum's), 2^-20 of the
    exponential and the sums, and `weight`, the rounding of weights to their parts; an output by that times the sum of w
    |v|, 2^-21 a step of its own sum over the keys (taken together as 2^-14: up to 128 steps), and its rounding to bf16,
    half a step 2^-8."""
    return (2 * spread[..., None] * steps * 2.0 ** -21 + 2.0 ** -20 + weight + 2.0 ** -14) * size + 2.0 ** -8 * np.abs(out)
