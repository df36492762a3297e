"""Kept blocks, their attention and the verification of drafts, plainly in float64 (numpy)."""
import numpy as np

BLOCK, D, TOP = 16, 128, 448.0

# Every e4m3fn code's value.
_c = np.arange(256)
_e, _m = (_c >> 3) & 15, _c & 7
CODES = np.where(_e == 0, _m / 8 * 2.0 ** -6, (1 + _m / 8) * 2.0 ** (_e.astype(float) - 7)) * np.where(_c & 128, -1.0, 1.0)
CODES[[0x7F, 0xFF]] = np.nan


def narrow(y):
    """The codes nearest to y (|y| <= 448 after clamping), ties to even, NaN for what is not finite."""
    y = np.asarray(y, np.float64)
    a = np.minimum(np.abs(np.where(np.isfinite(y), y, 0)), TOP)
    e = np.where(a > 0, np.maximum(np.frexp(a)[1] - 1, -6), -6)
    q = np.rint(a / 2.0 ** (e - 3)).astype(np.int64)  # 8..16 of a normal, 0..8 of a subnormal
    code = q + (e + 6) * 8  # a carry out of the mantissa (16, or 8 of a subnormal) steps the exponent
    code = np.where(np.signbit(y), code | 128, code)
    return np.where(np.isfinite(y), code, np.where(np.signbit(y), 0xFF, 0x7F)).astype(np.uint8)


def exponent(amax):
    """The least e with amax <= 448 * 2^e, of -100 .. 119."""
    if amax == 0:
        return -100
    e = int(np.ceil(np.log2(amax / TOP)))
    while amax <= TOP * 2.0 ** (e - 1):
        e -= 1
    while amax > TOP * 2.0 ** e:
        e += 1
    return min(max(e, -100), 119)


def turned(x, gain, angles, positions, halves, eps):
    """x [rows, heads, 128] through RmsNorm and the rotation by table rows [.., 64, 2]."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gain, np.float64)
    if angles is None:
        return x
    c, s = (np.asarray(angles, np.float64)[positions][:, None, :, i] for i in (0, 1))
    out = np.empty_like(x)
    a, b = (x[..., :64], x[..., 64:]) if halves else (x[..., 0::2], x[..., 1::2])
    y, z = a * c - b * s, a * s + b * c
    if halves:
        out[..., :64], out[..., 64:] = y, z
    else:
        out[..., 0::2], out[..., 1::2] = y, z
    return out


def kept_row(slot, pos, *, keys, table=None, kept_pages=0, page=16):
    """The kept row of a position (a block's 16 rows are consecutive)."""
    return slot * keys + pos if table is None else int(table[slot * kept_pages + pos // page]) * page + pos % page


def append(blocks, scales, which, new, slots, positions, skip=(), **where):
    """New rows [rows, kv, 128] into blocks [blocks, kv, 16, 128] of codes (K's layout) and their scales
    [blocks, kv, 2] at `which`, in place. Rows in `skip` are refused."""
    groups = {}
    for r in range(len(slots)):
        if r not in skip:
            row = kept_row(int(slots[r]), int(positions[r]), **where)
            groups.setdefault(row // BLOCK, []).append((row % BLOCK, r))
    for b, rows in groups.items():
        for h in range(new.shape[1]):
            x = {o: new[r, h] for o, r in rows}
            amax = max(float(np.max(np.abs(v), initial=0, where=np.isfinite(v))) for v in x.values())
            e = exponent(amax)
            if 0 not in x:
                was = int(np.log2(scales[b, h, which])) if scales[b, h, which] > 0 else -100
                e = max(e, min(max(was, -100), 119))
                for o in range(BLOCK):
                    if o not in x and e > was:
                        held = blocks[b, h, o]
                        blocks[b, h, o] = np.where(np.isnan(CODES[held]), held, narrow(CODES[held] * 2.0 ** (max(was, -100) - e)))
            for o, v in x.items():
                blocks[b, h, o] = narrow(np.where(np.isfinite(v), v / 2.0 ** e, v))
            scales[b, h, which] = 2.0 ** e


def attend(q, k, v, scales, slots, positions, *, scale, back=None, **where):
    """out [rows, heads, 128] and, per (row, head), the largest sum of |q_i k_i| * scale and the largest
    |v| among its keys. k [blocks, kv, 16, 128], v [blocks, kv, 128, 16] codes."""
    rows, heads, _ = q.shape
    kv = k.shape[1]
    group = heads // kv
    out = np.zeros((rows, heads, D))
    spread, size = np.zeros((rows, heads)), np.zeros((rows, heads))
    at = {}
    for r in range(rows):
        s, p = int(slots[r]), int(positions[r])
        lo = 0 if back is None else max(0, p - back)
        for j in range(lo, p + 1):
            if (s, j) not in at:
                at[s, j] = kept_row(s, j, **where)
        held = np.array([at[s, j] for j in range(lo, p + 1)])
        b, o = held // BLOCK, held % BLOCK
        kk = CODES[k[b, :, o]] * scales[b, :kv, 0, None]  # [keys, kv, 128]
        vv = CODES[v[b, :, :, o]] * scales[b, :kv, 1, None]
        for h in range(heads):
            x = kk[:, h // group] @ q[r, h].astype(np.float64) * scale
            spread[r, h] = np.max(np.abs(kk[:, h // group]) @ np.abs(q[r, h]).astype(np.float64)) * abs(scale)
            size[r, h] = np.max(np.abs(vv[:, h // group]))
            w = np.exp(x - x.max())
            out[r, h] = (w / w.sum()) @ vv[:, h // group]
    return out, spread, size


def verify(logits, drafts, uniforms=None, *, counts=None, first=None, probs=None, temperature=1.0):
    """(tokens, accepted) of include/tessera_hip.h's tessera_hip_verify, a sequence at a time."""
    seqs, most = drafts.shape
    rows, width = logits.shape
    tokens, accepted = np.full((seqs, most + 1), width), np.zeros(seqs, int)
    for s in range(seqs):
        n = most if counts is None else int(counts[s])
        at = s * (most + 1) if first is None else int(first[s])
        if n > most or at + n >= rows:
            continue
        temp = float(np.asarray(temperature, np.float32).reshape(-1)[s if np.ndim(temperature) else 0])
        greedy = uniforms is None or not temp > 0

        def spread(t):
            x = logits[at + t].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            best = int(np.argmax(x)) if x.max() > -np.inf else width
            e = np.where(x == x.max(), 1.0, np.exp(np.where(x == x.max(), 0, x - x.max()) / (temp if temp > 0 else 1.0))) \
                if best < width else np.zeros(width)
            return e, best

        for t in range(n + 1):
            e, best = spread(t)
            z = e.sum()
            if t == n:
                w = e
            else:
                d = int(drafts[s, t])
                d = d if 0 <= d < width else width
                if greedy:
                    take = d == best < width
                else:
                    chance = 1.0 if probs is None else float(probs[s, t, d]) if d < width else 0.0
                    chance = chance if chance > 0 else 0.0
                    take = d < width and float(uniforms[s, t]) * chance * z < e[d]
                if take:
                    tokens[s, t] = d
                    continue
                if probs is None:
                    w = np.where(np.arange(width) == d, 0, e)
                else:
                    q = probs[s, t].astype(np.float64)
                    w = np.maximum(e - np.where(q > 0, q, 0) * z, 0)
                if not w.sum() > 0:
                    w = e
            accepted[s] = t
            if greedy:
                tokens[s, t] = best
            elif w.sum() > 0:
                upto = np.cumsum(w)
                over = np.nonzero((upto > float(uniforms[s, most]) * upto[-1]) & (w > 0))[0]
                tokens[s, t] = over[0] if len(over) else np.nonzero(w > 0)[0][-1]
            break
    return tokens, accepted
