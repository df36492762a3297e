"""append_rows on the GPU against the float64 form: blocks and bf16 rows, every layout and refusal."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import abi, kv, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 1e-6


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def table_of(r, slots, pages_each, page, spare=2):
    pages = slots * pages_each + spare
    return r.permutation(pages)[:slots * pages_each].astype(np.int32), pages


def angle_table(keys):
    a = np.arange(keys)[:, None] * 1e4 ** (-np.arange(64) / 64)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def check_codes(got, want, value, scale, exact):
    """Codes against the float64 form's: equal where the value was not computed, else off by the rounding
    of a value that is itself off by the f32 steps before it (sum of squares, root, three products and
    two sums: under 16 halves of 2^-24 of the pair's size, 4 |value| or the block's largest / 448)."""
    if exact:
        assert np.array_equal(got, want)
        return
    v = K.CODES[got] * scale
    half = np.maximum(np.abs(value) * 2.0 ** -4, scale * 2.0 ** -10)
    slack = np.abs(value).max(-1, keepdims=True) * 2 * 2.0 ** -20
    assert np.all(np.abs(v - value) <= half + slack)
    assert np.mean(got != want) < 1e-3


CASES = [
    # (rows of each slot, positions before, heads, kv heads, page)
    ([1], [0], 2, 1, 16),
    ([1, 1, 1], [15, 16, 700], 16, 8, 16),
    ([16], [0], 8, 8, 16),
    ([17, 5, 33], [3, 14, 0], 10, 5, 32),
    ([3, 2, 9, 4], [0, 31, 29, 60], 24, 3, 64),
    ([130, 70], [0, 47], 16, 8, 16),
    ([1100], [9], 4, 2, 64),
    ([1] * 33, list(range(33)), 5, 1, 16),
]


@pytest.mark.parametrize("rows,past,heads,kvh,page", CASES)
@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("norm,turn,halves", [(True, True, True), (False, True, False), (False, False, True)])
def test_blocks(rows, past, heads, kvh, page, x, norm, turn, halves):
    r = rng(sum(rows) + heads + page)
    each = max(-(-(p + n) // page) for p, n in zip(past, rows))
    table, pages = table_of(r, len(rows), each, page)
    keys = each * page
    slots = np.repeat(np.arange(len(rows)), rows).astype(np.int32)
    positions = np.concatenate([p + np.arange(n) for p, n in zip(past, rows)]).astype(np.int32)
    n = len(slots)
    blocks = pages * page // 16
    old = r.integers(0, 256, (2, blocks, kvh, 16, 128)).astype(np.uint8)  # NaN codes too
    scales = np.zeros((blocks, kvh, 2))
    scales[:] = 2.0 ** r.integers(-9, -4, scales.shape)
    even = (kvh + 1) // 2 * 2
    held = np.full((blocks, even, 2), 7.0, np.float32)
    held[:, :kvh] = scales
    qkv = r.standard_normal((n, (heads + 2 * kvh) * 128)).astype(np.float32) * np.exp(r.standard_normal((n, 1)))
    t = dev(qkv.astype(np.float32), torch.float32 if x == "f32" else torch.bfloat16)
    qkv = t.float().cpu().numpy()
    v3 = t.view(n, heads + 2 * kvh, 128)
    gains = [(1 + 0.1 * r.standard_normal(128)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    angles = angle_table(keys) if turn else None
    k8, v8 = dev(old[0]), dev(old[1].transpose(0, 1, 3, 2))
    s8, status = dev(held), torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = rules.append_rows(v3[:, heads:heads + kvh], v3[:, heads + kvh:], k8, v8, dev(slots), dev(positions),
                              q=v3[:, :heads], keys=keys, q_gain=None if not norm else dev(gains[0]),
                              k_gain=None if not norm else dev(gains[1]), angles=None if not turn else dev(angles),
                              halves=halves, eps=EPS, scales=s8, table=dev(table), kept_pages=each, page=page,
                              status=status)
    where = dict(keys=keys, table=table, kept_pages=each, page=page)
    ref = qkv.reshape(n, -1, 128)
    want_q = K.turned(ref[:, :heads], gains[0], angles, positions, halves, EPS)
    got_q = q_out.float().cpu().numpy()
    # f32: norm (2^-24 each for the sum's 8 steps, root, quotient, two products) and the rotation's three.
    size = np.abs(want_q).max(-1, keepdims=True)
    assert np.all(np.abs(got_q - want_q) <= size * 2 * (2.0 ** -20) + (np.abs(want_q) * 2.0 ** -8 if x == "bf16" else 0))
    new = {0: K.turned(ref[:, heads:heads + kvh], gains[1], angles, positions, halves, EPS),
           1: ref[:, heads + kvh:].astype(np.float64)}
    got = {0: k8.cpu().numpy(), 1: v8.cpu().numpy().transpose(0, 1, 3, 2)}
    got_s = s8.cpu().numpy()
    for which in (0, 1):
        want_c, want_s = old[which].copy(), scales.copy()
        K.append(want_c, want_s, which, new[which], slots, positions, **where)
        # A largest value within the f32 error of a border may take the next power of two.
        assert np.array_equal(got_s[:, :kvh, which], want_s[..., which])
        exact = which == 1 or (not norm and not turn)
        rows_at = [K.kept_row(int(s), int(p), **where) for s, p in zip(slots, positions)]
        touched = np.array(rows_at)
        b, o = touched // 16, touched % 16
        check_codes(got[which][b, :, o], want_c[b, :, o], new[which], want_s[b][..., which, None], exact)
        rest = np.ones(want_c.shape[:1] + (16,), bool)
        rest[b, o] = False
        keep = got[which].transpose(0, 2, 1, 3)[rest], want_c.transpose(0, 2, 1, 3)[rest]
        assert np.array_equal(K.CODES[keep[0]], K.CODES[keep[1]], equal_nan=True)
    assert np.array_equal(got_s[:, kvh:], held[:, kvh:]) and int(status) == 0


@pytest.mark.parametrize("rows,norm,turn,halves", [(2050, True, True, True), (2050, True, True, False), (1500, True, False, True),
                                                   (1500, False, True, True), (0, True, True, True)])
def test_codes_are_the_nearest(rows, norm, turn, halves):
    """Codes and scales equal the 64-bit form's: a value is 2^-52 or so off before it is rounded, which none of a
    million comes that near a border of the codes to notice. rows 0: one row each of 900 slots."""
    r = rng(rows + halves)
    kvh, page = 4, 16
    slots, keys = (np.zeros(rows, np.int32), 2064) if rows else (np.arange(900, dtype=np.int32), 32)
    positions = np.arange(rows, dtype=np.int32) if rows else r.integers(0, 32, 900).astype(np.int32)
    n = len(slots)
    x = (r.standard_normal((n, kvh, 128)) * np.exp(2 * r.standard_normal((n, kvh, 1)))).astype(np.float32)
    gain = (1 + 0.1 * r.standard_normal(128)).astype(np.float32) if norm else None
    angles = angle_table(keys) if turn else None
    pages = (int(slots.max()) + 1) * keys // page
    k8, v8, s8 = rules.kept8(pages, kvh, page)
    rules.append_rows(dev(x), dev(x), k8, v8, dev(slots), dev(positions), keys=keys, scales=s8, page=page, halves=halves,
                      k_gain=None if not norm else dev(gain), angles=None if not turn else dev(angles), eps=EPS)
    blocks, scales = np.zeros((pages, kvh, 16, 128), np.uint8), np.zeros((pages, kvh, 2))
    K.append(blocks, scales, 0, K.turned(x, gain, angles, positions, halves, float(np.float32(EPS))), slots, positions, keys=keys)
    assert np.array_equal(s8.cpu().numpy()[:, :, 0], scales[..., 0])
    assert np.array_equal(k8.cpu().numpy(), blocks)


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("halves", [True, False])
def test_bf16_rows_as_the_separate_stages_keep_them(x, halves):
    """With gains and Halves pairs: what qk_norm_rope_append keeps; else the float64 form, rounded."""
    r = rng(7)
    heads, kvh, page, rows, past = 16, 8, 16, [40, 3, 1], [0, 13, 64]
    each = 8
    table, pages = table_of(r, 3, each, page)
    slots = np.repeat(np.arange(3), rows).astype(np.int32)
    positions = np.concatenate([p + np.arange(n) for p, n in zip(past, rows)]).astype(np.int32)
    n = len(slots)
    t = dev(r.standard_normal((n, (heads + 2 * kvh) * 128)).astype(np.float32), torch.float32 if x == "f32" else torch.bfloat16)
    gain = dev((1 + 0.1 * r.standard_normal((2, 128))).astype(np.float32))
    angles = rules.rope_table(each * page, 1e4)
    kept = [torch.full((pages * page, kvh, 128), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    v3 = t.view(n, heads + 2 * kvh, 128)
    args = dict(keys=each * page, table=dev(table), kept_pages=each, page=page)
    q = rules.append_rows(v3[:, heads:heads + kvh], v3[:, heads + kvh:], kept[0], kept[1], dev(slots), dev(positions),
                          q=v3[:, :heads], q_gain=gain[0], k_gain=gain[1], angles=angles, halves=halves, eps=EPS, **args)
    ref = t.float().cpu().numpy().reshape(n, -1, 128)
    g = gain.cpu().numpy()
    where = dict(keys=each * page, table=table, kept_pages=each, page=page)
    at = np.array([K.kept_row(int(s), int(p), **where) for s, p in zip(slots, positions)])
    for got, want in ((kept[0], K.turned(ref[:, heads:heads + kvh], g[1], angles.cpu().numpy(), positions, halves, EPS)),
                      (kept[1], ref[:, heads + kvh:])):
        y = got.float().cpu().numpy()
        size = np.abs(want).max(-1, keepdims=True)
        assert np.all(np.abs(y[at] - want) <= np.abs(want) * 2.0 ** -8 + size * 2.0 ** -19)
        rest = np.ones(len(y), bool)
        rest[at] = False
        assert np.all(y[rest] == 3.0)
    if x == "f32" and halves:
        out = torch.empty(n, heads, 128, device="cuda")
        rules.qk_norm_rope_append(t, gain[0], gain[1], out, kept[2], kept[3], dev(slots), dev(positions), heads=heads,
                                  kv_heads=kvh, eps=EPS, theta=1e4, **args)
        assert torch.equal(q, out) and torch.equal(kept[0], kept[2]) and torch.equal(kept[1], kept[3])


def test_non_finite_values_mark_their_own_codes():
    """Infinities and NaN become NaN codes and leave the scale and every other code as without them."""
    r = rng(8)
    k8, v8, s8 = rules.kept8(2, 2)
    i = torch.arange(16, dtype=torch.int32, device="cuda")
    x = dev(r.standard_normal((16, 2, 128)).astype(np.float32))
    x[:, :, 5] = x[:, :, 5].clamp(-1, 1)
    rules.append_rows(x, x, k8, v8, torch.zeros_like(i), i, keys=32, scales=s8)
    clean = k8.clone(), v8.clone(), s8.clone()
    y = x.clone()
    y[3, 0, 5], y[4, 1, 5], y[5, 0, 5] = float("inf"), float("-inf"), float("nan")
    rules.append_rows(y, y, k8, v8, torch.zeros_like(i), i, keys=32, scales=s8)
    assert torch.equal(s8, clean[2])
    for got, was in ((k8, clean[0]), (v8.transpose(2, 3), clean[1].transpose(2, 3))):
        differ = (got != was).nonzero().cpu().tolist()
        assert sorted(differ) == [[0, 0, 3, 5], [0, 0, 5, 5], [0, 1, 4, 5]]
        assert all((int(got[tuple(d)]) & 0x7F) == 0x7F for d in differ)


@pytest.mark.parametrize("size,e", [(0.0, -100), (1e-38, -100), (448.0, 0), (448.0001, 1), (3e38, 119)])
def test_scales_at_their_bounds(size, e):
    k8, v8, s8 = rules.kept8(1, 1)
    i = torch.arange(16, dtype=torch.int32, device="cuda")
    x = torch.full((16, 1, 128), size, device="cuda")
    rules.append_rows(x, -x, k8, v8, torch.zeros_like(i), i, keys=16, scales=s8)
    assert s8[0, 0].tolist() == [2.0 ** e] * 2
    want = int(K.narrow(min(size / 2.0 ** e, 448.0)))
    assert torch.all(k8 == want) and torch.all((v8 & 0x7F) == want)


def test_scales_grow_and_begin_anew():
    """One position at a time: a wider row moves the codes there to its scale; position 0 forgets them."""
    k8, v8, s8 = rules.kept8(1, 1)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    want_c, want_s = np.zeros((1, 1, 16, 128), np.uint8), np.zeros((1, 1, 2))
    r = rng(9)
    for pos, size in ((0, 1.0), (1, 0.5), (2, 300.0), (3, 1e6), (4, 1.0), (0, 1e-3), (1, 2.0)):
        x = (r.standard_normal((1, 1, 128)) * size).astype(np.float32)
        rules.append_rows(dev(x), dev(x), k8, v8, slot, torch.full_like(slot, pos), keys=16, scales=s8)
        K.append(want_c, want_s, 0, x.astype(np.float64), [0], [pos], keys=16)
        assert s8[0, 0, 0].item() == want_s[0, 0, 0] == s8[0, 0, 1].item()
        assert np.array_equal(k8.cpu().numpy(), want_c)
        assert np.array_equal(v8.cpu().numpy().transpose(0, 1, 3, 2), want_c)


def test_refused_rows_are_kept_nowhere():
    """Positions and slots out of range, bad pages, a block met twice: their status bits, nothing written,
    the rows beside them as alone."""
    r = rng(10)
    page, each, kvh, heads = 16, 3, 2, 4
    table = np.array([0, 1, 2, 3, 99, 5], np.int32)  # slot 1's second page does not exist
    x = r.standard_normal((9, heads + 2 * kvh, 128)).astype(np.float32)
    slots = np.array([0, 0, 1, 2, 0, 0, 0, 1, 0], np.int32)
    positions = np.array([46, 47, 17, 3, 48, 4, 5, 40, 4], np.int32)  # row 4: past the slot; row 8: as row 5
    bits = {2: abi.TS_STATUS_PAGE, 3: abi.TS_STATUS_PAGE, 4: abi.TS_STATUS_POSITION, 8: abi.TS_STATUS_TWICE}

    def run(rows):
        k8, v8, s8 = rules.kept8(6, kvh)
        k8.fill_(1)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        t = dev(x[rows])
        q = rules.append_rows(t[:, heads:heads + kvh], t[:, heads + kvh:], k8, v8, dev(slots[rows]), dev(positions[rows]),
                              q=t[:, :heads], keys=48, scales=s8, table=dev(table), kept_pages=each, page=page,
                              status=status)
        return k8, v8, s8, q, int(status)

    good = run([0, 1, 5, 6, 7])
    assert good[4] == 0
    for bad, bit in bits.items():
        rows = sorted([0, 1, 5, 6, 7, bad])
        got = run(rows)
        assert got[4] == bit
        assert all(torch.equal(a, b) for a, b in zip(got[:3], good[:3]))
        if bad == 4:
            assert torch.isnan(got[3][rows.index(4)]).all() and not torch.isnan(got[3][rows.index(5)]).any()
    assert run(list(range(9)))[4] == sum(set(bits.values()))


def test_in_place_q_other_streams_and_one_row_views():
    """q rotated in place; a call on another stream than the tensors' own; rows of a transposed buffer."""
    r = rng(11)
    heads, kvh, n = 6, 3, 5
    q, k = (dev(r.standard_normal((n, h, 128)).astype(np.float32)) for h in (heads, kvh))
    i = torch.arange(n, dtype=torch.int32, device="cuda")
    angles = rules.rope_table(16, 1e4)
    want = rules.kept8(1, kvh)
    out = rules.append_rows(k, k, want[0], want[1], torch.zeros_like(i), i, q=q, angles=angles, keys=16, scales=want[2])
    got = rules.kept8(1, kvh)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        same = rules.append_rows(k, k, got[0], got[1], torch.zeros_like(i), i, q=q, q_out=q, angles=angles, keys=16,
                                 scales=got[2])
    side.synchronize()
    assert same is q and torch.equal(q, out) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_pages_copy_whole():
    """Kept blocks' pages through the page copies: codes and scales."""
    r = rng(12)
    k8, v8, s8 = rules.kept8(4, 3, page=32)
    for t in (k8, v8):
        t.copy_(dev(r.integers(0, 255, tuple(t.shape)).astype(np.uint8)))
    s8.copy_(dev(r.random(tuple(s8.shape)).astype(np.float32)))
    was = [t.clone() for t in (k8, v8, s8)]
    kv.copy_kept8(k8, v8, s8, [(0, 3, 20), (2, 1, 32)], page=32)
    for t, w in zip((k8, v8, s8), was):
        t, w = t.view(4, 2, -1), w.view(4, 2, -1)
        assert torch.equal(t[3], w[0]) and torch.equal(t[1], w[2]) and torch.equal(t[0], w[0]) and torch.equal(t[2], w[2])
