"""append_latent, linear_heads, attend_latent and flash_latent on the GPU against the float64 forms."""
import numpy as np
import pytest

import latent_ref as L
from helpers import rng
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
WIDTHS = {"wide": (512, 64, 128, 128), "narrow": (256, 32, 64, 64)}  # rank, rope, nope, value
HALF = 2.0 ** -8  # of a bf16 step, relative


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def ints(a):
    return dev(np.asarray(a).astype(np.uint32).view(np.int32))


def f64(t):
    return t.double().cpu().numpy()


# --- append -------------------------------------------------------------------------------------

def check_append(c, q, out, kept, before, slots, positions, where, *, rank, gain, angles, halves, eps, bad, dense):
    """A value of the latent: the sum of squares (rank steps), the root and two products, each f32: (rank + 8) 2^-24 of
    it at most; of the rotation: three f32 roundings of the pair, 3 2^-24 (|a| + |b|); then half a step of bf16."""
    cc, n = f64(c), c.shape[0]
    at = np.where(bad, 0, positions)
    latent = cc[:, :rank] if gain is None else L.normed(cc[:, :rank], f64(gain), eps)
    turn = f64(angles)[at] if angles is not None else None
    part, size = (cc[:, rank:], 0) if angles is None else L.turned(cc[:, rank:], turn, halves)
    row = np.concatenate([latent, part], -1)
    slack = np.concatenate([np.abs(latent) * (rank + 8) * 2.0 ** -24, np.broadcast_to(size * 3 * 2.0 ** -24, part.shape)], -1)
    want = f64(before)
    limit = np.zeros_like(want)
    for i in range(n):
        if not bad[i]:
            w = L.kept_row(int(slots[i]), int(positions[i]), **where)
            want[w], limit[w] = row[i], slack[i] + np.abs(row[i]) * HALF
    got = f64(kept)
    assert np.all(np.abs(got - want) <= limit)
    if dense is not None:
        got = np.concatenate([f64(dense[0]), f64(dense[1])], -1)
        assert np.isnan(got[bad]).all()
        assert np.all((np.abs(got - row) <= slack + np.abs(row) * HALF)[~bad])
    if q is not None:
        want, size = (f64(q), 0) if angles is None else L.turned(f64(q), turn[:, None], halves)
        got = f64(out)
        assert np.isnan(got[bad]).all()
        limit = np.broadcast_to(size * 3 * 2.0 ** -24, want.shape) + np.abs(want) * (HALF if out.dtype == BF16 else 0)
        assert np.all((np.abs(got - want) <= limit)[~bad])


@pytest.mark.parametrize("rank,rope,heads", [(512, 64, 16), (512, 64, 128), (256, 32, 5), (8, 16, 1), (1024, 128, 3), (520, 64, 9)])
@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("form", ["decode", "prompt", "dense table", "bare"])
def test_append(rank, rope, heads, x, halves, form):
    r = rng(rank + heads)
    page, each, seqs = 32, 4, 5
    where = dict(keys=each * page, table=r.permutation(seqs * each).astype(np.int32), kept_pages=each, page=page)
    slots, positions = np.arange(seqs), r.integers(0, each * page, seqs)
    if form == "prompt":
        slots, positions = np.repeat([3, 0], [50, 37]), np.concatenate([np.arange(50) + 11, np.arange(37)])
    if form == "dense table":
        where = dict(keys=100)
        positions = positions % 100
    n = len(slots)
    wide = dev(r.standard_normal((n, rank + rope + 24)), x)
    c = wide[:, :rank + rope] if form != "bare" else wide[:, :rank + rope].contiguous()
    q = dev(r.standard_normal((n, heads, 40 + rope)), x)[..., 40:]
    out = torch.zeros(n, heads, rank + rope, dtype=BF16 if halves else F32, device="cuda")[..., rank:]
    gain = None if form == "bare" else dev(1 + 0.1 * r.standard_normal(rank), F32)
    angles = None if form == "bare" else rules.rope_table(130, 1e4, width=rope)
    kept = dev(r.standard_normal((seqs * each * page, rank + rope)), BF16)
    before = kept.clone()
    dense = None if form == "decode" else (torch.zeros(n, rank, dtype=BF16, device="cuda"),
                                           torch.zeros(n, rope, dtype=BF16, device="cuda"))
    kw = dict(where)
    if "table" in kw:
        kw["table"] = dev(kw["table"])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = rules.append_latent(c, kept, ints(slots), ints(positions), rank=rank, gain=gain, angles=angles, halves=halves,
                              eps=1e-5, q=q, q_out=out if form != "bare" else None, status=status,
                              c_out=dense and dense[0], r_out=dense and dense[1], **kw)
    assert int(status) == 0 and (form == "bare" or got.data_ptr() == out.data_ptr())
    check_append(c, q, got, kept, before, slots, positions, where, rank=rank, gain=gain, angles=angles, halves=halves,
                 eps=1e-5, bad=np.zeros(n, bool), dense=dense)
    if form != "bare":  # the absorbed part beside the rotated one is not touched
        assert int(out._base[..., :rank].count_nonzero()) == 0


@pytest.mark.parametrize("x", [F32, BF16])
def test_append_of_rows_without_a_place(x):
    """Positions past the slot or its table's pages, slots and pages that are not there."""
    r = rng(5)
    page, each, rank, rope, heads = 16, 3, 256, 32, 3
    table = np.array([0, 1, 2, 3, 99, 5], np.int32)  # slot 1's second page does not exist
    slots = np.array([0, 0, 1, 2, 0, 0, 1, 0xFFFFFFFF, 1], np.uint32)
    positions = np.array([46, 47, 17, 3, 48, 0xFFFFFFFF, 40, 3, 3], np.uint32)
    bad = np.array([0, 0, 1, 1, 1, 1, 0, 1, 0], bool)
    n = len(slots)
    c, q = dev(r.standard_normal((n, rank + rope)), x), dev(r.standard_normal((n, heads, rope)), x)
    kept = dev(r.standard_normal((6 * page, rank + rope)), BF16)
    before = kept.clone()
    angles, gain = rules.rope_table(64, 1e4, width=rope), dev(np.ones(rank), F32)
    dense = torch.zeros(n, rank, dtype=BF16, device="cuda"), torch.zeros(n, rope, dtype=BF16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = rules.append_latent(c, kept, ints(slots), ints(positions), keys=64, rank=rank, gain=gain, angles=angles, q=q,
                              c_out=dense[0], r_out=dense[1], table=dev(table), kept_pages=each, page=page, status=status)
    assert int(status) == abi.TS_STATUS_POSITION | abi.TS_STATUS_PAGE
    check_append(c, q, out, kept, before, slots, positions, dict(keys=64, table=table, kept_pages=each, page=page), rank=rank,
                 gain=gain, angles=angles, halves=True, eps=1e-6, bad=bad, dense=dense)
    for rows, bit in (([2], abi.TS_STATUS_PAGE), ([3], abi.TS_STATUS_PAGE), ([4], abi.TS_STATUS_POSITION)):
        status.zero_()
        rules.append_latent(c[rows], kept, ints(slots[rows]), ints(positions[rows]), keys=64, rank=rank, table=dev(table),
                            kept_pages=each, page=page, status=status)
        assert int(status) == bit


@pytest.mark.parametrize("halves", [True, False])
def test_append_in_place_and_not_finite(halves):
    """q rotated where it lies; infinities and NaN stay in their pair or row, and the rows beside them are as ever."""
    r = rng(6)
    n, rank, rope, heads = 9, 512, 64, 4
    c, q = dev(r.standard_normal((n, rank + rope)), BF16), dev(r.standard_normal((n, heads, 128 + rope)), BF16)
    angles, gain = rules.rope_table(32, 1e4, width=rope), dev(np.ones(rank), F32)
    i = torch.arange(n, dtype=torch.int32, device="cuda")
    kw = dict(keys=32, rank=rank, gain=gain, angles=angles, halves=halves)
    kept, clean = (torch.zeros(32, rank + rope, dtype=BF16, device="cuda") for _ in range(2))
    want = rules.append_latent(c, clean, torch.zeros_like(i), i, q=q[..., 128:], **kw)
    part = q[..., 128:]
    front = q[..., :128].clone()
    got = rules.append_latent(c, kept, torch.zeros_like(i), i, q=part, q_out=part, **kw)
    assert got.data_ptr() == part.data_ptr() and torch.equal(got, want) and torch.equal(q[..., :128], front)
    c[2, 7], c[4, rank + 3], c[5, rank + 1] = float("nan"), float("inf"), float("nan")
    rules.append_latent(c, kept, torch.zeros_like(i), i, **kw)
    same = torch.ones_like(kept, dtype=torch.bool)
    same[2, :rank] = False
    for row, at in ((4, 3), (5, 1)):
        same[row, rank + at] = False
        same[row, rank + ((at + 32) % 64 if halves else at ^ 1)] = False
    assert torch.equal(kept[same], clean[same]) and not torch.isfinite(kept[~same]).any()


# --- products a head ------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,heads,n,k", [(1, 16, 512, 128), (1, 1, 1, 8), (33, 5, 130, 72), (64, 3, 128, 512), (65, 4, 31, 24),
                                            (200, 2, 33, 640), (7, 128, 64, 256), (31, 3, 7, 136), (129, 1, 256, 64)])
@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("out", [F32, BF16])
def test_linear_heads(rows, heads, n, k, x, out):
    """An output's k products are exact and summed at 2^-21 a step of 16 (three times as many of f32 x, whose three parts
    drop 2^-24), all of the sum of |x w|; then half a step of bf16."""
    r = rng(rows + n + k)
    gap = 8 if (rows + n) % 2 else 0
    xs = dev(r.standard_normal((rows, heads, k + gap)), x)[..., :k]
    w = dev(r.standard_normal((heads, n + 3, k)) / 8, BF16)[:, 2:n + 2] if heads > 1 else dev(r.standard_normal((1, n, k)) / 8, BF16)
    held = torch.full((rows, heads, n + gap), 7.0, dtype=out, device="cuda")
    got = rules.linear_heads(xs, w, out=held[..., :n]) if gap else rules.linear_heads(xs, w, out_dtype=out)
    a, b = f64(xs), f64(w)
    want, size = np.einsum("rhk,hnk->rhn", a, b), np.einsum("rhk,hnk->rhn", np.abs(a), np.abs(b))
    steps = (k / 16 + 1) * (3 if x == F32 else 1)
    limit = size * (steps * 2.0 ** -21 + 2.0 ** -24) + (HALF * np.abs(want) if out == BF16 else 0)
    assert got.dtype == out and np.all(np.abs(f64(got) - want) <= limit)
    assert not gap or bool((held[..., n:] == 7.0).all())


@pytest.mark.parametrize("rows,heads,n,k", [(1100, 128, 40, 72), (130, 520, 130, 136), (4100, 16, 200, 320)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_linear_heads_of_many_rows(rows, heads, n, k, out):
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(rows, heads, k, generator=g, device="cuda").to(BF16)
    w = torch.randn(heads, n, k, generator=g, device="cuda").to(BF16)
    got = rules.linear_heads(x, w, out_dtype=out).double()
    xd, wd = x.double().transpose(0, 1).contiguous(), w.double().transpose(1, 2).contiguous()
    want = torch.bmm(xd, wd).transpose(0, 1)
    size = torch.bmm(xd.abs(), wd.abs()).transpose(0, 1)
    # k / 16 accumulating products and one more rounding, 2^-21 each, and bf16's half step.
    limit = (k / 16 + 1) * 2.0 ** -21 * size + (HALF * want.abs() if out is BF16 else 0)
    assert bool(((got - want).abs() <= limit).all())


@pytest.mark.parametrize("x", [F32, BF16])
def test_linear_heads_not_finite_and_layouts(x):
    """An infinity or NaN reaches its row alone (f32 ones too, though they enter in parts); heads may lie outside rows."""
    r = rng(8)
    xs, w = dev(r.standard_normal((40, 3, 64)), x), dev(np.abs(r.standard_normal((3, 48, 64))) + 0.1, BF16)
    want = rules.linear_heads(xs, w)
    xs[3, 1, 5], xs[39, 2, 63] = float("inf"), float("nan")
    got = rules.linear_heads(xs, w)
    assert bool((got[3, 1] == float("inf")).all()) and bool(torch.isnan(got[39, 2]).all())
    mask = torch.ones_like(got, dtype=torch.bool)
    mask[3, 1] = mask[39, 2] = False
    assert torch.equal(got[mask], want[mask])
    turned = xs.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty(3, 40, 48, device="cuda").transpose(0, 1)
    assert torch.equal(rules.linear_heads(turned, w, out=out).nan_to_num(5.0), got.nan_to_num(5.0))


# --- the absorbed form ----------------------------------------------------------------------------

def cache(r, lengths, width, page, dense=False, wild=True):
    """Kept rows of random values for slots of `lengths` positions; everything past them is NaN, or infinite."""
    each = max(1, -(-max(lengths) // page))
    pages = len(lengths) * each + (0 if dense else 2)
    table = r.permutation(pages).astype(np.int32)[:len(lengths) * each]
    where = dict(keys=each * page) if dense else dict(keys=each * page, table=table, kept_pages=each, page=page)
    kept = np.where(r.random((pages * page, 1)) < 0.5, np.nan, np.inf) * np.ones(width) if wild else np.zeros((pages * page, width))
    for s, n in enumerate(lengths):
        for j in range(n):
            kept[L.kept_row(s, j, **where)] = r.standard_normal(width)
    return dev(kept, BF16), where


def attend(q, kept, slots, positions, where, rank, **kw):
    args = dict(where)
    if "table" in args:
        args["table"] = dev(args["table"])
    return rules.attend_latent(q, kept, ints(slots), ints(positions), rank=rank, **args, **kw)


def check_attend(got, q, kept, slots, positions, where, *, rank, scale, back=None, one_part=True):
    out, size, spread = L.attend(f64(q), f64(kept), slots, positions, rank=rank, scale=scale, back=back, **where)
    limit = L.bound(out, size, spread, q.shape[-1] / 32 + 1, HALF if one_part else 2.0 ** -16)
    with np.errstate(invalid="ignore"):
        assert np.all(np.abs(f64(got) - out) <= limit), np.nanmax(np.abs(f64(got) - out) / limit)


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads", [1, 5, 16, 17, 32, 40, 64, 100, 128, 150])
@pytest.mark.parametrize("lengths", [[1], [2, 33, 31, 32, 64, 65], [700, 1, 300, 129]])
@pytest.mark.parametrize("dense", [False, True])
def test_decode_rows(widths, heads, lengths, dense):
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(heads + len(lengths))
    page = 16 if heads % 2 else 64
    kept, where = cache(r, lengths, rank + rope, page, dense)
    q = dev(r.standard_normal((len(lengths), heads, rank + rope)), BF16)
    slots, positions = np.arange(len(lengths)), np.array(lengths) - 1
    kw = dict(rank=rank, scale=(nope + rope) ** -0.5)
    got = attend(q, kept, slots, positions, where, **kw)
    check_attend(got, q, kept, slots, positions, where, **kw)
    assert torch.equal(got, attend(q, kept, slots, positions, where, **kw))  # the same call, the same bits


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads,run", [(16, 5), (32, 5), (2, 9), (16, 40), (5, 70), (128, 3), (8, 2), (1, 16)])
@pytest.mark.parametrize("back", [None, 0, 20, 500])
@pytest.mark.parametrize("hint", [1, 0])
def test_rows_that_stand_together(widths, heads, run, back, hint):
    """Drafted rows and chunks of ragged sequences, with and without a window, whatever `run` says of them."""
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(heads * run)
    counts = r.integers(1, run + 1, 5)
    lengths = counts + r.integers(0, 400, 5)
    kept, where = cache(r, list(lengths), rank + rope, 32)
    slots = np.repeat(r.permutation(5), counts)
    at = {s: lengths[s] - c for s, c in zip(range(5), counts)}
    positions, seen = [], {}
    lengths_of = dict(enumerate(lengths))
    for s in slots:
        seen[s] = seen.get(s, 0) + 1
    done = {}
    for s in slots:
        done[s] = done.get(s, 0) + 1
        positions.append(max(0, lengths_of[s] - seen[s]) + done[s] - 1)
    positions = np.minimum(np.array(positions), np.array([lengths_of[s] - 1 for s in slots]))
    q = dev(r.standard_normal((len(slots), heads, rank + rope)), BF16)
    kw = dict(rank=rank, scale=(nope + rope) ** -0.5, **({} if back is None else {"back": back}))
    got = attend(q, kept, slots, positions, where, run=run if hint else 3, max_position=int(max(positions)), **kw)
    check_attend(got, q, kept, slots, positions, where, **kw)


@pytest.mark.parametrize("heads,run", [(16, 1), (16, 6), (32, 1), (100, 2)])
def test_any_order_of_rows(heads, run):
    """Rows of many slots in any order, some twice, tiles of several slots."""
    r = rng(heads + run)
    rank, rope = 512, 64
    lengths = list(r.integers(1, 200, 9))
    kept, where = cache(r, lengths, rank + rope, 16)
    slots = r.integers(0, 9, 31)
    positions = np.array([r.integers(0, lengths[s]) for s in slots])
    q = dev(r.standard_normal((31, heads, rank + rope)), BF16)
    got = attend(q, kept, slots, positions, where, rank=rank, scale=0.07, run=run)
    check_attend(got, q, kept, slots, positions, where, rank=rank, scale=0.07)


@pytest.mark.parametrize("widths,heads,seqs,run", [("wide", 16, 300, 1), ("wide", 2, 1100, 1), ("narrow", 64, 600, 1),
                                                   ("wide", 128, 270, 1), ("narrow", 16, 150, 3), ("wide", 16, 3, 120)])
def test_many_tiles(widths, heads, seqs, run):
    """More tiles than groups run at once, than share their keys, and tiles of many groups."""
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(seqs)
    lengths = list(r.integers(run, run + 150, seqs))
    lengths[seqs // 2] = 1500
    kept, where = cache(r, lengths, rank + rope, 16, wild=False)
    slots = np.repeat(np.arange(seqs), run)
    positions = np.concatenate([n - run + np.arange(run) for n in lengths])
    q = dev(r.standard_normal((len(slots), heads, rank + rope)), BF16)
    got = attend(q, kept, slots, positions, where, rank=rank, scale=0.07, run=run)
    few = r.choice(len(slots), 60, replace=False)
    few[0] = seqs // 2 * run
    check_attend(got[dev(few)], q[dev(few)], kept, slots[few], positions[few], where, rank=rank, scale=0.07)


@pytest.mark.parametrize("heads,run", [(16, 1), (4, 4), (32, 4), (128, 1)])
@pytest.mark.parametrize("scale", [0.0, -0.05, 3.0])
def test_scales(heads, run, scale):
    """No scale (every key alike), a negative one, and one that leaves a single key."""
    r = rng(heads)
    rank, rope = 512, 64
    kept, where = cache(r, [90], rank + rope, 16)
    slots, positions = np.zeros(run, int), 90 - run + np.arange(run)
    q = dev(r.standard_normal((run, heads, rank + rope)), BF16)
    got = attend(q, kept, slots, positions, where, rank=rank, scale=scale, run=run)
    check_attend(got, q, kept, slots, positions, where, rank=rank, scale=scale)


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads,run", [(16, 5), (4, 4), (3, 7), (32, 3), (16, 30), (128, 2)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_not_finite_in_masked_places(widths, heads, run, value):
    """A value that is not finite in a row's key reaches the rows that see it, and only its own d of them; rows before it
    (and behind a window) are as without it."""
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(heads + run)
    kept, where = cache(r, [120 + run, 60], rank + rope, 16)
    slots = np.concatenate([np.zeros(run, int), [1]])
    positions = np.concatenate([120 + np.arange(run), [59]])
    # A latent's value that q does not look at (its own q value is 0), so that scores stay finite.
    d = 37
    q = r.standard_normal((run + 1, heads, rank + rope))
    q[..., d] = 0
    q = dev(q, BF16)
    kw = dict(rank=rank, scale=0.05, run=run, back=100)
    want = attend(q, kept, slots, positions, where, **kw)
    # One key that the first row alone sees, before the others' windows, and one that only the last does.
    for key, sees in ((20, positions - 100 <= 20), (120 + run - 1, positions == 120 + run - 1)):
        sees = sees & (slots == 0)
        x = kept.clone()
        x[L.kept_row(0, key, **where), d] = value
        got = attend(q, x, slots, positions, where, **kw)
        # (0 times infinity: the key's score is NaN, and with it all of the row.)
        assert bool(torch.isnan(got[dev(np.flatnonzero(sees))]).all())
        others = dev(np.flatnonzero(~sees))
        assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("heads,run", [(16, 1), (3, 7), (32, 3), (128, 2)])
def test_a_score_of_minus_infinity(heads, run):
    """A key at minus infinity of q has no weight: its infinite value alone is NaN (0 times infinity), the row's others are
    the other keys'."""
    r = rng(heads)
    rank, rope, d = 512, 64, 37
    kept, where = cache(r, [120 + run], rank + rope, 16)
    slots, positions = np.zeros(run, int), 120 + np.arange(run)
    q = dev(np.abs(r.standard_normal((run, heads, rank + rope))) + 0.1, BF16)
    for key in (50, 119 + run):
        x = kept.clone()
        x[L.kept_row(0, key, **where), d] = -float("inf")
        got = f64(attend(q, x, slots, positions, where, rank=rank, scale=0.02, run=run))
        sees = positions >= key
        assert np.isnan(got[sees, :, d]).all() and not np.isnan(got[~sees]).any()
        out, size, spread = L.attend(f64(q), f64(x), slots, positions, rank=rank, scale=0.02, **where)
        spread = np.full_like(spread, (np.abs(f64(q)).sum(-1) * 6 * 0.02).max())  # (no row's value is past 6)
        limit = L.bound(out, size, spread, 19, HALF)
        rest = np.arange(rank) != d
        assert np.all((np.abs(got - out) <= limit)[:, :, rest])


@pytest.mark.parametrize("heads,run", [(16, 1), (16, 5), (40, 3)])
def test_refused_rows(heads, run):
    """Positions past the slot or max_position, slots and pages that are not there: NaN and their bits; the rows beside
    them are as ever."""
    r = rng(heads)
    rank, rope, page = 256, 32, 16
    kept, where = cache(r, [100, 100, 100], rank + rope, page)
    table = where["table"].copy()
    table[where["kept_pages"] + 3] = 999  # slot 1's keys 48 .. 63
    where = dict(where, table=table)
    slots = np.array([0, 1, 1, 3, 2, 0, 2, 0xFFFFFFFF], np.uint32)
    positions = np.array([99, 40, 70, 5, 200, 0xFFFFFFFF, 98, 0], np.uint32)
    bad = np.array([0, 0, 1, 1, 1, 1, 0, 1], bool)
    q = dev(r.standard_normal((8, heads, rank + rope)), BF16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(q, kept, slots, positions, where, rank=rank, scale=0.1, run=run, max_position=111, status=status)
    assert int(status) == abi.TS_STATUS_POSITION | abi.TS_STATUS_PAGE
    assert torch.isnan(got[dev(bad)]).all()
    good = np.flatnonzero(~bad)
    check_attend(got[dev(good)], q[dev(good)], kept, slots[good], positions[good], where, rank=rank, scale=0.1)
    for row, bit in ((2, abi.TS_STATUS_PAGE), (3, abi.TS_STATUS_PAGE), (4, abi.TS_STATUS_POSITION), (0, 0)):
        status.zero_()
        attend(q[row:row + 1], kept, slots[row:row + 1], positions[row:row + 1], where, rank=rank, scale=0.1,
               max_position=200, status=status)
        assert int(status) == bit
    got = attend(q[:1], kept, [0], [99], where, rank=rank, scale=0.1, max_position=98, status=status)
    assert int(status) == abi.TS_STATUS_POSITION and torch.isnan(got).all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB, a long slot at its end: split over all groups."""
    rank, rope, page, n = 512, 64, 64, 20000
    pages = (5 << 30) // (page * 1152)
    kept = torch.zeros(pages * page, rank + rope, dtype=BF16, device="cuda")
    each = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    kept[-each * page:] = torch.randn(each * page, rank + rope, generator=g, device="cuda").to(BF16)
    table = torch.arange(pages - each, pages, dtype=torch.int32, device="cuda")
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    for heads in (16, 128):
        q = torch.randn(1, heads, rank + rope, generator=g, device="cuda").to(BF16)
        got = rules.attend_latent(q, kept, i, i + n - 1, keys=each * page, rank=rank, scale=0.07, table=table,
                                  kept_pages=each, page=page)
        k = kept[-each * page:][:n].double()
        w = torch.softmax(q[0].double() @ k.T * 0.07, -1)
        want, size = w @ k[:, :rank], w @ k[:, :rank].abs()
        # The bound of the module's form, its scores' size taken as sqrt(576) 6 times 6 (six deviations of each).
        limit = 2 * 0.07 * 576 * 36 * 19 * 2.0 ** -21 * size + (2.0 ** -20 + HALF + 2.0 ** -13) * size + HALF * want.abs()
        assert bool(((got[0].double() - want).abs() <= limit).all())
        assert float((got[0].double() - want).norm() / want.norm()) < 4e-3  # weights and outputs half a bf16 step each
    c = torch.randn(1, rank + rope, generator=g, device="cuda")
    rules.append_latent(c, kept, i, i + n - 1, keys=each * page, rank=rank, table=table, kept_pages=each, page=page)
    assert torch.equal(kept[-each * page + n - 1], c[0].to(BF16))


# Slots that could hold more keys, which lets a group take 32, 64 or 128 columns: (heads, run, positions a slot).
WIDE_TILES = [(32, 1, 1 << 17), (128, 1, 1 << 12), (128, 1, 1 << 17), (16, 64, 1 << 13), (16, 64, 1 << 16), (5, 70, 1 << 16),
              (40, 33, 1 << 16), (100, 9, 1 << 17), (150, 1, 1 << 17)]


def roomier(where, keys):
    """The same slots with places for `keys` positions, whose pages are not held."""
    table = where["table"].reshape(-1, where["kept_pages"])
    each = keys // (where["keys"] // where["kept_pages"])
    more = np.full((len(table), each - table.shape[1]), 2 ** 31 - 1, np.int32)
    return dict(keys=keys, table=np.concatenate([table, more], 1).reshape(-1), kept_pages=each)


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads,run,keys", WIDE_TILES)
@pytest.mark.parametrize("back", [None, 30])
def test_wide_tiles(widths, heads, run, keys, back):
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(heads + run)
    lengths = [run + 300, run, run + 31, run + 64, run + 1, run + 450, run + 2, run + 99]
    kept, where = cache(r, lengths, rank + rope, 16)
    where = roomier(where, keys)
    counts = np.array([run, 1, max(1, run - 3), run, 1, run, 1, max(1, run // 2)])
    slots = np.repeat(np.arange(8), counts)
    positions = np.concatenate([n - c + np.arange(c) for n, c in zip(lengths, counts)])
    q = dev(r.standard_normal((len(slots), heads, rank + rope)), BF16)
    kw = dict(rank=rank, scale=(nope + rope) ** -0.5, **({} if back is None else {"back": back}))
    got = attend(q, kept, slots, positions, where, run=run, max_position=keys - 1, **kw)
    check_attend(got, q, kept, slots, positions, where, **kw)
    assert torch.equal(got, attend(q, kept, slots, positions, where, run=run, max_position=keys - 1, **kw))
    # In another order, a tile of many slots; some rows refused.
    order = r.permutation(len(slots))[:60]
    slots, positions, q = slots[order].copy(), positions[order].copy(), q[dev(order)]
    slots[5], positions[3] = 8, keys
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(q, kept, slots, positions, where, run=run, max_position=keys - 1, status=status, **kw)
    bad = np.isin(np.arange(len(slots)), [5, 3])
    assert torch.isnan(got[dev(np.flatnonzero(bad))]).all()
    assert int(status) == abi.TS_STATUS_PAGE | abi.TS_STATUS_POSITION
    good = np.flatnonzero(~bad)
    check_attend(got[dev(good)], q[dev(good)], kept, slots[good], positions[good], where, **kw)


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads,run,keys,back", [(8, 16, 1 << 17, None), (16, 64, 1 << 16, None), (3, 90, 1 << 17, None),
                                                 (40, 33, 1 << 16, None), (16, 2000, 1 << 12, 100)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_wide_tiles_not_finite_in_masked_places(widths, heads, run, keys, back, value):
    """As with narrow ones: a value that is not finite reaches the rows that see its key alone."""
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(heads + run)
    kept, where = cache(r, [120 + run, 60], rank + rope, 16)
    where = roomier(where, keys)
    slots = np.concatenate([np.zeros(run, int), [1]])
    positions = np.concatenate([120 + np.arange(run), [59]])
    d = 37
    q = r.standard_normal((run + 1, heads, rank + rope))
    q[..., d] = 0
    q = dev(q, BF16)
    kw = dict(rank=rank, scale=0.05, **({} if back is None else {"back": back}))
    call = dict(kw, run=run, max_position=keys - 1)
    want = attend(q, kept, slots, positions, where, **call)
    few = np.unique(np.concatenate([[0, run], r.integers(0, run, 30)]))
    check_attend(want[dev(few)], q[dev(few)], kept, slots[few], positions[few], where, **kw)
    for key in (23, 121, 120 + run // 2, 120 + run - 1):
        sees = (positions - (back or keys) <= key) & (positions >= key) & (slots == 0)
        x = kept.clone()
        x[L.kept_row(0, key, **where), d] = value
        got = attend(q, x, slots, positions, where, **call)
        assert bool(torch.isnan(got[dev(np.flatnonzero(sees))]).all())
        others = dev(np.flatnonzero(~sees))
        assert torch.equal(got[others], want[others])


@pytest.mark.parametrize("rows", [2, 63, 64, 65, 130, 512, 513])
@pytest.mark.parametrize("heads,run", [(16, 5), (32, 2), (5, 9)])
def test_rows_of_many_short_runs(rows, heads, run):
    """Runs of any length at any place, as many tiles as may be told from the slots, and more."""
    rank, rope = 256, 32
    r = rng(rows + heads)
    counts = []
    while sum(counts) < rows:
        counts.append(min(int(r.integers(1, run + 2)), rows - sum(counts)))
    lengths = [int(c + r.integers(0, 50)) for c in counts]
    kept, where = cache(r, lengths, rank + rope, 16)
    where = roomier(where, 1 << 14)
    slots = np.repeat(np.arange(len(counts)), counts)
    positions = np.concatenate([n - c + np.arange(c) for n, c in zip(lengths, counts)])
    q = dev(r.standard_normal((rows, heads, rank + rope)), BF16)
    got = attend(q, kept, slots, positions, where, rank=rank, scale=0.1, run=run, max_position=(1 << 14) - 1)
    check_attend(got, q, kept, slots, positions, where, rank=rank, scale=0.1)


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads", [5, 16])
def test_decode_rows_take_weights_in_two_parts(widths, heads):
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(heads)
    lengths = [900, 1, 333]
    kept, where = cache(r, lengths, rank + rope, 16)
    q = dev(r.standard_normal((3, heads, rank + rope)), BF16)
    slots, positions = np.arange(3), np.array(lengths) - 1
    kw = dict(rank=rank, scale=(nope + rope) ** -0.5)
    check_attend(attend(q, kept, slots, positions, where, **kw), q, kept, slots, positions, where, one_part=False, **kw)


# --- the expanded form ----------------------------------------------------------------------------

def check_flash(got, q, k, v, r, **kw):
    out, size, spread = L.flash(f64(q), f64(k), f64(v), f64(r), **kw)
    limit = L.bound(out, size, spread, q.shape[-1] / 16 + 1, HALF)
    here = ~np.isnan(out)
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(f64(got) - out) <= limit)[here])
    return here


def flash_inputs(r, rows, keys, heads, widths):
    _, rope, nope, value = WIDTHS[widths]
    kv = dev(r.standard_normal((keys, heads, nope + value)), BF16)
    return (dev(r.standard_normal((rows, heads, nope + rope)), BF16), kv[..., :nope], kv[..., nope:],
            dev(r.standard_normal((keys, rope)), BF16))


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads", [1, 5, 16])
@pytest.mark.parametrize("rows,more", [([1], [0]), ([31, 1, 33], [0, 7, 0]), ([129, 0, 2, 64], [0, 5, 300, 0]),
                                       ([300, 40], [0, 90]), ([40, 9], [-30, 3])])
@pytest.mark.parametrize("back", [None, 0, 50])
def test_flash(widths, heads, rows, more, back):
    """Ragged sequences: none, one and many rows, more keys than rows, fewer (whose first rows see none and are 0)."""
    _, rope, nope, _ = WIDTHS[widths]
    r = rng(heads + sum(rows))
    if heads == 16 and sum(rows) > 200:
        rows, more = rows[-1:], more[-1:]
    keys = [a + b for a, b in zip(rows, more)]
    first, key_first = np.concatenate([[0], np.cumsum(rows)]), np.concatenate([[0], np.cumsum(keys)])
    x = flash_inputs(r, first[-1], key_first[-1], heads, widths)
    kw = dict(scale=(nope + rope) ** -0.5, **({} if back is None else {"back": back}))
    got = rules.flash_latent(*x, first=ints(first), key_first=ints(key_first), **kw)
    assert check_flash(got, *x, first=first, key_first=key_first, **kw).all()
    assert torch.equal(got, rules.flash_latent(*x, first=ints(first), key_first=ints(key_first), **kw))
    if len(rows) == 1:
        assert torch.equal(got, rules.flash_latent(*x, **kw))
    if not any(more):
        assert torch.equal(got, rules.flash_latent(*x, first=ints(first), **kw))


@pytest.mark.parametrize("seqs", [70, 300])
def test_flash_many_sequences(seqs):
    """More sequences than lanes, and than the tiles that are ordered."""
    r = rng(seqs)
    rows = r.integers(0, 9, seqs)
    rows[seqs // 3] = 200
    first = np.concatenate([[0], np.cumsum(rows)])
    x = flash_inputs(r, first[-1], first[-1], 2, "narrow")
    got = rules.flash_latent(*x, first=ints(first), scale=0.1)
    assert check_flash(got, *x, first=first, key_first=first, scale=0.1).all()


def test_flash_rows_behind_the_last_sequence_and_bad_bounds():
    """Left as they were: rows behind the last sequence, rows of sequences whose bounds descend or pass the tensors."""
    r = rng(4)
    x = flash_inputs(r, 90, 100, 3, "narrow")
    out = torch.full((90, 3, 64), 7.0, dtype=BF16, device="cuda")
    # Sequences: 0 .. 20 fine; 20 .. 50 with keys that pass the tensor; 50 .. 70 fine.
    first, key_first = np.array([0, 20, 50, 70]), np.array([0, 30, 2 ** 31, 2 ** 31 + 5])
    rules.flash_latent(*x, first=ints(first), key_first=ints(key_first), scale=0.1, out=out)
    check_flash(out[:20], x[0][:20], *x[1:], first=[0, 20], key_first=[0, 30], scale=0.1)
    assert bool((out[20:] == 7.0).all())
    first = np.array([0, 20, 10, 95, 60])
    out.fill_(7.0)
    rules.flash_latent(*x, first=ints(first), key_first=ints([0, 30, 40, 50, 60]), scale=0.1, out=out)
    check_flash(out[:20], x[0][:20], *x[1:], first=[0, 20], key_first=[0, 30], scale=0.1)
    assert bool((out[20:] == 7.0).all())


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_flash_not_finite_in_masked_places(widths, value):
    """A value that is not finite reaches the rows that see its key, and only its own d of them."""
    r = rng(11)
    q, k, v, rr = flash_inputs(r, 150, 150, 2, widths)
    first = ints([0, 100, 150])
    kw = dict(scale=0.1, first=first, back=60)
    want = rules.flash_latent(q, k, v, rr, **kw)
    for key in (40, 99, 100, 149):
        x = v.clone()
        x[key, 1, 9] = value
        got = rules.flash_latent(q, k, x, rr, **kw)
        i = np.arange(150)
        sees = (i >= key) & (i - 60 <= key) & ((i < 100) == (key < 100))
        mask = torch.ones_like(got, dtype=torch.bool)
        mask[dev(np.flatnonzero(sees)), 1, 9] = False
        assert torch.equal(got[mask], want[mask])
        hit = got[~mask]
        assert bool(torch.isnan(hit).all()) if value != value else bool((hit == value).all())


def test_flash_scales_and_layouts():
    r = rng(12)
    q, k, v, rr = flash_inputs(r, 70, 70, 4, "wide")
    for scale in (0.0, -0.1, 2.0):
        got = rules.flash_latent(q, k, v, rr, scale=scale)
        check_flash(got, q, k, v, rr, first=[0, 70], key_first=[0, 70], scale=scale)
    want = rules.flash_latent(q, k, v, rr, scale=0.1)
    wide = torch.zeros(70, 4 * 192 + 64, dtype=BF16, device="cuda")
    wide[:, :768] = q.flatten(1)
    kept = torch.zeros(70, 576, dtype=BF16, device="cuda")
    kept[:, 512:] = rr
    outside = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    got = rules.flash_latent(wide[:, :768].unflatten(1, (4, 192)), outside(k), outside(v), kept[:, 512:], scale=0.1)
    assert torch.equal(got, want)
