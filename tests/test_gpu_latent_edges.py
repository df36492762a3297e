"""Calls of latent attention at the edges of what its entry points take, on the GPU."""
import numpy as np
import pytest

import latent_ref as L
from helpers import rng
from tessera_amd import abi, rules
from test_gpu_latent import BF16, F32, HALF, WIDTHS, attend, cache, check_attend, check_flash, dev, f64, flash_inputs, ints, roomier

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("widths", ["wide", "narrow"])
def test_flash_of_broadcast_rows(widths):
    """q, k, v and r that are one row for all."""
    r = rng(21)
    q, k, v, rr = flash_inputs(r, 1, 1, 3, widths)
    many = [x.expand(n, *x.shape[1:]) for x, n in ((q, 150), (k, 170), (v, 170), (rr, 170))]
    got = rules.flash_latent(*many, scale=0.1)
    assert torch.equal(got, rules.flash_latent(*(x.contiguous() for x in many), scale=0.1))
    check_flash(got, *many, first=[0, 150], key_first=[0, 170], scale=0.1)
    one = rules.flash_latent(q, *many[1:], scale=0.1)  # (a row by itself has no distance either)
    assert torch.equal(one, got[149:])


def test_append_with_heads_outside_rows():
    """q_out [heads, rows, rope] seen as [rows, heads, rope]; rows that lie on one another are refused."""
    r = rng(22)
    n, rank, rope, heads = 11, 256, 32, 5
    c, q = dev(r.standard_normal((n, rank + rope)), F32), dev(r.standard_normal((n, heads, rope)), F32)
    angles, i = rules.rope_table(64, 1e4, width=rope), torch.arange(n, dtype=torch.int32, device="cuda")
    kept = torch.zeros(64, rank + rope, dtype=BF16, device="cuda")
    kw = dict(keys=64, rank=rank, angles=angles, q=q)
    want = rules.append_latent(c, kept, i * 0, i, **kw)
    out = torch.zeros(heads, n, rope, device="cuda").transpose(0, 1)
    assert torch.equal(rules.append_latent(c, kept, i * 0, i, q_out=out, **kw), want)
    for bad in (torch.zeros(1, heads, rope, device="cuda").expand(n, -1, -1),
                torch.zeros(n * heads * rope, device="cuda").as_strided((n, heads, rope), (rope, rope, 1))):
        with pytest.raises(abi.HipError, match="meet"):
            rules.append_latent(c, kept, i * 0, i, q_out=bad, **kw)


# Rows of one slot far apart, whose windows leave keys between them that no row sees: (heads, run, rows), which
# take 16, 32, 64 and 128 columns a group with `back` 700 and 8192 positions a slot.
APART = [(2, 16, 16), (2, 5, 80), (2, 5, 500), (8, 5, 500), (40, 3, 300), (40, 64, 512)]


def two_windows(r, rows, width, page=16, back=700, keys=8192):
    """Positions near 800 and near 6000 in turn, and kept rows whose table holds the pages of their windows alone."""
    positions = np.where(np.arange(rows) % 2 == 0, 800, 6000) + np.arange(rows) // 2 % 40
    seen = np.zeros(keys // page, bool)
    for p in set(positions):
        seen[(p - back) // page:p // page + 1] = True
    held = np.flatnonzero(seen)
    table = np.full(len(seen), 2 ** 31 - 1, np.int32)
    table[held] = r.permutation(len(held))
    kept = dev(r.standard_normal((len(held) * page, width)), BF16)
    return positions, kept, dict(keys=keys, table=table, kept_pages=len(seen), page=page)


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads,run,rows", APART)
def test_pages_between_windows_need_not_be_held(widths, heads, run, rows):
    """A page that no row sees is no row's refusal, wherever the rows that share its loads stand."""
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(rows + heads)
    positions, kept, where = two_windows(r, rows, rank + rope)
    q = dev(r.standard_normal((rows, heads, rank + rope)), BF16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(rank=rank, scale=(nope + rope) ** -0.5, back=700)
    got = attend(q, kept, np.zeros(rows, int), positions, where, run=run, max_position=8191, status=status, **kw)
    few = np.unique(np.concatenate([np.arange(6), r.integers(0, rows, 20)]))
    check_attend(got[dev(few)], q[dev(few)], kept, np.zeros(len(few), int), positions[few], where, **kw)
    assert int(status) == 0
    finite = bool(torch.isfinite(got).all())
    assert finite


@pytest.mark.parametrize("rows,heads,n,k", [(5, 3, 130, 72), (40, 40, 200, 136), (100, 3, 40, 72), (100, 2, 130, 200)])
@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("out", [F32, BF16])
def test_linear_heads_of_weights_that_are_not_finite(rows, heads, n, k, x, out):
    """An infinite weight makes its outputs infinite, but where x is 0 or the signs of two of them differ; NaN makes them NaN."""
    r = rng(rows + n)
    xs, w = r.standard_normal((rows, heads, k)), dev(r.standard_normal((heads, n, k)), BF16)
    xs[:, :, 9] = np.where(np.arange(rows)[:, None] % 2 == 0, 1.5, -2.0)  # (8 bits: the lower parts of an f32 are 0)
    xs[3, :, 9] = 0.0
    xs = dev(xs, x)
    want = f64(rules.linear_heads(xs, w, out_dtype=out))
    w[:, 1, 9], w[0, 3, 9], w[1, n - 1, 70], w[0, 5, 1] = float("inf"), -float("inf"), float("inf"), float("nan")
    w[1, 7, 8], w[1, 7, 9] = float("inf"), -float("inf")
    a, b = f64(xs), f64(w)
    with np.errstate(invalid="ignore"):
        bad = np.einsum("rhk,hnk->rhn", a, b)
    got = f64(rules.linear_heads(xs, w, out_dtype=out))
    odd = ~np.isfinite(bad)
    assert np.array_equal(got[odd], bad[odd], equal_nan=True) and np.array_equal(got[~odd], want[~odd])
    assert np.isinf(bad).sum() > rows and np.isnan(bad[3, 0, 1]) and np.isnan(bad[:, 0, 5]).all()


@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("rank", [512, 1024, 8])
def test_append_of_rows_past_the_range_of_their_squares(x, rank):
    """A finite row is normed whatever its size: squares of values from 2^64 on (or their sum) pass f32's range."""
    r = rng(rank)
    rope, n = 32, 6
    c = r.standard_normal((n, rank + rope))
    c[1] *= 2.0 ** 66
    c[2] *= 2.0 ** 122
    c[3, :rank] = 2.0 ** 63 * np.sign(c[3, :rank])  # (each square holds, their sum does not)
    c[4, :rank] = 0
    c[4, 5] = -3e38
    c[5, 3] = np.inf
    c = dev(c, x)
    gain = dev(1 + 0.1 * r.standard_normal(rank), F32)
    kept = torch.zeros(16, rank + rope, dtype=BF16, device="cuda")
    i = torch.arange(n, dtype=torch.int32, device="cuda")
    rules.append_latent(c, kept, i * 0, i, keys=16, rank=rank, gain=gain, eps=1e-5)
    want = L.normed(f64(c)[:5, :rank], f64(gain), 1e-5)
    # As check_append's: (rank + 8) steps of f32 and the rounding to bf16.
    assert np.all(np.abs(f64(kept)[:5, :rank] - want) <= np.abs(want) * ((rank + 8) * 2.0 ** -24 + HALF))
    got = f64(kept)[5, :rank]
    assert np.isnan(got[3]) and not np.delete(got, 3).any()


# More than 64 rows and columns over several chunks of 64 k, whole and begun: two buffers of f32 x, three of bf16.
@pytest.mark.parametrize("rows,heads,n,k", [(65, 3, 130, 72), (100, 2, 129, 136), (200, 4, 335, 328), (97, 32, 128, 512), (129, 2, 65, 128),
                                            (190, 1, 200, 192), (70, 5, 257, 640), (128, 2, 128, 1000)])
@pytest.mark.parametrize("x", [F32, BF16])
@pytest.mark.parametrize("out", [F32, BF16])
def test_linear_heads_of_many_chunks(rows, heads, n, k, x, out):
    """The bound of the products a head: k / 16 accumulating steps and one more at 2^-21 each of the sum of |x w|, three
    times as many of f32 x, whose parts drop 2^-24; then half a step of bf16."""
    r = rng(rows + n + k)
    gap = 8 if n % 2 else 0
    xs = dev(r.standard_normal((rows, heads, k + 8)), x)[..., :k]
    w = dev(r.standard_normal((heads, n, k)) / 8, BF16)
    held = torch.full((rows, heads, n + gap), 7.0, dtype=out, device="cuda")
    got = rules.linear_heads(xs, w, out=held[..., :n])
    a, b = f64(xs), f64(w)
    want, size = (np.matmul(p.transpose(1, 0, 2), q.transpose(0, 2, 1)).transpose(1, 0, 2) for p, q in ((a, b), (np.abs(a), np.abs(b))))
    steps = (k / 16 + 1) * (3 if x == F32 else 1)
    limit = size * (steps * 2.0 ** -21 + 2.0 ** -24) + (HALF * np.abs(want) if out == BF16 else 0)
    assert np.all(np.abs(f64(got) - want) <= limit)
    assert bool((held[..., n:] == 7.0).all())


# (heads, run, rows, positions a slot), which take 16, 32, 64 and 128 columns a group: keys of few tiles in whole parts and in
# equal runs, tiles cut where the slot changes, several blocks of heads, groups that each have a tile alone.
LOST = [(16, 1, 6, 1 << 13), (16, 1, 300, 1 << 13), (2, 16, 32, 1 << 13), (32, 1, 6, 1 << 17), (32, 1, 300, 1 << 13), (2, 3, 6, 1 << 17),
        (8, 16, 640, 1 << 13), (64, 1, 300, 1 << 13), (150, 1, 6, 1 << 17), (8, 5, 10, 1 << 17), (5, 33, 500, 1 << 13), (16, 16, 640, 1 << 13),
        (128, 1, 6, 1 << 17), (128, 1, 300, 1 << 13), (40, 3, 9, 1 << 17), (16, 33, 528, 1 << 13), (32, 33, 528, 1 << 13),
        (1024, 1, 300, 1 << 13)]


@pytest.mark.parametrize("widths", ["wide", "narrow"])
@pytest.mark.parametrize("heads,run,rows,keys", LOST)
@pytest.mark.parametrize("back", [None, 3000])
def test_lost_pages(widths, heads, run, rows, keys, back):
    """A page that is not held makes the rows that see its keys NaN, and sets the bit; the rows beside them, of shorter and of
    other sequences over the same pages, keep their bits. Pages at the start, at the end, in either block of a step, behind
    the blocks that are looked up at once (16 or 32 rounds)."""
    rank, rope, nope, _ = WIDTHS[widths]
    r = rng(rows + heads)
    n, page = 5000, 16
    held = -(-n // page)
    table = np.full((3, keys // page), 2 ** 31 - 1, np.int32)
    table[:, :held] = r.permutation(held)
    where = dict(keys=keys, kept_pages=keys // page, page=page)
    kept = dev(r.standard_normal((held * page, rank + rope)), BF16)
    index = np.arange(rows) // run
    starts = np.where(np.arange(index[-1] + 1) % 5 == 3, r.integers(0, 200, index[-1] + 1), r.integers(3800, n - run + 1, index[-1] + 1))
    starts[0] = n - run
    positions = starts[index] + np.arange(rows) % run
    slots = np.where(index % 3 == 2, 1 + index % 2, 0)
    q = dev(r.standard_normal((rows, heads, rank + rope)), BF16)
    kw = dict(rank=rank, scale=(nope + rope) ** -0.5, **({} if back is None else {"back": back}))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = dict(kw, run=run, max_position=keys - 1, status=status)
    want = attend(q, kept, slots, positions, dict(where, table=table.reshape(-1)), **call)
    few = np.unique([0, rows - 1, rows // 2])
    check_attend(want[dev(few)], q[dev(few)], kept, slots[few], positions[few], dict(where, table=table.reshape(-1)), **kw)
    assert int(status) == 0
    last = int(positions[slots == 0].max()) // page
    for lost in ([0], [1], [150], [151], [255, 256, 257], [last - 1], [last]):
        fewer = table.copy()
        fewer[0, lost] = held
        sees = np.zeros(rows, bool)
        for b in lost:
            sees |= (slots == 0) & (positions >= b * page) & (positions - (keys if back is None else back) <= b * page + page - 1)
        status.zero_()
        got = attend(q, kept, slots, positions, dict(where, table=fewer.reshape(-1)), **call)
        assert bool(torch.isnan(got[dev(np.flatnonzero(sees))]).all()), lost
        others = dev(np.flatnonzero(~sees))
        same = torch.equal(got[others], want[others])
        assert same and int(status) == (abi.TS_STATUS_PAGE if sees.any() else 0), lost


def flash_forms(q, k, v, r, *, scale, first, key_first, back):
    """latent_ref.flash on the GPU, in 64 bits, a head of a sequence at once."""
    out, size = (torch.full((*q.shape[:2], v.shape[-1]), float("nan"), dtype=torch.float64, device="cuda") for _ in range(2))
    spread = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    for a, b, ka, kb in zip(first[:-1], first[1:], key_first[:-1], key_first[1:]):
        pos = (kb - ka) - (b - a) + torch.arange(b - a, device="cuda")[:, None]
        key = torch.arange(kb - ka, device="cuda")
        sees = (key <= pos) & (key >= pos - back)
        for h in range(q.shape[1]):
            x, rows, vv = q[a:b, h].double(), torch.cat([k[ka:kb, h], r[ka:kb]], -1).double().T.contiguous(), v[ka:kb, h].double()
            w = torch.softmax((x @ rows * scale).masked_fill(~sees, -float("inf")), -1).nan_to_num(0.0)
            out[a:b, h], size[a:b, h] = w @ vv, w @ vv.abs()
            spread[a:b, h] = ((x.abs() @ rows.abs()) * sees).amax(-1) * abs(scale)
    return out.cpu().numpy(), size.cpu().numpy(), spread.cpu().numpy()


@pytest.mark.parametrize("rows,more", [([8300], [0]), ([4100, 5300], [77, 0]), ([90, 9000, 40], [0, 300, 9]), ([600] * 15, [0] * 15),
                                       ([2000, 7000], [-1000, 0])])
@pytest.mark.parametrize("widths,heads", [("narrow", 1), ("narrow", 8), ("wide", 2)])
@pytest.mark.parametrize("back", [None, 40])
def test_flash_of_long_sequences(rows, more, widths, heads, back):
    """More than the 64 tiles that are ordered at once, of a sequence or a few: every row is written, once and rightly."""
    _, rope, nope, value = WIDTHS[widths]
    keys = [a + b for a, b in zip(rows, more)]
    first, key_first = np.concatenate([[0], np.cumsum(rows)]), np.concatenate([[0], np.cumsum(keys)])
    g = torch.Generator(device="cuda").manual_seed(sum(rows))
    new = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF16)  # noqa: E731
    behind = 50
    q, k, v, r = new(first[-1] + behind, heads, nope + rope), new(key_first[-1], heads, nope), new(key_first[-1], heads, value), new(key_first[-1], rope)
    out = torch.full((len(q), heads, value), 7.0, dtype=BF16, device="cuda")
    kw = dict(scale=(nope + rope) ** -0.5, **({} if back is None else {"back": back}))
    got = rules.flash_latent(q, k, v, r, first=ints(first), key_first=ints(key_first), out=out, **kw)
    assert bool((got[first[-1]:] == 7.0).all())
    want, size, spread = flash_forms(q, k, v, r, first=first, key_first=key_first, scale=kw["scale"], back=1 << 30 if back is None else back)
    got, want, size, spread = f64(got)[:first[-1]], want[:first[-1]], size[:first[-1]], spread[:first[-1]]
    # (latent_ref.bound's 2^-14 is of 128 steps of 64 keys; 2^-13 more for up to 256.)
    limit = L.bound(want, size, spread, (nope + rope) / 16 + 1, HALF) + 2.0 ** -13 * size
    assert np.all(np.abs(got - want) <= limit)
