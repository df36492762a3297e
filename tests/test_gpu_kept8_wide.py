"""attend_kept8 in every one of its kernels, on the GPU against float64: tiles of 16, 64, 128 and 256 columns, keys
shared among groups or not, tiles in order of their cost or as they come; NaN codes, lost pages and refused rows in
each, for both types of q."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SCALE, PAGE = 128 ** -0.5, 16
TYPES = [("f32", torch.float32), ("bf16", torch.bfloat16)]


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Kept:
    """Blocks of slots of `lengths` positions, under a shuffled table; what is past them may be any byte."""

    def __init__(self, r, lengths, kvh, spare=1):
        self.each, self.kvh = -(-max(lengths) // PAGE), kvh
        self.pages = len(lengths) * self.each + spare
        self.table = r.permutation(self.pages)[:len(lengths) * self.each].astype(np.int32)
        g = torch.Generator(device="cuda").manual_seed(int(r.integers(1 << 30)))
        self.k, self.v, self.scales = rules.kept8(self.pages, kvh, PAGE)
        for t in (self.k, self.v):
            t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
        self.scales.copy_(torch.exp2(torch.randint(-8, -5, self.scales.shape, generator=g, device="cuda").float()))
        for s, n in enumerate(lengths):  # NaN codes behind each slot's last position
            if n % 16:
                b = int(self.table[s * self.each + n // 16])
                self.k[b, :, n % 16:], self.v[b, :, :, n % 16:] = 0x7F, 0xFF

    def block(self, s, j, table=None):
        """Block and place in it of position(s) j of slot s."""
        j = np.asarray(j)
        return (self.table if table is None else table)[s * self.each + j // 16], j % 16

    def attend(self, q, slots, positions, *, table=None, most=None, **kw):
        kw.setdefault("out_dtype", q.dtype)
        return rules.attend_kept8(q, self.k, self.v, self.scales, dev(np.asarray(slots, np.int32)),
                                  dev(np.asarray(positions, np.int32)), keys=self.each * PAGE, scale=SCALE, page=PAGE,
                                  table=dev(self.table if table is None else table), kept_pages=self.each,
                                  max_position=int(np.max(positions)) if most is None else most, **kw)

    def exact(self, q, slots, positions, back=None):
        """Outputs in float64, and per (row, head) the largest sum of |q_i k_i| SCALE and |v| among its keys."""
        q, group = q.double(), q.shape[1] // self.kvh
        codes = dev(K.CODES)
        out = torch.zeros_like(q)
        spread, size = (torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda") for _ in range(2))
        for s in np.unique(slots):
            rows = dev(np.nonzero(np.asarray(slots) == s)[0])
            pos = dev(np.asarray(positions)[np.asarray(slots) == s].astype(np.int64))
            b, o = (dev(np.asarray(x, np.int64)) for x in self.block(s, np.arange(int(pos.max()) + 1)))
            j = torch.arange(len(b), device="cuda")
            hidden = j[None] > pos[:, None]
            if back is not None:
                hidden |= j[None] < pos[:, None] - back
            hidden = hidden.repeat_interleave(group, 0)
            for h in range(self.kvh):
                kk = codes[self.k[b, h, o].long()] * self.scales[b, h, 0, None].double()
                vv = codes[self.v[b, h, :, o].long()] * self.scales[b, h, 1, None].double()
                at = slice(h * group, (h + 1) * group)
                qq = q[rows, at].reshape(-1, 128)
                w = torch.softmax((torch.mm(qq, kk.T.contiguous()) * SCALE).masked_fill(hidden, -torch.inf), -1)
                out[rows, at] = torch.mm(w, vv).view(-1, group, 128)
                big = torch.mm(qq.abs(), kk.abs().T.contiguous()).masked_fill(hidden, 0) * SCALE
                spread[rows, at] = big.amax(-1).view(-1, group)
                size[rows, at] = vv.abs().amax(-1).expand(len(big), -1).masked_fill(hidden, 0).amax(-1).view(-1, group)
        return out, spread, size


def within(got, want, spread, size, f32):
    """Where |got - want| keeps the bound. A score: f32 q in three bf16 parts (2^-24), 128 products summed at 2^-21
    each accumulating step (12 of them; of bf16 q 4). A weight is off by twice that, by 2^-20 of its exponential and
    the sums and by its rounding (three parts 2^-24; one, half a step of bf16, 2^-8); the output by that times the
    largest |v|, plus its own rounding."""
    score = spread * (2.0 ** -24 + 12 * 2.0 ** -21 if f32 else 4 * 2.0 ** -21)
    bound = (2 * score + 2.0 ** -20 + (2.0 ** -24 if f32 else 2.0 ** -8)) * size + (0 if f32 else 2.0 ** -8 * size)
    return (got.double() - want).abs() <= bound[..., None]


# (heads, kv heads, rows of each slot, positions kept before them, the hint `run`): what runs is said beside each.
FORMS = {
    "16": (4, 2, [3, 2, 3], [100, 0, 61], 3),                     # 16 columns, shared keys
    "64": (16, 2, [6, 3, 5], [100, 0, 61], 5),                    # 64 columns, shared keys (bf16: one buffer of codes)
    "64 alone": (8, 1, [5] * 260, list(range(260)), 5),           # 64 columns, a group a tile: more than 256 tiles
    "128": (4, 2, [90, 33, 70], [20, 0, 61], 90),                 # 128 columns, shared keys
    "128 ordered": (64, 32, [300, 260, 100], [0, 7, 400], 300),   # 128 columns, the widest tile first
    "256 ordered": (16, 8, [2300, 1000, 2048, 2900], [0, 37, 500, 3], 2048),  # 256 columns (bf16; f32: 128)
    "256 of three": (24, 8, [3000, 2500], [0, 1], 3000),          # 255 of 256 columns used
    "256 many": (128, 2, [1100], [30], 1100),                     # 275 tiles of four rows: in the order they come
    "256 border": (16, 8, [3100, 3044], [0, 9], 3000),             # as few rows as take 256 columns
    "256 heads": (128, 128, [700, 300, 24], [0, 100, 1000], 512), # one head a kv head, 256 rows a tile
}


@pytest.mark.parametrize("name,dtype", TYPES)
@pytest.mark.parametrize("back", [None, 37, 700])
@pytest.mark.parametrize("form", FORMS)
def test_against_float64(form, back, name, dtype):
    """Ragged rows: tiles that end in another sequence than they begin in, of costs from one step to many."""
    heads, kvh, rows, past, run = FORMS[form]
    r = rng(len(form) * 100 + heads + (back or 0))
    kept = Kept(r, [p + n for p, n in zip(past, rows)], kvh)
    slots = np.repeat(np.arange(len(rows)), rows)
    positions = np.concatenate([p + np.arange(n) for p, n in zip(past, rows)])
    q = dev(r.standard_normal((len(slots), heads, 128)).astype(np.float32), dtype)
    out = kept.attend(q, slots, positions, run=run, **({} if back is None else {"back": back}))
    want, spread, size = kept.exact(q, slots, positions, back)
    assert bool(within(out, want, spread, size, name == "f32").all())


SMALL = {  # (heads, kv heads, slots, rows of each)
    "16": (4, 2, 3, 4), "64": (16, 2, 3, 7), "128": (4, 2, 3, 90), "256": (128, 64, 3, 384),
}


@pytest.mark.parametrize("name,dtype", TYPES)
@pytest.mark.parametrize("form", SMALL)
def test_nan_codes_reach_the_rows_that_see_them(form, name, dtype):
    """A NaN key spoils what sees it, a NaN value its own column of that; everything else keeps the bound."""
    heads, kvh, slots_n, run = SMALL[form]
    r, n, back, group = rng(run), 70 + run, 40, heads // kvh
    kept = Kept(r, [n] * slots_n, kvh)
    slots, positions = np.repeat(np.arange(slots_n), run), np.tile(np.arange(n - run, n), slots_n)
    q = dev(r.standard_normal((len(slots), heads, 128)).astype(np.float32), dtype)
    want, spread, size = kept.exact(q, slots, positions, back)
    for at in (n - 1, n - run // 2 - 1, n - run - 20, 0):
        b, o = kept.block(1, at)
        was = kept.k[b, 1, o, 7].item(), kept.v[b, 0, 9, o].item()
        kept.k[b, 1, o, 7], kept.v[b, 0, 9, o] = 0xFF, 0x7F
        got = kept.attend(q, slots, positions, run=run, back=back)
        kept.k[b, 1, o, 7], kept.v[b, 0, 9, o] = was
        sees = dev((slots == 1) & (positions >= at) & (positions - back <= at))
        nan = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
        nan[:, group:2 * group] = sees[:, None, None]
        nan[:, :group, 9] = sees[:, None]
        assert torch.equal(torch.isnan(got), nan)
        assert bool((within(got, want, spread, size, name == "f32") | nan).all())


@pytest.mark.parametrize("name,dtype", TYPES)
@pytest.mark.parametrize("form", SMALL)
def test_refused_rows_and_lost_pages(form, name, dtype):
    """Positions past the slot or the stated bound, slots and pages out of range: NaN and a status bit; the rows
    beside them, of the same tile or another, keep the bound."""
    heads, kvh, slots_n, run = SMALL[form]
    r, n = rng(run + 1), max(128, -(-run // 16) * 16)
    kept = Kept(r, [n] * slots_n, kvh)
    slots, positions = np.repeat(np.arange(slots_n), run), np.tile(np.arange(n - run, n), slots_n)
    q = dev(r.standard_normal((len(slots), heads, 128)).astype(np.float32), dtype)
    want, spread, size = kept.exact(q, slots, positions)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def spoilt(bit, lost, slots=slots, positions=positions, **kw):
        status.zero_()
        got = kept.attend(q, slots, positions, run=run, status=status, **kw)
        assert int(status) == bit and torch.isnan(got[dev(lost)]).all()
        assert bool(within(got, want, spread, size, name == "f32")[dev(~lost)].all())

    one = np.arange(len(slots)) % 7 == 3  # rows in the midst of others
    spoilt(abi.TS_STATUS_POSITION, one, positions=np.where(one, positions + n, positions), most=n - 1)
    spoilt(abi.TS_STATUS_POSITION, one, positions=np.where(one, 0x7FFFFFFF, positions))
    spoilt(abi.TS_STATUS_POSITION, positions > n - 2, most=n - 2)
    spoilt(abi.TS_STATUS_PAGE, one, slots=np.where(one, slots_n, slots))
    spoilt(abi.TS_STATUS_PAGE, one, slots=np.where(one, -1, slots))
    spoilt(abi.TS_STATUS_PAGE, np.ones(len(slots), bool), slots=np.full(len(slots), slots_n))
    table = kept.table.copy()
    table[kept.each + n // 16 - 1] = kept.pages
    spoilt(abi.TS_STATUS_PAGE, (slots == 1) & (positions >= n - 16), table=table)
    table = kept.table.copy()
    table[0] = -1
    spoilt(abi.TS_STATUS_PAGE, slots == 0, table=table)


@pytest.mark.parametrize("name,dtype", TYPES)
@pytest.mark.parametrize("form", SMALL)
def test_calls_on_two_streams(form, name, dtype):
    """Two calls at once on two streams, each with scratch of its own: the bits of one alone."""
    heads, kvh, slots_n, run = SMALL[form]
    r, n = rng(run + 2), 600 + run
    kept = Kept(r, [n] * slots_n, kvh)
    slots, positions = np.repeat(np.arange(slots_n), run), np.tile(np.arange(n - run, n), slots_n)
    qs = [dev(r.standard_normal((len(slots), heads, 128)).astype(np.float32), dtype) for _ in range(2)]
    alone = [kept.attend(q, slots, positions, run=run) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(3):
        got = []
        for q, stream in zip(qs, streams):
            with torch.cuda.stream(stream):
                got.append(kept.attend(q, slots, positions, run=run))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


@pytest.mark.parametrize("heads,kvh,run", [(1, 1, 1), (16, 8, 1), (32, 2, 1), (8, 2, 4), (6, 2, 5)])
def test_weights_of_bf16_decode_rows_hold_16_bits(heads, kvh, run):
    """Tiles of up to 16 columns, f32 out: bf16 q's weights are off by half a step of two bf16 parts (2^-8 2^-8) where
    one would be off by 2^-8."""
    r = rng(heads + run)
    kept = Kept(r, [5, 40, 700, 3000], kvh)
    slots = np.repeat(np.arange(4), run)
    positions = np.concatenate([n - run + np.arange(run) for n in (5, 40, 700, 3000)])
    q = dev(r.standard_normal((len(slots), heads, 128)).astype(np.float32), torch.bfloat16)
    out = kept.attend(q, slots, positions, run=run, out_dtype=torch.float32)
    want, spread, size = kept.exact(q, slots, positions)
    bound = (2 * spread * 4 * 2.0 ** -21 + 2.0 ** -20 + 2.0 ** -16) * size
    assert bool(((out.double() - want).abs() <= bound[..., None]).all())
