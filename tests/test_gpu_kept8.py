"""attend_kept8 on the GPU against the float64 form over the same blocks."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def build(r, lengths, kvh, page, dense=False):
    """Blocks of random values for slots of `lengths` positions; everything past them is any byte."""
    each = max(1, -(-max(lengths) // page))
    pages = len(lengths) * each + (0 if dense else 1)
    table = np.arange(pages).astype(np.int32) if dense else r.permutation(pages).astype(np.int32)[:len(lengths) * each]
    blocks = pages * page // 16
    k, v = (r.integers(0, 256, s).astype(np.uint8) for s in ((blocks, kvh, 16, 128), (blocks, kvh, 128, 16)))
    even = (kvh + 1) // 2 * 2
    scales = np.exp2(r.integers(-9, -6, (blocks, even, 2))).astype(np.float32)
    where = dict(keys=each * page, table=table, kept_pages=each, page=page)
    for s, n in enumerate(lengths):
        for j in range(n):
            row = K.kept_row(s, j, **where)
            b, o = row // 16, row % 16
            k[b, :, o] = K.narrow(r.standard_normal((kvh, 128)) / scales[b, :kvh, 0, None])
            v[b, :, :, o] = K.narrow(r.standard_normal((kvh, 128)) / scales[b, :kvh, 1, None])
    if dense:
        where = dict(keys=each * page)
    return k, v, scales, where, pages


def call(q, k, v, scales, slots, positions, where, page, **kw):
    args = dict(where)
    if "table" in args:
        args["table"] = dev(args["table"])
    args["page"] = page
    return rules.attend_kept8(q, dev(k), dev(v), dev(scales), dev(np.asarray(slots, np.int32)),
                              dev(np.asarray(positions, np.int32)), scale=kw.pop("scale", SCALE), **args, **kw)


def bound(spread, size, f32):
    """A score's error: f32 q enters as three bf16 parts, |q| 2^-24 off at most, and 128 products are summed
    at 2^-21 each accumulating step (4 a part): spread (2^-24 + 12 2^-21), of bf16 q spread 4 2^-21. A weight
    is then off by twice that (its own and the sum's), by 2^-20 of the exponential and the sums and by its
    rounding (three parts 2^-24, one 2^-9, half a step of bf16 2^-8); the output by that times the largest
    |v|, plus its own rounding."""
    score = spread * (2.0 ** -24 + 12 * 2.0 ** -21 if f32 else 4 * 2.0 ** -21)
    return (2 * score + 2.0 ** -20 + (2.0 ** -24 if f32 else 2.0 ** -8)) * size + (0 if f32 else 2.0 ** -8 * size)


def check(out, want, spread, size, f32):
    got = out.float().cpu().numpy()
    assert np.all(np.abs(got - want) <= bound(spread, size, f32)[..., None])
    # Over all of it the errors average: their norm is far below the bound.
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel < (1e-5 if f32 else 4e-3), rel


TYPES = [("f32", torch.float32, True), ("bf16", torch.bfloat16, False)]


@pytest.mark.parametrize("name,dtype,f32", TYPES)
@pytest.mark.parametrize("heads,kvh,page", [(1, 1, 16), (16, 8, 16), (10, 2, 64), (24, 8, 32), (64, 1, 16), (33, 3, 16)])
def test_decode_rows(heads, kvh, page, name, dtype, f32):
    """One row a slot, from a single key to several parts; ratios that do not divide the 16 columns."""
    r = rng(heads + page)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 300, 1025]
    k, v, scales, where, _ = build(r, lengths, kvh, page)
    n = len(lengths)
    q = dev(r.standard_normal((n, heads, 128)).astype(np.float32), dtype)
    slots, positions = np.arange(n)[::-1], (np.array(lengths) - 1)[::-1]
    out = call(q, k, v, scales, slots, positions, where, page, out_dtype=dtype)
    check(out, *K.attend(q.float().cpu().numpy(), k, v, scales, slots, positions, scale=SCALE, **where), f32)


@pytest.mark.parametrize("name,dtype,f32", TYPES)
@pytest.mark.parametrize("heads,kvh,run,back", [(16, 8, 5, None), (8, 1, 8, None), (6, 2, 3, 100), (16, 8, 40, None),
                                               (4, 4, 130, 33), (64, 8, 9, 0), (40, 8, 17, 64)])
def test_runs_of_rows(heads, kvh, run, back, name, dtype, f32):
    """Drafted rows and prompt chunks: `run` rows of each slot over shared keys, with windows."""
    r = rng(run + heads)
    lengths = [run, run + 16, 2 * run + 77]
    k, v, scales, where, _ = build(r, lengths, kvh, 16)
    slots = np.repeat(np.arange(3), run)
    positions = np.concatenate([n - run + np.arange(run) for n in lengths])
    q = dev(r.standard_normal((3 * run, heads, 128)).astype(np.float32), dtype)
    kw = {} if back is None else {"back": back}
    out = call(q, k, v, scales, slots, positions, where, 16, run=run, out_dtype=dtype, **kw)
    check(out, *K.attend(q.float().cpu().numpy(), k, v, scales, slots, positions, scale=SCALE, back=back, **where), f32)


@pytest.mark.parametrize("run", [1, 2, 7, 64, 1000])
@pytest.mark.parametrize("name,dtype,f32", TYPES)
def test_any_run_hint_and_any_order(run, name, dtype, f32):
    """Ragged rows of many slots, packed and shuffled, under hints that fit none of them."""
    r = rng(run)
    lengths = [40, 1, 90, 17, 200, 33]
    k, v, scales, where, _ = build(r, lengths, 2, 32)
    slots = np.repeat(np.arange(6), [30, 1, 44, 17, 2, 20])
    positions = np.concatenate([n - m + np.arange(m) for n, m in zip(lengths, [30, 1, 44, 17, 2, 20])])
    if run == 7:
        order = r.permutation(len(slots))
        slots, positions = slots[order], positions[order]
    q = dev(r.standard_normal((len(slots), 6, 128)).astype(np.float32), dtype)
    out = call(q, k, v, scales, slots, positions, where, 32, run=run, out_dtype=dtype)
    check(out, *K.attend(q.float().cpu().numpy(), k, v, scales, slots, positions, scale=SCALE, **where), f32)


@pytest.mark.parametrize("run", [1, 4, 100])
def test_dense_rows(run):
    r = rng(3)
    lengths = [120, 128]
    k, v, scales, where, _ = build(r, lengths, 3, 16, dense=True)
    slots = np.repeat([0, 1], run)
    positions = np.concatenate([n - run + np.arange(run) for n in lengths])
    q = dev(r.standard_normal((2 * run, 6, 128)).astype(np.float32))
    out = call(q, k, v, scales, slots, positions, where, 16, run=run)
    check(out, *K.attend(q.cpu().numpy(), k, v, scales, slots, positions, scale=SCALE, **where), True)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
@pytest.mark.parametrize("run", [1, 70])
def test_scales_of_the_scores(scale, run):
    r = rng(4)
    k, v, scales, where, _ = build(r, [200], 1, 16)
    positions = 199 - run + 1 + np.arange(run)
    q = dev(r.standard_normal((run, 2, 128)).astype(np.float32))
    out = call(q, k, v, scales, np.zeros(run), positions, where, 16, run=run, scale=scale)
    want, spread, size = K.attend(q.cpu().numpy(), k, v, scales, np.zeros(run), positions, scale=scale, **where)
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound(spread, size, True)[..., None])


@pytest.mark.parametrize("run", [1, 6, 80])
def test_nan_reaches_only_the_rows_that_see_it(run):
    """A NaN key spoils the rows that see it, a NaN value its own column of theirs; the rows before it and
    those whose window has left it are as without it."""
    r = rng(5)
    n, back = 150, 40
    k, v, scales, where, _ = build(r, [n], 2, 16)
    positions = np.arange(n - run, n)
    q = dev(r.standard_normal((run, 4, 128)).astype(np.float32))
    clean = call(q, k, v, scales, np.zeros(run), positions, where, 16, run=run, back=back).cpu().numpy()
    for at in (n - 1, n - run // 2 - 1, max(0, n - run - 20)):
        row = K.kept_row(0, at, **where)
        b, o = row // 16, row % 16
        sees = (positions >= at) & (positions - back <= at)
        k2, v2 = k.copy(), v.copy()
        k2[b, 1, o, 7] = 0xFF
        v2[b, 0, 9, o] = 0x7F
        got = call(q, k2, v2, scales, np.zeros(run), positions, where, 16, run=run, back=back).cpu().numpy()
        want = np.zeros(clean.shape, bool)
        want[sees, 2:] = True
        want[sees, :2, 9] = True
        assert np.array_equal(np.isnan(got), want)
        assert np.allclose(got[~want], clean[~want], rtol=0, atol=1e-5)


@pytest.mark.parametrize("run", [1, 5, 90])
def test_refused_rows(run):
    """Positions past the slot, the table or the stated bound, slots and pages out of range: NaN and a
    status bit; the slots beside them as alone."""
    r = rng(6)
    k, v, scales, where, pages = build(r, [128, 128, 128], 2, 16)
    each = where["kept_pages"]
    q = dev(r.standard_normal((3 * run, 4, 128)).astype(np.float32))
    slots = np.repeat(np.arange(3), run)
    positions = np.tile(np.arange(128 - run, 128), 3)
    clean = call(q, k, v, scales, slots, positions, where, 16, run=run, max_position=127)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def spoilt(bit, slots=slots, positions=positions, where=where, most=127, lost=None):
        status.zero_()
        got = call(q, k, v, scales, slots, positions, where, 16, run=run, max_position=most, status=status)
        assert int(status) == bit
        lost = np.arange(3 * run) // run == 1 if lost is None else lost
        assert torch.isnan(got[dev(lost)]).all() and torch.equal(got[dev(~lost)], clean[dev(~lost)])

    bad = positions.copy()
    bad[run:2 * run] += 128 + run
    spoilt(abi.TS_STATUS_POSITION, positions=bad)
    spoilt(abi.TS_STATUS_POSITION, positions=bad, most=10000)
    out = slots.copy()
    out[run:2 * run] = 3
    spoilt(abi.TS_STATUS_PAGE, slots=out)
    table = where["table"].copy()
    table[each + 7] = pages
    # Rows that see none of the missing page's keys (112 on) are as they were.
    spoilt(abi.TS_STATUS_PAGE, where=dict(where, table=table), lost=(slots == 1) & (positions >= 112))


@pytest.mark.parametrize("name,dtype,f32", TYPES)
@pytest.mark.parametrize("seqs,run,heads,kvh,back", [(70, 1, 2, 1, None), (200, 1, 6, 3, 150), (260, 1, 2, 1, None),
                                                     (90, 3, 16, 1, None), (258, 3, 12, 1, 100), (20, 40, 4, 2, None)])
def test_many_ragged_sequences(seqs, run, heads, kvh, back, name, dtype, f32):
    """More sequences than one lane each of a wave, than the groups that share keys take, and tiles that begin
    in one sequence and end in another: lengths of `run` to 640, shared out in runs that begin and end anywhere."""
    r = rng(seqs + run)
    page, each = 16, 40
    blocks = seqs * each
    table = r.permutation(blocks).astype(np.int32)
    k, v = (r.integers(0, 256, s).astype(np.uint8) for s in ((blocks, kvh, 16, 128), (blocks, kvh, 128, 16)))
    for x in (k, v):
        x[(x & 0x7F) == 0x7F] = 0
    scales = np.exp2(r.integers(-9, -6, (blocks, (kvh + 1) // 2 * 2, 2))).astype(np.float32)
    where = dict(keys=each * page, table=table, kept_pages=each, page=page)
    counts = r.integers(1, run + 1, seqs)  # rows of each sequence
    lengths = np.maximum(r.integers(1, 641, seqs), counts)
    slots = np.repeat(r.permutation(seqs), counts)
    positions = np.concatenate([lengths[s] - n + np.arange(n) for s, n in zip(range(seqs), counts)])
    q = dev((r.standard_normal((len(slots), heads, 128)) / 8).astype(np.float32), dtype)
    kw = {} if back is None else {"back": back}
    out = call(q, k, v, scales, slots, positions, where, page, out_dtype=dtype, run=run, **kw)
    check(out, *K.attend(q.float().cpu().numpy(), k, v, scales, slots, positions, scale=SCALE, back=back, **where), f32)


def test_many_parts_and_offsets_past_32_bits():
    """A cache of more than 4 GiB of codes, a long slot at its end: split over many groups."""
    kvh, page, n = 8, 64, 20000
    pages = (5 << 30) // (page * kvh * 128)
    k, v, scales = rules.kept8(pages, kvh, page=page)
    each = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    blocks = each * page // 16
    for t in (k, v):
        x = torch.randn(blocks, *t.shape[1:], generator=g, device="cuda") * 60
        t[-blocks:] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[-blocks:] = 2.0 ** -6
    table = torch.arange(pages - each, pages, dtype=torch.int32, device="cuda")
    q = torch.randn(1, 16, 128, generator=g, device="cuda")
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = rules.attend_kept8(q, k, v, scales, i, i + n - 1, keys=each * page, scale=SCALE, table=table, kept_pages=each,
                             page=page)
    kk = k[-blocks:].view(torch.float8_e4m3fn).double().transpose(0, 1).reshape(kvh, -1, 128)[:, :n] / 64
    vv = v[-blocks:].view(torch.float8_e4m3fn).double().transpose(2, 3).transpose(0, 1).reshape(kvh, -1, 128)[:, :n] / 64
    x = torch.matmul(kk, q.double().view(kvh, 2, 128).transpose(1, 2).contiguous()).transpose(1, 2) * SCALE
    want = torch.matmul(torch.softmax(x, -1), vv).reshape(1, 16, 128)
    assert float((out - want).norm() / want.norm()) < 1e-5


def test_captured_and_replayed():
    """One captured call replayed over changing inputs equals the eager one, bit for bit; two graphs share
    no scratch."""
    r = rng(9)
    k, v, scales, where, _ = build(r, [3000, 900], 2, 16)
    kd, vd, sd, table = dev(k), dev(v), dev(scales), dev(where["table"])
    q = [dev(r.standard_normal((2, 8, 128)).astype(np.float32)) for _ in range(2)]
    slots, positions = dev(np.arange(2, dtype=np.int32)), dev(np.array([2999, 899], np.int32))
    kw = dict(keys=where["keys"], scale=SCALE, table=table, kept_pages=where["kept_pages"], max_position=2999)
    run = lambda i: rules.attend_kept8(q[i], kd, vd, sd, slots, positions, **kw)  # noqa: E731
    run(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(i))
        graphs.append(g)
    for i in range(3):
        for j in range(2):
            q[j].copy_(dev(r.standard_normal((2, 8, 128)).astype(np.float32)))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert torch.equal(outs[j], run(j))
