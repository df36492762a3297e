"""append_rows beyond 1024 rows of a call, where a group looks at 16 rows: decode rows, drafts and prompts mixed."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 1e-6


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


FORMS = {
    "decode": lambda r: [1] * 1300,
    "drafts": lambda r: r.integers(1, 10, 300).tolist(),
    "mixed": lambda r: r.choice([1, 1, 1, 2, 5, 16, 17, 33, 90], 200).tolist(),
    "edge": lambda r: [1] * 1025,
}


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("kept", ["e4m3", "bf16"])
@pytest.mark.parametrize("form,heads,kvh", [("decode", 2, 1), ("decode", 6, 3), ("decode", 16, 8), ("drafts", 5, 5),
                                            ("drafts", 16, 8), ("mixed", 6, 2), ("mixed", 9, 9), ("edge", 4, 2)])
def test_many_short_runs(form, heads, kvh, kept, x):
    """Runs that begin and end anywhere in a group's 16 rows, every one at a position of its own: q, the codes and the
    scales, and what no row of the call writes."""
    r = rng(heads * 10 + kvh)
    counts = FORMS[form](r)
    slots_n, page = len(counts), 32
    past = r.integers(0, 40, slots_n)
    each = int(max(p + n for p, n in zip(past, counts)) // page + 1)
    keys, pages = each * page, slots_n * each + 1
    assert sum(counts) > 1024
    table = r.permutation(pages)[:slots_n * each].astype(np.int32)
    order = r.permutation(slots_n)
    slots = np.concatenate([np.full(counts[s], s) for s in order]).astype(np.int32)
    positions = np.concatenate([past[s] + np.arange(counts[s]) for s in order]).astype(np.int32)
    n, where = len(slots), dict(keys=keys, table=table, kept_pages=each, page=page)
    t = dev((r.standard_normal((n, heads + 2 * kvh, 128)) * np.exp(r.standard_normal((n, 1, 1)))).astype(np.float32),
            torch.float32 if x == "f32" else torch.bfloat16)
    gain = (1 + 0.1 * r.standard_normal((2, 128))).astype(np.float32)
    angles = rules.rope_table(keys, 1e4)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    blocks = pages * page // 16
    if kept == "e4m3":
        old = r.integers(0, 256, (2, blocks, kvh, 16, 128)).astype(np.uint8)
        scales = 2.0 ** r.integers(-9, -4, (blocks, kvh, 2))
        held = np.zeros((blocks, (kvh + 1) // 2 * 2, 2), np.float32)
        held[:, :kvh] = scales
        k, v, s8 = dev(old[0]), dev(old[1].transpose(0, 1, 3, 2)), dev(held)
    else:
        k, v = (torch.full((pages * page, kvh, 128), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        s8 = None
    q = rules.append_rows(t[:, heads:heads + kvh], t[:, heads + kvh:], k, v, dev(slots), dev(positions), q=t[:, :heads],
                          q_gain=dev(gain[0]), k_gain=dev(gain[1]), angles=angles, eps=EPS, scales=s8, status=status,
                          keys=keys, table=dev(table), kept_pages=each, page=page)
    assert int(status) == 0
    ref, turns = t.float().cpu().numpy(), angles.cpu().numpy()
    eps = float(np.float32(EPS))
    want_q = K.turned(ref[:, :heads], gain[0], turns, positions, True, eps)
    new = [K.turned(ref[:, heads:heads + kvh], gain[1], turns, positions, True, eps), ref[:, heads + kvh:].astype(np.float64)]

    def near(got, want, rounding):
        # f32 steps of the norm and the rotation (2^-20 of twice the row's largest), and the type's rounding.
        size = np.abs(want).max(-1, keepdims=True)
        return np.all(np.abs(got - want) <= size * 2 * 2.0 ** -20 + np.abs(want) * rounding)

    assert near(q.float().cpu().numpy(), want_q, 2.0 ** -8 if x == "bf16" else 0)
    if kept == "e4m3":
        got = k.cpu().numpy(), v.cpu().numpy().transpose(0, 1, 3, 2)
        for which in (0, 1):
            want_c, want_s = old[which].copy(), scales.copy()
            K.append(want_c, want_s, which, new[which], slots, positions, **where)
            assert np.array_equal(s8.cpu().numpy()[:, :kvh, which], want_s[..., which])
            assert np.array_equal(K.CODES[got[which]], K.CODES[want_c], equal_nan=True)
    else:
        at = np.array([K.kept_row(int(s), int(p), **where) for s, p in zip(slots, positions)])
        rest = np.ones(pages * page, bool)
        rest[at] = False
        for got, want in zip((k, v), new):
            y = got.float().cpu().numpy()
            assert near(y[at], want, 2.0 ** -8) and np.all(y[rest] == 3.0)


@pytest.mark.parametrize("kept", ["e4m3", "bf16"])
def test_refusals_among_many_rows(kept):
    """Beyond 1024 rows: a block met again far behind its first rows, positions and slots out of range in the midst
    of a group's 16 rows. Nothing of them is kept, the others are as without them."""
    r = rng(77)
    kvh, keys, slots_n = 3, 64, 1200
    slots = r.permutation(slots_n).astype(np.int32)
    positions = r.integers(0, keys, slots_n).astype(np.int32)
    x = dev(r.standard_normal((slots_n + 3, kvh, 128)).astype(np.float32))
    where = np.array([5, 700, 1190])  # before these rows of the call
    extra_slots = np.array([slots_n, slots[3], slots[2]], np.int32)
    extra_positions = np.array([0, keys, positions[2]], np.int32)

    def run(slots, positions, x):
        if kept == "e4m3":
            k, v, s = rules.kept8(slots_n * keys // 16, kvh)
        else:
            (k, v), s = (torch.zeros(slots_n * keys, kvh, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)), None
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        rules.append_rows(x, x, k, v, dev(slots), dev(positions), keys=keys, scales=s, status=status)
        return k, v, s, int(status)

    good = run(slots, positions, x[:slots_n])
    at = np.insert(np.arange(slots_n), where, np.arange(slots_n, slots_n + 3))
    got = run(np.insert(slots, where, extra_slots), np.insert(positions, where, extra_positions), x[dev(at)])
    assert good[3] == 0 and got[3] == abi.TS_STATUS_POSITION | abi.TS_STATUS_PAGE | abi.TS_STATUS_TWICE
    assert all(a is b or torch.equal(a, b) for a, b in zip(got[:3], good[:3]))
