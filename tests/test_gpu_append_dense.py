"""append_rows into dense kept rows (no page table): bf16 rows of any count, blocks of any page."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


@pytest.mark.parametrize("keys,slots_n", [(1, 1), (5, 1), (5, 7), (20, 1), (20, 3), (100, 2), (47, 40)])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_bf16_rows_of_any_count(keys, slots_n, x):
    """Slots of `keys` positions one behind the other: a slot's first 16 rows begin anywhere, runs of rows cross
    borders of 16 positions. Each value is its rounding (half a step of bf16, 2^-8), the rest as it was; a row past
    its slot is refused and leaves the next slot's first row alone."""
    r = rng(keys + slots_n)
    kvh, heads = 3, 6
    kept = [torch.full((slots_n * keys, kvh, 128), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    past = r.integers(0, keys, slots_n)
    counts = [int(r.integers(1, keys - p + 1)) for p in past]
    slots = np.repeat(np.arange(slots_n), counts).astype(np.int32)
    positions = np.concatenate([p + np.arange(n) for p, n in zip(past, counts)]).astype(np.int32)
    slots, positions = np.append(slots, 0).astype(np.int32), np.append(positions, -(-keys // 16) * 16).astype(np.int32)
    n = len(slots)
    t = dev(r.standard_normal((n, heads + 2 * kvh, 128)).astype(np.float32), torch.float32 if x == "f32" else torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = rules.append_rows(t[:, heads:heads + kvh], t[:, heads + kvh:], *kept, dev(slots), dev(positions), q=t[:, :heads],
                          keys=keys, status=status)
    assert int(status) == abi.TS_STATUS_POSITION and torch.isnan(q[-1]).all() and torch.equal(q[:-1], t[:-1, :heads])
    at = slots[:-1].astype(np.int64) * keys + positions[:-1]
    for got, want in zip(kept, (t[:-1, heads:heads + kvh], t[:-1, heads + kvh:])):
        y, w = got.double().cpu().numpy(), want.double().cpu().numpy()
        assert np.all(np.abs(y[at] - w) <= np.abs(w) * 2.0 ** -8)
        rest = np.ones(len(y), bool)
        rest[at] = False
        assert np.all(y[rest] == 3.0)


@pytest.mark.parametrize("page", [16, 64])
def test_blocks_that_are_not_whole_pages(page):
    """Dense blocks have no pages: 10 of them serve under any page, for appends and attention."""
    r = rng(page)
    kvh, keys = 2, 80
    k8, v8, s8 = rules.kept8(10, kvh)
    slots = np.repeat(np.arange(2), keys).astype(np.int32)
    positions = np.tile(np.arange(keys), 2).astype(np.int32)
    x = r.standard_normal((2 * keys, kvh, 128)).astype(np.float32)
    rules.append_rows(dev(x), dev(x), k8, v8, dev(slots), dev(positions), keys=keys, scales=s8, page=page)
    blocks, scales = np.zeros((10, kvh, 16, 128), np.uint8), np.zeros((10, kvh, 2))
    K.append(blocks, scales, 0, x.astype(np.float64), slots, positions, keys=keys)
    assert np.array_equal(k8.cpu().numpy(), blocks) and np.array_equal(s8.cpu().numpy()[..., 0], scales[..., 0])
    assert np.array_equal(v8.cpu().numpy().transpose(0, 1, 3, 2), blocks)
    q = dev(r.standard_normal((2, 4, 128)).astype(np.float32))
    i, p = np.arange(2, dtype=np.int32), np.array([79, 40], np.int32)
    out = rules.attend_kept8(q, k8, v8, s8, dev(i), dev(p), keys=keys, scale=128 ** -0.5, page=page)
    want, spread, size = K.attend(q.cpu().numpy(), k8.cpu().numpy(), v8.cpu().numpy(), s8.cpu().numpy().astype(float), i, p,
                                  scale=128 ** -0.5, keys=keys)
    # A score: q in three bf16 parts (2^-24), 12 accumulating steps at 2^-21; a weight twice that, its exponential
    # and its own rounding (2^-20).
    bound = (2 * spread * (2.0 ** -24 + 12 * 2.0 ** -21) + 2.0 ** -20) * size
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound[..., None])
