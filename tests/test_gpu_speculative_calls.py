"""Calls of the 8-bit cache's operators that are empty, refused or unusually laid out, through rules."""
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


def test_empty_batches():
    """No rows, no sequences: empty outputs, nothing written."""
    k8, v8, s8 = rules.kept8(2, 2)
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    x = torch.empty(0, 8, 128, device="cuda")
    q = rules.append_rows(x[:, 4:6], x[:, 6:], k8, v8, i, i, q=x[:, :4], keys=32, scales=s8)
    assert q.shape == (0, 4, 128) and int(k8.count_nonzero()) == int(s8.count_nonzero()) == 0
    rows = torch.zeros(32, 2, 128, dtype=torch.bfloat16, device="cuda")
    assert rules.append_rows(x[:, 4:6], x[:, 6:], rows, rows.clone(), i, i, keys=32) is None
    assert rules.attend_kept8(q, k8, v8, s8, i, i, keys=32, scale=1.0).shape == (0, 4, 128)
    u = torch.empty(0, 4, device="cuda")
    for logits in (torch.empty(0, 50, device="cuda"), torch.zeros(4, 50, device="cuda")):
        for uniforms in (None, u):
            tokens, accepted = rules.verify(logits, torch.empty(0, 3, dtype=torch.int32, device="cuda"), uniforms)
            assert tokens.shape == (0, 4) and accepted.shape == (0,)


def test_sequences_without_a_row_of_logits_are_refused():
    status, one = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for uniforms in (None, torch.zeros(2, 2, device="cuda")):
        status.zero_()
        tokens, accepted = rules.verify(torch.empty(0, 50, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda"),
                                        uniforms, counts=one, first=one, status=status)
        assert tokens.tolist() == [[50, 50]] * 2 and accepted.tolist() == [0, 0] and int(status) == abi.TS_STATUS_POSITION


@pytest.mark.parametrize("many", [0, 1200])
@pytest.mark.parametrize("kept", ["e4m3", "bf16"])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_q_of_rows_without_a_place_is_nan(out, kept, many):
    """Positions past the slot or past its table's pages, slots and pages that are not there: kept nowhere, q NaN;
    the rows beside them, and one refused for meeting a block twice, have theirs."""
    r = rng(3 + many)
    page, each, kvh, heads = 16, 3, 2, 5
    table = np.array([0, 1, 2, 3, 99, 5], np.int32)  # slot 1's second page does not exist
    slots = np.array([0, 0, 1, 2, 0, 0, 1, 0, 0xFFFFFFFF], np.uint32).astype(np.int32)
    # 60 and 47 + 1 are within `keys` but not within the table's three pages.
    positions = np.array([46, 47, 17, 3, 48, 60, 40, 45, 3], np.int32)
    bad = np.array([0, 0, 1, 1, 1, 1, 0, 0, 1], bool)
    bits = abi.TS_STATUS_POSITION | abi.TS_STATUS_PAGE | abi.TS_STATUS_TWICE
    # Beyond 1024 rows a wave takes four of them: others, of a slot that is not there, before these.
    slots, positions = np.append(np.full(many, 7, np.int32), slots), np.append(np.zeros(many, np.int32), positions)
    bad = np.append(np.ones(many, bool), bad)
    n = len(slots)
    x = dev(r.standard_normal((n, heads + 2 * kvh, 128)).astype(np.float32))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    if kept == "e4m3":
        k, v, scales = rules.kept8(6, kvh)
    else:
        k, v, scales = *(torch.zeros(96, kvh, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)), None
    angles = rules.rope_table(64, 1e4)
    q_out = torch.empty(n, heads, 128, dtype=out, device="cuda")
    q = rules.append_rows(x[:, heads:heads + kvh], x[:, heads + kvh:], k, v, dev(slots), dev(positions), q=x[:, :heads],
                          keys=64, scales=scales, table=dev(table), kept_pages=each, page=page, status=status,
                          angles=angles, q_out=q_out)
    assert int(status) == bits
    got = q.double().cpu().numpy()
    assert np.isnan(got[bad]).all()
    want = K.turned(x[:, :heads].cpu().numpy(), None, angles.cpu().numpy(), np.where(bad, 0, positions), True, 0)
    size = np.abs(want).max(-1, keepdims=True)
    # Three f32 steps of the rotation (2^-24 each of the pair's size), and the rounding of bf16.
    slack = size * 2.0 ** -21 + np.abs(want) * (2.0 ** -8 if out == torch.bfloat16 else 0)
    assert np.all((np.abs(got - want) <= slack)[~bad])


@pytest.mark.parametrize("width,off,apart", [(4096, 1, 4097), (777, 3, 777), (1028, 5, 1031), (1, 1, 1)])
@pytest.mark.parametrize("greedy", [False, True])
def test_bf16_logits_at_odd_elements(width, off, apart, greedy):
    """Rows of bf16 logits that begin at an odd element, whole fours wide or not."""
    r = rng(width + off)
    seqs, most = 4, 3
    rows = seqs * (most + 1)
    held = torch.full((off + rows * apart,), 60.0, dtype=torch.bfloat16, device="cuda")
    x = held[off:].view(rows, apart)[:, :width]
    x.copy_(dev((3 * r.standard_normal((rows, width))).astype(np.float32)))
    assert x.data_ptr() % 4 == 2
    at = x.float().cpu().numpy()
    drafts = at.argmax(-1).reshape(seqs, most + 1)[:, :most].astype(np.int32)
    drafts[1, 1] = (drafts[1, 1] + 1) % width
    u = None if greedy else r.random((seqs, most + 1)).astype(np.float32)
    tokens, accepted = rules.verify(x, dev(drafts), None if greedy else dev(u))
    want_t, want_a = K.verify(at, drafts, u)
    assert np.array_equal(accepted.cpu().numpy(), want_a) and np.array_equal(tokens.cpu().numpy(), want_t)


@pytest.mark.parametrize("dtype", [torch.int32, torch.uint32])
def test_positions_of_either_type_without_a_stated_bound(dtype):
    """Their maximum is found of int32 and uint32 positions, beside rows that are refused (2^32 - 1)."""
    r = rng(31)
    k8, v8, s8 = rules.kept8(4, 1)
    x = dev(r.standard_normal((64, 1, 128)).astype(np.float32))
    i = torch.arange(64, dtype=torch.int32, device="cuda")
    rules.append_rows(x, x, k8, v8, torch.zeros_like(i), i, keys=64, scales=s8)
    q = dev(r.standard_normal((3, 2, 128)).astype(np.float32))
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    positions = torch.tensor([63, -1, 5], dtype=torch.int32, device="cuda")
    want = rules.attend_kept8(q, k8, v8, s8, slots, positions, keys=64, scale=0.1, max_position=63)
    got = rules.attend_kept8(q, k8, v8, s8, slots.view(dtype), positions.view(dtype), keys=64, scale=0.1)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    got = rules.attend_kept8(q[1:2], k8, v8, s8, slots[:1].view(dtype), positions[1:2].view(dtype), keys=64, scale=0.1)
    assert torch.isnan(got).all()


@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("halves", [True, False])
def test_values_that_pass_f32_on_the_way_to_their_codes(one, halves):
    """A rotation (or a gain) that takes finite values past f32's range: as the formula has it, the largest code of
    the largest scale, of their sign, and no NaN; what was infinite or NaN before is a NaN code."""
    r = rng(41)
    n = 1 if one else 16
    x = (r.standard_normal((n, 1, 128)) * 1e30).astype(np.float32)
    pairs = ([3, 67], [5, 69]) if halves else ([6, 7], [10, 11])
    x[:, 0, pairs[0]] = 3.3e38, -3.3e38
    x[:, 0, pairs[1]] = -3.3e38, 3.3e38
    x[0, 0, 20], x[-1, 0, 31] = np.inf, np.nan
    turn = np.zeros((16, 64, 2), np.float32)
    turn[...] = np.sqrt(0.5)
    i = np.arange(n, dtype=np.int32)
    k8, v8, s8 = rules.kept8(1, 1)
    rules.append_rows(dev(x), dev(x), k8, v8, dev(np.zeros(n, np.int32)), dev(i), keys=16, scales=s8, angles=dev(turn),
                      halves=halves)
    blocks, scales = np.zeros((1, 1, 16, 128), np.uint8), np.zeros((1, 2, 2))
    want = K.turned(x, None, turn, i, halves, 0)
    assert np.abs(want[np.isfinite(want)]).max() > np.finfo(np.float32).max
    K.append(blocks, scales, 0, want, np.zeros(n), i, keys=16)
    got = k8.cpu().numpy()
    assert s8[0, 0, 0].item() == scales[0, 0, 0] == 2.0 ** 119
    assert np.array_equal(K.CODES[got], K.CODES[blocks], equal_nan=True) and np.isnan(K.CODES[got[0, 0, :n]]).sum() == 4
