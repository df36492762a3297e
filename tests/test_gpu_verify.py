"""verify on the GPU against the float64 form: tokens and counts are equal."""
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


def problem(r, seqs, most, width, kind, ragged=True):
    """Logits with a few likely tokens, drafts of a drafter near the target."""
    counts = r.integers(0, most + 1, seqs).astype(np.int32) if ragged else np.full(seqs, most, np.int32)
    first = np.concatenate([[0], np.cumsum(counts + 1)])
    rows = int(first[-1])
    logits = (2 * r.standard_normal((rows, width))).astype(np.float32)
    logits[np.arange(rows), r.integers(0, width, rows)] += 8
    logits[np.arange(rows), r.integers(0, width, rows)] += 7
    at = np.minimum(first[:-1, None] + np.minimum(np.arange(most), counts[:, None]), rows - 1)
    near = logits[at] + 0.5 * r.standard_normal((seqs, most, width)).astype(np.float32)
    e = np.exp(near - near.max(-1, keepdims=True, initial=-1e30)) if most else near
    probs = (e / e.sum(-1, keepdims=True)).astype(np.float32) if most else near
    if kind == "probs":
        x = r.random((seqs, most, 1))
        drafts = np.minimum((probs.astype(np.float64).cumsum(-1) < x).sum(-1), width - 1)
    else:
        drafts = near.argmax(-1) if most else np.zeros((seqs, 0))
    u = r.random((seqs, most + 1)).astype(np.float32)
    return logits, drafts.astype(np.int32), u, counts, first[:-1].astype(np.int32), probs


def compare(logits, drafts, u, dtype=torch.float32, **kw):
    x = dev(logits, dtype)
    on = {k: dev(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    if "probs" in on:
        on["draft_probs"] = on.pop("probs")
    tokens, accepted = rules.verify(x, dev(drafts), None if u is None else dev(u), **on)
    want_t, want_a = K.verify(x.float().cpu().numpy(), drafts, u, **kw)
    assert np.array_equal(accepted.cpu().numpy(), want_a)
    assert np.array_equal(tokens.cpu().numpy(), want_t)
    return want_t, want_a


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["probs", "point", "greedy"])
@pytest.mark.parametrize("seqs,most,width", [(1, 1, 1), (1, 4, 50), (7, 3, 255), (3, 8, 4096), (5, 5, 4097), (2, 64, 1000),
                                            (4, 4, 50257), (2, 2, 151936), (300, 1, 33), (3, 0, 777)])
def test_against_float64(seqs, most, width, kind, dtype):
    r = rng(seqs * 1000 + most + width)
    logits, drafts, u, counts, first, probs = problem(r, seqs, most, width, kind)
    kw = dict(counts=counts, first=first)
    if kind == "probs":
        kw["probs"] = probs
    temperature = 1.0 if kind == "greedy" else [0.5, 1.0, 1.75][seqs % 3]
    compare(logits, drafts, None if kind == "greedy" else u, dtype, temperature=temperature, **kw)


def test_without_counts_and_first():
    r = rng(1)
    logits, drafts, u, _, _, probs = problem(r, 6, 3, 900, "probs", ragged=False)
    compare(logits, drafts, u, probs=probs)
    compare(logits, drafts, None)


def test_each_sequence_its_temperature():
    """0, negative and NaN are greedy, beside sampled sequences of the same call."""
    r = rng(2)
    logits, drafts, u, counts, first, probs = problem(r, 6, 4, 5000, "probs")
    t = np.array([0.0, 0.7, -1.0, 2.0, np.nan, 1.0], np.float32)
    compare(logits, drafts, u, counts=counts, first=first, probs=probs, temperature=t)


def test_masked_infinite_and_nan_logits():
    """-inf and NaN have no probability, a row of nothing else none to pick; +inf shares the whole; ties
    go to the lowest index."""
    r = rng(3)
    width = 9000
    logits, drafts, u, _, _, _ = problem(r, 8, 2, width, "point", ragged=False)
    logits[0, 10:] = -np.inf
    logits[1] = np.nan
    logits[1, 4500] = 1.0
    drafts[0] = 3, 4500
    logits[3] = -np.inf
    logits[6] = np.nan
    logits[9, [7, 8000]] = np.inf
    drafts[3] = 8000, 1
    logits[12] = 0.0
    logits[15] = -3.0e38
    drafts[6, 0] = width  # no token of the vocabulary
    drafts[7, 1] = -1
    compare(logits, drafts, u)
    compare(logits, drafts, None)


@pytest.mark.parametrize("edge", [0.0, float(np.nextafter(np.float32(1), np.float32(0)))])
def test_uniforms_at_their_ends(edge):
    """u = 0 takes every draft that has a chance and the first index with weight; u just below 1 the last."""
    r = rng(4)
    logits, drafts, u, counts, first, probs = problem(r, 5, 3, 10000, "probs")
    logits[:, :3] = -np.inf
    logits[:, -2:] = -np.inf
    compare(logits, drafts, np.full_like(u, edge), counts=counts, first=first, probs=probs)


def test_draft_probabilities_that_are_none():
    """NaN and negative ones count as 0; a drafter surer than the target everywhere leaves p itself."""
    r = rng(5)
    logits, drafts, u, counts, first, probs = problem(r, 6, 2, 3000, "probs")
    probs[0], probs[1, :, ::2], probs[2, :, 1::2] = 2.0, np.nan, -1.0
    compare(logits, drafts, u, counts=counts, first=first, probs=probs)


def test_sequences_out_of_range_are_refused():
    """More drafts than there is room for, rows past the last: nothing accepted, `width` throughout, the
    status bit; the others as alone."""
    r = rng(6)
    logits, drafts, u, counts, first, probs = problem(r, 5, 3, 600, "probs", ragged=False)
    counts[1], first[3] = 4, len(logits) - 3
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for uniforms in (u, None):
        status.zero_()
        tokens, accepted = rules.verify(dev(logits), dev(drafts), None if uniforms is None else dev(uniforms),
                                        counts=dev(counts), first=dev(first), draft_probs=dev(probs), status=status)
        want_t, want_a = K.verify(logits, drafts, uniforms, counts=counts, first=first, probs=probs)
        assert np.array_equal(tokens.cpu().numpy(), want_t) and np.array_equal(accepted.cpu().numpy(), want_a)
        assert int(status) == abi.TS_STATUS_POSITION and want_t[1].tolist() == [600] * 4 == want_t[3].tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,off_x,off_q", [(4096, 0, 1), (4096, 1, 0), (1028, 4, 4), (4, 0, 0), (2052, 2, 3)])
def test_any_alignment(width, off_x, off_q, dtype):
    """Logits and probabilities that begin anywhere; rows of whole fours and a last run that is not full."""
    r = rng(width + off_x)
    logits, drafts, u, counts, first, probs = problem(r, 6, 4, width, "probs")
    x = torch.empty(logits.size + 8, dtype=dtype, device="cuda")[2 * off_x:][:logits.size].view(logits.shape)
    q = torch.empty(probs.size + 4, device="cuda")[off_q:][:probs.size].view(probs.shape)
    x.copy_(dev(logits))
    q.copy_(dev(probs))
    tokens, accepted = rules.verify(x, dev(drafts), dev(u), counts=dev(counts), first=dev(first), draft_probs=q)
    want_t, want_a = K.verify(x.float().cpu().numpy(), drafts, u, counts=counts, first=first, probs=probs)
    assert np.array_equal(accepted.cpu().numpy(), want_a) and np.array_equal(tokens.cpu().numpy(), want_t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_apart(dtype):
    """Rows of a padded product (odd distance), and given outputs."""
    r = rng(7)
    logits, drafts, u, counts, first, probs = problem(r, 4, 3, 777, "probs")
    wide = torch.zeros(len(logits), 801, dtype=dtype, device="cuda")
    wide[:, :777] = dev(logits)
    view = wide[:, :777]
    tokens = torch.full((4, 4), -5, dtype=torch.int32, device="cuda")
    got = rules.verify(view, dev(drafts), dev(u), counts=dev(counts), first=dev(first), draft_probs=dev(probs), tokens=tokens)
    want = K.verify(view.float().cpu().numpy(), drafts, u, counts=counts, first=first, probs=probs)
    assert got[0] is tokens and np.array_equal(tokens.cpu().numpy(), want[0])
    assert np.array_equal(got[1].cpu().numpy(), want[1])


def test_captured_and_replayed():
    r = rng(8)
    logits, drafts, u, counts, first, probs = problem(r, 6, 4, 20000, "probs")
    x, ud = dev(logits), dev(u)
    args = dict(counts=dev(counts), first=dev(first), draft_probs=dev(probs))
    dd = dev(drafts)
    rules.verify(x, dd, ud, **args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tokens, accepted = rules.verify(x, dd, ud, **args)
    for _ in range(3):
        ud.copy_(dev(r.random(u.shape).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        want = rules.verify(x, dd, ud, **args)
        assert torch.equal(tokens, want[0]) and torch.equal(accepted, want[1])
