"""verify over rows of several pieces a chunk, several runs a wave and more than 1024 runs, on the GPU against float64."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import rules
from test_gpu_verify import problem

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def compare(x, drafts, u, **kw):
    """x: logits on the GPU."""
    on = {("draft_probs" if k == "probs" else k): dev(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    tokens, accepted = rules.verify(x, dev(drafts), None if u is None else dev(u), **on)
    want_t, want_a = K.verify(x.float().cpu().numpy(), drafts, u, **kw)
    assert np.array_equal(accepted.cpu().numpy(), want_a)
    assert np.array_equal(tokens.cpu().numpy(), want_t)


# (sequences, drafts each, width): pieces a chunk, chunks a row; runs of the draw, waves a sequence.
LONG = [(14, 3, 151936),  # 2, 38; 594, 288
        (40, 1, 151937),  # 2, 38; 594, 96
        (64, 3, 20000),   # 1, 10; 79, 64
        (70, 15, 16500),  # 4, 3; 65, 48
        (1100, 3, 8191),  # 8, 1; 32, 16
        (300, 6, 6145),   # 4, 1; 25, 16
        (2, 1, 600001)]   # 1, 293; 2344, 2048


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["probs", "point", "greedy"])
@pytest.mark.parametrize("seqs,most,width", LONG)
def test_against_float64(seqs, most, width, kind, dtype):
    r = rng(seqs + most + width)
    if kind == "probs" and seqs * most * width > 2e7:
        seqs = max(2, int(2e7 / most / width))  # (the 64-bit form of the probabilities fills the host)
    logits, drafts, u, counts, first, probs = problem(r, seqs, most, width, kind)
    kw = dict(counts=counts, first=first, temperature=1.0 if kind == "greedy" else 0.75)
    if kind == "probs":
        kw["probs"] = probs
    compare(dev(logits, dtype), drafts, None if kind == "greedy" else u, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [8192, 8190])
@pytest.mark.parametrize("greedy", [False, True])
def test_maxima_that_move_from_piece_to_piece(greedy, width, dtype):
    """Four pieces a chunk, one chunk a row: the maximum rises with each, falls, lies in the last, is infinite in
    one, and pieces without any logit lie before, between and behind. Drafts and picks among the ties."""
    seqs, most = 1040, 1
    r, rows = rng(width), 2 * seqs
    x = r.standard_normal((rows, width)).astype(np.float32)
    ramp = np.linspace(-30, 30, width, dtype=np.float32)
    kinds = np.arange(rows) // 2 % 10  # of a sequence's two rows
    x[kinds == 1] += ramp
    x[kinds == 2] -= ramp
    x[kinds == 3, -1] = 50
    x[kinds == 4, 5000] = np.inf
    x[kinds == 4, 3] = np.inf
    x[kinds == 5, :4096] = -np.inf
    x[kinds == 6, 2048:6144] = np.nan
    x[kinds == 7, 2048:] = -np.inf
    x[kinds == 8] = -np.inf
    x[kinds == 9] = 0.0
    t = dev(x, dtype)
    at = t.float().cpu().numpy()
    first_of = np.where(np.isnan(at), -np.inf, at).argmax(-1)[::2]
    drafts = np.where(r.random(seqs) < 0.7, first_of, r.integers(0, width, seqs)).astype(np.int32)[:, None]
    u = r.random((seqs, most + 1)).astype(np.float32)
    compare(t, drafts, None if greedy else u, temperature=1.5)


def test_picks_all_along_a_row():
    """The token at u's place in the running sum, for u over the whole of [0, 1): every run of every wave is drawn."""
    seqs, width = 256, 40000
    x = np.zeros((seqs, width), np.float32)
    u = ((np.arange(seqs) + 0.5) / seqs).astype(np.float32)[:, None]
    drafts = np.zeros((seqs, 0), np.int32)
    tokens, accepted = rules.verify(dev(x), dev(drafts), dev(u))
    want = np.floor(u[:, 0].astype(np.float64) * width).astype(int)  # the first index with index + 1 > u width
    assert np.array_equal(tokens.cpu().numpy()[:, 0], want) and not accepted.any()


def test_two_calls_at_once():
    """On two streams, each with scratch of its own: what each gives alone."""
    r = rng(11)
    problems = [problem(r, 6, 4, 50000, "probs") for _ in range(2)]
    on = [[dev(a) for a in p] for p in problems]

    def call(p):
        logits, drafts, u, counts, first, probs = p
        return rules.verify(logits, drafts, u, counts=counts, first=first, draft_probs=probs)

    alone = [call(p) for p in on]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in on]
    for _ in range(5):
        got = []
        for p, stream in zip(on, streams):
            with torch.cuda.stream(stream):
                got.append(call(p))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(alone, got) for a, b in zip(x, y))
