"""Speculative decoding over an 8-bit paged cache, as a server runs it: pages from the pool, a fork, appended
rows, attention of drafted rows, verification, truncation to what was accepted."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import kv, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE, EACH, KVH, HEADS, WIDTH, MOST = 16, 12, 2, 6, 300, 4
KEYS, SCALE = PAGE * EACH, 128 ** -0.5
WHERE = dict(keys=KEYS, kept_pages=EACH, page=PAGE)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Model:
    """One layer of attention whose next token is, but for e^-40 or so, the successor of the last one."""

    def __init__(self, r):
        self.embed = (r.standard_normal((WIDTH, HEADS + 2 * KVH, 128)) * np.exp(r.standard_normal((WIDTH, 1, 1)))).astype(np.float32)
        self.after = r.permutation(WIDTH)
        self.head = dev((r.standard_normal((HEADS * 128, WIDTH)) / 64).astype(np.float32))
        a = np.arange(KEYS)[:, None] * 1e4 ** (-np.arange(64) / 64)
        self.angles = np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)

    def logits(self, out, tokens):
        x = out.flatten(1) @ self.head
        x = 4 * torch.tanh(x)
        x[torch.arange(len(tokens)), dev(self.after[tokens])] += 48
        return x


class Server:
    def __init__(self, r, slots):
        self.m, self.pool = Model(r), kv.Pool(slots * EACH, PAGE)
        self.k, self.v, self.scales = rules.kept8(slots * EACH, KVH, PAGE)
        self.table = np.full((slots, EACH), 0xFFFFFFFF, np.uint32)
        self.angles = dev(self.m.angles)
        self.kept = {}  # (slot, position): the token kept there

    def pages(self, slot, run):
        held = self.pool.pages(run)
        self.table[slot] = 0xFFFFFFFF
        self.table[slot, :len(held)] = held

    def grow(self, slot, run, rows):
        copies = self.pool.grow(run, rows)
        if copies:
            kv.copy_kept8(self.k, self.v, self.scales, copies, page=PAGE)
        self.pages(slot, run)
        return len(copies)

    def rows(self, slots, positions, tokens, run, back=None):
        """The tokens' rows appended and attended to, checked; their outputs."""
        slots, positions = np.asarray(slots, np.int32), np.asarray(positions, np.int32)
        x = dev(self.m.embed[tokens])
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        table = dev(self.table.reshape(-1).view(np.int32))
        on = dict(table=table, status=status, **WHERE)
        q = rules.append_rows(x[:, HEADS:HEADS + KVH], x[:, HEADS + KVH:], self.k, self.v, dev(slots), dev(positions),
                              q=x[:, :HEADS], angles=self.angles, scales=self.scales, **on)
        out = rules.attend_kept8(q, self.k, self.v, self.scales, dev(slots), dev(positions), scale=SCALE, run=run,
                                 max_position=int(positions.max()), **on)
        assert int(status) == 0
        for s, p, t in zip(slots, positions, tokens):
            self.kept[int(s), int(p)] = int(t)
        k, v, scales = self.k.cpu().numpy(), self.v.cpu().numpy(), self.scales.cpu().numpy()
        at = dict(table=self.table.reshape(-1), **WHERE)
        # The kept rows are the tokens': a code is half a step off (2^-4, or of the subnormals 2^-10 of the scale;
        # growing scales round again, each half as much as the next), on top of the rotation's f32 steps.
        for s in set(slots.tolist()):
            n = int(positions[slots == s].max()) + 1
            t = np.array([self.kept[s, p] for p in range(n)])
            row = np.array([K.kept_row(s, p, **at) for p in range(n)])
            b, o = row // 16, row % 16
            x = self.m.embed[t]
            for want, codes, which in ((K.turned(x[:, HEADS:HEADS + KVH], None, self.m.angles, np.arange(n), True, 0),
                                        k[b, :, o], 0),
                                       (x[:, HEADS + KVH:].astype(float), v[b, :, :, o], 1)):
                unit = scales[b, :KVH, which, None].astype(float)
                slack = np.abs(want).max(-1, keepdims=True) * 2.0 ** -19
                assert np.all(np.abs(K.CODES[codes] * unit - want) <= np.abs(want) * 2.0 ** -4 + unit * 2.0 ** -9 + slack)
        want, spread, size = K.attend(q.cpu().numpy(), k, v, scales, slots, positions, scale=SCALE, **at)
        # A score: q in three bf16 parts (2^-24), 12 accumulating steps at 2^-21; a weight twice that, its
        # exponential and its own rounding (2^-20).
        bound = (2 * spread * (2.0 ** -24 + 12 * 2.0 ** -21) + 2.0 ** -20) * size
        assert np.all(np.abs(out.cpu().numpy() - want) <= bound[..., None])
        return out


@pytest.mark.parametrize("greedy", [False, True])
def test_drafts_of_a_forked_sequence(greedy):
    r = rng(21)
    server = Server(r, 2)
    prompt = r.integers(0, WIDTH, 41)
    first = server.pool.reserve(1, len(prompt), KEYS)
    server.pages(0, first)
    server.rows(np.zeros(41), np.arange(41), prompt, 41)
    # A second sequence goes on from the first 38 of them: its third page is copied as it grows.
    second = server.pool.fork(first, 38, KEYS)
    server.kept.update({(1, p): int(prompt[p]) for p in range(38)})
    runs, past = [first, second], [41, 38]
    last = [int(server.m.after[prompt[40]]), int(server.m.after[prompt[37]])]
    copied = 0
    for step in range(7):
        counts = r.integers(0, MOST + 1, 2).astype(np.int32)
        right = [int(r.integers(0, n + 1)) for n in counts]
        drafts = np.zeros((2, MOST), np.int32)
        slots, positions, tokens = [], [], []
        for s in range(2):
            t = last[s]
            for i in range(counts[s]):
                good = int(server.m.after[t])
                drafts[s, i] = t = good if i < right[s] else (good + 1 + int(r.integers(0, WIDTH - 1))) % WIDTH
            copied += server.grow(s, runs[s], past[s] + int(counts[s]) + 1)
            slots += [s] * (counts[s] + 1)
            positions += range(past[s], past[s] + counts[s] + 1)
            tokens += [last[s], *drafts[s, :counts[s]].tolist()]
        out = server.rows(slots, positions, np.array(tokens), MOST + 1)
        logits = server.m.logits(out, np.array(tokens))
        u = None if greedy else r.random((2, MOST + 1)).astype(np.float32)
        starts = np.array([0, counts[0] + 1], np.int32)
        got, accepted = rules.verify(logits, dev(drafts), None if greedy else dev(u), counts=dev(counts), first=dev(starts))
        got, accepted = got.cpu().numpy(), accepted.cpu().numpy()
        want_t, want_a = K.verify(logits.cpu().numpy(), drafts, u, counts=counts, first=starts)
        assert np.array_equal(got, want_t) and np.array_equal(accepted, want_a)
        assert accepted.tolist() == right
        for s in range(2):
            n = int(accepted[s])
            assert got[s, n] == server.m.after[tokens[starts[s] + n]]
            past[s] += n + 1
            server.pool.truncate(runs[s], past[s])
            last[s] = int(got[s, n])
        assert server.pool.consistent()
    assert copied >= 1
    for run in runs:
        server.pool.release(run)


def test_a_captured_step_beside_eager_ones():
    """A step of the three captured into one graph (two rows a sequence, each drafting one token), replayed
    over inputs written in place, with eager steps on another stream between the replays."""
    r = rng(22)
    m = Model(r)
    slots_n, past = 5, np.array([3, 15, 16, 40, 100], np.int32)

    def state():
        k, v, scales = rules.kept8(slots_n * EACH, KVH, PAGE)
        table = r.permutation(slots_n * EACH).astype(np.int32)
        return k, v, scales, dev(table)

    k, v, scales, table = state()
    slots = dev(np.repeat(np.arange(slots_n, dtype=np.int32), 2))
    pos = torch.empty(2 * slots_n, dtype=torch.int32, device="cuda")
    x = torch.empty(2 * slots_n, HEADS + 2 * KVH, 128, device="cuda")
    bias = torch.zeros(2 * slots_n, WIDTH, device="cuda")
    drafts = torch.empty(slots_n, 1, dtype=torch.int32, device="cuda")
    u = torch.empty(slots_n, 2, device="cuda")
    angles = dev(m.angles)

    def fill(at, tokens, uniforms):
        pos.copy_(dev((at[:, None] + np.arange(2)).reshape(-1).astype(np.int32)))
        x.copy_(dev(m.embed[tokens.reshape(-1)]))
        bias.zero_()
        bias[torch.arange(2 * slots_n), dev(m.after[tokens.reshape(-1)])] = 3
        drafts.copy_(dev(tokens[:, 1:].astype(np.int32)))
        u.copy_(dev(uniforms))

    def step(k, v, scales):
        q = rules.append_rows(x[:, HEADS:HEADS + KVH], x[:, HEADS + KVH:], k, v, slots, pos, q=x[:, :HEADS],
                              angles=angles, scales=scales, table=table, **WHERE)
        out = rules.attend_kept8(q, k, v, scales, slots, pos, scale=SCALE, run=2, table=table, max_position=KEYS - 1, **WHERE)
        return out, rules.verify(torch.addmm(bias, out.flatten(1), m.head), drafts, u)

    # Prompts, then a warm-up whose rows the first step writes again.
    for s in range(slots_n):
        n = int(past[s])
        rows = dev(m.embed[r.integers(0, WIDTH, n)])
        rules.append_rows(rows[:, HEADS:HEADS + KVH], rows[:, HEADS + KVH:], k, v, dev(np.full(n, s, np.int32)),
                          dev(np.arange(n, dtype=np.int32)), angles=angles, scales=scales, table=table, **WHERE)
    tokens = r.integers(0, WIDTH, (8, slots_n, 2))
    uniforms = r.random((8, slots_n, 2)).astype(np.float32)
    fill(past, tokens[0], uniforms[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(k.clone(), v.clone(), scales.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, (got, accepted) = step(k, v, scales)
    for i in range(8):
        fill(past + 2 * i, tokens[i], uniforms[i])
        k2, v2, s2 = k.clone(), v.clone(), scales.clone()
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):  # beside the replay, over copies
            out2, (got2, accepted2) = step(k2, v2, s2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(got, got2) and torch.equal(accepted, accepted2)
        assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(scales, s2)
    assert torch.isfinite(out).all()
