"""Latent attention as a layer uses it: prompts by the expanded form, decoding by the absorbed one over pages of the pool."""
import numpy as np
import pytest

from helpers import rng
from tessera_amd import kv, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
RANK, ROPE, NOPE, VALUE, HEADS, PAGE = 512, 64, 128, 128, 16, 16
SCALE = (NOPE + ROPE) ** -0.5


class Layer:
    """The attention of one layer, from its product rows on: c [rows, rank + rope] and q [rows, heads, nope + rope]."""

    def __init__(self, seed, pages):
        g = torch.Generator(device="cuda").manual_seed(seed)
        new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.up = (new(HEADS, NOPE + VALUE, RANK) * RANK ** -0.5).to(BF16)
        self.absorb = self.up[:, :NOPE].transpose(1, 2).contiguous()   # [heads, rank, nope], laid out once
        self.gain = 1 + 0.1 * new(RANK)
        self.angles = rules.rope_table(512, 1e4, width=ROPE)
        self.kept = torch.zeros(pages * PAGE, RANK + ROPE, dtype=BF16, device="cuda")
        self.g = g

    def inputs(self, rows):
        return (torch.randn(rows, RANK + ROPE, generator=self.g, device="cuda").to(BF16),
                torch.randn(rows, HEADS, NOPE + ROPE, generator=self.g, device="cuda").to(BF16))

    def prompt(self, c, q, slots, positions, first, **where):
        n = len(c)
        c_out, r_out = torch.empty(n, RANK, dtype=BF16, device="cuda"), torch.empty(n, ROPE, dtype=BF16, device="cuda")
        q = q.clone()
        rules.append_latent(c, self.kept, slots, positions, rank=RANK, gain=self.gain, angles=self.angles, halves=False,
                            q=q[..., NOPE:], q_out=q[..., NOPE:], c_out=c_out, r_out=r_out, **where)
        kv_rows = rules.linear(c_out, self.up.flatten(0, 1), out_dtype=BF16).view(n, HEADS, NOPE + VALUE)
        return rules.flash_latent(q, kv_rows[..., :NOPE], kv_rows[..., NOPE:], r_out, scale=SCALE, first=first)

    def decode(self, c, q, slots, positions, run=1, max_position=None, **where):
        latent = torch.empty(len(c), HEADS, RANK + ROPE, dtype=BF16, device="cuda")
        rules.append_latent(c, self.kept, slots, positions, rank=RANK, gain=self.gain, angles=self.angles, halves=False,
                            q=q[..., NOPE:], q_out=latent[..., RANK:], **where)
        rules.linear_heads(q[..., :NOPE], self.absorb, out=latent[..., :RANK])
        o = rules.attend_latent(latent, self.kept, slots, positions, rank=RANK, scale=SCALE, run=run,
                                max_position=max_position, **where)
        return rules.linear_heads(o, self.up[:, NOPE:], out_dtype=torch.float32)


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def place(lengths, pages, seed):
    each = max(-(-n // PAGE) for n in lengths)
    table = rng(seed).permutation(pages)[:len(lengths) * each].astype(np.int32)
    return dict(keys=each * PAGE, table=torch.from_numpy(table).cuda(), kept_pages=each, page=PAGE)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_expanded_and_absorbed_forms_agree():
    """A batch of prompts by the expanded form, and the same rows by the absorbed one over what was kept. Each rounds to
    bf16 at other places (kv or absorbed q, weights, latent sums, out: 2^-8 at most each, of independent signs): the
    norms of their difference is within 4 half steps."""
    layer = Layer(1, 64)
    lengths = [70, 1, 33]
    where = place(lengths, 64, 1)
    slots = i32(np.repeat([0, 1, 2], lengths).tolist())
    positions = i32([j for n in lengths for j in range(n)])
    c, q = layer.inputs(sum(lengths))
    a = layer.prompt(c, q, slots, positions, i32([0, 70, 71, 104]), **where)
    kept = layer.kept.clone()
    b = layer.decode(c, q, slots, positions, run=70, **where)
    assert torch.equal(layer.kept, kept)  # the same rows again
    assert rel(a, b) < 4 * 2.0 ** -8
    one = torch.cat([layer.decode(c[i:i + 1], q[i:i + 1], slots[i:i + 1], positions[i:i + 1], **where) for i in (0, 69, 70, 103)])
    assert rel(one, b[[0, 69, 70, 103]]) < 2 * 2.0 ** -8


def test_forked_pages():
    """A sequence forked from another's pages goes on as the other would: its begun page is copied by the pool's copies."""
    layer = Layer(2, 16)
    pool = kv.Pool(16, PAGE)
    a = pool.reserve(1, 40, 64)
    pool.grow(a, 40)
    c, q = layer.inputs(41)
    each = 4

    def table_of(*runs):
        t = np.zeros((len(runs), each), np.int32)
        for i, run in enumerate(runs):
            p = pool.pages(run)
            t[i, :len(p)] = p
        return dict(keys=each * PAGE, table=torch.from_numpy(t).cuda(), kept_pages=each, page=PAGE)

    layer.prompt(c[:40], q[:40], i32([0] * 40), i32(list(range(40))), i32([0, 40]), **table_of(a))
    b = pool.fork(a, 40, 64)
    copies = pool.grow(b, 41)
    assert len(copies) == 1
    kv.copy_pages([layer.kept], copies, page=PAGE, pages=16)
    pool.grow(a, 41)
    where = table_of(a, b)
    two = layer.decode(c[[40, 40]], q[[40, 40]], i32([0, 1]), i32([40, 40]), **where)
    assert torch.equal(two[0], two[1])


def test_captured_decode_steps():
    """Two captured steps of different rows replayed in turn, with eager ones between, equal the eager ones bit for bit."""
    lengths = [200, 37, 90]
    where = place(lengths, 64, 3)
    layer, eager = Layer(3, 64), Layer(3, 64)
    slots = i32(np.repeat([0, 1, 2], lengths).tolist())
    positions = i32([j for n in lengths for j in range(n)])
    c, q = layer.inputs(sum(lengths))
    for x in (layer, eager):
        x.prompt(c, q, slots, positions, i32([0, 200, 237, 327]), **where)
    s, p = i32([0, 1, 2]), i32([199, 36, 89])
    steps = [layer.inputs(3) for _ in range(2)]
    run = lambda x, i: x.decode(*steps[i], s, p, max_position=207, **where)  # noqa: E731
    run(layer, 0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(layer, i))
        graphs.append(g)
    for n in range(3):
        for i in range(2):
            for t in steps[i]:
                t.copy_(torch.randn(t.shape, generator=eager.g, device="cuda"))
        p.copy_(i32([199 + n, 36 + n, 89 + n]))
        for i in range(2):
            graphs[i].replay()
            torch.cuda.synchronize()
            want = run(eager, i)
            assert torch.equal(outs[i], want) and torch.equal(layer.kept, eager.kept)


def test_on_another_stream():
    layer = Layer(4, 32)
    where = place([50], 32, 4)
    c, q = layer.inputs(50)
    args = (i32([0] * 50), i32(list(range(50))))
    want = layer.prompt(c, q, *args, i32([0, 50]), **where)
    again = layer.decode(c[-1:], q[-1:], args[0][-1:], args[1][-1:], **where)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer.prompt(c, q, *args, i32([0, 50]), **where)
        step = layer.decode(c[-1:], q[-1:], args[0][-1:], args[1][-1:], **where)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(step, again)


def test_empty_batches():
    layer = Layer(5, 4)
    none = i32([])
    c, q = layer.inputs(0)
    where = place([64], 4, 5)
    assert layer.decode(c, q, none, none, **where).shape == (0, HEADS, VALUE)
    kv_rows = torch.empty(0, HEADS, NOPE + VALUE, dtype=BF16, device="cuda")
    r = torch.empty(0, ROPE, dtype=BF16, device="cuda")
    for first in (None, i32([0]), i32([0, 0, 0])):
        out = rules.flash_latent(q, kv_rows[..., :NOPE], kv_rows[..., NOPE:], r, scale=SCALE, first=first)
        assert out.shape == (0, HEADS, VALUE)
    # Rows without any key are zero.
    q = layer.inputs(3)[1]
    out = rules.flash_latent(q, kv_rows[..., :NOPE], kv_rows[..., NOPE:], r, scale=SCALE, first=i32([0, 3]), key_first=i32([0, 0]))
    assert int(out.count_nonzero()) == 0 and int(layer.kept.count_nonzero()) == 0
