"""Timed operators of latent attention: keys and values of all heads come from one row a position, a
normed latent of `rank` values and a rotated key part of `rope`, kept in bf16 pages. Each operator as a
plain torch form and, with `own`, through the public entry points (tessera_amd.rules).

Kept rows [pages * page, rank + rope] bf16; position j of slot s is row
table[s, j // page] * page + j % page.

  append  product rows [rows, rank + rope] -> RmsNorm of the latent, rotation of the key part, kept; the
          rotated part of q; on request the kept rows back to back as well
  heads   a product a head: out[r, h] = w[h] x[r, h] (q into the latent space, latent sums out of it)
  attend  the absorbed form: softmax(q . row * scale) over the kept rows, times their latents
  flash   the expanded form: every head's own keys (and the shared rotated part) and values, prompts

Sizes are those of this repository's benchmark (16 heads, 32 sequences of 512 .. 8192 kept rows, prompts
of 2048) and of the ranges around them; widths 512 + 64 with heads of 128 + 64 and 128, or half of each.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e4
SIZE = {"f32": 4, "bf16": 2}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
# rank, rotated part, a head's own key part, a head's value
WIDTHS = {"wide": (512, 64, 128, 128), "narrow": (256, 32, 64, 64)}


def listed():
    return [
        # One new token of one chat: the smallest append, launches and latency.
        {"name": "append_1", "op": "append", "seqs": 1, "rows": 1, "ragged": False, "least": 700, "most": 700,
         "heads": 16, "widths": "wide", "x": "bf16", "out": "bf16", "norm": True, "halves": False, "dense": False,
         "page": 16},
        # A loaded server's decode step, all heads on one card, f32 product rows.
        {"name": "append_128", "op": "append", "seqs": 128, "rows": 1, "ragged": False, "least": 1, "most": 6000,
         "heads": 128, "widths": "wide", "x": "f32", "out": "bf16", "norm": True, "halves": True, "dense": False,
         "page": 64},
        # Prompts batched back to back, whose kept rows the expanded form's product takes as well.
        {"name": "append_prefill_6x2048", "op": "append", "seqs": 6, "rows": 2048, "ragged": True, "least": 0,
         "most": 0, "heads": 16, "widths": "wide", "x": "bf16", "out": "bf16", "norm": True, "halves": False,
         "dense": True, "page": 16},
        # q of a decode batch into the latent space: the weights' bytes.
        {"name": "heads_in_32", "op": "heads", "rows": 32, "heads": 128, "k": 128, "n": 512, "gap": 64, "x": "bf16",
         "out": "bf16"},
        # A chunk's latent sums out of it, to the f32 rows that this framework's products take.
        {"name": "heads_out_1024", "op": "heads", "rows": 1024, "heads": 32, "k": 512, "n": 128, "gap": 0, "x": "bf16",
         "out": "f32"},
        # One chat's decode step: one row, the keys split.
        {"name": "attend_1x4000", "op": "attend", "seqs": 1, "rows": 1, "ragged": False, "least": 4000, "most": 4000,
         "heads": 16, "widths": "wide", "back": -1, "page": 16},
        # Decode attention of a loaded server, one card's share of the heads.
        {"name": "attend_32x8192_h16", "op": "attend", "seqs": 32, "rows": 1, "ragged": False, "least": 512,
         "most": 8192, "heads": 16, "widths": "wide", "back": -1, "page": 16},
        # The same with all heads on the card.
        {"name": "attend_32x8192_h128", "op": "attend", "seqs": 32, "rows": 1, "ragged": False, "least": 512,
         "most": 8192, "heads": 128, "widths": "wide", "back": -1, "page": 64},
        # Drafted rows checked at once, up to 5 a sequence.
        {"name": "attend_draft_24x5", "op": "attend", "seqs": 24, "rows": 5, "ragged": True, "least": 1000,
         "most": 9001, "heads": 32, "widths": "wide", "back": -1, "page": 16},
        # Later chunks of prompts over their kept rows.
        {"name": "attend_chunk_2x512", "op": "attend", "seqs": 2, "rows": 512, "ragged": False, "least": 2500,
         "most": 4600, "heads": 16, "widths": "wide", "back": -1, "page": 16},
        # Prompts of 2048 rows over their own keys.
        {"name": "flash_4x2048", "op": "flash", "seqs": 4, "rows": 2048, "ragged": False, "past": 0, "heads": 16,
         "widths": "wide", "back": -1},
        # Ragged prompts behind a shared beginning, a window, half the widths, an odd number of heads.
        {"name": "flash_ragged_5x900", "op": "flash", "seqs": 5, "rows": 900, "ragged": True, "past": 333, "heads": 5,
         "widths": "narrow", "back": 700},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "heads", "attend", "attend", "flash"])
    heads = rng.choice([1, 2, 4, 5, 8, 16, 16, 20, 32, 64, 128])
    widths = rng.choice(["wide", "wide", "narrow"])
    page = rng.choice([16, 16, 32, 64])
    if op == "append":
        form = rng.choice(["decode", "draft", "prefill"])
        seqs = _log(rng, 1, 256) if form != "prefill" else _log(rng, 1, 4)
        rows = 1 if form == "decode" else rng.randint(2, 9) if form == "draft" else _log(rng, 17, 600)
        least = 0 if form == "prefill" else rng.randint(0, 300)
        return {"op": op, "seqs": seqs, "rows": rows, "ragged": rows > 1 and rng.random() < 0.7, "least": least,
                "most": least + (rng.randint(0, 600) if form == "prefill" else _log(rng, 1, 4000)),
                "heads": min(heads, 16) if form == "prefill" else heads, "widths": widths,
                "x": rng.choice(["f32", "bf16"]), "out": rng.choice(["f32", "bf16", "bf16"]),
                "norm": rng.random() < 0.8, "halves": rng.random() < 0.5, "dense": rng.random() < 0.4, "page": page}
    if op == "heads":
        k, n = rng.choice([(128, 512), (512, 128), (64, 256), (256, 64), (8 * rng.randint(1, 80), rng.randint(1, 640))])
        return {"op": op, "rows": _log(rng, 1, max(1, 32000 // heads)), "heads": heads, "k": k, "n": n,
                "gap": rng.choice([0, 64]), "x": rng.choice(["f32", "bf16", "bf16"]), "out": rng.choice(["f32", "bf16"])}
    if op == "attend":
        form = rng.choice(["decode", "decode", "draft", "long", "chunk"])
        c = {"op": op, "ragged": False, "heads": heads, "widths": widths,
             "back": rng.choice([-1, -1, -1, _log(rng, 1, 2000)]), "page": page}
        if form == "chunk":
            rows = _log(rng, 33, 400)
            c.update(seqs=rng.randint(1, 2), rows=rows, ragged=rng.random() < 0.7, least=rows,
                     most=rows + rng.randint(0, 2500), heads=min(heads, 16))
        elif form == "long":
            least = _log(rng, 10000, 100000)
            c.update(seqs=rng.randint(1, 2), rows=1, least=least, most=least + rng.randint(0, 5000))
        else:
            rows = 1 if form == "decode" else rng.randint(2, 6)
            least = _log(rng, rows, 2500)
            c.update(seqs=_log(rng, 1, 24), rows=rows, ragged=rows > 1 and rng.random() < 0.5, least=least,
                     most=least + _log(rng, 1, 3000), heads=heads if rows == 1 else min(heads, 32))
        return c
    rows = _log(rng, 1, 1500)
    return {"op": op, "seqs": rng.randint(1, 4), "rows": rows, "ragged": rng.random() < 0.6,
            "past": rng.choice([0, 0, rng.randint(1, 500)]), "heads": min(heads, 16), "widths": widths,
            "back": rng.choice([-1, -1, -1, _log(rng, 1, 1000)])}


# ---------------------------------------------------------------------------------------------
# Shapes of a case: how many rows and kept positions each sequence has. The same multiset for
# every seed (spread evenly over the range), in an order of the seed's own.
# ---------------------------------------------------------------------------------------------

def _spread(least, most, n):
    return [least + (most - least) * i // max(1, n - 1) if n > 1 else most for i in range(n)]


def _lengths(c, seed):
    """(new rows, positions before them) of each sequence."""
    rows = _spread(max(1, c["rows"] // 2), c["rows"], c["seqs"]) if c["ragged"] else [c["rows"]] * c["seqs"]
    if c["op"] == "flash":
        past = _spread(c["past"] // 2, c["past"], c["seqs"])
    else:
        held = _spread(c["least"], c["most"], c["seqs"])  # append: before the rows; attend: with them
        past = held if c["op"] == "append" else [max(0, h - r) for h, r in zip(held, rows)]
    order = list(range(c["seqs"]))
    random.Random(seed).shuffle(order)
    return [rows[i] for i in order], [past[i] for i in order]


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _paged(c, seed):
    """slots, positions, the page table and its sizes, for rows packed back to back."""
    rows, past = _lengths(c, seed)
    page, r = c["page"], np.random.default_rng(seed)
    most = max(p + n for p, n in zip(past, rows))
    kept_pages = -(-most // page)
    counts = [-(-(p + n) // page) for p, n in zip(past, rows)]
    pages = sum(counts)
    free = r.permutation(pages)
    table = np.zeros((c["seqs"], kept_pages), np.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = free[at:at + n]
        at += n
    slots = np.repeat(np.arange(c["seqs"], dtype=np.int32), rows)
    starts = np.concatenate([[0], np.cumsum(rows)])
    index = np.arange(starts[-1]) - np.repeat(starts[:-1], rows)
    positions = (index + np.repeat(past, rows)).astype(np.int32)
    return {"rows": rows, "past": past, "keys": kept_pages * page, "kept_pages": kept_pages, "pages": pages,
            "most": most, "table": _dev(table), "slots": _dev(slots), "positions": _dev(positions),
            "index": _dev(index)}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _kept_rows(c, s):
    """Each new row's kept row."""
    pos = s["positions"].long()
    return s["table"][s["slots"].long(), pos // c["page"]].long() * c["page"] + pos % c["page"]


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------

def _prepare_append(c, seed):
    rank, rope, nope, _ = WIDTHS[c["widths"]]
    s, g = _paged(c, seed), _generator(seed)
    n = sum(s["rows"])
    s["c"] = _normal(g, (n, rank + rope), TYPE[c["x"]])
    s["q"] = _normal(g, (n, c["heads"], nope + rope), TYPE[c["x"]])
    # The rotated part goes to where the attention's q has it: behind the absorbed one.
    s["q_out"] = torch.zeros(n, c["heads"], rank + rope, dtype=TYPE[c["out"]], device="cuda")[..., rank:]
    s["gain"] = 1 + 0.1 * torch.randn(rank, generator=g, device="cuda") if c["norm"] else None
    angle = torch.arange(s["keys"], dtype=torch.float64, device="cuda")[:, None] * THETA ** (
        -torch.arange(rope // 2, dtype=torch.float64, device="cuda") * 2 / rope)
    s["angles"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    s["kept"] = _normal(g, (s["pages"] * c["page"], rank + rope), torch.bfloat16)
    if c["dense"]:
        s["c_out"] = torch.zeros(n, rank, dtype=torch.bfloat16, device="cuda")
        s["r_out"] = torch.zeros(n, rope, dtype=torch.bfloat16, device="cuda")
    return s


def _turned(x, cs, halves):
    """x [..., rope] rotated by cs [..., rope / 2, 2]."""
    if halves:
        a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
        return torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)


def _append(c, s):
    rank, rope, nope, _ = WIDTHS[c["widths"]]
    out = {"q": s["q_out"], "kept": s["kept"]}
    if c["dense"]:
        out.update(c=s["c_out"], r=s["r_out"])
    if own:
        from tessera_amd import rules
        rules.append_latent(s["c"], s["kept"], s["slots"], s["positions"], keys=s["keys"], rank=rank, gain=s["gain"],
                            angles=s["angles"], halves=c["halves"], eps=EPS, q=s["q"][..., nope:], q_out=s["q_out"],
                            c_out=out.get("c"), r_out=out.get("r"), table=s["table"], kept_pages=s["kept_pages"],
                            page=c["page"])
        return out
    x = s["c"].float()
    latent, turn = x[:, :rank], s["angles"][s["positions"].long()]
    if s["gain"] is not None:
        latent = latent * (s["gain"] / torch.sqrt((latent * latent).mean(-1, keepdim=True) + EPS))
    row = torch.cat([latent, _turned(x[:, rank:], turn, c["halves"])], -1).to(torch.bfloat16)
    s["kept"][_kept_rows(c, s)] = row
    s["q_out"].copy_(_turned(s["q"][..., nope:].float(), turn[:, None], c["halves"]))
    if c["dense"]:
        s["c_out"].copy_(row[:, :rank])
        s["r_out"].copy_(row[:, rank:])
    return out


def _exact_append(c, seed):
    rank, rope, nope, _ = WIDTHS[c["widths"]]
    s = _prepare_append(c, seed)
    unit = torch.view_as_complex(s["angles"].double())[s["positions"].long()]

    def turned(t, z):
        pairs = t.unflatten(-1, (2, rope // 2)).transpose(-1, -2) if c["halves"] else t.unflatten(-1, (rope // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        return (y.transpose(-1, -2) if c["halves"] else y).flatten(-2)

    x = s["c"].double()
    latent = x[:, :rank]
    if c["norm"]:
        latent = latent / (latent.square().mean(-1, keepdim=True) + EPS).sqrt() * s["gain"].double()
    row = torch.cat([latent, turned(x[:, rank:], unit)], -1)
    kept = s["kept"].double()
    kept[_kept_rows(c, s)] = row
    out = {"q": turned(s["q"][..., nope:].double(), unit[:, None]), "kept": kept}
    if c["dense"]:
        out.update(c=row[:, :rank], r=row[:, rank:])
    return out


def _work_append(c):
    rank, rope, _, _ = WIDTHS[c["widths"]]
    n = sum(_lengths(c, 0)[0])
    row = (rank + rope) * (SIZE[c["x"]] + (4 if c["dense"] else 2))
    q = c["heads"] * rope * (SIZE[c["x"]] + SIZE[c["out"]])
    return {"bytes": n * (row + q + rope * 4 + 8) + (rank * 4 if c["norm"] else 0),
            "flops": n * (rank * (4 if c["norm"] else 0) + (c["heads"] + 1) * rope * 3)}


# ---------------------------------------------------------------------------------------------
# heads
# ---------------------------------------------------------------------------------------------

def _prepare_heads(c, seed):
    g = _generator(seed)
    rows, heads, k, n, gap = c["rows"], c["heads"], c["k"], c["n"], c["gap"]
    # x is the front of wider rows (q's own part before the rotated one), and so is out.
    x = _normal(g, (rows, heads, k + gap), TYPE[c["x"]])[..., :k]
    w = _normal(g, (heads, n, k), torch.bfloat16) * k ** -0.5
    out = torch.zeros(rows, heads, n + gap, dtype=TYPE[c["out"]], device="cuda")[..., :n]
    return {"x": x, "w": w, "out": out}


def _heads(c, s):
    if own:
        from tessera_amd import rules
        return rules.linear_heads(s["x"], s["w"], out=s["out"])
    y = torch.matmul(s["x"].float().transpose(0, 1), s["w"].float().transpose(1, 2).contiguous())
    s["out"].copy_(y.transpose(0, 1))
    return s["out"]


def _exact_heads(c, seed):
    s = _prepare_heads(c, seed)
    return torch.stack([s["x"][:, h].double() @ s["w"][h].double().T for h in range(c["heads"])], 1)


def _work_heads(c):
    each = c["rows"] * c["heads"]
    return {"bytes": each * (c["k"] * SIZE[c["x"]] + c["n"] * SIZE[c["out"]]) + c["heads"] * c["n"] * c["k"] * 2,
            "flops": 2 * each * c["n"] * c["k"]}


# ---------------------------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------------------------

def _scale(c):
    _, rope, nope, _ = WIDTHS[c["widths"]]
    return (nope + rope) ** -0.5


def _prepare_attend(c, seed):
    rank, rope, _, _ = WIDTHS[c["widths"]]
    s, g = _paged(c, seed), _generator(seed)
    s["kept"] = _normal(g, (s["pages"] * c["page"], rank + rope), torch.bfloat16)
    s["q"] = _normal(g, (sum(s["rows"]), c["heads"], rank + rope), torch.bfloat16)
    s["window"] = c["back"] if c["back"] >= 0 else 2 ** 32 - 1
    return s


def _attend(c, s):
    rank = WIDTHS[c["widths"]][0]
    if own:
        from tessera_amd import rules
        back = {"back": c["back"]} if c["back"] >= 0 else {}
        return rules.attend_latent(s["q"], s["kept"], s["slots"], s["positions"], keys=s["keys"], rank=rank,
                                   scale=_scale(c), table=s["table"], kept_pages=s["kept_pages"], page=c["page"],
                                   max_position=s["most"] - 1, run=c["rows"], **back)
    seqs, most, heads = c["seqs"], max(s["rows"]), c["heads"]
    slots, index = s["slots"].long(), s["index"]
    q = torch.zeros(seqs, most, heads, s["q"].shape[-1], device="cuda")
    q[slots, index] = s["q"].float()
    at = torch.zeros(seqs, most, dtype=torch.long, device="cuda")
    at[slots, index] = s["positions"].long()
    row = (s["table"].long()[:, :, None] * c["page"] + torch.arange(c["page"], device="cuda")).flatten(1)
    kept = s["kept"][row].float()                                # [seqs, positions, rank + rope]
    scores = torch.matmul(q.flatten(1, 2), kept.transpose(1, 2).contiguous()) * _scale(c)
    key = torch.arange(scores.shape[-1], device="cuda")
    seen = (key <= at[..., None]) & (key >= at[..., None] - s["window"])
    scores = scores.view(seqs, most, heads, -1).masked_fill_(~seen[:, :, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(1, 2), kept[..., :rank].contiguous()).view(seqs, most, heads, rank)
    return o[slots, index].to(torch.bfloat16)


def _exact_attend(c, seed):
    rank = WIDTHS[c["widths"]][0]
    s = _prepare_attend(c, seed)
    out, row = [], 0
    for slot, (n, past) in enumerate(zip(s["rows"], s["past"])):
        held = torch.arange(past + n, device="cuda")
        kept = s["kept"][s["table"][slot].long()[held // c["page"]] * c["page"] + held % c["page"]].double()
        for at in range(0, n, 128):
            pos = past + torch.arange(at, min(at + 128, n), device="cuda")
            lo, hi = max(0, past + at - s["window"]), past + min(at + 128, n)
            q = s["q"][row + at:row + min(at + 128, n)].double()
            logit = (q.flatten(0, 1) @ kept[lo:hi].T).view(len(pos), c["heads"], -1) * _scale(c)
            keys = held[lo:hi]
            hidden = (keys > pos[:, None]) | (keys < pos[:, None] - s["window"])
            w = torch.softmax(logit.masked_fill(hidden[:, None], -math.inf), -1)
            out.append((w.flatten(0, 1) @ kept[lo:hi, :rank]).view(len(pos), c["heads"], rank))
        row += n
    return torch.cat(out)


def _seen(c):
    """Positions that some row of its sequence sees, and (row, key) pairs."""
    kept = pairs = 0
    for n, p in zip(*_lengths(c, 0)):
        kept += n + (p if c["back"] < 0 else min(p, c["back"]))
        most = p + n if c["back"] < 0 else c["back"] + 1
        pairs += sum(min(p + i + 1, most) for i in range(n))
    return kept, pairs


def _work_attend(c):
    rank, rope, _, _ = WIDTHS[c["widths"]]
    kept, pairs = _seen(c)
    n = sum(_lengths(c, 0)[0])
    return {"bytes": 2 * kept * (rank + rope) + 2 * n * c["heads"] * (2 * rank + rope),
            "flops": 2 * (2 * rank + rope) * c["heads"] * pairs}


# ---------------------------------------------------------------------------------------------
# flash
# ---------------------------------------------------------------------------------------------

def _prepare_flash(c, seed):
    _, rope, nope, value = WIDTHS[c["widths"]]
    g = _generator(seed)
    rows, past = _lengths(c, seed)
    n, keys = sum(rows), sum(rows) + sum(past)
    offsets = lambda lengths: _dev(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32))  # noqa: E731
    # One product gives every head's key part and value side by side.
    kv = _normal(g, (keys, c["heads"], nope + value), torch.bfloat16)
    return {"rows": rows, "past": past, "q": _normal(g, (n, c["heads"], nope + rope), torch.bfloat16),
            "k": kv[..., :nope], "v": kv[..., nope:], "r": _normal(g, (keys, rope), torch.bfloat16),
            "first": offsets(rows), "key_first": offsets([a + b for a, b in zip(rows, past)]),
            "window": c["back"] if c["back"] >= 0 else 2 ** 32 - 1}


def _flash(c, s):
    if own:
        from tessera_amd import rules
        back = {"back": c["back"]} if c["back"] >= 0 else {}
        return rules.flash_latent(s["q"], s["k"], s["v"], s["r"], scale=_scale(c), first=s["first"],
                                  key_first=s["key_first"], **back)
    out, row, key = [], 0, 0
    for n, past in zip(s["rows"], s["past"]):
        q = s["q"][row:row + n].float().transpose(0, 1)
        here = slice(key, key + past + n)
        k = torch.cat([s["k"][here].float(), s["r"][here, None].float().expand(-1, c["heads"], -1)], -1)
        scores = torch.matmul(q, k.permute(1, 2, 0).contiguous()) * _scale(c)
        j = torch.arange(past + n, device="cuda")
        at = past + torch.arange(n, device="cuda")[:, None]
        scores.masked_fill_((j > at) | (j < at - s["window"]), -math.inf)
        scores -= scores.amax(-1, keepdim=True)
        p = scores.exp_()
        p /= p.sum(-1, keepdim=True)
        out.append(torch.matmul(p, s["v"][here].float().transpose(0, 1).contiguous()).transpose(0, 1))
        row, key = row + n, key + past + n
    return torch.cat(out).to(torch.bfloat16)


def _exact_flash(c, seed):
    s = _prepare_flash(c, seed)
    nope = s["k"].shape[-1]
    out = torch.empty(s["q"].shape[0], c["heads"], s["v"].shape[-1], dtype=torch.float64, device="cuda")
    row = key = 0
    for n, past in zip(s["rows"], s["past"]):
        r = s["r"][key:key + past + n].double()
        for h in range(c["heads"]):
            k, v = s["k"][key:key + past + n, h].double(), s["v"][key:key + past + n, h].double()
            for at in range(0, n, 512):
                q = s["q"][row + at:row + min(n, at + 512), h].double()
                logit = (q[:, :nope] @ k.T + q[:, nope:] @ r.T) * _scale(c)
                ahead = torch.arange(past + n, device="cuda") - (past + at + torch.arange(len(q), device="cuda")[:, None])
                logit[(ahead > 0) | (ahead < -s["window"])] = -math.inf
                out[row + at:row + at + len(q), h] = torch.softmax(logit, -1) @ v
        row, key = row + n, key + past + n
    return out


def _work_flash(c):
    _, rope, nope, value = WIDTHS[c["widths"]]
    kept, pairs = _seen(c)
    n = sum(_lengths(c, 0)[0])
    return {"bytes": 2 * kept * (c["heads"] * (nope + value) + rope) + 2 * n * c["heads"] * (nope + rope + value),
            "flops": 2 * (nope + rope + value) * c["heads"] * pairs}


# ---------------------------------------------------------------------------------------------

def prepare(case, seed):
    s = {"append": _prepare_append, "heads": _prepare_heads, "attend": _prepare_attend,
         "flash": _prepare_flash}[case["op"]](case, seed)
    s["case"] = case
    return s


def run(state):
    return {"append": _append, "heads": _heads, "attend": _attend, "flash": _flash}[state["case"]["op"]](state["case"],
                                                                                                       state)


def exact(case, seed):
    return {"append": _exact_append, "heads": _exact_heads, "attend": _exact_attend,
            "flash": _exact_flash}[case["op"]](case, seed)


def work(case):
    return {"append": _work_append, "heads": _work_heads, "attend": _work_attend, "flash": _work_flash}[case["op"]](case)
