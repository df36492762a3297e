"""Timed operators of speculative decoding over an 8-bit paged cache: appending rows, attention
over the kept blocks, and the verification of drafted tokens, each as a plain torch form and,
with `own`, through the public entry points (tessera_amd.rules).

Kept blocks: 16 positions of one kv head, e4m3 codes times one power-of-two scale for K and one
for V. k [blocks, kv_heads, 16, 128], v [blocks, kv_heads, 128, 16] (positions innermost), scales
[blocks, kv_heads rounded up to even, 2] f32. Position j of slot s lives in block
table[s, j // page] * (page / 16) + (j % page) // 16.

  append  product rows -> q/k RmsNorm (optional), rotation, k and v into kept blocks (or bf16
          kept rows [positions, kv_heads, 128]), q out
  attend  softmax(q . k * scale) v over the kept blocks, one or several rows a sequence
  verify  drafted tokens against the target's distribution, from given uniform numbers

Sizes are those of this repository's benchmark (a Qwen3-0.6B-shaped decoder's heads and
vocabulary, paged GQA attention) and of the ranges around them.
"""
import math
import random

import numpy as np
import torch

own = False

D = 128        # head width
BLOCK = 16     # positions a kept block holds
TOP = 448.0    # largest e4m3 value
EPS = 1e-6
THETA = 1e6
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One new token of one chat: the smallest append, launches and latency.
        {"name": "append_e4m3_1", "op": "append", "seqs": 1, "rows": 1, "ragged": False, "least": 700, "most": 700,
         "heads": 16, "kv_heads": 8, "x": "f32", "kept": "e4m3", "norm": True, "halves": True, "page": 16},
        # A loaded server's decode step of a model without q/k norms, bf16 kept rows, adjacent pairs.
        {"name": "append_bf16_200", "op": "append", "seqs": 200, "rows": 1, "ragged": False, "least": 1, "most": 4000,
         "heads": 32, "kv_heads": 8, "x": "bf16", "kept": "bf16", "norm": False, "halves": False, "page": 16},
        # Drafted rows of a serving batch: blocks that already hold rows, several rows each.
        {"name": "append_e4m3_draft_48x5", "op": "append", "seqs": 48, "rows": 5, "ragged": True, "least": 30,
         "most": 6000, "heads": 64, "kv_heads": 8, "x": "bf16", "kept": "e4m3", "norm": False, "halves": True,
         "page": 64},
        # Prompts of up to 2048 rows batched back to back into the 8-bit cache.
        {"name": "append_e4m3_prefill_6x2048", "op": "append", "seqs": 6, "rows": 2048, "ragged": True, "least": 0,
         "most": 0, "heads": 16, "kv_heads": 8, "x": "f32", "kept": "e4m3", "norm": True, "halves": True,
         "page": 16},
        # One chat's decode step: few groups, the keys split.
        {"name": "attend_1x4000", "op": "attend", "seqs": 1, "rows": 1, "ragged": False, "least": 4000, "most": 4000,
         "heads": 16, "kv_heads": 8, "q": "f32", "out": "f32", "back": -1, "page": 16},
        # Decode attention of a loaded server: 32 sequences of 512..8192 kept rows.
        {"name": "attend_32x8192", "op": "attend", "seqs": 32, "rows": 1, "ragged": False, "least": 512, "most": 8192,
         "heads": 16, "kv_heads": 8, "q": "f32", "out": "f32", "back": -1, "page": 16},
        # Drafted rows checked at once: 5 rows a sequence over shared keys, 8 heads a kv head.
        {"name": "attend_draft_24x5", "op": "attend", "seqs": 24, "rows": 5, "ragged": False, "least": 1000,
         "most": 9001, "heads": 64, "kv_heads": 8, "q": "bf16", "out": "bf16", "back": -1, "page": 16},
        # Two long documents, one new token each, few kv heads.
        {"name": "attend_2x131000", "op": "attend", "seqs": 2, "rows": 1, "ragged": False, "least": 120001,
         "most": 131000, "heads": 32, "kv_heads": 4, "q": "bf16", "out": "bf16", "back": -1, "page": 64},
        # Prompts of 2048 rows prefilled over their own keys.
        {"name": "attend_prefill_4x2048", "op": "attend", "seqs": 4, "rows": 2048, "ragged": False, "least": 2048,
         "most": 2048, "heads": 16, "kv_heads": 8, "q": "bf16", "out": "bf16", "back": -1, "page": 16},
        # Later chunks of ragged prompts, a window of 1000 keys, f32 rows.
        {"name": "attend_chunk_3x700", "op": "attend", "seqs": 3, "rows": 700, "ragged": True, "least": 900,
         "most": 5000, "heads": 16, "kv_heads": 8, "q": "f32", "out": "f32", "back": 1000, "page": 16},
        # One chat's greedy drafts, checked against the vocabulary: the smallest verification.
        {"name": "verify_greedy_1x4", "op": "verify", "seqs": 1, "drafts": 4, "ragged": False, "vocab": 151936,
         "logits": "f32", "probs": False, "greedy": True, "temperature": 1.0},
        # A serving batch's sampled drafts against the drafter's distributions, ragged.
        {"name": "verify_32x4", "op": "verify", "seqs": 32, "drafts": 4, "ragged": True, "vocab": 151936,
         "logits": "f32", "probs": True, "greedy": False, "temperature": 0.75},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "verify"])
    kv = rng.choice([1, 2, 3, 4, 8, 8, 8])
    group = rng.choice([1, 2, 2, 4, 5, 8])
    page = rng.choice([16, 16, 32, 64])
    if op == "append":
        form = rng.choice(["decode", "draft", "prefill"])
        seqs = _log(rng, 1, 256) if form != "prefill" else _log(rng, 1, 4)
        rows = 1 if form == "decode" else rng.randint(2, 9) if form == "draft" else _log(rng, 17, 600)
        least = 0 if form == "prefill" else rng.randint(0, 300)
        return {"op": op, "seqs": seqs, "rows": rows, "ragged": rows > 1 and rng.random() < 0.7, "least": least,
                "most": least + (rng.randint(0, 600) if form == "prefill" else _log(rng, 1, 4000)),
                "heads": kv * group, "kv_heads": kv, "x": rng.choice(["f32", "bf16"]),
                "kept": rng.choice(["e4m3", "e4m3", "bf16"]), "norm": rng.random() < 0.5,
                "halves": rng.random() < 0.7, "page": page}
    if op == "attend":
        form = rng.choice(["decode", "draft", "long", "prefill"])
        typed = rng.choice(["f32", "bf16"])
        c = {"op": op, "ragged": False, "heads": kv * group, "kv_heads": kv, "q": typed, "out": typed,
             "back": rng.choice([-1, -1, -1, _log(rng, 1, 2000)]), "page": page}
        if form == "prefill":
            rows = _log(rng, 65, 900)
            c.update(seqs=rng.randint(1, 2), rows=rows, ragged=rng.random() < 0.7, least=rows,
                     most=rows + rng.randint(0, 1500), heads=kv * min(group, 4))
        elif form == "long":
            least = _log(rng, 10000, 60000)
            c.update(seqs=rng.randint(1, 2), rows=1, least=least, most=least + rng.randint(0, 5000))
        else:
            rows = 1 if form == "decode" else rng.randint(2, 9)
            least = _log(rng, rows, 2500)
            c.update(seqs=_log(rng, 1, 32), rows=rows, ragged=rows > 1 and rng.random() < 0.5, least=least,
                     most=least + _log(rng, 1, 2000))
        return c
    drafts = rng.randint(1, 8)
    greedy = rng.random() < 0.3
    return {"op": op, "seqs": _log(rng, 1, 12), "drafts": drafts, "ragged": rng.random() < 0.6,
            "vocab": _log(rng, 50, 152000), "logits": rng.choice(["f32", "f32", "bf16"]),
            "probs": not greedy and rng.random() < 0.6, "greedy": greedy,
            "temperature": rng.choice([0.5, 0.75, 1.0, 1.0, 1.25])}


# ---------------------------------------------------------------------------------------------
# Shapes of a case: how many rows and kept positions each sequence has. The same multiset for
# every seed (spread evenly over the range), in an order of the seed's own.
# ---------------------------------------------------------------------------------------------

def _spread(least, most, n):
    return [least + (most - least) * i // max(1, n - 1) if n > 1 else most for i in range(n)]


def _lengths(c, seed):
    """(new rows, positions kept before them) of each sequence."""
    rows = _spread(max(1, c["rows"] // 2), c["rows"], c["seqs"]) if c["ragged"] else [c["rows"]] * c["seqs"]
    held = _spread(c["least"], c["most"], c["seqs"])  # append: before the rows; attend: with them
    past = held if c["op"] == "append" else [max(0, h - r) for h, r in zip(held, rows)]
    order = list(range(c["seqs"]))
    random.Random(seed).shuffle(order)
    return [rows[i] for i in order], [past[i] for i in order]


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
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return {"rows": rows, "past": past, "keys": kept_pages * page, "kept_pages": kept_pages, "pages": pages,
            "most": most, "table": dev(table), "slots": dev(slots), "positions": dev(positions), "slots_np": slots,
            "index_np": index, "positions_np": positions, "table_np": table}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _scale_of(amax):
    """2^e, e the least of -100 .. 119 with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax / TOP)  # amax / TOP = m 2^e, 0.5 <= m < 1
    # amax / 448 rounds: compare the product, which is exact in f32, instead.
    e = torch.where(amax <= torch.ldexp(torch.full_like(amax, TOP), e - 1), e - 1, e)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -100).clamp(-100, 119))


def _codes(x):
    return x.clamp(-TOP, TOP).to(torch.float8_e4m3fn)


def _kept8(g, blocks, kv):
    """Kept blocks as appends leave them: normal values with a few wide channels."""
    even = (kv + 1) // 2 * 2
    k = torch.empty(blocks, kv, BLOCK, D, dtype=torch.uint8, device="cuda")
    v = torch.empty(blocks, kv, D, BLOCK, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(blocks, even, 2, device="cuda")
    wide = torch.exp(0.5 * torch.randn(kv, 1, D, generator=g, device="cuda"))
    for at in range(0, blocks, 4096):
        n = min(4096, blocks - at)
        x = torch.randn(n, kv, BLOCK, D, generator=g, device="cuda") * wide
        s = _scale_of(x.abs().amax(dim=(2, 3)))
        k[at:at + n] = _codes(x / s[:, :, None, None]).view(torch.uint8)
        scales[at:at + n, :kv, 0] = s
        x = torch.randn(n, kv, D, BLOCK, generator=g, device="cuda")
        s = _scale_of(x.abs().amax(dim=(2, 3)))
        v[at:at + n] = _codes(x / s[:, :, None, None]).view(torch.uint8)
        scales[at:at + n, :kv, 1] = s
    return k, v, scales


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------

def _prepare_append(c, seed):
    p, g = _paged(c, seed), _generator(seed)
    kv, heads, n = c["kv_heads"], c["heads"], len(p["slots_np"])
    s = dict(p)
    s["qkv"] = _rows(g, (n, (heads + 2 * kv) * D), TYPE[c["x"]])
    s["q_gain"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda") if c["norm"] else None
    s["k_gain"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda") if c["norm"] else None
    angle = torch.arange(p["keys"], dtype=torch.float64, device="cuda")[:, None] * THETA ** (
        -torch.arange(D // 2, dtype=torch.float64, device="cuda") * 2 / D)
    s["angles"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    if c["kept"] == "e4m3":
        per = c["page"] // BLOCK
        s["k"], s["v"], s["scales"] = _kept8(g, p["pages"] * per, kv)
        # The scheduler's list of the blocks that these rows write, and each row's place in it.
        pos = p["positions_np"]
        block = p["table_np"][p["slots_np"], pos // c["page"]].astype(np.int64) * per + pos % c["page"] // BLOCK
        touched, place = np.unique(block, return_inverse=True)
        s["touched"], s["place"] = torch.from_numpy(touched).cuda(), torch.from_numpy(place.reshape(-1)).cuda()
    else:
        s["k"] = _rows(g, (p["pages"] * c["page"], kv, D), torch.bfloat16)
        s["v"] = _rows(g, (p["pages"] * c["page"], kv, D), torch.bfloat16)
        s["scales"] = None
    return s


def _turned(x, gain, angles, pos, halves):
    """RmsNorm (with a gain) and the rotation of rows x [rows, heads, 128]."""
    if gain is not None:
        x = x * (gain / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS))
    cs = angles[pos][:, None].to(x.dtype)
    if halves:
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)


def _into_blocks(kept, scales, new, touched, place, offset, swap):
    """New rows [rows, kv, 128] into blocks `touched` of one kept tensor; `scales` its [blocks, kv]."""
    nb, kv = touched.numel(), new.shape[1]
    old = kept[touched].view(torch.float8_e4m3fn)
    old = old.transpose(2, 3) if swap else old                      # [nb, kv, 16, 128]
    started = torch.zeros(nb, dtype=torch.int, device="cuda").index_add(0, place, (offset == 0).int()) > 0
    written = torch.zeros(nb, BLOCK, dtype=torch.bool, device="cuda")
    written[place, offset] = True
    finite = torch.where(torch.isfinite(new), new.abs(), 0).amax(-1)  # [rows, kv]
    need = torch.zeros(nb, kv, device="cuda").scatter_reduce(0, place[:, None].expand(-1, kv), finite, "amax")
    was = scales[touched]
    scale = torch.where(started[:, None], _scale_of(need), torch.maximum(_scale_of(need), was))
    value = torch.where(started[:, None, None, None], old.float() * scale[:, :, None, None],
                        old.float() * was[:, :, None, None])
    value[place, :, offset] = torch.where(torch.isfinite(new), new, math.nan)
    code = _codes(value / scale[:, :, None, None]).view(torch.uint8)
    keep = (started[:, None] & ~written)[:, None, :, None]           # rows that the new start leaves as they were
    code = torch.where(keep, old.contiguous().view(torch.uint8), code)
    kept[touched] = code.transpose(2, 3) if swap else code
    scales[touched] = scale


def _append(c, s):
    heads, kv = c["heads"], c["kv_heads"]
    x = s["qkv"].view(-1, heads + 2 * kv, D)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if own:
        from tessera_amd import rules
        out = rules.append_rows(k, v, s["k"], s["v"], s["slots"], s["positions"], q=q, q_gain=s["q_gain"],
                                k_gain=s["k_gain"], angles=s["angles"], halves=c["halves"], eps=EPS,
                                scales=s["scales"], keys=s["keys"], table=s["table"],
                                kept_pages=s["kept_pages"], page=c["page"])
    else:
        pos = s["positions"].long()
        out = _turned(q.float(), s["q_gain"], s["angles"], pos, c["halves"]).to(x.dtype)
        k = _turned(k.float(), s["k_gain"], s["angles"], pos, c["halves"])
        if c["kept"] == "e4m3":
            _into_blocks(s["k"], s["scales"][:, :kv, 0], k, s["touched"], s["place"], pos % BLOCK, False)
            _into_blocks(s["v"], s["scales"][:, :kv, 1], v.float(), s["touched"], s["place"], pos % BLOCK, True)
        else:
            row = s["table"][s["slots"].long(), pos // c["page"]].long() * c["page"] + pos % c["page"]
            s["k"][row] = k.to(torch.bfloat16)
            s["v"][row] = v.to(torch.bfloat16)
    if c["kept"] == "bf16":
        return {"q": out, "k": s["k"], "v": s["v"]}
    return {"q": out, "k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn),
            "scales": s["scales"]}


def _e4m3_64(y):
    """The e4m3 value nearest to y (float64, |y| <= 448), ties to even."""
    e = torch.frexp(y.abs())[1] - 1                       # 2^e <= |y| < 2^(e + 1)
    step = torch.ldexp(torch.ones_like(y), e.clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _exact_append(c, seed):
    s = _prepare_append(c, seed)
    heads, kv = c["heads"], c["kv_heads"]
    x = s["qkv"].double().view(-1, heads + 2 * kv, D)
    pos = s["positions"].long()
    turn = torch.view_as_complex(s["angles"].double())[pos][:, None]

    def turned(t, gain):
        if gain is not None:
            t = t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * gain.double()
        pairs = t.unflatten(-1, (2, D // 2)).transpose(-1, -2) if c["halves"] else t.unflatten(-1, (D // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return (z.transpose(-1, -2) if c["halves"] else z).flatten(-2)

    out = {"q": turned(x[:, :heads], s["q_gain"])}
    new = {"k": turned(x[:, heads:heads + kv], s["k_gain"]), "v": x[:, heads + kv:]}
    if c["kept"] == "bf16":
        row = s["table"].long()[s["slots"].long(), pos // c["page"]] * c["page"] + pos % c["page"]
        for name in ("k", "v"):
            out[name] = s[name].double()
            out[name][row] = new[name]
        return out
    scales = s["scales"].double()
    off, place, nb = pos % BLOCK, s["place"], s["touched"].numel()
    for which, name in enumerate(("k", "v")):
        held = s[name].view(torch.float8_e4m3fn).double()
        view = held if name == "k" else held.transpose(2, 3)
        # Every touched block as [16 positions] of new values, NaN where none is written.
        grid = torch.full((nb, BLOCK, kv, D), math.nan, dtype=torch.float64, device="cuda")
        grid[place, off] = new[name]
        grid = grid.transpose(1, 2)
        fresh = ~grid.isnan()
        amax = torch.where(fresh, grid.abs(), 0).amax((2, 3))
        need = torch.exp2(torch.ceil(torch.log2((amax / TOP).clamp(min=2.0 ** -110))).clamp(-100, 119))
        first = fresh[:, 0, 0, 0][:, None]
        was = scales[s["touched"], :kv, which]
        scale = torch.where(first, need, torch.maximum(need, was))
        before = view[s["touched"]]
        rebased = _e4m3_64(before * (was / scale)[:, :, None, None])
        rest = torch.where(first[:, :, None, None], before, rebased)
        view[s["touched"]] = torch.where(fresh, _e4m3_64(torch.nan_to_num(grid) / scale[:, :, None, None]), rest)
        scales[s["touched"], :kv, which] = scale
        out[name] = held
    out["scales"] = scales
    return out


def _work_append(c):
    rows, _ = _lengths(c, 0)
    n, per = sum(rows), D * SIZE[c["x"]]
    moved = n * (2 * c["heads"] + 2 * c["kv_heads"]) * per + n * 2 * c["kv_heads"] * D * SIZE[c["kept"]]
    # Blocks already begun are read and rewritten where their scale grows; counted are their scales alone.
    blocks = sum(-(-r // BLOCK) for r in rows) if c["kept"] == "e4m3" else 0
    return {"bytes": moved + n * (D // 2) * 8 + blocks * c["kv_heads"] * 16,
            "flops": n * (c["heads"] + 2 * c["kv_heads"]) * D * 4}


# ---------------------------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------------------------

def _prepare_attend(c, seed):
    p, g = _paged(c, seed), _generator(seed)
    s = dict(p)
    s["k"], s["v"], s["scales"] = _kept8(g, p["pages"] * (c["page"] // BLOCK), c["kv_heads"])
    s["q"] = _rows(g, (len(p["slots_np"]), c["heads"], D), TYPE[c["q"]])
    s["index"] = torch.from_numpy(p["index_np"]).cuda()
    s["window"] = c["back"] if c["back"] >= 0 else 2 ** 32 - 1
    return s


def _dequantised(c, s, name, which, dtype):
    """[seqs, kv_heads, kept positions, 128] of every slot's table row."""
    per = c["page"] // BLOCK
    block = (s["table"].long()[:, :, None] * per + torch.arange(per, device="cuda")).flatten(1)
    x = s[name][block].view(torch.float8_e4m3fn).to(dtype)     # [seqs, blocks, kv, 16, 128] (v: 128, 16)
    x = x.transpose(3, 4) if name == "v" else x
    x = x * s["scales"][block][:, :, :c["kv_heads"], which].to(dtype)[..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(c, s):
    if own:
        from tessera_amd import rules
        back = {"back": c["back"]} if c["back"] >= 0 else {}
        return rules.attend_kept8(s["q"], s["k"], s["v"], s["scales"], s["slots"], s["positions"], keys=s["keys"],
                                  scale=1 / math.sqrt(D), table=s["table"], kept_pages=s["kept_pages"],
                                  page=c["page"], max_position=s["most"] - 1, run=c["rows"], out_dtype=TYPE[c["out"]], **back)
    kv, seqs, most = c["kv_heads"], c["seqs"], max(s["rows"])
    group, slots, index = c["heads"] // kv, s["slots"].long(), s["index"]
    q = torch.zeros(seqs, most, c["heads"], D, device="cuda")
    q[slots, index] = s["q"].float()
    at = torch.zeros(seqs, most, dtype=torch.long, device="cuda")
    at[slots, index] = s["positions"].long()
    q = q.view(seqs, most, kv, group, D).permute(0, 2, 1, 3, 4).reshape(seqs, kv, most * group, D)
    k = _dequantised(c, s, "k", 0, torch.float32)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D)
    del k
    key = torch.arange(scores.shape[-1], device="cuda")
    seen = (key <= at[..., None]) & (key >= at[..., None] - s["window"])
    scores = scores.view(seqs, kv, most, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, kv, most * group, -1), _dequantised(c, s, "v", 1, torch.float32))
    o = o.view(seqs, kv, most, group, D).permute(0, 2, 1, 3, 4).reshape(seqs, most, c["heads"], D)
    return o[slots, index].to(TYPE[c["out"]])


def _exact_attend(c, seed):
    s = _prepare_attend(c, seed)
    kv, group, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    out, row = [], 0
    for slot, (n, past) in enumerate(zip(s["rows"], s["past"])):
        held = torch.arange(past + n, device="cuda")
        block = s["table"][slot].long()[held // page] * (page // BLOCK) + held % page // BLOCK
        ks, vs = s["scales"].double()[block, :kv, :1], s["scales"].double()[block, :kv, 1:]
        k = s["k"][block, :, held % BLOCK].view(torch.float8_e4m3fn).double() * ks
        v = s["v"][block, :, :, held % BLOCK].view(torch.float8_e4m3fn).double() * vs
        for at in range(0, n, 256):
            here = torch.arange(at, min(at + 256, n), device="cuda")
            pos = past + here
            lo, hi = max(0, past + at - s["window"]), past + min(at + 256, n)
            q = s["q"][row + here].double().view(len(here), kv, group, D).permute(1, 2, 0, 3)
            logit = torch.matmul(q, k[lo:hi].permute(1, 2, 0)[:, None].contiguous()) * D ** -0.5
            keys = held[lo:hi]
            hidden = (keys[None] > pos[:, None]) | (keys[None] < pos[:, None] - s["window"])
            w = torch.softmax(logit.masked_fill(hidden, -math.inf), -1)
            o = torch.matmul(w, v[lo:hi].transpose(0, 1)[:, None].contiguous())
            out.append(o.permute(2, 0, 1, 3).reshape(len(here), kv * group, D))
        row += n
    return torch.cat(out)


def _work_attend(c):
    rows, past = _lengths(c, 0)
    kept = pairs = 0
    for n, p in zip(rows, past):
        first = p if c["back"] < 0 else min(p, c["back"])
        # Positions that some row of the sequence sees, and (row, key) pairs.
        kept += min(p + n, n + first)
        most = p + n if c["back"] < 0 else c["back"] + 1
        pairs += sum(min(p + i + 1, most) for i in range(n))
    n = sum(rows)
    return {"bytes": kept * c["kv_heads"] * 2 * (D + 4 / BLOCK) + n * c["heads"] * D * (SIZE[c["q"]] + SIZE[c["out"]]),
            "flops": 4 * D * c["heads"] * pairs}


# ---------------------------------------------------------------------------------------------
# verify
# ---------------------------------------------------------------------------------------------

def _counts(c, seed):
    n = _spread(0, c["drafts"], c["seqs"]) if c["ragged"] and c["seqs"] > 1 else [c["drafts"]] * c["seqs"]
    random.Random(seed).shuffle(n)
    return n


def _prepare_verify(c, seed):
    g, counts, r = _generator(seed), _counts(c, seed), np.random.default_rng(seed)
    seqs, most, vocab = c["seqs"], c["drafts"], c["vocab"]
    first = np.concatenate([[0], np.cumsum([n + 1 for n in counts])])
    rows = int(first[-1])
    # A few tokens of each row carry most of its mass; the drafter's logits are near the target's.
    logits = 2.0 * torch.randn(rows, vocab, generator=g, device="cuda")
    hot = torch.randint(vocab, (rows, min(vocab, 24)), generator=g, device="cuda")
    bump = 9.0 + 3.0 * torch.randn(hot.shape, generator=g, device="cuda")
    logits.scatter_(1, hot, bump)
    logits = logits.to(TYPE[c["logits"]])
    at = first[:-1, None] + np.minimum(np.arange(most)[None], np.array(counts)[:, None])
    near = logits.float()[torch.from_numpy(at).cuda()] / c["temperature"]
    if not c["greedy"]:
        near += 0.7 * torch.randn(near.shape, generator=g, device="cuda")
    probs = torch.softmax(near, -1)
    if c["greedy"]:
        drafts = near.argmax(-1)
        miss = torch.rand(seqs, most, generator=g, device="cuda") < 0.25
        drafts = torch.where(miss, torch.randint(vocab, (seqs, most), generator=g, device="cuda"), drafts)
    elif c["probs"]:
        drafts = torch.multinomial(probs.view(-1, vocab), 1, generator=g).view(seqs, most)
    else:
        drafts = probs.argmax(-1)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()  # noqa: E731
    return {"logits": logits, "drafts": drafts.int().contiguous(), "counts": dev(np.array(counts)),
            "first": dev(first[:-1]), "probs": probs.contiguous() if c["probs"] else None,
            "uniforms": None if c["greedy"] else torch.rand(seqs, most + 1, generator=g, device="cuda")}


def _verify(c, s):
    if own:
        from tessera_amd import rules
        tokens, accepted = rules.verify(s["logits"], s["drafts"], s["uniforms"], counts=s["counts"], first=s["first"],
                                        draft_probs=s["probs"], temperature=c["temperature"])
        return {"tokens": tokens, "accepted": accepted}
    seqs, most, vocab = c["seqs"], c["drafts"], c["vocab"]
    drafts, counts, first = s["drafts"].long(), s["counts"].long(), s["first"].long()
    step = torch.arange(most, device="cuda")
    live = step < counts[:, None]
    row = first[:, None] + torch.minimum(step, counts[:, None])
    token = torch.arange(vocab, device="cuda")
    if c["greedy"]:
        x = s["logits"]
        best = torch.where(x == x.amax(-1, keepdim=True), token, vocab).amin(-1)
        accepted = ((best[row] == drafts) & live).long().cumprod(1).sum(1)
        pick = best[first + accepted]
    else:
        x = s["logits"].double() / c["temperature"]
        e = (x - x.amax(-1, keepdim=True)).exp_()
        z = e.sum(-1)
        p = e[row, drafts] / z[row]
        q = s["probs"].gather(2, drafts[..., None])[..., 0].double() if c["probs"] else 1.0
        u = s["uniforms"].double()
        accepted = ((u[:, :most] * q < p) & live).long().cumprod(1).sum(1)
        here = first + accepted
        refused = (accepted < counts)[:, None]
        at = accepted.clamp(max=most - 1)
        seq = torch.arange(seqs, device="cuda")
        drafted = s["probs"][seq, at].double() if c["probs"] else (token == drafts[seq, at][:, None]).double()
        w = e[here] / z[here][:, None]
        rest = (w - drafted).clamp_(min=0) if c["probs"] else w * (1 - drafted)
        rest = torch.where(refused, rest, w)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
        upto = rest.cumsum(-1)
        pick = (upto <= u[:, most:] * upto[:, -1:]).sum(-1)
        last = torch.where(rest > 0, token, -1).amax(-1)
        pick = torch.minimum(pick, last)
    at = torch.arange(most + 1, device="cuda")
    kept = torch.where(at < accepted[:, None], torch.nn.functional.pad(drafts, (0, 1)), vocab)
    tokens = torch.where(at == accepted[:, None], pick[:, None], kept)
    return {"tokens": tokens.int(), "accepted": accepted.int()}


def _work_verify(c):
    rows = sum(n + 1 for n in _counts(c, 0))
    size = SIZE[c["logits"]]
    drafter = c["seqs"] * c["vocab"] * 4 if c["probs"] else 0
    return {"bytes": rows * c["vocab"] * size + drafter + c["seqs"] * (c["drafts"] + 1) * 12,
            "flops": rows * c["vocab"] * (1 if c["greedy"] else 4)}


# ---------------------------------------------------------------------------------------------

def prepare(case, seed):
    s = {"append": _prepare_append, "attend": _prepare_attend, "verify": _prepare_verify}[case["op"]](case, seed)
    s["case"] = case
    return s


def run(state):
    return {"append": _append, "attend": _attend, "verify": _verify}[state["case"]["op"]](state["case"], state)


def exact(case, seed):
    if case["op"] == "append":
        return _exact_append(case, seed)
    return _exact_attend(case, seed) if case["op"] == "attend" else None


def work(case):
    return {"append": _work_append, "attend": _work_attend, "verify": _work_verify}[case["op"]](case)
