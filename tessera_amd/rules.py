"""Host-side mirror of the reference's lowering-rule kernels, over torch device tensors.

Each function is named for the reference rule whose kernel it launches
(``tiled``, ``lanes``, ``linear``, ``attend_rows``, ``flash_rows``, ``rms_norm``,
``rope``, ``argmax``, ``top_k``, ``gather``; ``append_rows``, ``attend_kept8``, ``verify`` and the latent ones
have no rule of the reference beside them) and takes the same operands in the
same order as that rule's Launch (reads, epilogue operands, output, counts:
engine/plan/lower/src/abi.rs:148-153, product.rs:70-76, rule.rs:92-110).
torch only provides device memory and the current stream; every computation is
a call into libtessera_hip.so through ``tessera_amd.abi``. Errors raise
``abi.HipError`` with the library's message.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import abi

_DT = {torch.float32: abi.TS_F32, torch.bfloat16: abi.TS_BF16, torch.uint8: abi.TS_E4M3,
       torch.float8_e4m3fn: abi.TS_E4M3}


def _ptr(t):
    return None if t is None else t.data_ptr()


# torch's own call for a raw stream handle, without the Stream object around it; not public.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


class Workspace:
    """Scratch of one thread's calls: a new tensor for each call, so that calls on several
    streams or threads share none (the allocator's cache keeps it in stream order, and a call
    that is being captured gets it from the graph's own memory). Not cleared: the kernels write
    what they read. `buf` is the last one (the routing of a picked product can be read there)."""

    def __init__(self, device="cuda"):
        self.device = device
        self.buf = None

    def get(self, nbytes: int):
        if nbytes == 0:
            return None, 0
        self.buf = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return self.buf.data_ptr(), nbytes


_ws = threading.local()


def workspace(device) -> Workspace:
    """The calling thread's."""
    key = str(device)
    ws = _ws.__dict__.get(key)
    if ws is None:
        ws = _ws.__dict__[key] = Workspace(device)
    return ws


BLOCK_FORMS = {"q8_0": abi.TS_Q8_0, "mxfp8": abi.TS_MXFP8, "int4_g32": abi.TS_INT4_G32, "q4_0": abi.TS_Q4_0,
               "nvfp4": abi.TS_NVFP4, "mxfp4": abi.TS_MXFP4, "int4_g128": abi.TS_INT4_G128}


def chain(stages, operands=(), *, sum_at=0, spans=None):
    """A stage chain (ts_after) for a product's epilogue or for map(): `stages` in order,
    each "add", "mul", ("scale", by) or an activation name ("gelu_tanh", "silu",
    "sigmoid", "relu", "softplus", "exp", "tanh"); `operands` the f32 tensors the Add /
    Mul stages read, in order; `sum_at` which of the chain's reads is the sum (or map's
    input). engine/plan/lower/src/kernels/map.rs:40-59,125-185. The tensors must stay
    alive until the call has been enqueued (the struct holds their addresses)."""
    c = abi.After()
    if len(stages) > abi.TS_MAP_STAGES or len(operands) > abi.TS_MAP_OPERANDS:
        raise ValueError(f"at most {abi.TS_MAP_STAGES} stages and {abi.TS_MAP_OPERANDS} operands")
    for i, st in enumerate(stages):
        if st == "add":
            c.stage[i].op = abi.TS_MAP_ADD
        elif st == "mul":
            c.stage[i].op = abi.TS_MAP_MUL
        elif isinstance(st, tuple) and st[0] == "scale":
            c.stage[i].op, c.stage[i].by = abi.TS_MAP_SCALE, float(st[1])
        else:
            c.stage[i].op, c.stage[i].act = abi.TS_MAP_ACT, abi.ACTS[st]
    for j, t in enumerate(operands):
        if t.dtype != torch.float32:
            raise ValueError("chain operands are f32")
        c.operand[j] = t.data_ptr()
        c.spans[j] = (spans or [0] * len(operands))[j]
    c.count, c.sum = len(stages), sum_at
    c._keep = list(operands)
    return c


def linear_args(x, w, out, *, w_scale=None, gain=None, a0=None, stages=0, eps=1e-6, w_form=None):
    m, k = x.shape
    # Block forms: w is the packed tensor (uint8: head, then each row's blocks).
    w_dtype = _DT[w.dtype] if w_form is None else abi.TS_F32_PARTS if w_form == "f32_parts" else BLOCK_FORMS[w_form]
    # One call with every field in order: a ctypes attribute at a time costs more than the launch.
    return abi.LinearArgs(x.data_ptr(), w.data_ptr(), None if w_scale is None else w_scale.data_ptr(),
                          None if gain is None else gain.data_ptr(), None if a0 is None else a0.data_ptr(),
                          out.data_ptr(), None, 0, m, out.shape[1], k, _DT[x.dtype], w_dtype, _DT[out.dtype], stages,
                          eps)


def _linear(fn: str, x, w, *, out=None, out_dtype=torch.float32, w_scale=None, gain=None, a0=None,
            silu_mul=False, eps=1e-6, w_form=None, rows=None, after=None):
    """rows: the weight rows of a packed block-form tensor (w is then flat bytes).
    after: a chain() run on each sum before the store."""
    m = x.shape[0]
    wr = rows if w_form is not None and w_form != "f32_parts" else w.shape[0]
    if wr is None:
        raise ValueError("a block-form weight tensor needs rows=")
    n = wr // 2 if silu_mul or w_form == "f32_parts" else wr
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=x.device)
    stages = (abi.TS_AFTER_ADD if a0 is not None else 0) | (abi.TS_AFTER_SILU_MUL if silu_mul else 0) | \
        (abi.TS_BEFORE_RMS_NORM if gain is not None else 0)
    a = linear_args(x, w, out, w_scale=w_scale, gain=gain, a0=a0, stages=stages, eps=eps, w_form=w_form)
    if after is not None:
        a.after = C.addressof(after)
    if m > 4:  # the products of fewer rows take no workspace
        need = abi.workspace_of(fn, a)
        if need:
            scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
            a.workspace, a.workspace_bytes = scratch.data_ptr(), need
    abi.call(fn, C.byref(a), _stream())
    return out


def pack_f32(w):
    """f32 weights [n, k] to the TS_F32_PARTS layout ([2n, k] bf16: high parts, then
    low parts), once at load; pass the result with w_form="f32_parts"."""
    n, k = w.shape
    out = torch.empty((2 * n, k), dtype=torch.bfloat16, device=w.device)
    abi.call("tessera_hip_pack_f32", C.byref(abi.PackArgs(_ptr(w), _ptr(out), n, k)), _stream())
    return out


def linear(x, w, **kw):
    """tiled or lanes by row count (the cost select between the two rules). k is split by the row
    count too: the last bits of a row's sums can differ with the number of rows beside it."""
    return _linear("tessera_hip_linear", x, w, **kw)


def lanes(x, w, **kw):
    """Few-row product (rule "lanes"/"thin"): m <= 64."""
    return _linear("tessera_hip_lanes", x, w, **kw)


def tiled(x, w, **kw):
    """Matrix-unit product (rule "tiled")."""
    return _linear("tessera_hip_tiled", x, w, **kw)


def picked(x, w, ids, *, n=None, repeat=1, first=0, offset=0, silu_mul=False, w_scale=None, out=None,
           out_dtype=torch.float32, after=None):
    """Rule "picked": row r multiplies matrix ids[r] - first of the set w [count, stride, k]
    (rows offset..offset+n, or the gate/up pair with silu_mul); x row r // repeat."""
    count, stride, k = w.shape
    rows = ids.numel()
    if n is None:
        n = (stride - offset) // 2 if silu_mul else stride - offset
    if out is None:
        out = torch.empty((rows, n), dtype=out_dtype, device=x.device)
    a = abi.PickedArgs()
    a.x, a.w, a.w_scale, a.ids, a.out = _ptr(x), _ptr(w), _ptr(w_scale), _ptr(ids), _ptr(out)
    a.rows, a.n, a.k, a.count, a.stride, a.offset, a.repeat, a.first = rows, n, k, count, stride, offset, repeat, first
    a.x_dtype, a.w_dtype, a.out_dtype = _DT[x.dtype], _DT[w.dtype], _DT[out.dtype]
    a.stages = abi.TS_AFTER_SILU_MUL if silu_mul else 0
    if after is not None:
        a.after = C.addressof(after)
    need = abi.load().tessera_hip_picked_workspace(C.byref(a))
    a.workspace, a.workspace_bytes = workspace(x.device).get(need)
    abi.call("tessera_hip_picked", C.byref(a), _stream())
    return out


def map(x, stages, operands=(), *, sum_at=0, spans=None, out=None):
    """Rule "map": out = chain(x) elementwise over f32 x (map.rs:60-65,187-260)."""
    if out is None:
        out = torch.empty_like(x)
    a = abi.MapArgs()
    a.x, a.out, a.len = _ptr(x), _ptr(out), x.numel()
    a.after = chain(stages, operands, sum_at=sum_at, spans=spans)
    abi.call("tessera_hip_map", C.byref(a), _stream())
    return out


def take(x, ids, out=None):
    rows, width = x.shape
    picks = ids.shape[-1]
    if out is None:
        out = torch.empty(ids.shape, dtype=torch.float32, device=x.device)
    abi.call("tessera_hip_take", C.byref(abi.TakeArgs(_ptr(x), _ptr(ids), _ptr(out), rows, width, picks)), _stream())
    return out


def softmax(x, out=None):
    width = x.shape[-1]
    rows = x.numel() // width
    if out is None:
        out = torch.empty_like(x)
    abi.call("tessera_hip_softmax", C.byref(abi.SoftmaxArgs(_ptr(x), _ptr(out), rows, width)), _stream())
    return out


def mix(x, weights=None, out=None):
    """Weighted sum over axis 1 of x [outer, count, inner] (mean without weights)."""
    outer, count = x.shape[0], x.shape[1]
    inner = x.numel() // (outer * count)
    if out is None:
        out = torch.empty((outer,) + tuple(x.shape[2:]), dtype=torch.float32, device=x.device)
    abi.call("tessera_hip_mix", C.byref(abi.MixArgs(_ptr(x), _ptr(weights), _ptr(out), outer, count, inner)),
             _stream())
    return out


def moe_layer(h, router, w_in, w_out, *, top=8, shared_in=None, shared_out=None, inner_dtype=torch.bfloat16,
              scores=None):
    """One MoE MLP as the reference composes it (engine/models/src/decoder.rs:73-84):
    scores = h . router^T; ids = top_k(scores); gates = softmax(take(scores, ids));
    inner = silu(h . gate_e) * (h . up_e) per pick; y = mix(inner . out_e, gates);
    plus the shared expert's SwiGLU when given. `scores` given: the router product is
    skipped (router may be None). The last bits of a token's scores can differ with the number
    of tokens (linear splits k by the row count), so near ties may pick another expert.
    Returns (y, ids, gates)."""
    tokens = h.shape[0]
    if scores is None:
        scores = linear(h, router)
    ids = top_k(scores, top)
    gates = softmax(take(scores, ids))
    ffn = w_out.shape[2]
    inner = picked(h, w_in, ids, n=ffn, repeat=top, silu_mul=True, out_dtype=inner_dtype)
    y_picks = picked(inner, w_out, ids, out_dtype=torch.float32)
    y = mix(y_picks.view(tokens, top, -1), gates)
    if shared_in is not None:
        s_inner = linear(h, shared_in, silu_mul=True, out_dtype=inner_dtype)
        y = linear(s_inner, shared_out, a0=y, out=y)
    return y, ids, gates


def rows_args(q, k, v, out, slots, positions, *, keys, scale, table=None, kept_pages=0, page=16,
              back=abi.U32_MAX, max_position=None, status=None, shape=None):
    # attend_step, whose q is in its product rows, passes the shape in place of q
    rows, heads, width = shape or q.shape
    if max_position is None:
        max_position = int(positions.max().item()) if rows else 0
    # status: int32 device word, TS_STATUS_* bits of refused rows
    return abi.RowsArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(slots), _ptr(positions), _ptr(table), None, 0, rows,
                        keys, heads, k.shape[-2], width, back, kept_pages, page, scale,
                        abi.TS_F32 if q is None else _DT[q.dtype], _DT[k.dtype], _DT[out.dtype], max_position,
                        _ptr(status))


def attend_rows(q, k, v, slots, positions, *, keys, scale, table=None, kept_pages=0, page=16,
                back=abi.U32_MAX, max_position=None, out=None, status=None):
    """Decode rows over kept K/V (rule "attend"/attend_rows; split-KV)."""
    if out is None:
        out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    a = rows_args(q, k, v, out, slots, positions, keys=keys, scale=scale, table=table,
                  kept_pages=kept_pages, page=page, back=back, max_position=max_position, status=status)
    need = abi.load().tessera_hip_attend_rows_workspace(C.byref(a))
    a.workspace, a.workspace_bytes = workspace(q.device).get(need)
    abi.call("tessera_hip_attend_rows", C.byref(a), _stream())
    return out


def rope_table(positions, theta, width=128, device="cuda"):
    """(cos, sin) of every (position, pair) angle (the "angles" stage)."""
    t = torch.empty((positions, width // 2, 2), dtype=torch.float32, device=device)
    abi.call("tessera_hip_rope_table", C.byref(abi.AnglesArgs(_ptr(t), positions, width, theta)), _stream())
    return t


def attend_step(qkv, q_gain, k_gain, k, v, slots, positions, *, heads, keys, scale, eps, theta, table=None,
                kept_pages=0, page=16, back=abi.U32_MAX, max_position=None, out=None, angles=None):
    """Fused decode step: q/k RmsNorm + RoPE from raw product rows, append, attend."""
    rows = qkv.shape[0]
    if angles is None:
        angles = rope_table(keys, theta, device=qkv.device)
    if out is None:
        out = torch.empty((rows, heads, 128), dtype=torch.float32, device=qkv.device)
    a = rows_args(None, k, v, out, slots, positions, keys=keys, scale=scale, table=table, kept_pages=kept_pages,
                  page=page, back=back, max_position=max_position, shape=(rows, heads, 128))
    need = abi.load().tessera_hip_attend_rows_workspace(C.byref(a))
    a.workspace, a.workspace_bytes = workspace(qkv.device).get(need)
    st = abi.StepArgs(a, _ptr(qkv), _ptr(q_gain), _ptr(k_gain), _ptr(angles), angles.shape[0], eps)
    abi.call("tessera_hip_attend_step", C.byref(st), _stream())
    return out


def flash_rows(q, k, v, slots, positions, *, keys, scale, table=None, kept_pages=0, page=16,
               back=abi.U32_MAX, max_position=None, out=None, status=None):
    """Prefill rows over kept K/V (rule "flash"/flash_rows); rows may be packed ragged.
    max_position (an upper bound on positions) defaults to their maximum (a host read:
    pass it when capturing a graph)."""
    if out is None:
        out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    a = rows_args(q, k, v, out, slots, positions, keys=keys, scale=scale, table=table,
                  kept_pages=kept_pages, page=page, back=back, max_position=max_position, status=status)
    abi.call("tessera_hip_flash_rows", C.byref(a), _stream())
    return out


MASKS = {"causal": lambda n: (abi.U32_MAX, 0, 1), "bidirectional": lambda n: (abi.U32_MAX, abi.U32_MAX, 0),
         "within": lambda n: (n, n, 0), "back": lambda n: (n, 0, 1)}


def flash(q, k, v, *, scale, mask="causal", n=0, out=None):
    """Rule "flash" on whole sequences: q [seqs, rows, heads, 128] (f32 or bf16), k / v
    [seqs, keys, kv_heads, 128] bf16, any mask of engine/ir/graph/src/node.rs:162-181
    ("causal", "bidirectional", "within" n, "back" n)."""
    seqs, rows, heads, width = q.shape
    keys, kvh = k.shape[1], k.shape[2]
    if out is None:
        out = torch.empty((seqs, rows, heads, width), dtype=torch.float32, device=q.device)
    back, ahead, causal = MASKS[mask](n)
    a = abi.FlashArgs(_ptr(q), _ptr(k), _ptr(v), _ptr(out), seqs, rows, keys, heads, kvh, width, back, ahead,
                      causal, scale, _DT[q.dtype], _DT[k.dtype], _DT[out.dtype])
    abi.call("tessera_hip_flash", C.byref(a), _stream())
    return out


def rms_norm(x, gain, eps, out=None):
    rows, width = x.reshape(-1, x.shape[-1]).shape
    if out is None:
        out = torch.empty_like(x)
    abi.call("tessera_hip_rms_norm", C.byref(abi.NormArgs(_ptr(x), _ptr(gain), _ptr(out), rows, width, eps)),
             _stream())
    return out


def rope(x, positions, theta, halves=True):
    """In place on x [rows, heads, width]."""
    rows, heads, width = x.shape
    a = abi.RopeArgs(_ptr(x), _ptr(positions), rows, heads, width, theta, 1 if halves else 0)
    abi.call("tessera_hip_rope", C.byref(a), _stream())
    return x


def qk_norm_rope_append(qkv, q_gain, k_gain, q_out, k_cache, v_cache, slots, positions, *, heads,
                        kv_heads, keys, eps, theta, table=None, kept_pages=0, page=16):
    rows = qkv.shape[0]
    a = abi.QkArgs(_ptr(qkv), _ptr(q_gain), _ptr(k_gain), _ptr(q_out), _ptr(k_cache), _ptr(v_cache),
                   _ptr(slots), _ptr(positions), _ptr(table), rows, heads, kv_heads, 128, keys, kept_pages,
                   page, eps, theta)
    abi.call("tessera_hip_qk_norm_rope_append", C.byref(a), _stream())
    return q_out


def gather(table, ids, first=0, out=None):
    count = ids.numel()
    rows, width = table.shape
    if out is None:
        out = torch.empty((count, width), dtype=torch.float32, device=table.device)
    a = abi.GatherArgs(_ptr(table), _ptr(ids), _ptr(out), count, rows, width, first)
    abi.call("tessera_hip_gather", C.byref(a), _stream())
    return out


def argmax(x, ids=None):
    rows, width = x.shape
    if ids is None:
        ids = torch.empty(rows, dtype=torch.int32, device=x.device)
    a = abi.ArgmaxArgs(_ptr(x), _ptr(ids), None, 0, rows, width)
    a.workspace, a.workspace_bytes = workspace(x.device).get(abi.load().tessera_hip_argmax_workspace(C.byref(a)))
    abi.call("tessera_hip_argmax", C.byref(a), _stream())
    return ids


def linear_argmax(x, w, *, gain=None, eps=1e-6, keys=None):
    """The few-row product with the greedy pick folded in (TS_AFTER_ARGMAX): (logits,
    ids). `keys` (int64 [m], zero) may be passed to reuse; it is zero again after."""
    m, n = x.shape[0], w.shape[0]
    out = torch.empty((m, n), dtype=torch.float32, device=x.device)
    if keys is None:
        keys = torch.zeros(m, dtype=torch.int64, device=x.device)
    stages = abi.TS_AFTER_ARGMAX | (abi.TS_BEFORE_RMS_NORM if gain is not None else 0)
    a = linear_args(x, w, out, gain=gain, stages=stages, eps=eps)
    a.workspace, a.workspace_bytes = _ptr(keys), keys.numel() * 8
    abi.call("tessera_hip_lanes", C.byref(a), _stream())
    ids = torch.empty(m, dtype=torch.int32, device=x.device)
    abi.call("tessera_hip_argmax_keys", C.byref(abi.KeysArgs(_ptr(keys), _ptr(ids), m, n)), _stream())
    return out, ids


def top_k(x, k, ids=None):
    rows, width = x.shape
    if ids is None:
        ids = torch.empty((rows, k), dtype=torch.int32, device=x.device)
    abi.call("tessera_hip_top_k", C.byref(abi.TopKArgs(_ptr(x), _ptr(ids), rows, width, k)), _stream())
    return ids


# ---------------------------------------------------------------------------------------------
# Speculative decoding over an 8-bit cache: kept blocks, appends, attention, verification.
# ---------------------------------------------------------------------------------------------

KEPT_BLOCK = 16  # positions a kept block holds
_INTS = (torch.int32, torch.uint32)
_CODES = (torch.uint8, torch.float8_e4m3fn)
_F32 = (torch.float32,)
_ROWS = (torch.float32, torch.bfloat16)


def _checked(what, on, *tensors):
    """Each (name, tensor, its types, its elements or -1): contiguous and on GPU `on`; None passes. (The
    operators below look at their tensors in one expression, and come here to say what is wrong: a loop
    over ten tensors costs as much as the launch.)"""
    if on < 0:
        raise ValueError(f"{what}: tensors not on a GPU")
    for name, t, types, count in tensors:
        if t is not None and (t.get_device() != on or t.dtype not in types or not t.is_contiguous() or
                              (count >= 0 and t.numel() != count)):
            raise ValueError(f"{what}: {name} must be contiguous, on GPU {on}, of " +
                             " or ".join(str(d).replace("torch.", "") for d in types) +
                             (f", {count} elements" if count >= 0 else ""))


def _call_on(on, fn, args):
    """The call on GPU `on`'s current stream, whichever device is current."""
    if on == torch.cuda.current_device():
        code = fn(args, _stream() if _raw_stream is None else _raw_stream(on))
    else:
        with torch.cuda.device(on):
            code = fn(args, _stream())
    if code:
        abi.check(code, fn.__name__)


def kept8(pages, kv_heads, page=16, device="cuda"):
    """Kept blocks of `pages` pages, all zero: (k, v, scales) as include/tessera_hip.h lays them out
    (16 positions of one kv head a block: e4m3 codes times a power of two)."""
    blocks = pages * page // KEPT_BLOCK
    k = torch.zeros((blocks, kv_heads, KEPT_BLOCK, 128), dtype=torch.uint8, device=device)
    v = torch.zeros((blocks, kv_heads, 128, KEPT_BLOCK), dtype=torch.uint8, device=device)
    return k, v, torch.zeros((blocks, (kv_heads + 1) // 2 * 2, 2), dtype=torch.float32, device=device)


def _kept8_blocks(what, k, v, scales, kv_heads):
    """How many blocks there are; the shapes are kept8()'s."""
    blocks, *one = k.shape
    if one != [kv_heads, KEPT_BLOCK, 128] or v.shape != (blocks, kv_heads, 128, KEPT_BLOCK) or \
            scales.shape != (blocks, (kv_heads + 1) // 2 * 2, 2):
        raise ValueError(f"{what}: kept blocks of {kv_heads} heads as kept8() makes them")
    return blocks


def _slots(what, table, kept_pages, held, keys):
    """Slots that the table (or the dense kept rows) holds."""
    if table is None:
        return held // keys if keys else 0
    slots, rest = divmod(table.numel(), kept_pages) if kept_pages > 0 else (0, 1)
    if rest:
        raise ValueError(f"{what}: a table of {table.numel()} entries is not whole slots of {kept_pages}")
    return slots


def _pages(table, held, page):
    """Pages that `held` kept rows are; of dense ones, which no page divides, a begun last one too."""
    page = max(page, 1)
    return held // page if table is not None else -(-held // page)


def append_rows(k, v, k_kept, v_kept, slots, positions, *, keys, q=None, q_gain=None, k_gain=None, angles=None,
                halves=True, eps=1e-6, scales=None, table=None, kept_pages=0, page=16, q_out=None, status=None):
    """New rows k, v [rows, kv_heads, 128] (views of a product's rows serve: only the rows' distance is
    free) into the kept rows, q [rows, heads, 128] rotated to q_out (of q's type unless given). With
    gains q / k pass through RmsNorm, with `angles` (rope_table's, at least `keys` positions) through the
    rotation. `scales` given: k_kept, v_kept are kept8() blocks; else bf16 rows [*, kv_heads, 128].
    Rows of one call that fall into one block of 16 positions stand together, in order; later ones that do
    not are kept nowhere, which only status tells. Rows without a place (position, slot or page) are kept
    nowhere and their q is NaN. status: int32 device word, TS_STATUS_* bits of rows that were not kept.
    Returns q_out."""
    what = "append_rows"
    rows, kv_heads, width = shape = k.shape
    on, x = k.get_device(), k.dtype
    (k_stride, k_head, k_one), (v_stride, v_head, v_one) = k.stride(), v.stride()
    if x not in _ROWS or v.dtype is not x or v.shape != shape or v.get_device() != on or k_one != 1 or v_one != 1 or \
            ((k_head != width or v_head != width) and kv_heads > 1):
        raise ValueError("append_rows: k and v must be rows of one type (f32 or bf16), width and device, a row's "
                         "heads back to back")
    heads = q_stride = q_type = 0
    if q is not None:
        heads = q.size(1)
        q_stride, q_head, q_one = q.stride()
        if q.dtype is not x or q.shape != (rows, heads, width) or q.get_device() != on or q_one != 1 or \
                (q_head != width and heads > 1):
            raise ValueError("append_rows: q must be rows as k's, a row's heads back to back")
        if q_out is None:
            q_out = q.new_empty(rows, heads, width)
        else:
            _checked(what, on, ("q_out", q_out, _ROWS, rows * heads * width))
        q_type = _DT[q_out.dtype]
    if rows == 1:  # any distance will do
        q_stride, k_stride, v_stride = heads * width, kv_heads * width, kv_heads * width
    elif (q_stride | k_stride | v_stride) >> 32:
        raise ValueError("append_rows: rows more than 2^32 elements apart")
    if scales is not None:
        held = _kept8_blocks(what, k_kept, v_kept, scales, kv_heads) * KEPT_BLOCK
        kept, kv = _CODES, abi.TS_E4M3
    else:
        held = k_kept.numel() // (kv_heads * width) if kv_heads else 0
        kept, kv = (torch.bfloat16,), abi.TS_BF16
        if k_kept.shape != v_kept.shape or k_kept.shape[-2:] != (kv_heads, width):
            raise ValueError("append_rows: kept rows are bf16 [rows, kv_heads, 128], or blocks with their scales")
    f32 = torch.float32
    if not (on >= 0 and k_kept.get_device() == v_kept.get_device() == slots.get_device() == positions.get_device() == on
            and k_kept.dtype in kept and v_kept.dtype in kept and slots.dtype in _INTS and positions.dtype in _INTS
            and slots.numel() == positions.numel() == rows and k_kept.is_contiguous() and v_kept.is_contiguous()
            and slots.is_contiguous() and positions.is_contiguous()
            and (table is None or table.get_device() == on and table.dtype in _INTS and table.is_contiguous())
            and (scales is None or scales.get_device() == on and scales.dtype is f32 and scales.is_contiguous())
            and (angles is None or angles.get_device() == on and angles.dtype is f32 and angles.is_contiguous())
            and (q_gain is None or q_gain.get_device() == on and q_gain.dtype is f32 and q_gain.numel() == width and q_gain.is_contiguous())
            and (k_gain is None or k_gain.get_device() == on and k_gain.dtype is f32 and k_gain.numel() == width and k_gain.is_contiguous())
            and (status is None or status.get_device() == on and status.dtype in _INTS)):
        _checked(what, on, ("k_kept", k_kept, kept, -1), ("v_kept", v_kept, kept, -1), ("slots", slots, _INTS, rows),
                 ("positions", positions, _INTS, rows), ("table", table, _INTS, -1), ("scales", scales, _F32, -1),
                 ("angles", angles, _F32, -1), ("q_gain", q_gain, _F32, width), ("k_gain", k_gain, _F32, width),
                 ("status", status, _INTS, -1))
    a = abi.AppendArgs(None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
                       None if q_gain is None else q_gain.data_ptr(), None if k_gain is None else k_gain.data_ptr(),
                       None if angles is None else angles.data_ptr(), None if q is None else q_out.data_ptr(),
                       k_kept.data_ptr(), v_kept.data_ptr(), None if scales is None else scales.data_ptr(),
                       slots.data_ptr(), positions.data_ptr(), None if table is None else table.data_ptr(),
                       None if status is None else status.data_ptr(), rows, heads, kv_heads, width, q_stride,
                       k_stride, v_stride, keys, _slots(what, table, kept_pages, held, keys), kept_pages, page,
                       _pages(table, held, page), 0 if angles is None else angles.numel() // width, halves, _DT[x],
                       q_type, kv, eps)
    _call_on(on, abi.load().tessera_hip_append_rows, a)
    return q_out


def attend_kept8(q, k, v, scales, slots, positions, *, keys, scale, table=None, kept_pages=0, page=16,
                 back=abi.U32_MAX, run=1, max_position=None, out=None, out_dtype=torch.float32, status=None):
    """Attention of q [rows, heads, 128] (f32 or bf16) over kept8() blocks: decode rows, several drafted
    rows of a sequence, prompts. run: how many rows of a slot stand together (a hint: it groups rows and
    picks the kernel). max_position (an upper bound on positions) defaults to their maximum (a host
    read: pass it when capturing a graph). out f32 or bf16."""
    what = "attend_kept8"
    rows, heads, width = q.shape
    kv_heads, on = k.shape[1], q.get_device()
    held = _kept8_blocks(what, k, v, scales, kv_heads) * KEPT_BLOCK
    if out is None:
        out = q.new_empty(rows, heads, width) if out_dtype is q.dtype else q.new_empty(q.shape, dtype=out_dtype)
    elif out.shape != q.shape:
        raise ValueError("attend_kept8: out must have q's shape")
    if not (on >= 0 and k.get_device() == v.get_device() == scales.get_device() == slots.get_device()
            == positions.get_device() == out.get_device() == on and q.dtype in _ROWS and out.dtype in _ROWS
            and k.dtype in _CODES and v.dtype in _CODES and scales.dtype is torch.float32 and slots.dtype in _INTS
            and positions.dtype in _INTS and slots.numel() == positions.numel() == rows and q.is_contiguous()
            and k.is_contiguous() and v.is_contiguous() and scales.is_contiguous() and slots.is_contiguous()
            and positions.is_contiguous() and out.is_contiguous()
            and (table is None or table.get_device() == on and table.dtype in _INTS and table.is_contiguous())
            and (status is None or status.get_device() == on and status.dtype in _INTS)):
        _checked(what, on, ("q", q, _ROWS, -1), ("k", k, _CODES, -1), ("v", v, _CODES, -1),
                 ("scales", scales, _F32, -1), ("slots", slots, _INTS, rows), ("positions", positions, _INTS, rows),
                 ("table", table, _INTS, -1), ("out", out, _ROWS, -1), ("status", status, _INTS, -1))
    if max_position is None:
        # (as int32, which has a maximum; a position from 2^31 on is past any slot's)
        max_position = int(positions.view(torch.int32).max().item()) if rows else 0
    a = abi.Kept8Args(abi.RowsArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), slots.data_ptr(),
                                   positions.data_ptr(), None if table is None else table.data_ptr(), None, 0, rows,
                                   keys, heads, kv_heads, width, back, kept_pages, page, scale, _DT[q.dtype],
                                   abi.TS_E4M3, _DT[out.dtype], max_position,
                                   None if status is None else status.data_ptr()),
                      scales.data_ptr(), _slots(what, table, kept_pages, held, keys), _pages(table, held, page), run)
    lib = abi.load()
    need = lib.tessera_hip_attend_kept8_workspace(a)
    if need:
        scratch = slots.new_empty((need + 3) // 4)
        a.rows.workspace, a.rows.workspace_bytes = scratch.data_ptr(), need
    _call_on(on, lib.tessera_hip_attend_kept8, a)
    return out


def verify(logits, drafts, uniforms=None, *, counts=None, first=None, draft_probs=None, temperature=1.0, tokens=None,
           accepted=None, status=None):
    """Drafted tokens [seqs, most] against the target's logits [rows, width] (f32 or bf16; rows any
    distance apart): sequence s's rows are first[s] .. first[s] + counts[s] (without them s * (most + 1)
    and most). uniforms [seqs, most + 1] f32 in [0, 1): one a draft, the last for the token after the
    accepted ones; None: greedy. draft_probs f32 [seqs, most, width]: the drafter's probabilities; None: it
    had only the one token. temperature: a number or f32 [seqs] (<= 0: greedy).
    Returns (tokens [seqs, most + 1], accepted [seqs]) of drafts' type: the accepted drafts, the next token,
    then `width`."""
    what = "verify"
    rows, width = logits.shape
    seqs, most = drafts.shape
    on = logits.get_device()
    per = temperature if isinstance(temperature, torch.Tensor) else None
    stride, inner = logits.stride()
    if rows <= 1:
        stride = width
    if (inner != 1 and width > 1) or stride < width or stride >> 32 or logits.dtype not in _ROWS:
        raise ValueError("verify: logits are f32 or bf16, a row's back to back, rows apart")
    if tokens is None:
        tokens = drafts.new_empty(seqs, most + 1)
    if accepted is None:
        accepted = drafts.new_empty(seqs)
    if draft_probs is not None and draft_probs.shape != (seqs, most, width):
        raise ValueError(f"verify: draft_probs must be f32 {[seqs, most, width]}")
    f32, each = torch.float32, seqs * (most + 1)
    if not (on >= 0 and drafts.get_device() == tokens.get_device() == accepted.get_device() == on
            and drafts.dtype in _INTS and tokens.dtype in _INTS and accepted.dtype in _INTS and drafts.is_contiguous()
            and tokens.is_contiguous() and accepted.is_contiguous() and tokens.numel() == each
            and accepted.numel() == seqs
            and (uniforms is None or uniforms.get_device() == on and uniforms.dtype is f32
                 and uniforms.numel() == each and uniforms.is_contiguous())
            and (draft_probs is None or draft_probs.get_device() == on and draft_probs.dtype is f32
                 and draft_probs.is_contiguous())
            and (counts is None or counts.get_device() == on and counts.dtype in _INTS and counts.numel() == seqs
                 and counts.is_contiguous())
            and (first is None or first.get_device() == on and first.dtype in _INTS and first.numel() == seqs
                 and first.is_contiguous())
            and (per is None or per.get_device() == on and per.dtype is f32 and per.numel() == seqs
                 and per.is_contiguous())
            and (status is None or status.get_device() == on and status.dtype in _INTS)):
        _checked(what, on, ("drafts", drafts, _INTS, -1), ("uniforms", uniforms, _F32, each),
                 ("draft_probs", draft_probs, _F32, -1), ("temperature", per, _F32, seqs),
                 ("counts", counts, _INTS, seqs), ("first", first, _INTS, seqs), ("tokens", tokens, _INTS, each),
                 ("accepted", accepted, _INTS, seqs), ("status", status, _INTS, -1))
    a = abi.VerifyArgs(logits.data_ptr(), drafts.data_ptr(), None if uniforms is None else uniforms.data_ptr(),
                       None if draft_probs is None else draft_probs.data_ptr(), None if per is None else per.data_ptr(),
                       None if counts is None else counts.data_ptr(), None if first is None else first.data_ptr(),
                       tokens.data_ptr(), accepted.data_ptr(), None, 0, None if status is None else status.data_ptr(),
                       seqs, most, rows, width, stride, _DT[logits.dtype], 0.0 if per is not None else temperature)
    lib = abi.load()
    need = lib.tessera_hip_verify_workspace(a)
    if need:
        scratch = drafts.new_empty((need + 3) // 4)
        a.workspace, a.workspace_bytes = scratch.data_ptr(), need
    _call_on(on, lib.tessera_hip_verify, a)
    return tokens, accepted


# ---------------------------------------------------------------------------------------------
# Latent attention: one kept row a position for all heads, absorbed and expanded forms.
# ---------------------------------------------------------------------------------------------

_BF16 = (torch.bfloat16,)


def _rows_of(what, name, t, on, dtype, heads=None):
    """The distances (of rows, of heads) of t [rows, heads, width], any of them where there is one row or head."""
    rows, n, width = t.shape
    row, head, one = t.stride()
    if t.get_device() != on or t.dtype is not dtype or (one != 1 and width > 1) or (heads is not None and n != heads):
        raise ValueError(f"{what}: {name} must be [rows, heads, width] of {str(dtype).replace('torch.', '')} on GPU {on}, a "
                         "head's values back to back")
    if n <= 1:
        head = 0
    if rows <= 1:
        row = 0
    if row >> 32 or head >> 32:
        raise ValueError(f"{what}: {name} rows or heads more than 2^32 elements apart")
    return row, head


def append_latent(c, kept, slots, positions, *, keys, rank, gain=None, angles=None, halves=True, eps=1e-6, q=None,
                  q_out=None, c_out=None, r_out=None, table=None, kept_pages=0, page=16, status=None):
    """New rows of latent attention: c [rows, rank + rope] (f32 or bf16; rows a row or more apart), its latent through
    RmsNorm (with `gain` [rank]) and its last `rope` values through the rotation (with `angles`, rope_table's of width
    `rope`, at least `keys` positions, or any scaled ones of its shape) into kept [*, rank + rope] bf16. q [rows, heads,
    rope] (a view of wider heads serves) is rotated to q_out (a view too, f32 or bf16; made in q's type if not given).
    c_out [rows, rank], r_out [rows, rope] bf16: the kept rows' values back to back. Rows without a place (position,
    slot or page) are kept nowhere, their outputs are NaN, and status (int32 device word) tells of them. No two rows of
    a call are for one place. Returns q_out."""
    what = "append_latent"
    rows, width = c.shape
    on, x = c.get_device(), c.dtype
    rope = width - rank
    stride, one = c.stride()
    if rows <= 1:
        stride = width
    if x not in _ROWS or (one != 1 and width > 1) or stride >> 32:
        raise ValueError("append_latent: c must be rows of f32 or bf16, a row's values back to back")
    if kept.shape[-1] != width:
        raise ValueError(f"append_latent: kept rows of {kept.shape[-1]} values for rows of {width}")
    held = kept.numel() // width if width else 0
    heads = q_row = q_head = o_row = o_head = q_type = 0
    if q is not None:
        heads = q.shape[1]
        q_row, q_head = _rows_of(what, "q", q, on, x)
        if q_out is None:
            q_out = q.new_empty(rows, heads, rope)
        elif q_out.dtype not in _ROWS:
            raise ValueError("append_latent: q_out must be f32 or bf16")
        o_row, o_head = _rows_of(what, "q_out", q_out, on, q_out.dtype, heads)
        if q.shape != (rows, heads, rope) or q_out.shape != (rows, heads, rope):
            raise ValueError(f"append_latent: q and q_out must be {[rows, heads, rope]}")
        q_type = _DT[q_out.dtype]
    if not (on >= 0 and kept.get_device() == slots.get_device() == positions.get_device() == on
            and kept.dtype is torch.bfloat16 and kept.is_contiguous() and slots.dtype in _INTS and positions.dtype in _INTS
            and slots.numel() == positions.numel() == rows and slots.is_contiguous() and positions.is_contiguous()
            and (table is None or table.get_device() == on and table.dtype in _INTS and table.is_contiguous())
            and (gain is None or gain.get_device() == on and gain.dtype is torch.float32 and gain.numel() == rank
                 and gain.is_contiguous())
            and (angles is None or angles.get_device() == on and angles.dtype is torch.float32 and angles.is_contiguous())
            and (c_out is None or c_out.get_device() == on and c_out.dtype is torch.bfloat16
                 and c_out.numel() == rows * rank and c_out.is_contiguous())
            and (r_out is None or r_out.get_device() == on and r_out.dtype is torch.bfloat16
                 and r_out.numel() == rows * rope and r_out.is_contiguous())
            and (status is None or status.get_device() == on and status.dtype in _INTS)):
        _checked(what, on, ("kept", kept, _BF16, -1), ("slots", slots, _INTS, rows), ("positions", positions, _INTS, rows),
                 ("table", table, _INTS, -1), ("gain", gain, _F32, rank), ("angles", angles, _F32, -1),
                 ("c_out", c_out, _BF16, rows * rank), ("r_out", r_out, _BF16, rows * rope), ("status", status, _INTS, -1))
    a = abi.AppendLatentArgs(c.data_ptr(), None if q is None else q.data_ptr(), None if gain is None else gain.data_ptr(),
                             None if angles is None else angles.data_ptr(), None if q is None else q_out.data_ptr(),
                             kept.data_ptr(), None if c_out is None else c_out.data_ptr(),
                             None if r_out is None else r_out.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                             None if table is None else table.data_ptr(), None if status is None else status.data_ptr(),
                             rows, heads, rank, rope, stride, q_row, q_head, o_row, o_head, keys,
                             _slots(what, table, kept_pages, held, keys), kept_pages, page, _pages(table, held, page),
                             0 if angles is None or not rope else angles.numel() // rope, halves, _DT[x], q_type, eps)
    _call_on(on, abi.load().tessera_hip_append_latent, a)
    return q_out


def linear_heads(x, w, *, out=None, out_dtype=torch.float32):
    """A product a head: out[r, h] = w[h] x[r, h]. x [rows, heads, k] f32 or bf16 and out [rows, heads, n] f32 or bf16
    may be views of wider rows and heads (no two of out's pieces meet); w [heads, n, k] bf16, heads n k or more apart. (q
    into the latent space with w [heads, rank, nope], latent sums out of it with w [heads, value, rank].)"""
    what = "linear_heads"
    on, dtype = x.get_device(), x.dtype
    rows, heads, k = x.shape
    n = w.shape[1]
    x_row, x_head = _rows_of(what, "x", x, on, dtype)
    w_head = w.stride(0) if heads > 1 else 0
    if out is None:
        out = x.new_empty(rows, heads, n, dtype=out_dtype)
    elif rows and out.data_ptr() == x.data_ptr():
        raise ValueError("linear_heads: out lies where x does")
    o_row, o_head = _rows_of(what, "out", out, on, out.dtype, heads)
    if on < 0 or dtype not in _ROWS or out.dtype not in _ROWS or out.shape != (rows, heads, n):
        raise ValueError(f"linear_heads: x and out [rows, heads, *] must be f32 or bf16 on a GPU, out {[rows, heads, n]}")
    if w.shape != (heads, n, k) or w.get_device() != on or w.dtype is not torch.bfloat16 or \
            (w.stride(2) != 1 and k > 1) or (w.stride(1) != k and n > 1):
        raise ValueError(f"linear_heads: w must be bf16 {[heads, n, k]} on GPU {on}, a head's rows back to back")
    a = abi.HeadsArgs(x.data_ptr(), w.data_ptr(), out.data_ptr(), rows, heads, n, k, x_row, x_head, o_row, o_head, w_head,
                      _DT[dtype], _DT[out.dtype])
    _call_on(on, abi.load().tessera_hip_linear_heads, a)
    return out


def attend_latent(q, kept, slots, positions, *, keys, rank, scale, table=None, kept_pages=0, page=16, back=abi.U32_MAX,
                  run=1, max_position=None, out=None, status=None):
    """The absorbed form of latent attention: q [rows, heads, rank + rope] bf16 (the absorbed part, then the rotated one)
    over kept [*, rank + rope] bf16; out [rows, heads, rank] bf16, each row's weighted sum of latents. run: how many rows
    of a slot stand together (a hint: it groups rows and picks the kernel). max_position (an upper bound on positions)
    defaults to their maximum (a host read: pass it when capturing a graph)."""
    what = "attend_latent"
    rows, heads, width = q.shape
    on = q.get_device()
    if kept.shape[-1] != width:
        raise ValueError(f"attend_latent: kept rows of {kept.shape[-1]} values for q of {width}")
    held = kept.numel() // width if width else 0
    if out is None:
        out = q.new_empty(rows, heads, rank)
    elif out.shape != (rows, heads, rank):
        raise ValueError(f"attend_latent: out must be {[rows, heads, rank]}")
    elif rows and out.data_ptr() == q.data_ptr():
        raise ValueError("attend_latent: out lies where q does")
    bf16 = torch.bfloat16
    if not (on >= 0 and kept.get_device() == slots.get_device() == positions.get_device() == out.get_device() == on
            and q.dtype is bf16 and kept.dtype is bf16 and out.dtype is bf16 and slots.dtype in _INTS
            and positions.dtype in _INTS and slots.numel() == positions.numel() == rows and q.is_contiguous()
            and kept.is_contiguous() and slots.is_contiguous() and positions.is_contiguous() and out.is_contiguous()
            and (table is None or table.get_device() == on and table.dtype in _INTS and table.is_contiguous())
            and (status is None or status.get_device() == on and status.dtype in _INTS)):
        _checked(what, on, ("q", q, _BF16, -1), ("kept", kept, _BF16, -1), ("slots", slots, _INTS, rows),
                 ("positions", positions, _INTS, rows), ("table", table, _INTS, -1), ("out", out, _BF16, -1),
                 ("status", status, _INTS, -1))
    if max_position is None:
        # (as int32, which has a maximum; a position from 2^31 on is past any slot's)
        max_position = int(positions.view(torch.int32).max().item()) if rows else 0
    a = abi.LatentArgs(abi.RowsArgs(q.data_ptr(), kept.data_ptr(), None, out.data_ptr(), slots.data_ptr(),
                                    positions.data_ptr(), None if table is None else table.data_ptr(), None, 0, rows, keys,
                                    heads, 1, width, back, kept_pages, page, scale, abi.TS_BF16, abi.TS_BF16, abi.TS_BF16,
                                    max_position, None if status is None else status.data_ptr()),
                       rank, _slots(what, table, kept_pages, held, keys), _pages(table, held, page), run)
    lib = abi.load()
    need = lib.tessera_hip_attend_latent_workspace(a)
    if need:
        scratch = slots.new_empty((need + 3) // 4)
        a.rows.workspace, a.rows.workspace_bytes = scratch.data_ptr(), need
    _call_on(on, lib.tessera_hip_attend_latent, a)
    return out


def flash_latent(q, k, v, r, *, scale, first=None, key_first=None, back=abi.U32_MAX, out=None):
    """The expanded form of latent attention over whole sequences packed back to back, causal, ends aligned (a row of a
    sequence of n rows and m keys stands at m - n + its number) and with a window of `back` keys before its own: q [rows,
    heads, nope + rope] bf16 (rows a row or more apart, or one broadcast row), k [keys, heads, nope] and v [keys, heads, value] bf16 (views of
    one product's rows serve), r [keys, rope] bf16: the keys' rotated part, all heads'. first [seqs + 1]: each sequence's
    first row, then the end (None: one sequence); key_first: the same of the keys (None: first's). Returns out [rows,
    heads, value] bf16; rows outside the sequences are left as they were, rows that see no key are zero."""
    what = "flash_latent"
    rows, heads, width = q.shape
    on, bf16 = q.get_device(), torch.bfloat16
    key_rows, _, nope = k.shape
    value, rope = v.shape[-1], r.shape[-1]
    q_row, q_head = _rows_of(what, "q", q, on, bf16)
    k_row, k_head = _rows_of(what, "k", k, on, bf16, heads)
    v_row, v_head = _rows_of(what, "v", v, on, bf16, heads)
    if (heads > 1 and q_head != width) or width != nope + rope or v.shape[0] != key_rows:
        raise ValueError("flash_latent: q [rows, heads, nope + rope] with a row's heads back to back, k [keys, heads, nope], "
                         "v [keys, heads, value] and r [keys, rope]")
    if r.shape != (key_rows, rope) or r.get_device() != on or r.dtype is not bf16 or (r.stride(1) != 1 and rope > 1):
        raise ValueError(f"flash_latent: r must be bf16 {[key_rows, rope]} on GPU {on}, a row's values back to back")
    r_row = r.stride(0) if key_rows > 1 else 0
    if r_row >> 32:
        raise ValueError("flash_latent: r rows more than 2^32 elements apart")
    if out is None:
        out = q.new_empty(rows, heads, value)
    elif out.shape != (rows, heads, value):
        raise ValueError(f"flash_latent: out must be {[rows, heads, value]}")
    elif rows and out.data_ptr() == q.data_ptr():
        raise ValueError("flash_latent: out lies where q does")
    if first is None and key_first is not None:
        raise ValueError("flash_latent: key_first without first")
    seqs = 1 if first is None else first.numel() - 1
    if seqs < 0:
        raise ValueError("flash_latent: first must hold each sequence's first row and the end")
    if not (on >= 0 and out.get_device() == on and out.dtype is bf16 and out.is_contiguous()
            and (first is None or first.get_device() == on and first.dtype in _INTS and first.is_contiguous())
            and (key_first is None or key_first.get_device() == on and key_first.dtype in _INTS
                 and key_first.numel() == seqs + 1 and key_first.is_contiguous())):
        _checked(what, on, ("out", out, _BF16, -1), ("first", first, _INTS, -1), ("key_first", key_first, _INTS, seqs + 1))
    a = abi.FlashLatentArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), r.data_ptr(), out.data_ptr(),
                            None if first is None else first.data_ptr(), None if key_first is None else key_first.data_ptr(),
                            rows, key_rows, seqs, heads, nope, rope, value, q_row, k_row, k_head, v_row,
                            v_head, r_row, back, scale)
    _call_on(on, abi.load().tessera_hip_flash_latent, a)
    return out
