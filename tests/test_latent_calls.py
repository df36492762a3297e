"""What the entry points of latent attention hand to the library, seen on the CPU: the call itself is caught."""
import ctypes as C

import pytest

from tessera_amd import abi, rules
from test_latent_ref import _append, _attend, _flash, _heads, _no_gpu, _refused

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0."""

    def get_device(self):
        return 0


def t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


@pytest.fixture
def called(monkeypatch):
    """The arguments of the calls that would have been made."""
    calls = []
    monkeypatch.setattr(rules, "_call_on", lambda on, fn, args: calls.append(args))
    return calls


def test_flash_takes_one_q_row_for_all_rows(called):
    """A q that is broadcast over its rows has no distance between them, and is not read past its one row."""
    q, kv, r = t(1, 4, 192).expand(7, -1, -1), t(9, 4, 256), t(9, 64)
    rules.flash_latent(q, kv[..., :128], kv[..., 128:], r, scale=1.0)
    rules.flash_latent(q[:1], kv[..., :128], kv[..., 128:], r, scale=1.0)
    rules.flash_latent(t(7, 4 * 192 + 8)[:, :768].unflatten(1, (4, 192)), kv[..., :128], kv[..., 128:], r, scale=1.0)
    assert [a.q_stride for a in called] == [0, 0, 776]


@pytest.mark.parametrize("rows,heads,row,head", [(3, 16, 0, 64), (2, 1, 0, 0), (2, 1, 32, 0), (3, 16, 64, 64), (3, 16, 1016, 64),
                                                 (3, 16, 64, 184)])
def test_append_refuses_q_out_whose_rows_meet(rows, heads, row, head):
    """Rows that lie on one another, or among another's heads, would be written by several waves at once."""
    _refused("tessera_hip_append_latent", _append(rows=rows, heads=heads, q_out_stride=row, q_out_head=head), b"meet")


@pytest.mark.parametrize("rows,heads,row,head", [(3, 16, 512, 512), (3, 16, 15 * 576 + 504, 576), (3, 16, 512, 2 * 512 + 504), (2, 1, 0, 0)])
def test_heads_refuses_out_whose_rows_meet(rows, heads, row, head):
    _refused("tessera_hip_linear_heads", _heads(rows=rows, heads=heads, out_stride=row, out_head=head), b"meet")


AT = 1 << 30  # (fake addresses, a range of its own for each tensor)


def _placed(kind):
    """A valid call whose tensors all lie apart, and its entry point."""
    at = lambda n: AT + (n << 24)  # noqa: E731
    if kind == "heads":  # x [3, 16, 128] and out [3, 16, 512] bf16, w [16, 512, 128]
        return _heads(x=at(0), w=at(1), out=at(2)), "tessera_hip_linear_heads"
    if kind == "append":  # c [3, 576], q and q_out [3, 16, 64] bf16, kept 32 pages of 16
        names = ("c", "q", "gain", "rope_table", "q_out", "kept", "c_out", "r_out", "slots", "positions", "kept_table")
        return _append(**{name: at(n) for n, name in enumerate(names)}), "tessera_hip_append_latent"
    if kind == "attend":  # q [2, 16, 576], out [2, 16, 512], 1024 pages of 16
        a = _attend(q=at(0), k=at(4), out=at(8), slots=at(9), positions=at(10), kept_table=at(11))
        a.rows.workspace, a.rows.workspace_bytes = at(12), 1 << 26
        return a, "tessera_hip_attend_latent"
    names = ("q", "k", "v", "r", "out", "first", "key_first")  # q [100, 16, 192], k and v [120, 16, 128], out [100, 16, 128]
    return _flash(**{name: at(n) for n, name in enumerate(names)}), "tessera_hip_flash_latent"


def _set(a, name, value):
    setattr(a.rows if hasattr(a, "rows") and hasattr(a.rows, "q") else a, name, value)


@pytest.mark.parametrize("kind,out,over,first", [
    ("heads", "out", "x", 0), ("heads", "out", "x", 16), ("heads", "out", "x", 2 * 6144 + 15 * 384 + 248), ("heads", "out", "w", 16 * 131072 - 8),
    ("heads", "out", "w", -3 * 16 * 1152 + 128 + 8), ("append", "q_out", "q", 16), ("append", "q_out", "q", -16),
    ("append", "q_out", "c", 1152 + 1136), ("append", "q_out", "kept", 512 * 1152 - 16), ("append", "c_out", "c", 0),
    ("append", "c_out", "c", -3 * 1024 + 16), ("append", "r_out", "q", 2 * 8192 + 15 * 384 + 112), ("append", "r_out", "c_out", 16),
    ("append", "kept", "c", -1024), ("append", "r_out", "gain", 16), ("append", "c_out", "slots", 0), ("append", "q_out", "kept_table", 112),
    ("attend", "out", "q", 0), ("attend", "out", "q", 2 * 16 * 1152 - 16), ("attend", "out", "k", 1024 * 16 * 1152 - 16),
    ("attend", "out", "k", -2 * 16 * 1024 + 16), ("attend", "out", "positions", 0), ("attend", "out", "workspace", 1024),
    ("flash", "out", "q", 16), ("flash", "out", "k", 119 * 8192 + 15 * 512 + 240), ("flash", "out", "v", -100 * 4096 + 16),
    ("flash", "out", "r", 0), ("flash", "out", "first", -16),
])
def test_outputs_over_inputs_are_refused(kind, out, over, first):
    """Wherever they begin: at the input's start, before it or within it."""
    a, fn = _placed(kind)
    at = getattr(a.rows if kind == "attend" else a, over)
    _set(a, out, at + first)
    _refused(fn, a, b"lies where")


@pytest.mark.parametrize("kind,out,over,first", [
    ("heads", "out", "x", 3 * 16 * 384), ("heads", "out", "w", 16 * 131072), ("append", "q_out", "q", 128), ("append", "q_out", "q", 0),
    ("append", "q_out", "q", 256), ("append", "c_out", "c", 3 * 1152), ("append", "r_out", "c_out", 3 * 1024),
    ("append", "kept", "c", -512 * 1152), ("attend", "out", "q", 2 * 16 * 1152), ("attend", "out", "k", -2 * 16 * 1024),
    ("flash", "out", "q", 100 * 16 * 384), ("flash", "out", "k", -100 * 4096), ("heads", "out", None, 0)])
def test_outputs_beside_inputs_are_taken(kind, out, over, first):
    """At their end, before their start, or (q_out and q, a head's 64 of 192 values) between a head's values."""
    _no_gpu()
    a, fn = _placed(kind)
    if over == "q" and kind == "append":
        a.q_out_stride, a.q_out_head = a.q_stride, a.q_head
    if over:
        _set(a, out, getattr(a.rows if kind == "attend" else a, over) + first)
    assert getattr(abi.load(), fn)(C.byref(a), None) not in (abi.TS_OK, abi.TS_ERR_ARG)  # (there is no GPU to run it)


@pytest.mark.parametrize("x_stride,x_head,out_stride,out_head,first,taken", [
    (16 * 192, 192, 16 * 192, 192, 128, True),    # heads of 128 and 64 in one row
    (16 * 192, 192, 16 * 192, 192, 120, False),
    (16 * 192, 128, 16 * 192, 64, 16 * 128, True),  # all heads' 128, then all heads' 64
    (16 * 192, 128, 16 * 192, 64, 16 * 128 - 8, False),
    (16 * 192, 128, 16 * 192, 64, 16 * 192, False),  # (the next row's x)
    (128, 192 * 3, 64, 192 * 3, 128 * 3, True),      # heads, rows, and in a head all rows' 128, then all rows' 64
    (128, 192 * 3, 64, 192 * 3, 128 * 3 - 8, False),
])
def test_parts_of_the_same_rows(x_stride, x_head, out_stride, out_head, first, taken):
    _no_gpu()
    a, fn = _placed("heads")
    a.n, a.k, a.w_head, a.out = 64, 128, 64 * 128, a.x + 2 * first
    a.x_stride, a.x_head, a.out_stride, a.out_head = x_stride, x_head, out_stride, out_head
    code = getattr(abi.load(), fn)(C.byref(a), None)
    assert code not in (abi.TS_OK, abi.TS_ERR_ARG) if taken else code == abi.TS_ERR_ARG


def test_flash_refuses_key_parts_too_far_apart(called):
    """A distance that 32 bits do not hold is refused, not cut."""
    q, kv = t(3, 4, 192), t(2, 4, 256)
    r = torch.empty((1 << 32) + 64, dtype=BF16, device="meta").as_subclass(OnGpu).as_strided((2, 64), (1 << 32, 1))
    with pytest.raises(ValueError, match="2\\^32 elements apart"):
        rules.flash_latent(q, kv[..., :128], kv[..., 128:], r, scale=1.0)
    assert not called
