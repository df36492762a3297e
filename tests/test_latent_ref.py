"""CPU checks of latent attention: the float64 forms, the structs, and the calls' refusals."""
import ctypes as C

import numpy as np
import pytest

import latent_ref as L
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")


def test_absorbed_and_expanded_forms_agree():
    """q taken into the latent space over the rows, against every head's own keys and values made of them."""
    r = np.random.default_rng(1)
    heads, rank, rope, nope, value, n = 3, 24, 8, 12, 10, 9
    rows = r.standard_normal((n, rank + rope))
    up_k, up_v = r.standard_normal((heads, nope, rank)), r.standard_normal((heads, value, rank))
    q = r.standard_normal((n, heads, nope + rope))
    k, v = np.einsum("hdr,nr->nhd", up_k, rows[:, :rank]), np.einsum("hdr,nr->nhd", up_v, rows[:, :rank])
    want, *_ = L.flash(q, k, v, rows[:, rank:], scale=0.2, first=[0, n], key_first=[0, n], back=5)
    absorbed = np.concatenate([np.einsum("hdr,nhd->nhr", up_k, q[..., :nope]), q[..., nope:]], -1)
    got, *_ = L.attend(absorbed, rows, np.zeros(n, int), np.arange(n), rank=rank, scale=0.2, back=5, keys=n)
    assert np.allclose(np.einsum("hdr,nhr->nhd", up_v, got), want, atol=1e-12)


def test_flash_form_is_softmax():
    r = np.random.default_rng(2)
    q, k, v, rr = (r.standard_normal(s) for s in ((7, 2, 6), (11, 2, 4), (11, 2, 5), (11, 2)))
    out, *_ = L.flash(q, k, v, rr, scale=0.3, first=[0, 7], key_first=[0, 11])
    qt, kt = torch.from_numpy(q).transpose(0, 1), torch.from_numpy(np.concatenate([k, np.repeat(rr[:, None], 2, 1)], -1)).transpose(0, 1)
    x = qt @ kt.transpose(1, 2) * 0.3
    x = x.masked_fill(torch.arange(11) > 4 + torch.arange(7)[:, None], -np.inf)
    want = (torch.softmax(x, -1) @ torch.from_numpy(v).transpose(0, 1)).transpose(0, 1)
    assert np.allclose(out, want.numpy(), atol=1e-12)


@pytest.mark.parametrize("halves", [True, False])
def test_rotation_form(halves):
    """As complex numbers."""
    r = np.random.default_rng(3)
    x, angle = r.standard_normal((5, 3, 8)), r.standard_normal((5, 1, 4))
    got, size = L.turned(x, np.stack([np.cos(angle), np.sin(angle)], -1), halves)
    a, b = (x[..., :4], x[..., 4:]) if halves else (x[..., 0::2], x[..., 1::2])
    z = (a + 1j * b) * np.exp(1j * angle)
    y, w = (got[..., :4], got[..., 4:]) if halves else (got[..., 0::2], got[..., 1::2])
    assert np.allclose(y + 1j * w, z) and np.all(np.abs(got) <= size + 1e-12)


STRUCTS = {"ts_append_latent_args": "AppendLatentArgs", "ts_heads_args": "HeadsArgs", "ts_latent_args": "LatentArgs",
           "ts_flash_latent_args": "FlashLatentArgs"}


def test_structs_match_the_compiler(tmp_path):
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    lines, want = ['#include <stddef.h>', '#include <stdio.h>', f'#include "{abi.HEADER}"', "int main(void) {"], []
    for cname, name in STRUCTS.items():
        st = getattr(abi, name)
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        want.append(C.sizeof(st))
        for field, _ in st._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {field}));')
            want.append(getattr(st, field).offset)
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == want


FAKE = 1 << 20  # 16-byte aligned, never dereferenced on these paths


def _no_gpu():
    if torch.cuda.device_count() > 0:
        pytest.skip("fake device addresses are only passed where no GPU could run them")


def _refused(fn, args, text, code=abi.TS_ERR_ARG):
    _no_gpu()
    lib = abi.load()
    assert getattr(lib, fn)(C.byref(args), None) == code
    assert text in lib.tessera_hip_last_error(), lib.tessera_hip_last_error()


def _append(**over):
    a = abi.AppendLatentArgs()
    for name in ("c", "q", "gain", "rope_table", "q_out", "kept", "c_out", "r_out", "slots", "positions", "kept_table"):
        setattr(a, name, FAKE)
    a.q_out = 2 * FAKE
    a.rows, a.heads, a.rank, a.rope, a.c_stride = 3, 16, 512, 64, 576
    a.q_stride, a.q_head, a.q_out_stride, a.q_out_head = 4096, 192, 1024, 64
    a.keys, a.slot_count, a.kept_pages, a.page, a.pages, a.rope_rows = 256, 2, 16, 16, 32, 256
    a.halves, a.x_dtype, a.q_out_dtype, a.eps = 1, abi.TS_BF16, abi.TS_BF16, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(c=None), b"null"), (dict(kept=None), b"null"), (dict(slots=None), b"null"), (dict(rank=0), b"rank 0"),
    (dict(rank=508), b"rank 508"), (dict(rank=1032), b"rank 1032"), (dict(rope=8), b"8 rotated"), (dict(rope=48), b"48 rotated"),
    (dict(rope=256), b"256 rotated"), (dict(x_dtype=abi.TS_E4M3), b"f32 or bf16"), (dict(page=24), b"page 24"),
    (dict(page=8), b"page 8"), (dict(slot_count=0), b"slots"), (dict(pages=0), b"0 pages"), (dict(rope_rows=255), b"255 rows"),
    (dict(c_stride=568), b"apart"), (dict(c_stride=580), b"16-byte"), (dict(c=FAKE + 8), b"aligned"),
    (dict(kept=FAKE + 8), b"aligned"), (dict(gain=FAKE + 4), b"aligned"), (dict(c_out=FAKE + 2), b"aligned"),
    (dict(q_out=None), b"q_out"), (dict(heads=0), b"0 heads"), (dict(q_head=196), b"16-byte"), (dict(q_out_head=36), b"16-byte"),
    (dict(q_out_head=32), b"heads 32 apart"), (dict(q_out_dtype=abi.TS_E4M3), b"q out"), (dict(q=FAKE + 8), b"aligned"),
    (dict(q_out=FAKE), b"in place"), (dict(kept_table=None, keys=300), b"kept rows hold"),
])
def test_append_refusals(over, text):
    _refused("tessera_hip_append_latent", _append(**over), text)


def _heads(**over):
    a = abi.HeadsArgs(FAKE, FAKE, FAKE, 3, 16, 512, 128, 16 * 192, 192, 16 * 576, 576, 512 * 128, abi.TS_BF16, abi.TS_BF16)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(x=None), b"null"), (dict(w=None), b"null"), (dict(out=None), b"null"), (dict(x_dtype=abi.TS_U32), b"x f32 or bf16"),
    (dict(out_dtype=abi.TS_E4M3), b"out f32 or bf16"), (dict(heads=0), b"0 heads"), (dict(n=0), b"n 0"), (dict(k=0), b"k 0"),
    (dict(k=100), b"k 100"), (dict(x_head=196), b"16-byte"), (dict(x_stride=3076), b"16-byte"), (dict(w_head=512 * 128 + 4), b"16-byte"),
    (dict(w_head=512 * 64), b"heads of w"), (dict(out_head=500), b"meet"), (dict(out_stride=500), b"meet"),
    (dict(x=FAKE + 8), b"aligned"), (dict(w=FAKE + 8), b"aligned"), (dict(out=FAKE + 1), b"aligned"),
])
def test_heads_refusals(over, text):
    _refused("tessera_hip_linear_heads", _heads(**over), text)


def _attend(rows=2, rank=512, slot_count=2, pages=1024, run=1, **over):
    r = abi.RowsArgs()
    r.q = r.k = r.out = r.slots = r.positions = r.kept_table = FAKE
    r.rows, r.keys, r.heads, r.kv_heads, r.width, r.back = rows, 8192, 16, 1, 576, abi.U32_MAX
    r.kept_pages, r.page, r.scale, r.max_position = 512, 16, 0.07, 8191
    r.q_dtype = r.kv_dtype = r.out_dtype = abi.TS_BF16
    for k, v in over.items():
        setattr(r, k, v)
    return abi.LatentArgs(r, rank, slot_count, pages, run)


@pytest.mark.parametrize("over,text", [
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(positions=None), b"null"), (dict(rank=256), b"256 of them"),
    (dict(width=544), b"576 and 512"), (dict(kv_heads=2), b"2 rows"), (dict(heads=0), b"0 heads"), (dict(heads=2000), b"2000 heads"),
    (dict(q_dtype=abi.TS_F32), b"bf16 supported"), (dict(kv_dtype=abi.TS_E4M3), b"bf16 supported"),
    (dict(out_dtype=abi.TS_F32), b"bf16 supported"), (dict(page=20), b"page 20"), (dict(slot_count=0), b"slots"),
    (dict(kept_table=None, keys=250), b"whole blocks"), (dict(kept_table=None), b"ok"), (dict(keys=1 << 31), b"positions a slot"),
    (dict(q=FAKE + 8), b"aligned"), (dict(k=FAKE + 8), b"aligned"), (dict(out=FAKE + 4), b"aligned"),
])
def test_attend_refusals(over, text):
    if text == b"ok":  # refused for its workspace alone
        _refused("tessera_hip_attend_latent", _attend(**over), b"workspace", abi.TS_ERR_WORKSPACE)
    else:
        _refused("tessera_hip_attend_latent", _attend(**over), text)


def test_attend_workspace():
    _no_gpu()
    lib = abi.load()
    a = _attend()
    need = lib.tessera_hip_attend_latent_workspace(C.byref(a))
    assert need > 0
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 8, need)):
        a.rows.workspace, a.rows.workspace_bytes = ws, size
        assert lib.tessera_hip_attend_latent(C.byref(a), None) == abi.TS_ERR_WORKSPACE


def _flash(**over):
    a = abi.FlashLatentArgs(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 100, 120, 2, 16, 128, 64, 128, 16 * 192, 4096, 256, 4096,
                            256, 64, abi.U32_MAX, 0.07)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(r=None), b"null"), (dict(out=None), b"null"),
    (dict(nope=64), b"64 + 64"), (dict(rope=32), b"128 + 32"), (dict(value=64), b"and 64 values"), (dict(heads=0), b"0 heads"),
    (dict(first=None), b"without their bounds"), (dict(first=None, seqs=1), b"without those of the rows"),
    (dict(q_stride=16 * 128), b"q rows"), (dict(q_stride=16 * 192 + 4), b"16-byte"), (dict(k_head=100), b"16-byte"),
    (dict(r_stride=68), b"16-byte"), (dict(v=FAKE + 8), b"aligned"), (dict(k_stride=1 << 26), b"apart"),
    (dict(rows=1 << 29), b"rows"),
])
def test_flash_refusals(over, text):
    _refused("tessera_hip_flash_latent", _flash(**over), text)


def test_more_rows_than_one_launch_takes():
    _refused("tessera_hip_append_latent", _append(rows=1 << 28), b"in one launch")
    _refused("tessera_hip_linear_heads", _heads(rows=1 << 30), b"in one launch")
    _refused("tessera_hip_attend_latent", _attend(rows=1 << 27), b"in one launch")
    _refused("tessera_hip_flash_latent", _flash(rows=1 << 28), b"in one launch")


def test_empty_calls_need_no_pointers():
    _no_gpu()
    lib = abi.load()
    a = _append(rows=0, c=None, q=None, q_out=None, slots=None, positions=None, c_out=None, r_out=None)
    assert lib.tessera_hip_append_latent(C.byref(a), None) == abi.TS_OK
    assert lib.tessera_hip_linear_heads(C.byref(_heads(rows=0, x=None, out=None)), None) == abi.TS_OK
    a = _attend(rows=0, q=None, out=None, slots=None, positions=None)
    assert lib.tessera_hip_attend_latent_workspace(C.byref(a)) == 0
    assert lib.tessera_hip_attend_latent(C.byref(a), None) == abi.TS_OK
    assert lib.tessera_hip_flash_latent(C.byref(_flash(rows=0, q=None, out=None)), None) == abi.TS_OK
    assert lib.tessera_hip_flash_latent(C.byref(_flash(seqs=0)), None) == abi.TS_OK
    for fn in (lib.tessera_hip_append_latent, lib.tessera_hip_linear_heads, lib.tessera_hip_attend_latent,
               lib.tessera_hip_flash_latent):
        assert fn(None, None) == abi.TS_ERR_ARG


def test_python_refuses_before_any_launch():
    """Types, shapes and devices that the entry points could not tell from pointers."""
    t = lambda *s, d=torch.bfloat16: torch.zeros(*s, dtype=d)  # noqa: E731
    i = t(3, d=torch.int32)
    with pytest.raises(ValueError, match="not on a GPU"):
        rules.append_latent(t(3, 576), t(64, 576), i, i, keys=64, rank=512)
    with pytest.raises(ValueError, match="f32 or bf16"):
        rules.append_latent(t(3, 576, d=torch.float16), t(64, 576), i, i, keys=64, rank=512)
    with pytest.raises(ValueError, match="kept rows of 575"):
        rules.append_latent(t(3, 576), t(64, 575), i, i, keys=64, rank=512)
    with pytest.raises(ValueError, match="q and q_out must be"):
        rules.append_latent(t(3, 576), t(64, 576), i, i, keys=64, rank=512, q=t(3, 4, 32))
    with pytest.raises(ValueError, match="back to back"):
        rules.append_latent(t(3, 576), t(64, 576), i, i, keys=64, rank=512, q=t(3, 64, 4).transpose(1, 2))
    with pytest.raises(ValueError, match="on a GPU"):
        rules.linear_heads(t(3, 4, 64), t(4, 32, 64))
    with pytest.raises(ValueError, match="back to back"):
        rules.linear_heads(t(3, 4, 128)[..., ::2], t(4, 32, 64))
    with pytest.raises(ValueError, match="not on a GPU"):
        rules.attend_latent(t(3, 4, 576), t(64, 576), i, i, keys=64, rank=512, scale=1.0)
    with pytest.raises(ValueError, match="kept rows of 288"):
        rules.attend_latent(t(3, 4, 576), t(64, 288), i, i, keys=64, rank=512, scale=1.0)
    with pytest.raises(ValueError, match="out must be"):
        rules.attend_latent(t(3, 4, 576), t(64, 576), i, i, keys=64, rank=512, scale=1.0, out=t(3, 4, 576))
    with pytest.raises(ValueError, match="nope"):
        rules.flash_latent(t(3, 4, 192), t(5, 4, 96), t(5, 4, 128), t(5, 64), scale=1.0)
    with pytest.raises(ValueError, match="key_first without first"):
        rules.flash_latent(t(3, 4, 192), t(5, 4, 128), t(5, 4, 128), t(5, 64), scale=1.0, key_first=t(2, d=torch.int32))
    with pytest.raises(ValueError, match="not on a GPU"):
        rules.flash_latent(t(3, 4, 192), t(5, 4, 128), t(5, 4, 128), t(5, 64), scale=1.0)
    x = t(3, 4, 64)
    with pytest.raises(ValueError, match="out lies where x"):
        rules.linear_heads(x, t(4, 64, 64), out=x)
    x = t(3, 4, 576)
    with pytest.raises(ValueError, match="out lies where q"):
        rules.attend_latent(x, t(64, 576), i, i, keys=64, rank=512, scale=1.0, out=x.flatten()[:3 * 4 * 512].view(3, 4, 512))
    x = t(3, 4, 192)
    with pytest.raises(ValueError, match="out lies where q"):
        rules.flash_latent(x, t(5, 4, 128), t(5, 4, 128), t(5, 64), scale=1.0, out=x.flatten()[:3 * 4 * 128].view(3, 4, 128))
