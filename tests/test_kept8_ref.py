"""CPU checks of the float64 forms that the GPU tests compare with, and of the calls' refusals."""
import ctypes as C

import numpy as np
import pytest

import kept8_ref as K
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")


def test_narrow_every_code_and_tie():
    """Every finite code is its own; between neighbours the nearer, the even one at a tie."""
    assert np.array_equal(K.narrow(K.CODES[:127]), np.arange(127))
    lo, hi = K.CODES[:126], K.CODES[1:127]
    mid = (lo + hi) / 2
    assert np.array_equal(K.narrow(mid), np.where(np.arange(126) % 2, np.arange(1, 127), np.arange(126)))
    assert np.array_equal(K.narrow(mid * (1 + 1e-12)), np.arange(1, 127))
    assert np.array_equal(K.narrow([500.0, -500.0, np.inf, -np.inf]), [0x7E, 0xFE, 0x7F, 0xFF])
    x = torch.randn(100000, generator=torch.Generator().manual_seed(1)) * 30
    got = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(K.narrow(x.numpy()), got)


def test_exponent_is_the_least():
    for amax in (1e-30, 3.0, 447.99, 448.0, np.nextafter(448.0, 500), 1e30):
        e = K.exponent(amax)
        assert amax <= 448.0 * 2.0 ** e and (e == -100 or amax > 448.0 * 2.0 ** (e - 1))
    assert K.exponent(0) == -100 and K.exponent(3e38) == 119


def test_attend_ref_is_softmax():
    """One head over dense blocks: torch's softmax over the dequantised keys."""
    r = np.random.default_rng(2)
    k = K.narrow(r.standard_normal((2, 1, 16, 128)) * 40)
    v = K.narrow(r.standard_normal((2, 1, 128, 16)) * 40)
    s = np.full((2, 2, 2), 2.0 ** -5)
    q = r.standard_normal((1, 2, 128)).astype(np.float32)
    out, _, _ = K.attend(q, k, v, s, [0], [20], scale=0.1, keys=32)
    kk = torch.from_numpy(K.CODES[k[:, 0]].reshape(32, 128) / 32)[:21]
    vv = torch.from_numpy(K.CODES[v[:, 0]].transpose(0, 2, 1).reshape(32, 128) / 32)[:21]
    want = torch.softmax(torch.from_numpy(q[0]).double() @ kk.T * 0.1, -1) @ vv
    assert np.allclose(out[0], want.numpy(), atol=1e-12)


def test_verify_ref_keeps_the_targets_distribution():
    """Accepted or redrawn, the first token is distributed as the target whatever the drafter's q."""
    r = np.random.default_rng(3)
    p, q = r.dirichlet(np.ones(6)), r.dirichlet(np.ones(6)).astype(np.float32)
    n = 20000
    drafts = r.choice(6, (n, 1), p=q / q.astype(np.float64).sum())
    u = r.random((n, 2)).astype(np.float32)
    logits = np.tile(np.log(p).astype(np.float32), (2 * n, 1))
    tokens, _ = K.verify(logits, drafts, u, probs=np.tile(q, (n, 1, 1)))
    share = np.bincount(tokens[:, 0], minlength=6) / n
    # A share's standard error is below sqrt(1/4 / n) = 0.0035: five of them.
    assert np.max(np.abs(share - p)) < 0.018


STRUCTS = {"ts_append_args": "AppendArgs", "ts_kept8_args": "Kept8Args", "ts_verify_args": "VerifyArgs"}


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


def _append(**over):
    a = abi.AppendArgs()
    a.q = a.k = a.v = a.q_out = a.k_kept = a.v_kept = a.scales = a.slots = a.positions = a.kept_table = FAKE
    a.rows, a.heads, a.kv_heads, a.width, a.keys, a.slot_count, a.kept_pages = 3, 16, 8, 128, 256, 2, 16
    a.q_stride, a.k_stride, a.v_stride, a.page, a.pages, a.halves = 2048, 1024, 1024, 16, 32, 1
    a.x_dtype, a.q_out_dtype, a.kv_dtype, a.eps = abi.TS_F32, abi.TS_F32, abi.TS_E4M3, 1e-6
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(k=None), b"null"), (dict(positions=None), b"null"), (dict(width=64), b"width 64"), (dict(kv_heads=0), b"kv heads"),
    (dict(scales=None), b"scales"), (dict(page=24), b"page 24"), (dict(page=8), b"page 8"), (dict(x_dtype=abi.TS_E4M3), b"f32 or bf16"),
    (dict(kv_dtype=abi.TS_F32), b"bf16 or e4m3"), (dict(k_stride=1022), b"apart"), (dict(v_stride=1026), b"16-byte"),
    (dict(k=FAKE + 4), b"aligned"), (dict(scales=FAKE + 8), b"aligned"), (dict(rope_table=FAKE, rope_rows=255), b"255 rows"),
    (dict(kept_table=None, keys=250), b"whole blocks"), (dict(kept_table=None, pages=31), b"kept rows hold"),
    (dict(q_out=None), b"q_out"), (dict(q_stride=1024), b"q rows"), (dict(q_out_dtype=abi.TS_E4M3), b"q out"),
    (dict(q_out_dtype=abi.TS_BF16), b"in place"), (dict(slot_count=0), b"slots"), (dict(pages=0), b"0 pages"),
])
def test_append_refusals(over, text):
    _no_gpu()
    lib = abi.load()
    a = _append(**over)
    assert lib.tessera_hip_append_rows(C.byref(a), None) == abi.TS_ERR_ARG
    assert text in lib.tessera_hip_last_error()


def _attend(rows=2, **over):
    r = abi.RowsArgs()
    r.q = r.k = r.v = r.out = r.slots = r.positions = r.kept_table = FAKE
    r.rows, r.keys, r.heads, r.kv_heads, r.width, r.back = rows, 8192, 16, 8, 128, abi.U32_MAX
    r.kept_pages, r.page, r.scale, r.max_position = 512, 16, 0.088, 8191
    r.q_dtype, r.kv_dtype, r.out_dtype = abi.TS_F32, abi.TS_E4M3, abi.TS_F32
    a = abi.Kept8Args(r, FAKE, 2, 1024, 1)
    for k, v in over.items():
        setattr(a if hasattr(abi.Kept8Args, k) and k != "rows" else a.rows, k, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(q=None), b"null"), (dict(scales=None), b"null"), (dict(width=64), b"width 64"), (dict(heads=12), b"12 heads"),
    (dict(heads=8 * 65), b"at most 64"), (dict(kv_dtype=abi.TS_BF16), b"e4m3"), (dict(q_dtype=abi.TS_E4M3), b"q and out"),
    (dict(out_dtype=abi.TS_E4M3), b"q and out"), (dict(page=20), b"page 20"), (dict(keys=0), b"positions"),
    (dict(kept_table=None, keys=8190), b"whole blocks"), (dict(k=FAKE + 8), b"aligned"), (dict(slot_count=0), b"slots"),
])
def test_attend_refusals(over, text):
    _no_gpu()
    lib = abi.load()
    a = _attend(**over)
    assert lib.tessera_hip_attend_kept8(C.byref(a), None) == abi.TS_ERR_ARG
    assert text in lib.tessera_hip_last_error()


def test_attend_workspace_is_asked_for_and_checked():
    _no_gpu()
    lib = abi.load()
    a = _attend()
    need = lib.tessera_hip_attend_kept8_workspace(C.byref(a))
    assert need > 0
    for workspace, size in ((None, need), (FAKE, need - 1), (FAKE + 8, need)):
        a.rows.workspace, a.rows.workspace_bytes = workspace, size
        assert lib.tessera_hip_attend_kept8(C.byref(a), None) == abi.TS_ERR_WORKSPACE
    a.rows.rows = 0
    assert lib.tessera_hip_attend_kept8_workspace(C.byref(a)) == 0
    assert lib.tessera_hip_attend_kept8(C.byref(a), None) == abi.TS_OK


def _verify(**over):
    a = abi.VerifyArgs()
    a.logits = a.drafts = a.uniforms = a.tokens = a.accepted = a.workspace = FAKE
    a.seqs, a.most, a.rows, a.width, a.stride, a.logits_dtype, a.temperature = 2, 4, 10, 1000, 1000, abi.TS_F32, 1.0
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,text", [
    (dict(logits=None), b"null"), (dict(drafts=None), b"null"), (dict(accepted=None), b"null"), (dict(most=65, rows=200), b"65 drafts"),
    (dict(logits_dtype=abi.TS_E4M3), b"f32 or bf16"), (dict(stride=999), b"apart"), (dict(width=0), b"logits"),
    (dict(rows=9), b"9 rows"), (dict(logits=FAKE + 2), b"aligned"),
])
def test_verify_refusals(over, text):
    _no_gpu()
    lib = abi.load()
    a = _verify(**over)
    assert lib.tessera_hip_verify(C.byref(a), None) == abi.TS_ERR_ARG
    assert text in lib.tessera_hip_last_error()


def test_verify_workspace_is_asked_for_and_checked():
    _no_gpu()
    lib = abi.load()
    a = _verify()
    a.workspace_bytes = lib.tessera_hip_verify_workspace(C.byref(a)) - 1
    assert lib.tessera_hip_verify(C.byref(a), None) == abi.TS_ERR_WORKSPACE
    a.seqs = 0
    assert lib.tessera_hip_verify(C.byref(a), None) == abi.TS_OK


def test_rules_refuse_what_is_not_on_a_gpu_or_misshapen():
    k = torch.zeros(2, 8, 128)
    i = torch.zeros(2, dtype=torch.int32)
    kk, kv, sc = rules.kept8(4, 8, device="cpu")
    assert kk.shape == (4, 8, 16, 128) and kv.shape == (4, 8, 128, 16) and sc.shape == (4, 8, 2)
    assert rules.kept8(2, 3, page=64, device="cpu")[2].shape == (8, 4, 2)
    with pytest.raises(ValueError, match="not on a GPU"):
        rules.append_rows(k, k, kk, kv, i, i, keys=32, scales=sc)
    with pytest.raises(ValueError, match="one type"):
        rules.append_rows(k, k.bfloat16(), kk, kv, i, i, keys=32, scales=sc)
    with pytest.raises(ValueError, match="back to back"):
        rules.append_rows(k.transpose(0, 1), k.transpose(0, 1), kk, kv, i, i, keys=32, scales=sc)
    with pytest.raises(ValueError, match="not on a GPU"):
        rules.attend_kept8(k, kk, kv, sc, i, i, keys=32, scale=1.0)
    with pytest.raises(ValueError, match="kept blocks"):
        rules.attend_kept8(k, kk, kv, sc[:, :4], i, i, keys=32, scale=1.0)
    with pytest.raises(ValueError, match="not on a GPU"):
        rules.verify(torch.zeros(3, 50), torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="rows apart"):
        rules.verify(torch.zeros(1, 50).expand(3, 50), torch.zeros(1, 2, dtype=torch.int32))


def test_rules_refuse_rows_further_apart_than_the_arguments_say():
    """A distance past 32 bits would be taken modulo 2^32 by the C structs."""
    far = torch.empty(3, (1 << 32) // 128 + 8, 128, device="meta")
    i = torch.zeros(3, dtype=torch.int32)
    kk, kv, sc = rules.kept8(4, 8, device="cpu")
    with pytest.raises(ValueError, match="apart"):
        rules.append_rows(far[:, :8], far[:, 8:16], kk, kv, i, i, keys=32, scales=sc)
    near = torch.zeros(3, 8, 128)
    with pytest.raises(ValueError, match="apart"):
        rules.append_rows(near, near, kk, kv, i, i, keys=32, scales=sc, q=far[:, :8])
    with pytest.raises(ValueError, match="apart"):
        rules.verify(far.view(3, -1)[:, :50], torch.zeros(1, 2, dtype=torch.int32))
