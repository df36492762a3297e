"""CPU checks of calls of the 8-bit cache's operators: what is empty, what is refused, where a call goes."""
import ctypes as C

import pytest

from tessera_amd import abi
from test_kept8_ref import FAKE, _append, _attend, _no_gpu, _verify

torch = pytest.importorskip("torch")


def test_no_rows_and_no_sequences_need_no_pointers():
    """Tensors without elements have no address."""
    _no_gpu()
    lib = abi.load()
    none = dict.fromkeys(("q", "k", "v", "q_out", "slots", "positions"))
    assert lib.tessera_hip_append_rows(C.byref(_append(rows=0, **none)), None) == abi.TS_OK
    assert lib.tessera_hip_append_rows(C.byref(_append(rows=0, **dict(none, q=FAKE))), None) == abi.TS_OK
    a = _attend(rows=0, q=None, out=None, slots=None, positions=None)
    assert lib.tessera_hip_attend_kept8_workspace(C.byref(a)) == 0
    assert lib.tessera_hip_attend_kept8(C.byref(a), None) == abi.TS_OK
    for uniforms in (None, FAKE):
        a = _verify(seqs=0, drafts=None, tokens=None, accepted=None, uniforms=uniforms, workspace=None)
        assert lib.tessera_hip_verify_workspace(C.byref(a)) == 0
        assert lib.tessera_hip_verify(C.byref(a), None) == abi.TS_OK
        a.rows, a.logits = 0, None
        assert lib.tessera_hip_verify(C.byref(a), None) == abi.TS_OK


def test_arguments_of_no_rows_are_still_checked():
    _no_gpu()
    lib = abi.load()
    assert lib.tessera_hip_append_rows(C.byref(_append(rows=0, width=64)), None) == abi.TS_ERR_ARG
    assert lib.tessera_hip_append_rows(C.byref(_append(rows=0, k_kept=None)), None) == abi.TS_ERR_ARG
    assert lib.tessera_hip_attend_kept8(C.byref(_attend(rows=0, page=20)), None) == abi.TS_ERR_ARG
    assert lib.tessera_hip_verify(C.byref(_verify(seqs=0, width=0)), None) == abi.TS_ERR_ARG
    assert lib.tessera_hip_verify(C.byref(_verify(logits=None)), None) == abi.TS_ERR_ARG
    for fn in (lib.tessera_hip_append_rows, lib.tessera_hip_attend_kept8, lib.tessera_hip_verify):
        assert fn(None, None) == abi.TS_ERR_ARG


def test_bf16_logits_may_begin_at_any_element():
    """f32 logits at any f32, bf16 ones at any bf16: past the alignment, the workspace is what is asked for."""
    _no_gpu()
    lib = abi.load()
    for dtype, at, want in ((abi.TS_BF16, 2, abi.TS_ERR_WORKSPACE), (abi.TS_BF16, 1, abi.TS_ERR_ARG),
                            (abi.TS_F32, 4, abi.TS_ERR_WORKSPACE), (abi.TS_F32, 2, abi.TS_ERR_ARG)):
        a = _verify(logits=FAKE + at, logits_dtype=dtype, workspace=None)
        assert lib.tessera_hip_verify(C.byref(a), None) == want


def test_page_copies_go_to_the_buffers_device(monkeypatch):
    """The copies of kept blocks (and kept rows) run on the stream of the device that holds them, whichever device is
    current: the launch is made under that device."""
    from tessera_amd import kv, rules
    under, launched = [], []

    class Device:
        def __init__(self, on):
            self.on = on

        def __enter__(self):
            under.append(self.on)

        def __exit__(self, *_):
            under.pop()

    class Stream:
        cuda_stream = 64

    class Library:
        def tessera_hip_kv_copy(self, args, stream):
            launched.append((list(under), stream.value))
            return abi.TS_OK

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: Stream)
    monkeypatch.setattr(kv, "lib", Library)
    k8, v8, s8 = rules.kept8(4, 2, device="cpu")
    kv.copy_kept8(k8, v8, s8, [(0, 3, 5)], page=16)
    kv.copy_pages([torch.zeros(64, 2, 128)], [(1, 2, 16)], page=16, pages=4)
    assert launched == [([torch.device("cpu")], 64)] * 3 and not under


@pytest.mark.parametrize("blocks,page,want", [(5, 32, (2, 8192)), (8, 64, (2, 16384)), (3, 16, (3, 4096))])
def test_copied_pages_are_whole_blocks(monkeypatch, blocks, page, want):
    """A page is page / 16 blocks, however many blocks are left over; pages that are not blocks are refused."""
    from tessera_amd import kv, rules
    copied = []
    monkeypatch.setattr(kv, "copy_pages", lambda buffers, copies, **kw: copied.extend((tuple(b.shape), kw["pages"]) for b in buffers))
    k8, v8, s8 = rules.kept8(blocks, 2, device="cpu")
    kv.copy_kept8(k8, v8, s8, [(0, 1, 7)], page=page)
    assert copied == [(want, want[0])] * 2 + [((want[0], page // 16 * 4), want[0])]
    for bad in (24, 8, 0):
        with pytest.raises(ValueError, match="whole blocks"):
            kv.copy_kept8(k8, v8, s8, [(0, 1, 7)], page=bad)


def test_the_stated_error_of_the_verifications_exponentials():
    """verify.hip's series for 2^f, its coefficients read from the source, against longdouble exponentials: at most
    1.1e-10 off, 2^0 exact; and what that does to the borders of a wide row's running sum."""
    import os
    import re

    import numpy as np
    with open(os.path.join(os.path.dirname(abi.__file__), "csrc", "verify.hip")) as f:
        source = f.read()
    body = source[source.index("TS_DEV double exp2_neg"):source.index("TS_DEV void weights")]
    magic, same, *series = (float(c) for c in re.findall(r"scalar\(([\d.e+-]+)\)", body))
    assert magic == same == 1.5 * 2 ** 52 and len(series) == 7

    def exp2(t):
        n = (t + magic) - magic
        f, r = t - n, np.float64(series[0])
        for c in series[1:]:
            r = r * f + c
        return np.ldexp(r * f + 1.0, n.astype(int))

    t = np.linspace(-3, 0, 3000001)
    exact = np.exp2(t.astype(np.longdouble))
    assert np.max(np.abs(exp2(t) / exact - 1)) < 1.101e-10 and exp2(np.zeros(1))[0] == 1.0
    r = np.random.default_rng(1)
    for temperature in (0.75, 1.0, 1.25):
        x = 2 * r.standard_normal(151936)
        x[r.integers(0, len(x), 24)] = 9 + 3 * r.standard_normal(24)
        y = (x - x.max()) * (np.log2(np.e) / temperature)
        a, b = exp2(y).astype(np.longdouble), np.exp2(y.astype(np.longdouble))
        moved = np.abs(np.cumsum(a) / a.sum() - np.cumsum(b) / b.sum())
        assert moved.max() < 6e-12 and moved.sum() < 6e-7
