"""Calls of the 8-bit cache's operators that are empty, refused or unusually laid out, through rules."""
import numpy as np
import pytest

import kept8_ref as K
from helpers import rng
from tessera_amd import abi, rules

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def test_empty_batches():
    """No rows, no sequences: empty outputs, nothing written."""
    k8, v8, s8 = rules.kept8(2, 2)
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    x = torch.empty(0, 8, 128, device="cuda")
    q = rules.append_rows(x[:, 4:6], x[:, 6:], k8, v8, i, i, q=x[:, :4], keys=32, scales=s8)
    assert q.shape == (0, 4, 128) and int(k8.count_nonzero()) == int(s8.count_nonzero()) == 0
    rows = torch.zeros(32, 2, 128, dtype=torch.bfloat16, device="cuda")
    assert rules.append_rows(x[:, 4:6], x[:, 6:], rows, rows.clone(), i, i, keys=32) is None
    assert rules.attend_kept8(q, k8, v8, s8, i, i, keys=32, scale=1.0).shape == (0, 4, 128)
    u = torch.empty(0, 4, device="cuda")
    for logits in (torch.empty(0, 50, device="cuda"), torch.zeros(4, 50, device="cuda")):
        for uniforms in (None, u):
            tokens, accepted = rules.verify(logits, torch.empty(0, 3, dtype=torch.int32, device="cuda"), uniforms)
            assert tokens.shape == (0, 4) and accepted.shape == (0,)


def test_sequences_without_a_row_of_logits_are_refused():
    status, one = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for uniforms in (None, torch.zeros(2, 2, device="cuda")):
        status.zero_()
        tokens, accepted = rules.verify(torch.empty(0, 50, device="cuda"), torch.zeros(2, 1, dtype=torch.int32, device="cuda"),
                                        uniforms, counts=one, first=one, status=status)
        assert tokens.tolist() == [[50, 50]] * 2 and accepted.tolist() == [0, 0] and int(status) == abi.TS_STATUS_POSITION
