"""What the entry points of latent attention hand to the library, seen on the CPU: the call itself is caught."""
import pytest

from tessera_amd import rules
from test_latent_ref import _append, _heads, _refused

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
