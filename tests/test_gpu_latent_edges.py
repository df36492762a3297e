"""Calls of latent attention at the edges of what its entry points take, on the GPU."""
import numpy as np
import pytest

import latent_ref as L
from helpers import rng
from tessera_amd import abi, rules
from test_gpu_latent import BF16, F32, HALF, WIDTHS, attend, cache, check_attend, check_flash, dev, f64, flash_inputs, ints, roomier

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("widths", ["wide", "narrow"])
def test_flash_of_broadcast_rows(widths):
    """q, k, v and r that are one row for all."""
    r = rng(21)
    q, k, v, rr = flash_inputs(r, 1, 1, 3, widths)
    many = [x.expand(n, *x.shape[1:]) for x, n in ((q, 150), (k, 170), (v, 170), (rr, 170))]
    got = rules.flash_latent(*many, scale=0.1)
    assert torch.equal(got, rules.flash_latent(*(x.contiguous() for x in many), scale=0.1))
    check_flash(got, *many, first=[0, 150], key_first=[0, 170], scale=0.1)
    one = rules.flash_latent(q, *many[1:], scale=0.1)  # (a row by itself has no distance either)
    assert torch.equal(one, got[149:])
