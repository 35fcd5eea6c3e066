"""gated_scan on the B200: states that decay to nothing, types that are widened.

Tolerances as in the tests beside this one, u = 2^-24: a gate within 2 u and a step's rounding u make 3 u a token of a
state's own size; half a step of bf16 is 2^-9 of a value."""
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2 import gated_scan, last_status  # noqa: E402
from training_ref import gated_ref  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _status():
    yield
    assert last_status() == 0


@pytest.mark.parametrize("L,C", [(300, 8), (2000, 8), (2000, 40), (5000, 16), (700, 4736)])
@pytest.mark.parametrize("gate", [-1.0, -0.05, -90.0])
def test_a_large_state_decays_to_nothing(L, C, gate):
    """1e38 forgotten over more than a segment's tokens: what is left of it is what the recurrence leaves, and of it and of
    the 3e37 on the way no more than 2^-149 where a product of gates is held above zero, or two roundings of 2^-150 among
    the smallest numbers: 2.6e38 x 2^-149 for both."""
    x, g = torch.zeros(1, L, C), torch.full((1, L, C), gate)
    h0, dl = torch.full((1, C), 1e38), torch.full((1, C), -1e38)
    x[:, L // 2] = 3e37
    ref = [t.double().requires_grad_(True) for t in (x, g, h0)]
    h_r, l_r = gated_ref(*ref)
    want = torch.autograd.grad(l_r, ref, dl.double())
    dev = [t.cuda().requires_grad_(True) for t in (x, g, h0)]
    h, last = gated_scan(*dev)
    got = torch.autograd.grad(last, dev, dl.cuda())
    far = 2.6e38 * 2.0 ** -149

    def near(a, b):
        a, b = a.detach().double().cpu(), b.detach()
        assert bool(((a - b).abs() <= 3 * U * (L + 1) * b.abs() + far).all())

    near(h, h_r)
    near(last, l_r)
    near(got[0], want[0])
    near(got[2], want[2])
