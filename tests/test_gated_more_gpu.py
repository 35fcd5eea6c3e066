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


HALF = {torch.float32: 0.0, torch.float64: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("L,C", [(1, 7), (130, 40), (1000, 33)])
@pytest.mark.parametrize("tx,tg", [(a, b) for a in HALF for b in HALF])
def test_types(tx, tg, L, C):
    """Any two floating types: taken as they are where both are fp32 or both bf16, else as fp32, and h and the gradients come
    back in their inputs' types, rounded once (half a step; fp64 inputs here are fp32's values).  fp32's own part of the
    error as in the tests beside this one: 48 u of the norm, twice that for gradients."""
    gen = torch.Generator().manual_seed(L)
    x, h0, dy = (torch.randn(2, L, C, generator=gen).to(tx) for _ in range(3))
    g, h0, dl = (-torch.rand(2, L, C, generator=gen) - 0.02).to(tg), h0[:, 0].float(), torch.randn(2, C, generator=gen)
    ref = [t.double().requires_grad_(True) for t in (x, g, h0)]
    h_r, l_r = gated_ref(*ref)
    want = torch.autograd.grad((h_r, l_r), ref, (dy.double(), dl.double()))
    dev = [t.cuda().requires_grad_(True) for t in (x, g, h0)]
    h, last = gated_scan(*dev)
    assert h.dtype == tx and last.dtype == torch.float32
    got = torch.autograd.grad((h, last), dev, (dy.cuda(), dl.cuda()))
    with torch.no_grad():
        h2, l2 = gated_scan(*dev)
    assert h2.dtype == tx and torch.equal(h, h2) and torch.equal(last, l2)

    def near(a, b, tol):
        assert float((a.detach().double().cpu() - b.detach()).norm()) <= tol * float(b.detach().norm())

    near(h, h_r, 48 * U + HALF[tx])
    near(last, l_r, 48 * U)
    for a, b, t in zip(got, want, (x, g, h0)):
        assert a.dtype == t.dtype
        near(a, b, 96 * U + HALF[t.dtype])


def test_whole_numbers():
    """Whole numbers are taken as fp32, and h comes back as that."""
    x, g = torch.tensor([[[2], [3], [4]]], device="cuda"), torch.zeros(1, 3, 1, device="cuda")
    h, last = gated_scan(x, g)
    assert h.dtype == torch.float32 and h.flatten().tolist() == [2.0, 5.0, 9.0] and float(last) == 9.0
