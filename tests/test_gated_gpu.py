"""gated_scan on the B200 against the recurrence in 64 bits.

Tolerances, with u = 2^-24 and before any run.  A gate is expf of g within 2 ulp (2 u relative, with the rounding
of g's own exponent) and a step one fused multiply-add (u): a state that remembers m = 1 / (1 - a) tokens carries
at most 3 u m of its own size; segments' factors are products of up to 32 x 256 gates, off by as much as the same
tokens' steps.  The tests' gates remember up to m = 60 tokens and errors of tokens are independent (sqrt m):
3 u * 8 * 2 (factor and state) = 48 u = 2.9e-6 relative to the output's norm, twice that for dg, the product of
two such values.  Half a step of bf16, 2^-8, covers a rounded output.
"""
import math
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
import atomic_gdn2  # noqa: E402
from atomic_gdn2 import gated_scan, last_status  # noqa: E402
from training_ref import gated_ref  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TOL = {torch.float32: 48 * U, torch.bfloat16: 48 * U + 2.0 ** -8}


@pytest.fixture(autouse=True, params=["binding", "python"])
def _path(request):
    """The common call through the compiled binding; with checks at once everything goes the Python way."""
    atomic_gdn2.set_checks("async" if request.param == "binding" else "sync")
    yield
    atomic_gdn2.set_checks("async")
    assert last_status() == 0


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double()
    assert a.shape == b.shape
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


def _inputs(B, L, C, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, L, C, generator=gen).to(dtype)
    g = -torch.exp(torch.randn(B, L, C, generator=gen) * 0.5 - 4.0 * torch.rand(C, generator=gen)).to(dtype)
    return x, g, torch.randn(B, C, generator=gen), torch.randn(B, L, C, generator=gen).to(dtype), torch.randn(B, C, generator=gen)


SIZES = [(1, 1, 1), (3, 2, 5), (2, 4, 64), (2, 5, 33), (1, 31, 7), (2, 32, 32), (1, 33, 96), (4, 130, 40), (2, 257, 31), (1, 1000, 34),
         (3, 513, 129), (1, 2500, 8), (1, 5000, 66), (40, 300, 32), (5, 777, 100)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("masks", ["", "lengths", "reset", "both"])
@pytest.mark.parametrize("B,L,C", SIZES)
def test_matches_the_recurrence(B, L, C, masks, dtype):
    x, g, h0, dy, dl = _inputs(B, L, C, dtype, B * 1000 + L + C)
    gen = torch.Generator().manual_seed(L)
    lengths = reset = None
    if masks in ("lengths", "both"):
        lengths = torch.randint(0, L + 1, (B,), generator=gen, dtype=torch.int32)
        lengths[0] = L
        if B > 1:
            lengths[1] = 0
    if masks in ("reset", "both"):
        reset = torch.rand(B, L, generator=gen) < 0.05
    ref = [t.double().requires_grad_(True) for t in (x, g, h0)]
    h_r, l_r = gated_ref(*ref, lengths, reset)
    grads_r = torch.autograd.grad((h_r, l_r), ref, (dy.double(), dl.double()))
    dev = [t.cuda().requires_grad_(True) for t in (x, g, h0)]
    kw = dict(lengths=None if lengths is None else lengths.cuda(), reset=None if reset is None else reset.cuda())
    h, last = gated_scan(*dev, **kw)
    grads = torch.autograd.grad((h, last), dev, (dy.cuda(), dl.cuda()))
    assert h.dtype == dtype and last.dtype == torch.float32
    assert _rel(h, h_r) < TOL[dtype] and _rel(last, l_r) < TOL[torch.float32]
    for n, a, b, t in zip(("dx", "dg", "dh0"), grads, grads_r, (x, g, h0)):
        assert a.dtype == t.dtype
        assert _rel(a, b) < 2 * TOL[t.dtype], n
    with torch.no_grad():
        h2, last2 = gated_scan(*dev, **kw)
    if L > 4:
        assert torch.equal(h2, h) and torch.equal(last2, last)
    else:  # a few tokens are walked, not joined
        assert _rel(h2, h_r) < TOL[dtype] and _rel(last2, l_r) < TOL[torch.float32]
