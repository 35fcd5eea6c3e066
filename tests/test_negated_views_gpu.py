"""Views whose values are their memory's negated (torch makes them of a conjugate's imaginary part): the training operators
read the values.  Equal, bit by bit, to the same call on copies."""
import pytest
import torch

from atomic_gdn2 import gated_scan, last_status, linear, set_checks
from atomic_gdn2.training import AdamW

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["binding", "python"])
def _path(request):
    set_checks("async" if request.param == "binding" else "sync")
    yield
    set_checks("async")
    assert last_status() == 0


def _negated(t):
    v = torch._neg_view(t.detach().neg().contiguous())
    assert v.is_neg() and v.is_contiguous() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [3, 200])
def test_linear(M, dtype):
    gen = torch.Generator(device="cuda").manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)
    x, w, b, r, dy = make(M, 64), make(64, 72), make(72), make(M, 72), make(M, 72)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = linear(*leaves[:3], act="gelu", residual=leaves[3])
    grads = torch.autograd.grad(want, leaves, dy)
    neg = [_negated(t).requires_grad_(True) for t in (x, w, b, r)]
    assert torch.equal(linear(*neg[:3], act="gelu", residual=neg[3]), want)
    with torch.no_grad():
        assert torch.equal(linear(*neg[:3], act="gelu", residual=neg[3]), want)
    y = linear(*leaves[:3], act="gelu", residual=leaves[3])
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(y, leaves, _negated(dy)), grads))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L", [1, 300])
def test_gated_scan(L, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)
    x, g, h0, dh, dl = make(2, L, 40), -make(2, L, 40).abs(), make(2, 40).float(), make(2, L, 40), make(2, 40).float()
    leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
    want = gated_scan(*leaves)
    grads = torch.autograd.grad(want, leaves, (dh, dl))
    neg = [_negated(t).requires_grad_(True) for t in (x, g, h0)]
    assert all(torch.equal(a, c) for a, c in zip(gated_scan(*neg), want))
    with torch.no_grad():
        assert all(torch.equal(a, c) for a, c in zip(gated_scan(*neg), want))
        with pytest.raises(ValueError):
            gated_scan(x, g, h0, h_out=_negated(h0))
    again = torch.autograd.grad(gated_scan(*leaves), leaves, (_negated(dh), _negated(dl)))
    assert all(torch.equal(a, c) for a, c in zip(again, grads))


def test_adamw():
    p, q = (torch.nn.Parameter(torch.ones(1, device="cuda")) for _ in range(2))
    (torch.complex(torch.ones(1, device="cuda"), p).conj() * torch.tensor([2 + 3j], device="cuda")).real.sum().backward()
    assert p.grad.is_neg()
    q.grad = p.grad.clone()
    for t in (p, q):
        AdamW([t], lr=0.1).step()
    assert torch.equal(p, q) and float(p.detach()) < 1.0
    bad = torch.nn.Parameter(_negated(torch.ones(3, device="cuda")))
    bad.grad = torch.ones(3, device="cuda")
    with pytest.raises(ValueError):
        AdamW([bad]).step()
