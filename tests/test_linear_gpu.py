"""linear on the B200 against 64 bits.

Tolerances, with u = 2^-24 and before any run.  fp32: the terms' products leave 2^-26 of each, the tensor cores sum
64 values in at most 24 additions that may truncate (2 u each of the partial sum) and the parts follow in rounded
additions: a sum of k products is off by (48 + k / 64) u of sum |a b|.  bf16: exact products, k / 16 + 8 truncating
additions: (k / 8 + 16) u of sum |a b|, and half a step of the output, 2^-8 of the value.  GELU's slope is at most
1.13, its own error 4 u.  bf16 gradients: dz is rounded (2^-8 of it) and GELU's slope is taken at a rounded z
(|slope'| <= 0.8: 0.8 * 2^-8 |z|): relative to sum |dz w| 2^-8 (1 + 0.8 |z|max |dy| / |dz|) -- checked in the norm,
where errors of different terms are independent: 3 * 2^-8 of the result's norm.
"""
import math
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
import atomic_gdn2  # noqa: E402
from atomic_gdn2 import last_status, linear  # noqa: E402
from training_ref import linear_ref  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True, params=["binding", "python"])
def _path(request):
    """The common call through the compiled binding; with checks at once everything goes the Python way."""
    atomic_gdn2.set_checks("async" if request.param == "binding" else "sync")
    yield
    atomic_gdn2.set_checks("async")
    assert last_status() == 0


def _close(y, ref, size, k, dtype, extra=0.0):
    """|y - ref| within the bound above; `size` is sum |a b|."""
    y, ref = y.detach().double(), ref.detach()
    bound = (48 + k / 64) * U * size if dtype == torch.float32 else (k / 8 + 16) * U * size + 2.0 ** -8 * ref.abs()
    over = ((y - ref).abs() - 1.2 * bound - 4 * U * ref.abs() - extra).max()
    assert float(over) <= 0, float(((y - ref).abs() / (bound + 1e-30)).max())


def _norm_close(y, ref, tol):
    y, ref = y.detach().double(), ref.detach()
    assert float((y - ref).norm()) <= tol * float(ref.norm()), float((y - ref).norm() / ref.norm())


SIZES = [(1, 1, 1), (1, 64, 64), (2, 100, 33), (7, 512, 130), (16, 129, 64), (17, 64, 128), (33, 65, 31), (128, 128, 128),
         (129, 200, 257), (200, 1000, 72), (256, 64, 256), (300, 513, 700), (64, 5000, 40), (1500, 96, 1300), (2100, 260, 1160)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_product(M, K, N, dtype):
    gen = torch.Generator(device="cuda").manual_seed(M + K + N)
    x = torch.randn(M, K, generator=gen, device="cuda").to(dtype)
    w = (torch.randn(K, N, generator=gen, device="cuda") / math.sqrt(K)).to(dtype)
    y = linear(x, w)
    assert y.dtype == dtype and y.shape == (M, N)
    _close(y, x.double() @ w.double(), x.double().abs() @ w.double().abs(), K, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_gradients(M, K, N, act, dtype):
    gen = torch.Generator(device="cuda").manual_seed(M + 2 * K + N)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, w, b, r, dy = (t.to(dtype) for t in (n(M, K), n(K, N) / math.sqrt(K), n(N), n(M, N), n(M, N)))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = linear(*leaves[:3], act=act, residual=leaves[3])
    ref = [t.double().requires_grad_(True) for t in (x, w, b, r)]
    y_r = linear_ref(*ref[:3], act, ref[3])
    grads = torch.autograd.grad(y, leaves, dy)
    grads_r = torch.autograd.grad(y_r, ref, dy.double())
    size = x.double().abs() @ w.double().abs()
    _close(y, y_r, size, K, dtype, extra=4 * U * (b.abs() + r.abs()) + (8 * U if act else 0.0))
    for name, a, g, k in zip(("dx", "dw", "db", "dr"), grads, grads_r, (N, M, M, 1)):
        assert a.dtype == dtype
        _norm_close(a, g, (48 + k / 64 + 64) * U if dtype == torch.float32 else 3 * 2.0 ** -8)
    with torch.no_grad():
        assert torch.equal(linear(*leaves[:3], act=act, residual=leaves[3]), y)
