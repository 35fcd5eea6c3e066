"""linear on the B200: long sums, the size of bf16 gradients' errors.  u = 2^-24."""
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2 import last_status, linear  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _status():
    yield
    assert last_status() == 0


def _product(a, b):
    """a b in 64 bits."""
    y = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device="cuda")
    for k in range(0, a.shape[1], 16384):
        y += a[:, k:k + 16384].double() @ b[k:k + 16384].double()
    return y


@pytest.mark.parametrize("what", ["forward", "dW"])
def test_long_bf16_sums(what):
    """262144 positive products, so that every error of the additions goes one way, in so many results that no sum is split:
    1024 products meet in truncating additions of 16 (144 u of the sum, as in the tests beside this one), these sums in
    at most 256 rounded additions (u each), and the result is rounded once: 400 u and half a step, 2^-8."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    make = lambda *s: (1.0 + torch.rand(*s, generator=gen, device="cuda")).bfloat16()
    n, long = 2048, 1 << 18
    if what == "forward":
        x, w = make(n, long), make(long, n)
        y, ref = linear(x, w), _product(x, w)
    else:
        x, dy, w = make(long, n), make(long, n), torch.zeros(n, n, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = torch.autograd.grad(linear(x, w), w, dy)[0]
        ref = _product(x.t(), dy)
    off = ((y.double() - ref) / ref).abs().max()
    assert float(off) <= 1.001 * (400 * U + 2.0 ** -8)


@pytest.mark.parametrize("M", [2, 40])
def test_rows_far_apart(M):
    """Rows 2^28 + 8 elements apart, of x and of W: copied, forward and backward."""
    ld = (1 << 28) + 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    store = torch.empty((M - 1) * ld + 64 if M < 3 else ld + 64, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((M, 64), (ld, 1)) if M < 3 else torch.empty(M, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.empty(64, 48, dtype=torch.bfloat16, device="cuda") if M < 3 else store.as_strided((2, 48), (ld, 1))
    x = x if M < 3 else x[:, :2]
    for t in (x, w):
        t.copy_(torch.randint(-4, 5, t.shape, generator=gen, device="cuda"))      # sums that are exact
    dy = torch.randint(-2, 3, (M, 48), generator=gen, device="cuda").bfloat16()
    want = x.double() @ w.double(), dy.double() @ w.double().t(), x.double().t() @ dy.double()
    assert torch.equal(linear(x, w).double(), want[0].bfloat16().double())
    x.requires_grad_(True), w.requires_grad_(True)
    y = linear(x, w)
    for a, b in zip((y, *torch.autograd.grad(y, (x, w), dy)), want):
        assert torch.equal(a.double(), b.bfloat16().double())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(3, 8, 40), (256, 1024, 512), (2048, 128, 1024)])
def test_gelu_of_huge_values(M, K, N, dtype):
    """Where z is so large that its square overflows GELU's slope is 1, or 0 to the left: finite gradients of finite inputs.
    One value of x and of W in each sum and powers of two, so that y and the gradients are exact."""
    x, w = torch.zeros(M, K, device="cuda", dtype=dtype), torch.zeros(K, N, device="cuda", dtype=dtype)
    x[:, 0] = 2.0 ** (50.0 + torch.arange(M, device="cuda") % 8)
    w[0] = 2.0 ** (30.0 + torch.arange(N, device="cuda") % 8) * (1 - 2.0 * (torch.arange(N, device="cuda") % 3 == 0))
    dy = torch.zeros(M, N, device="cuda", dtype=dtype)
    dy[:, N // 2:N // 2 + 3] = 1.0
    x.requires_grad_(True), w.requires_grad_(True)
    y = linear(x, w, act="gelu")
    z = x.detach().double() @ w.detach().double()
    assert torch.equal(y.double(), torch.clamp(z, min=0.0))
    dz = dy.double() * (z > 0)
    for a, b in zip(torch.autograd.grad(y, (x, w), dy), (dz @ w.detach().double().t(), x.detach().double().t() @ dz)):
        assert torch.equal(a.double(), b.to(dtype).double())


def test_bf16_gradients_through_gelu():
    """A value's rounding to bf16 is off by up to 2^-8 / m, m its mantissa: r = 2^-8 / sqrt(3) sqrt(mean of 1 / m^2), 0.425 2^-8,
    in the root of the mean square where mantissas are spread evenly over the logarithm.  A gradient has dz's rounding
    (r: its errors are independent), z's (|gelu''(z) z| <= 0.29 where gelu' has a mean square of 0.4: below r / 2) and its
    own (r): 1.5 r of its norm, 5 % for the spread.  The same of y, which is rounded once: r."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    M, K, N, r = 2048, 512, 2048, 0.425 * 2.0 ** -8
    x = torch.randn(M, K, generator=gen, device="cuda").bfloat16().requires_grad_(True)
    w = (torch.randn(K, N, generator=gen, device="cuda") / K ** 0.5).bfloat16().requires_grad_(True)
    dy = torch.randn(M, N, generator=gen, device="cuda").bfloat16()
    y = linear(x, w, act="gelu")
    ref = [t.detach().double().requires_grad_(True) for t in (x, w)]
    y_r = torch.nn.functional.gelu(ref[0] @ ref[1], approximate="tanh")
    off = lambda a, b: float((a.double() - b).norm() / b.norm())
    assert off(y.detach(), y_r.detach()) <= 1.05 * r
    for a, b in zip(torch.autograd.grad(y, (x, w), dy), torch.autograd.grad(y_r, ref, dy.double())):
        assert off(a, b) <= 1.05 * 1.5 * r


@pytest.mark.parametrize("M,K,N", [(300, 1025, 200), (300, 2048, 201), (1000, 3000, 1000), (2048, 1088, 2560), (2500, 4160, 2049),
                                   (130, 65536, 260), (257, 70001, 129), (2048, 1024, 2048)])
def test_bf16_sums_of_several_turns(M, K, N):
    """Whole numbers whose sums are exact in fp32, so that results are the exact ones, rounded once: sums of one and several
    turns, the last of them short, split and whole, in single CTAs and pairs, cut tiles, rows on odd places."""
    gen = torch.Generator(device="cuda").manual_seed(K)
    whole = lambda *s: torch.randint(-4, 5, s, generator=gen, device="cuda").bfloat16()
    x, w, b, r, dy = whole(M, K), whole(K, N), whole(N), whole(M, N), whole(M, N)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = linear(x, w, b, residual=r)
    want = [_product(x.detach(), w.detach()) + b.detach().double() + r.detach().double(), _product(dy, w.detach().t()),
            _product(x.detach().t(), dy), dy.double().sum(0), dy.double()]
    for a, e in zip((y, *torch.autograd.grad(y, leaves, dy)), want):
        assert torch.equal(a.detach(), e.bfloat16())
