"""The training operators together: the LM's step on them, and a layer whose mixer is the gated scan."""
import math
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2 import gated_scan, last_status, linear, make_blr_trainable, make_cfg  # noqa: E402
from atomic_gdn2.layer import GDN2Layer, lnorm  # noqa: E402
from atomic_gdn2.training import GDN2LM, AdamW, TrainStep, make_optimizer  # noqa: E402
from oracle_blr import make_oracle_blr, prologue_torch  # noqa: E402
from training_ref import gated_ref, linear_ref  # noqa: E402

pytestmark = pytest.mark.gpu
TOL = 1e-4   # fp32 operator tolerance (dot highest, solve / B3 bf16x3)


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm())


def test_layer_on_the_products():
    """test_lm_gpu's layer with linear in place of torch.addmm, against 64 bits."""
    cfg, D = make_cfg(), 128
    lay = GDN2Layer(256, 2, D, expansion=2, generator=torch.Generator().manual_seed(4), linear_fn=linear)
    ref = GDN2Layer(256, 2, D, expansion=2, prologue_fn=prologue_torch)
    ref.load_state_dict(lay.state_dict())
    ref, lay = ref.double(), lay.cuda()
    x = torch.randn(2, 256, 256, generator=torch.Generator().manual_seed(5))
    y = lay(x.cuda(), make_blr_trainable(cfg, 1 / math.sqrt(D)), cfg)
    (y * y).sum().backward()
    yr = ref(x.double(), make_oracle_blr(cfg, 1 / math.sqrt(D)), cfg)
    (yr * yr).sum().backward()
    assert last_status() == 0 and _rel(y, yr) < TOL
    for (n, p), (_, pr) in zip(lay.named_parameters(), ref.named_parameters()):
        assert _rel(p.grad, pr.grad) < TOL, n


@pytest.mark.parametrize("bits", [32, 8])
def test_lm_steps(bits):
    """TrainStep on the framework's products and optimizer beside torch's: gradients' norms and weights after three
    steps agree (32 bits: 1e-4 of the update; 8 bits: the first step's moments are not rounded yet), and a spike is
    skipped on both."""
    torch.backends.cuda.matmul.allow_tf32 = False
    cfg = make_cfg()
    kw = dict(d_model=128, n_heads=1, d_head=128, n_layers=2, seed=3)
    a, b = GDN2LM(cfg, linear_fn=linear, **kw).cuda(), GDN2LM(cfg, **kw).cuda()
    start = [p.detach().clone() for p in a.parameters()]
    sa = TrainStep(a, make_optimizer(a, 1e-3, state_bits=bits), lr=1e-3, warmup=0, total=10)
    sb = TrainStep(b, make_optimizer(b, 1e-3), lr=1e-3, warmup=0, total=10)
    gen = torch.Generator().manual_seed(1)
    for k in range(3):
        ids = torch.randint(0, 256, (2, 256), generator=gen).cuda()
        (la, na, oa), (lb, nb, ob) = sa(ids), sb(ids)
        assert bool(oa) and bool(ob) and _rel(la, lb) < 1e-4 and _rel(na, nb) < (1e-3 if bits == 32 else 1e-2)
        assert _rel(sa.gn_ema, sb.gn_ema) < (1e-3 if bits == 32 else 1e-2)
        if k == 0 or bits == 32:
            # where a gradient is next to nothing its sign decides the first update: compared in the norm
            moved = [(p.detach() - s, q.detach() - s) for p, q, s in zip(a.parameters(), b.parameters(), start)]
            assert sum(float((u - v).norm()) ** 2 for u, v in moved) < (2e-2 ** 2) * sum(float(v.norm()) ** 2 for _, v in moved)
    before = [p.detach().clone() for p in a.parameters()]
    sa.gn_ema = sa.gn_ema * 1e-4
    _, _, ok = sa(ids)
    assert not bool(ok) and all(torch.equal(p, q) for p, q in zip(before, a.parameters()))


class Mixer(torch.nn.Module):
    """A layer of the same shape as GDN2Layer with the elementwise recurrence as its mixer."""

    def __init__(self, d, c, gen):
        super().__init__()
        n = lambda *s: torch.nn.Parameter(torch.randn(*s, generator=gen) / math.sqrt(s[0]))
        self.proj_w, self.proj_b, self.o_w, self.o_b = n(d, 2 * c), n(2 * c), n(c, d), n(d)
        self.up_w, self.up_b, self.down_w, self.down_b = n(d, 2 * d), n(2 * d), n(2 * d, d), n(d)
        self.c = c

    def forward(self, x, lengths, reset, product, scan):
        y = product(lnorm(x), self.proj_w, self.proj_b)
        h, last = scan(y[..., :self.c], torch.nn.functional.logsigmoid(y[..., self.c:] + 3.0), None, lengths=lengths, reset=reset)
        x = product(h, self.o_w, self.o_b, residual=x)
        u = product(lnorm(x), self.up_w, self.up_b, act="gelu")
        return product(u, self.down_w, self.down_b, residual=x), last


@pytest.mark.parametrize("bits", [32, 8])
def test_a_layer_of_all_three(bits):
    """Projection, scan, projections with GELU and residuals, then a step: gradients against 64 bits, and the next
    forward answers from the states that the scan left."""
    gen = torch.Generator().manual_seed(2)
    m = Mixer(64, 96, gen)
    ref = Mixer(64, 96, gen).double()
    ref.load_state_dict(m.state_dict())
    m = m.cuda()
    x = torch.randn(3, 150, 64, generator=gen)
    lengths, reset = torch.tensor([150, 70, 0], dtype=torch.int32), torch.rand(3, 150, generator=gen) < 0.02
    y, last = m(x.cuda(), lengths.cuda(), reset.cuda(), linear, gated_scan)
    (y.square().sum() + last.sum()).backward()
    y_r, last_r = ref(x.double(), lengths, reset, lambda a, w, b, act=None, residual=None: linear_ref(a, w, b, act, residual),
                      lambda a, g, h0, lengths, reset: gated_ref(a, g, h0, lengths, reset))
    (y_r.square().sum() + last_r.sum()).backward()
    assert last_status() == 0 and _rel(y, y_r) < 1e-5 and _rel(last, last_r) < 1e-5
    for (n, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        assert _rel(p.grad, q.grad) < 1e-5, n
    opt = AdamW(m.parameters(), lr=1e-3, clip=1.0, state_bits=bits)
    was = [p.detach().clone() for p in m.parameters()]
    opt.step()
    norm = math.sqrt(sum(float((q.grad ** 2).sum()) for q in ref.parameters()))
    assert float(opt.grad_norm) == pytest.approx(norm, rel=1e-5) and bool(opt.step_made)
    # a first step is lr (g / (|g| + eps) + wd p)
    for p, w, q in zip(m.parameters(), was, ref.parameters()):
        g = q.grad / norm
        want = w.double().cpu() * (1 - 1e-4) - 1e-3 * g / (g.abs() + 1e-8)
        assert float(((p.detach().double().cpu() - want).norm()) / (want - w.double().cpu()).norm()) < 1e-2
    with torch.no_grad():                                             # a token more for each sequence
        h1, next_state = gated_scan(torch.ones(3, 1, 96, device="cuda"), torch.full((3, 1, 96), -0.1, device="cuda"), last.detach())
    assert _rel(next_state, math.exp(-0.1) * last_r + 1.0) < 1e-5 and torch.equal(h1[:, 0], next_state)
