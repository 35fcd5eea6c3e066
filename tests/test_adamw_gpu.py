"""training.AdamW on the B200.

The moments' operations are rounded to fp32 one by one, so moments and codes equal the restatement's bit by bit
where the clipping factor does; that and the norm's sum are fp64 on both sides, rounded once (1e-15 from the
border between two fp32 values they could differ: not at the seeds used).  A step's quotient is 16 u of it off
(u = 2^-24: division 4 u, root 2 u, the factors and products the rest) on either side, the difference and the decay
4 u of p; bf16 weights are rounded after each step, one side's to the neighbour now and then: 2^-7 of p a step.
"""
import copy
import math
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2.training import AdamW  # noqa: E402
from training_ref import BLOCK, adamw_ref, code_m, code_r, decode, encode, root  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [(3, 5), (1,), (256,), (257,), (64, 128), (8192,), (8193,), (100, 333), (0,), (2, 3, 4, 5)]


class Ref:
    """The same optimizer on the CPU, from the operator's definition."""

    def __init__(self, params, bits, wd, lr=1e-2, b1=0.9, b2=0.95, eps=1e-8, clip=None, spike=None):
        self.p = [p.detach().cpu().clone() for p in params]
        self.bits, self.wd, self.lr, self.b1, self.b2, self.eps, self.clip, self.spike = bits, wd, lr, b1, b2, eps, clip, spike
        self.t, self.ema = [0] * len(self.p), torch.zeros(())
        n = [p.numel() for p in self.p]
        if bits == 8:
            self.s = [[torch.zeros(k, dtype=torch.uint8), torch.zeros(-(-k // BLOCK)), torch.zeros(k, dtype=torch.uint8),
                       torch.zeros(-(-k // BLOCK))] for k in n]
        else:
            self.s = [[torch.zeros(k), torch.zeros(k)] for k in n]

    def step(self, grads, loss=None):
        coef, ok = torch.ones(()), loss is None or math.isfinite(loss)
        if self.clip or self.spike:
            sq = sum(float((g.double() ** 2).sum()) for g in grads if g is not None)
            n = torch.tensor(math.sqrt(sq) if math.isfinite(sq) else sq).float()
            ok = ok and bool(torch.isfinite(n)) and not (self.spike and self.ema > 0 and not n < torch.tensor(self.spike).float() * self.ema)
            if self.clip:
                coef = torch.tensor(self.clip).float() / torch.clamp(n, min=self.clip)
            if ok:
                self.ema = torch.tensor(0.98).float() * self.ema + torch.tensor(0.02).float() * n if self.ema > 0 else n
            self.norm = n
        self.ok = ok
        if not ok:
            return
        for i, g in enumerate(grads):
            if g is None or not g.numel():
                continue
            self.t[i] += 1
            m, v = decode(*self.s[i]) if self.bits == 8 else self.s[i]
            p, m, v = adamw_ref(self.p[i].flatten(), g.flatten(), m, v, self.t[i], self.lr, self.wd[i], self.b1, self.b2,
                                self.eps, coef)
            self.p[i] = p.view(self.p[i].shape).to(self.p[i].dtype)
            self.s[i] = [*encode(m, 448.0, code_m), *encode(root(v), 1.9375, code_r)] if self.bits == 8 else [m, v]


def _model(dtypes, seed=0):
    gen = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter((torch.randn(*s, generator=gen) * 0.1).to(dtypes[i % len(dtypes)]).cuda())
              for i, s in enumerate(SHAPES)]
    return params, gen


def _grads(params, gen, scale=1.0):
    return [(torch.randn(p.shape, generator=gen) * scale * 10.0 ** float(torch.randn((), generator=gen))).to(p.dtype) for p in params]


def _same(opt, params, ref):
    for i, p in enumerate(params):
        st = opt.state[p]
        a, b = p.detach().cpu().double(), ref.p[i].double()
        far = ref.t[i] * (8 * U * (b.abs() + 0.1) + 64 * U * 10 * ref.lr + (2.0 ** -7 * (b.abs() + 0.1) if p.dtype == torch.bfloat16 else 0))
        assert bool(((a - b).abs() <= far).all()), i
        names = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale") if ref.bits == 8 else ("exp_avg", "exp_avg_sq")
        for name, r in zip(names, ref.s[i]):
            assert torch.equal(st[name].cpu().flatten(), r), (i, name)
        assert float(st["step"]) == ref.t[i]


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip,spike", [(None, None), (1.0, None), (0.5, 5.0)])
def test_steps_equal_the_definition(dtypes, bits, clip, spike):
    params, gen = _model(dtypes)
    wd = [0.1 if p.ndim > 1 else 0.0 for p in params]
    opt = AdamW([dict(params=[p for p, w in zip(params, wd) if w], weight_decay=0.1),
                 dict(params=[p for p, w in zip(params, wd) if not w], weight_decay=0.0)], lr=1e-2, clip=clip,
                spike_factor=spike, state_bits=bits)
    ref = Ref(params, bits, wd, clip=clip, spike=spike)
    for k in range(4):
        grads = _grads(params, gen, 100.0 if k == 2 and spike else 1.0)
        if k == 1:
            grads[3] = None
        for p, g in zip(params, grads):
            p.grad = None if g is None else g.cuda()
        opt.step()
        ref.step(grads)
        if clip or spike:
            assert float(opt.grad_norm) == float(ref.norm) and bool(opt.step_made) == ref.ok
            assert float(opt.norm_mean) == float(ref.ema)
        if k == 2 and spike:
            assert not ref.ok
        for i, p in enumerate(params):                       # tensors without values have no step
            if not p.numel():
                opt.state[p]["step"].zero_()
        _same(opt, params, ref)
