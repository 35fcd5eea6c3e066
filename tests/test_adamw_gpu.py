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


def _train(opt, params, gen, n=3, scale=1.0):
    for _ in range(n):
        for p in params:
            p.grad = (torch.randn(p.shape, generator=gen) * scale).to(p.dtype).cuda()
        opt.step()


def test_against_torch():
    """The same weights as torch's AdamW after some steps (its order of operations differs: 2^-20 of a step each), and
    either's state_dict loads into the other."""
    a, gen = _model([torch.float32], 3)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
    mine, theirs = AdamW(a, **kw), torch.optim.AdamW(b, **kw)
    for k in range(6):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=gen).cuda()
            q.grad = p.grad.clone()
        mine.step()
        theirs.step()
        for p, q in zip(a, b):
            if p.numel():
                assert float((p.detach() - q.detach()).abs().max()) < 7 * (2.0 ** -20 * 0.1 + 4 * U)
        if k == 2:
            s = copy.deepcopy(mine.state_dict())
            mine.load_state_dict(theirs.state_dict())
            theirs.load_state_dict(s)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict(bits):
    params, gen = _model([torch.float32, torch.bfloat16], 4)
    opt = AdamW(params, lr=1e-2, clip=1.0, state_bits=bits)
    _train(opt, params, gen)
    saved = copy.deepcopy(opt.state_dict())
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = AdamW(twin, lr=1.0, clip=1.0, state_bits=bits)
    other.load_state_dict(saved)
    state = gen.get_state()
    _train(opt, params, gen)
    gen.set_state(state)
    _train(other, twin, gen)
    for p, q in zip(params, twin):
        assert torch.equal(p, q)
        for k, v in opt.state[p].items():
            assert torch.equal(v, other.state[q][k]) and v.dtype == other.state[q][k].dtype
    with pytest.raises(ValueError):
        AdamW(twin, state_bits=40 - bits).load_state_dict(saved)
    copied = copy.deepcopy(other)                                     # its weights and options with it
    assert copied.clip == 1.0 and copied.state_bits == bits and float(copied.grad_norm) == float(other.grad_norm)
    _train(copied, copied.param_groups[0]["params"], gen, 1)
    with pytest.raises(ValueError):
        copied.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2, device="cuda"))], lr=-1.0))


def test_moments():
    for bits in (8, 32):
        params, gen = _model([torch.float32], 5)
        params = [p for p in params if p.numel()]
        opt = AdamW(params, state_bits=bits)
        _train(opt, params, gen)
        got = opt.moments()
        for p, (m, v) in zip(params, got):
            st = opt.state[p]
            if bits == 8:
                a, b = decode(st["exp_avg"].cpu(), st["exp_avg_scale"].cpu(), st["exp_avg_sq"].cpu(), st["exp_avg_sq_scale"].cpu())
            else:
                a, b = st["exp_avg"].cpu().flatten(), st["exp_avg_sq"].cpu().flatten()
            assert m.shape == v.shape == p.shape and torch.equal(m.cpu().flatten(), a) and torch.equal(v.cpu().flatten(), b)
        out = [(torch.zeros_like(p), torch.zeros_like(p)) for p in params[:2]]
        assert opt.moments(params[:2], out=out) is out and torch.equal(out[1][0], got[1][0])
        with pytest.raises(ValueError):
            opt.moments(params, out=out)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than a table holds, with and without a norm."""
    gen = torch.Generator().manual_seed(6)
    sizes = [1 + (i * 37) % 700 for i in range(700)] + [20000]
    for clip in (None, 1.0):
        params = [torch.nn.Parameter(torch.randn(n, generator=gen).cuda()) for n in sizes]
        opt = AdamW(params, lr=1e-2, clip=clip, state_bits=bits, weight_decay=0.1)
        ref = Ref(params, bits, [0.1] * len(params), clip=clip)
        for _ in range(2):
            grads = [torch.randn(n, generator=gen) for n in sizes]
            for p, g in zip(params, grads):
                p.grad = g.cuda()
            opt.step()
            ref.step(grads)
            if clip:
                assert float(opt.grad_norm) == float(ref.norm)
        _same(opt, params, ref)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_views_and_orders(bits, dtype):
    """Weights that start anywhere, weights and gradients in other orders than each other's: every value takes its own step."""
    gen = torch.Generator().manual_seed(7)
    pool = torch.zeros(40000, dtype=dtype, device="cuda")
    shapes, at, params = [(17, 31), (3000,), (90, 100), (4, 6, 10)], 1, []
    for s in shapes:
        n = math.prod(s)
        params.append(torch.nn.Parameter(pool[at:at + n].view(s)))
        at += n + 3
    params[2] = torch.nn.Parameter(pool[at:at + 9000].view(100, 90).t())
    opt = AdamW(params, lr=1e-2, clip=1.0, state_bits=bits)
    order = lambda t: t.t() if t.shape == (90, 100) else t            # its memory's order
    twins = [torch.nn.Parameter(order(p.detach()).contiguous().clone()) for p in params]
    ref = Ref(twins, bits, [0.1] * 4, clip=1.0)
    for _ in range(3):
        grads = [torch.randn(s, generator=gen).to(dtype) for s in shapes]
        for i, (p, g) in enumerate(zip(params, grads)):
            g = g.cuda()
            p.grad = g if i else g.t().contiguous().t()               # a gradient in another order
        opt.step()
        ref.step([order(g) for g in grads])
    for i, p in enumerate(params):
        far = ref.t[i] * (8 * U * 0.2 + 64 * U * 0.1 + (2.0 ** -7 * 0.2 if dtype == torch.bfloat16 else 0))
        assert float((order(p.detach()).cpu().double() - ref.p[i].double()).abs().max()) <= far
    assert bool((pool[0] == 0).all()) and bool((pool[at + 9000:] == 0).all())


def test_guard():
    """Steps that are not made: the weights, moments, counts and the mean stay; the norm is told."""
    for bits in (32, 8):
        for bad in ("nan", "inf", "loss", "spike"):
            params, gen = _model([torch.float32], 8)
            opt = AdamW(params, lr=1e-2, clip=1.0, spike_factor=4.0, state_bits=bits)
            _train(opt, params, gen, 2)
            before = [p.detach().clone() for p in params], copy.deepcopy(opt.state_dict()["state"]), opt.norm_mean
            for p in params:
                p.grad = torch.randn(p.shape, generator=gen).cuda() * (100.0 if bad == "spike" else 1.0)
            if bad in ("nan", "inf"):
                params[5].grad[77] = float(bad)
            opt.step(loss=torch.tensor(float("nan") if bad == "loss" else 1.0, device="cuda"))
            assert not bool(opt.step_made) and float(opt.norm_mean) == float(before[2])
            assert math.isfinite(float(opt.grad_norm)) == (bad in ("loss", "spike"))
            assert all(torch.equal(a, p) for a, p in zip(before[0], params))
            for i, st in opt.state_dict()["state"].items():
                assert all(torch.equal(v, before[1][i][k]) for k, v in st.items())
            _train(opt, params, gen, 1)
            assert bool(opt.step_made)
    params, gen = _model([torch.float32], 9)                          # without clip or spike_factor only the loss counts
    opt = AdamW(params, lr=1e-2)
    _train(opt, params, gen, 1)
    was = params[0].detach().clone()
    opt.step(loss=torch.tensor(float("inf"), device="cuda"))
    assert torch.equal(params[0], was) and not bool(opt.step_made)
    params[0].grad.zero_()
    params[4].grad.fill_(float("nan"))
    opt.step()
    assert bool(torch.isnan(params[4]).all()) and bool(torch.isfinite(params[0]).all())


def test_clips_at_the_ends_of_the_range():
    """An infinite clip clips nothing (the guard stays), one below fp32's normal numbers leaves next to nothing."""
    for bits in (32, 8):
        for clip in (float("inf"), 1e300):
            params, gen = _model([torch.float32], 11)
            twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
            opt, plain = AdamW(params, lr=1e-2, clip=clip, state_bits=bits), AdamW(twin, lr=1e-2, state_bits=bits)
            for scale in (1.0, 100.0):
                for p, q, g in zip(params, twin, _grads(params, gen, scale)):
                    p.grad = g.cuda()
                    q.grad = p.grad.clone()
                opt.step()
                plain.step()
                assert bool(opt.step_made) and math.isfinite(float(opt.grad_norm))
            assert all(torch.equal(p, q) for p, q in zip(params, twin))
            params[4].grad.fill_(float("inf"))
            opt.step()
            assert not bool(opt.step_made) and all(torch.equal(p, q) for p, q in zip(params, twin))
        p = torch.nn.Parameter(torch.ones(300, device="cuda"))
        p.grad = torch.full_like(p, 3.0)
        opt = AdamW([p], lr=1e-2, eps=1.0, weight_decay=0.0, clip=1e-60, spike_factor=1e-60, state_bits=bits)
        opt.step()
        assert bool((p == 1.0).all()) and bool(opt.step_made)         # steps of 1e-38 or less
        opt.step()
        assert not bool(opt.step_made)                                # no norm is below 1e-60 of the mean


def test_zero_and_extreme_gradients():
    """A gradient of zeros has norm zero; gradients whose squares fp32 cannot hold are clipped like others."""
    for bits in (32, 8):
        params, gen = _model([torch.float32], 10)
        for scale in (0.0, 1e-30, 1e25):
            opt = AdamW(params, lr=1e-3, clip=1.0, state_bits=bits, weight_decay=0.0)
            grads = [torch.randn(p.shape, generator=gen) * scale for p in params]
            for p, g in zip(params, grads):
                p.grad = g.cuda()
            was = [p.detach().clone() for p in params]
            opt.step()
            want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
            assert float(opt.grad_norm) == pytest.approx(want, rel=1e-6, abs=0.0) and bool(opt.step_made)
            # a first step moves every weight by lr g / (|g| + eps): at most lr
            assert all(float((p - a).abs().max()) <= 1.001e-3 + 4 * U for p, a in zip(params, was) if p.numel())
            if scale == 0.0:
                assert all(torch.equal(p, a) for p, a in zip(params, was))


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_and_streams(bits):
    """A captured step, its rate in device memory, replays like eager steps; steps go to the current stream."""
    params, gen = _model([torch.float32], 11)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    rate = torch.full((), 1e-2, device="cuda")
    a, b = AdamW(params, lr=rate, clip=1.0, state_bits=bits), AdamW(twin, lr=1e-2, clip=1.0, state_bits=bits)
    for p, q in zip(params, twin):
        p.grad = torch.randn(p.shape, generator=gen).cuda()
        q.grad = p.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside the capture"):
        with torch.cuda.graph(graph):
            a.step()
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for k in range(3):
        lr = 1e-2 / (k + 1)
        rate.fill_(lr)
        b.param_groups[0]["lr"] = float(torch.tensor(lr))             # what fp32 holds of it
        for p, q in zip(params, twin):
            q.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(k))
            p.grad.copy_(q.grad)
        graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(5_000_000)
            b.step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(params, twin))
        assert float(a.grad_norm) == float(b.grad_norm) and float(a.state[params[0]]["step"]) == k + 2


def test_hooks_and_schedulers():
    """torch's hooks around a step, and its learning-rate schedulers, work as on its own optimizers."""
    params, gen = _model([torch.float32], 12)
    opt, seen = AdamW(params, lr=1e-2), []
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)
    _train(opt, params, gen, 1)
    sched.step()
    assert opt.param_groups[0]["lr"] == 5e-3
    opt.register_step_pre_hook(lambda o, a, k: seen.append("before"))
    opt.register_step_post_hook(lambda o, a, k: seen.append("after"))
    was = params[4].detach().clone()
    _train(opt, params, gen, 1)
    assert seen == ["before", "after"] and not torch.equal(was, params[4]) and float(opt.state[params[4]]["step"]) == 2


def test_refusals():
    cuda = lambda *s, dtype=torch.float32: torch.nn.Parameter(torch.zeros(*s, device="cuda", dtype=dtype))
    for p in (cuda(4, dtype=torch.float16), cuda(4, dtype=torch.float64), torch.nn.Parameter(torch.zeros(1, device="cuda").expand(5)),
              torch.nn.Parameter(torch.zeros(8, device="cuda")[::2])):
        p.grad = torch.zeros_like(p)
        with pytest.raises(ValueError):
            AdamW([p]).step()
    p = cuda(6, 2)
    p.grad = torch.zeros(6, 2, device="cuda").to_sparse()
    with pytest.raises(ValueError):
        AdamW([p]).step()
    p.grad = torch.zeros(6, 2, device="cuda")
    opt = AdamW([p], state_bits=8)
    opt.step()
    for name, bad in (("exp_avg", torch.zeros(6, 2, device="cuda")), ("exp_avg_scale", torch.zeros(2, device="cuda")),
                      ("step", torch.zeros(())), ("exp_avg_sq", torch.zeros(3, 2, dtype=torch.uint8, device="cuda"))):
        good = opt.state[p][name]
        opt.state[p][name] = bad
        with pytest.raises(ValueError):
            opt.step()
        opt.state[p][name] = good
    with pytest.raises(ValueError):
        opt.step(loss=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        AdamW([p], lr=torch.zeros(2, device="cuda")).step()
    version = p._version
    opt.step()
    assert p._version > version                                       # a change in place to autograd
    assert float(opt.step(lambda: (p * 2).sum().detach() + 1.0)) == 1.0
