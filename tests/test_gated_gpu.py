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


def _leaves(*ts):
    return [t.cuda().requires_grad_(True) for t in ts]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [37, 40])
@pytest.mark.parametrize("L", [1, 3, 70])
def test_views_of_one_projection(L, C, dtype):
    """x and g side by side in one tensor, odd offsets, transposed and broadcast inputs."""
    B = 3
    x, g, h0, dy, dl = _inputs(B, L, C, dtype, L)
    both = torch.cat([x, g], 2)
    flat = both.cuda()
    pad = torch.zeros(B * L * 2 * C + 1, dtype=dtype, device="cuda")[1:].view(B, L, 2 * C).copy_(flat)
    wide = torch.cat([flat, flat[..., :1]], 2)
    ref = [t.double().requires_grad_(True) for t in (x, g, h0)]
    h_r, l_r = gated_ref(*ref)
    want = torch.autograd.grad((h_r, l_r), ref[:2], (dy.double(), dl.double()))
    for src in (flat, pad, wide, flat.transpose(0, 1).contiguous().transpose(0, 1), flat.transpose(1, 2).contiguous().transpose(1, 2)):
        src = src.detach().requires_grad_(True)
        h, last = gated_scan(src[..., :C], src[..., C:2 * C], h0.cuda())
        assert _rel(h, h_r) < TOL[dtype] and _rel(last, l_r) < TOL[torch.float32]
        (d,) = torch.autograd.grad((h, last), src, (dy.cuda().transpose(0, 1).contiguous().transpose(0, 1), dl.cuda()))
        assert _rel(d[..., :C], want[0]) < 2 * TOL[dtype] and _rel(d[..., C:2 * C], want[1]) < 2 * TOL[dtype]
    gate = g[:1, :1].cuda().requires_grad_(True)                      # one row of gates for all tokens of all sequences
    h, last = gated_scan(x.cuda(), gate.expand(B, L, C), h0.cuda())
    one = g[:1, :1].double().requires_grad_(True)
    h_r, l_r = gated_ref(x.double(), one.expand(B, L, C), h0.double())
    assert _rel(h, h_r) < TOL[dtype]
    (d,), (d_r,) = torch.autograd.grad((h, last), gate, (dy.cuda(), dl.cuda())), torch.autograd.grad((h_r, l_r), one, (dy.double(), dl.double()))
    # the sum over tokens is torch's, in the inputs' type: a rounding for each of them, independent (sqrt)
    assert _rel(d, d_r) < 2 * TOL[dtype] * max(1.0, math.sqrt(B * L)) * float(gated_ref(x.double().abs(), one.detach().expand(B, L, C))[0].norm() / h_r.detach().norm())


@pytest.mark.parametrize("L", [1, 4, 40, 600])
def test_what_is_masked_does_not_matter(L):
    """NaN and infinities past the lengths and before a reset: outputs and gradients are those of zeros there."""
    B, C = 4, 40
    x, g, h0, dy, dl = _inputs(B, L, C, torch.float32, L)
    lengths = torch.tensor([L, 0, L // 2, max(1, L - 1)], dtype=torch.int32)
    past = (torch.arange(L)[None] >= lengths[:, None])[..., None]
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38])[torch.arange(B * L * C) % 4].view(B, L, C)
    clean = gated_ref(*(torch.where(past, torch.zeros(()), t).double() for t in (x, g)), h0.double(), lengths)
    dev = _leaves(torch.where(past, bad, x), torch.where(past, bad, g), h0)
    h, last = gated_scan(*dev, lengths=lengths.cuda())
    assert _rel(h, clean[0]) < TOL[torch.float32] and _rel(last, clean[1]) < TOL[torch.float32]
    assert bool((h[past.expand_as(h).cuda()] == 0).all()) and torch.equal(last[1].cpu(), h0[1])
    grads = torch.autograd.grad((h, last), dev, (torch.where(past, bad, dy).cuda(), dl.cuda()))
    ref = [torch.where(past, torch.zeros(()), t).double().requires_grad_(True) for t in (x, g)] + [h0.double().requires_grad_(True)]
    h_r, l_r = gated_ref(*ref, lengths)
    grads_r = torch.autograd.grad((h_r, l_r), ref, (torch.where(past, torch.zeros(()), dy).double(), dl.double()))
    for a, b in zip(grads, grads_r):
        assert _rel(a, b) < 2 * TOL[torch.float32]
    if L < 4:
        return
    t = L // 3                                                        # a state of NaN and infinities, then a reset
    reset = torch.zeros(B, L, dtype=torch.bool)
    reset[:, t] = True
    worse = torch.where(torch.arange(L)[None, :, None] < t, bad, x)
    h, last = gated_scan(worse.cuda(), g.cuda(), torch.full_like(h0, float("nan")).cuda(), reset=reset.cuda())
    h_r, l_r = gated_ref(x[:, t:].double(), g[:, t:].double(), None, None, reset[:, t:])
    assert _rel(h[:, t:], h_r) < TOL[torch.float32] and _rel(last, l_r) < TOL[torch.float32]
    assert not bool(torch.isfinite(h[:, :t]).all())


@pytest.mark.parametrize("C", [33, 64])
def test_values_that_are_not_finite(C):
    """An infinite state stays infinite through any number of tokens, a gate of -inf makes NaN of it (0 * inf) and forgets
    a finite one, a NaN stays in its channel."""
    B, L = 1, 3000
    x, g, _, _, _ = _inputs(B, L, C, torch.float32, 5)
    g[..., :8] = -3.0                                                 # products of gates underflow within a segment
    x[0, 10, 0] = float("inf")
    x[0, 20, 1] = float("-inf")
    x[0, 30, 2] = float("nan")
    g[0, 40, 3] = float("nan")
    g[0, 1500, 4] = -float("inf")
    x[0, 1000, 5], g[0, 1500, 5] = float("inf"), -float("inf")
    h, last = gated_scan(x.cuda(), g.cuda())
    h_r, l_r = gated_ref(x, g)                                        # the recurrence itself, in fp32
    h = h.cpu()
    assert torch.equal(torch.isnan(h), torch.isnan(h_r)) and torch.equal(torch.isinf(h), torch.isinf(h_r))
    assert torch.equal(h[torch.isinf(h)], h_r[torch.isinf(h_r)])
    fine = torch.isfinite(h_r)
    assert _rel(h[fine], h_r[fine]) < TOL[torch.float32]


def test_index_and_out():
    B, L, C = 6, 2, 48
    x, g, h0, _, _ = _inputs(B, L, C, torch.float32, 8)
    index = torch.tensor([3, 0, -1, 0, 5, 3])
    rows = torch.where((index >= 0)[:, None], h0[index.clamp(min=0)], torch.zeros(()))
    h_r, l_r = gated_ref(x.double(), g.double(), rows.double())
    for L2 in (2, 2):
        for cast in (torch.int32, torch.int64):
            h, last = gated_scan(x.cuda(), g.cuda(), h0.cuda(), h_index=index.cuda().to(cast))
            assert _rel(h, h_r) < TOL[torch.float32] and _rel(last, l_r) < TOL[torch.float32]
    long_x, long_g = x.repeat(1, 50, 1), g.repeat(1, 50, 1)
    h, last = gated_scan(long_x.cuda(), long_g.cuda(), h0.cuda(), h_index=index.cuda())
    assert _rel(h, gated_ref(long_x.double(), long_g.double(), rows.double())[0]) < TOL[torch.float32]
    for xs in ((x, g), (long_x, long_g)):                             # in place
        state = h0.cuda()
        version = state._version
        want = gated_scan(xs[0].cuda(), xs[1].cuda(), h0.cuda())
        h, last = gated_scan(xs[0].cuda(), xs[1].cuda(), state, h_out=state)
        assert last is state and state._version > version
        assert torch.equal(h, want[0]) and torch.equal(last, want[1])


def test_refusals():
    x = torch.zeros(2, 8, 16, device="cuda")
    h0 = torch.zeros(2, 16, device="cuda")
    need = x.clone().requires_grad_(True)
    for bad in (dict(x=x[0]), dict(g=x[:, :4]), dict(g=x.cpu()), dict(h0=h0[:1]), dict(h0=h0.cpu()), dict(h0=h0[:, :8]),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(lengths=torch.zeros(2, device="cuda")),
                dict(reset=torch.zeros(2, 8, device="cuda")), dict(reset=torch.zeros(2, 7, dtype=torch.bool, device="cuda")),
                dict(h_index=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(x=x[:0], g=x[:0]), dict(x=x[..., :0], g=x[..., :0]),
                dict(h_out=h0.cpu()), dict(h_out=h0.double()), dict(h0=h0, h_out=torch.zeros(40, device="cuda")[8:].view(2, 16)[:1]),
                dict(x=x.to(torch.complex64), g=x.to(torch.complex64))):
        a = dict(x=x, g=x, h0=None)
        a.update(bad)
        with pytest.raises(ValueError):
            gated_scan(a.pop("x"), a.pop("g"), a.pop("h0"), **a)
    pool = torch.zeros(48, device="cuda")
    with pytest.raises(ValueError):                                   # overlapping, not the same
        gated_scan(x, x, pool[:32].view(2, 16), h_out=pool[16:].view(2, 16))
    with pytest.raises(ValueError):
        gated_scan(x, x, h0, h_index=torch.zeros(2, dtype=torch.int32, device="cuda"), h_out=h0)
    wide = torch.zeros(2, 3, 64, device="cuda")                       # a state next to its inputs is fine, inside them not
    own = wide[:1, :, :16]
    for kw in (dict(x=own, g=own.clone()), dict(x=own.clone(), g=own)):
        for out in (wide[:1, 0, :16], wide[:1, 2, :16], wide[:1, 1, 8:24]):
            with pytest.raises(ValueError, match="overlaps"):
                gated_scan(**kw, h_out=out)
        gated_scan(**kw, h_out=wide[1:, 0, :16])
    for kw in (dict(h_index=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(h_out=torch.zeros_like(h0))):
        with pytest.raises(RuntimeError, match="no backward"):
            gated_scan(need, x, h0, **kw)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError):
            gated_scan(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), x)
    h, _ = gated_scan(need, x)
    (d,) = torch.autograd.grad(h.sum(), need, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        d.sum().backward()


def test_status():
    """A positive gate, a length and an index out of range are reported; what is taken then is the nearer bound."""
    x = torch.ones(2, 40, 8, device="cuda")
    atomic_gdn2.set_checks("sync")
    g = torch.zeros_like(x)
    g[1, 20, 3] = 0.5
    n = torch.tensor([41, -1], dtype=torch.int32, device="cuda")
    i = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    for a, kw, what in ((g, {}, "g > 0"), (x * 0, dict(lengths=n), "length"), (x * 0, dict(h0=torch.zeros(2, 8, device="cuda"), h_index=i), "index")):
        for first, L in ((19, 3), (0, 40)):
            with pytest.raises(RuntimeError, match=what):
                gated_scan(x[:, :L], a[:, first:first + L], kw.get("h0"), **{k: v for k, v in kw.items() if k != "h0"})
    atomic_gdn2.set_checks("off")
    h, last = gated_scan(x, x * 0, lengths=n)
    assert float(last[0, 0]) == 40.0 and float(last[1, 0]) == 0.0 and last_status() != 0
    need = x.clone().requires_grad_(True)
    gate = g.clone().requires_grad_(True)
    h, _ = gated_scan(need, gate)                                     # a gate above zero counts as zero, its gradient too
    d = torch.autograd.grad(h.sum(), gate)[0]
    assert float(h[1, 20, 3]) == 21.0 and float(d[1, 20, 3]) == 0.0 and float(d[1, 21, 3]) != 0.0
    for fl in atomic_gdn2.pipeline._flags.values():
        fl.take()


def test_some_gradients_only():
    B, L, C = 2, 50, 24
    x, g, h0, dy, dl = _inputs(B, L, C, torch.float32, 11)
    ref = [t.double().requires_grad_(True) for t in (x, g, h0)]
    h_r, l_r = gated_ref(*ref)
    for i in range(3):
        ts = [t.cuda().requires_grad_(j == i) for j, t in enumerate((x, g, h0))]
        h, last = gated_scan(*ts)
        for outs, outs_r, ds in (((h,), (h_r,), (dy,)), ((last,), (l_r,), (dl,))):
            a = torch.autograd.grad(outs, ts[i], [d.cuda() for d in ds], retain_graph=True)[0]
            b = torch.autograd.grad(outs_r, ref[i], [d.double() for d in ds], retain_graph=True)[0]
            assert _rel(a, b) < 2 * TOL[torch.float32]
    ts = _leaves(x, g)
    h, last = gated_scan(*ts)                                         # what is saved may not change before the backward
    with torch.no_grad():
        ts[0].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()
    e = torch.zeros(2, 0, 5, device="cuda", requires_grad=True)       # no tokens
    s = torch.randn(2, 5, device="cuda", requires_grad=True)
    h, last = gated_scan(e, e, s)
    assert h.shape == (2, 0, 5) and torch.equal(last, s)
    assert torch.equal(torch.autograd.grad(last.sum(), s)[0], torch.ones_like(s))


def test_gradients_against_differences():
    """In the direction of the gradient: (f(x + t d) - f(x - t d)) / 2 t = |grad|^2 / |grad| within t^2 and fp32's
    rounding of f (2^-24 |f| / t), both some 1e-4 of it at t = 2^-6."""
    B, L, C = 1, 45, 16
    x, g, h0, dy, dl = _inputs(B, L, C, torch.float32, 3)
    ts = _leaves(x, g - 0.05, h0)
    f = lambda *a: sum((o.double() * c.double()).sum() for o, c in zip(gated_scan(*a), (dy.cuda(), dl.cuda())))
    grads = torch.autograd.grad(f(*ts), ts)
    for i in range(3):
        d = grads[i] / grads[i].norm()
        t = 2.0 ** -6
        with torch.no_grad():
            up, down = ([u + s * t * d if j == i else u for j, u in enumerate(ts)] for s in (1, -1))
            slope = float(f(*up) - f(*down)) / (2 * t)
        assert abs(slope / float(grads[i].norm()) - 1) < 2e-3


def test_other_stream_and_graph():
    """Launches go to the current stream; a captured call, forward and backward, replays on new inputs."""
    B, L, C = 2, 200, 64
    x, g, h0, dy, dl = _inputs(B, L, C, torch.float32, 13)
    ts = _leaves(x, g, h0)
    cot = dy.cuda(), dl.cuda()
    want = gated_scan(*ts)
    want_d = torch.autograd.grad(want, ts, cot)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = gated_scan(*ts)
        got_d = torch.autograd.grad(got, ts, cot)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip((*want, *want_d), (*got, *got_d)):
        assert torch.equal(a, b)
    atomic_gdn2.set_checks("async")
    del want, got         # torch captures no backward while an eager graph of the same leaves lives
    graphs = []
    for _ in range(2):                                                # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gated_scan(*ts)
            d = torch.autograd.grad(out, ts, cot)
            with torch.no_grad():
                step = gated_scan(ts[0][:, :1], ts[1][:, :1], ts[2])
        graphs.append((graph, out, d, step))
    with torch.no_grad():
        ts[0].mul_(-2.0)
    for graph, *_ in graphs * 2:
        graph.replay()
    again = gated_scan(*ts)
    again_d = torch.autograd.grad(again, ts, cot)
    with torch.no_grad():
        step_want = gated_scan(ts[0][:, :1], ts[1][:, :1], ts[2])
    for _, out, d, step in graphs:
        for a, b in zip((*again, *again_d, *step_want), (*out, *d, *step)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,C", [(2, 100, 64), (3, 1, 64), (1, 37, 40), (40, 200, 256)])
def test_saved_tensors_that_come_back_in_another_order(B, L, C, dtype):
    """Saved on the host they come back contiguous, whatever the strides they had; other hooks may turn them, rows of
    an odd number of values to rows of an even one and back."""
    gen = torch.Generator(device="cuda").manual_seed(L)
    n = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, g, dh, h0, dlast = n(B, L, C).to(dtype), -n(B, L, C).abs().to(dtype), n(B, L, C).to(dtype), n(B, C), n(B, C)
    lengths = torch.randint(0, L + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
    reset = torch.rand(B, L, generator=gen, device="cuda") < 0.05
    views = ((x, g), (torch.cat([x, x], 2)[..., :C], torch.cat([g, g], 2)[..., :C]),
             (torch.cat([x, x[..., :1]], 2)[..., :C], g), (x, torch.cat([g, g[..., :3]], 2)[..., :C]))
    hooks = (None, torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(
        lambda t: t, lambda t: torch.cat([t, t[..., :1]], 2)[..., :C] if t.ndim == 3 else t),
        torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.mT.contiguous().mT if t.ndim == 3 else t))
    for x2, g2 in views:
        want = None
        for hook in hooks:
            ts = [t.detach().requires_grad_(True) for t in (x2, g2, h0)]
            with hook or torch.enable_grad():
                out = gated_scan(*ts, lengths=lengths, reset=reset)
            got = torch.autograd.grad(out, ts, (dh, dlast))
            want = want or got
            assert all(torch.equal(a, c) for a, c in zip(got, want))
    for back, match in ((lambda t: t.cpu(), "another device"), (lambda t: t[:, :0] if t.ndim == 3 else t, "size")):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            h, _ = gated_scan(*ts)
        with pytest.raises(RuntimeError, match=match):
            h.sum().backward()


def test_same_bits_every_time():
    for B, L, C in ((1, 20000, 40), (3, 1111, 700)):
        x, g, h0, dy, dl = _inputs(B, L, C, torch.float32, 17)
        ts = _leaves(x, g, h0)
        runs = []
        for _ in range(3):
            out = gated_scan(*ts)
            runs.append((*out, *torch.autograd.grad(out, ts, (dy.cuda(), dl.cuda()))))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_offsets_past_32_bits():
    """More than 2^31 values of x and h: the last tokens against the recurrence from the state before them."""
    L, C = 1 << 20, 2100
    x = torch.empty(1, L, C, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    g = torch.full((1, 1, C), -0.1, dtype=torch.bfloat16, device="cuda").expand(1, L, C)
    with torch.no_grad():
        h, last = gated_scan(x, g)
    # 300 tokens forget all but exp(-30) of what was before them
    h_r, l_r = gated_ref(x[:, -300:].double().cpu(), g[:, -300:].double().cpu())
    assert _rel(last, l_r) < TOL[torch.float32] + math.exp(-30)
    assert _rel(h[:, -50:], h_r[:, -50:]) < TOL[torch.bfloat16]
    n = torch.tensor([L - 3], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        h2, _ = gated_scan(x, g, lengths=n)
    assert torch.equal(h2[:, -50:-3], h[:, -50:-3]) and bool((h2[:, -3:] == 0).all())
