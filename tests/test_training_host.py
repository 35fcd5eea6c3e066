"""Host side of the training operators: refusals that need no GPU, and the 8-bit moments' formats."""
import ctypes
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2 import _lib, gated_scan, linear, make_cfg  # noqa: E402
from atomic_gdn2.training import GDN2LM, AdamW, TrainStep, make_optimizer  # noqa: E402
from training_ref import code_m, code_r, decode, encode, root  # noqa: E402


def test_operators_have_no_cpu_path():
    with pytest.raises(RuntimeError):
        linear(torch.zeros(2, 3), torch.zeros(3, 4))
    with pytest.raises(RuntimeError):
        gated_scan(torch.zeros(1, 2, 3), torch.zeros(1, 2, 3))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError):
        AdamW([p]).step()
    with pytest.raises(ValueError):
        gated_scan(torch.zeros(2, 3), torch.zeros(2, 3))


def test_adamw_refusals():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(lr=-1.0),
               dict(weight_decay=-1.0), dict(clip=0.0), dict(clip=-1.0), dict(spike_factor=0.0), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            AdamW(p, **kw)
    opt = AdamW(p)
    assert opt.step() is None                      # nothing has a gradient
    with pytest.raises(RuntimeError):
        opt.grad_norm
    with pytest.raises(ValueError):
        opt.moments(p)
    opt = AdamW([dict(params=p, lr=0.1), dict(params=[torch.nn.Parameter(torch.zeros(1))], eps=1e-3)])
    p[0].grad = torch.zeros(3)
    with pytest.raises(ValueError):
        opt.step()


def test_model_and_step_take_the_operators():
    """The options reach where they are used; without them everything is as it was."""
    m = GDN2LM(make_cfg(), d_model=32, n_heads=1, d_head=16, n_layers=1, blr_fn=lambda *a: None, linear_fn=linear)
    assert m.layers[0].linear_fn is linear and m.linear_fn is linear
    opt = make_optimizer(m, 1e-3, state_bits=8)
    assert isinstance(opt, AdamW) and opt.state_bits == 8 and [g["weight_decay"] for g in opt.param_groups] == [0.1, 0.0]
    step = TrainStep(m, opt, clip=0.7, spike_factor=3.0)
    assert opt.clip == 0.7 and opt.spike_factor == 3.0 and float(step.gn_ema) == 0.0
    plain = GDN2LM(make_cfg(), d_model=32, n_heads=1, d_head=16, n_layers=1, blr_fn=lambda *a: None)
    assert plain.linear_fn is None and isinstance(make_optimizer(plain, 1e-3), torch.optim.AdamW)


def test_a_state_of_other_options_is_refused():
    """What torch's Adam can be told and this optimizer does not do; refused before anything is loaded."""
    p = torch.nn.Parameter(torch.ones(3, 2))
    for kind, kw in ((torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.AdamW, dict(maximize=True)), (torch.optim.Adam, dict(weight_decay=0.1))):
        other = kind([p], lr=0.5, **kw)
        opt = AdamW([p], lr=0.25)
        with pytest.raises(ValueError):
            opt.load_state_dict(other.state_dict())
        assert opt.param_groups[0]["lr"] == 0.25 and "amsgrad" not in opt.param_groups[0]
        with pytest.raises(ValueError):
            AdamW([dict(params=[p], **{k: v for k, v in other.param_groups[0].items() if k != "params"})])
    opt = AdamW([p], lr=0.25)
    for kind, kw in ((torch.optim.AdamW, dict(foreach=True)), (torch.optim.Adam, dict(weight_decay=0.0))):
        opt.load_state_dict(kind([p], lr=0.5, **kw).state_dict())
        assert opt.param_groups[0]["lr"] == 0.5
    back = torch.optim.AdamW([p])
    back.load_state_dict(opt.state_dict())
    bad = opt.state_dict()
    bad["param_groups"][0]["betas"] = (0.9, 1.0)
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)


def test_moment_codes():
    """Half a step: 1/16 of an e4m3 value, 1/32 of a root, each next to the smallest normal numbers of the format;
    zeros stay zeros, and roots above zero stay above zero."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(1000, generator=gen) * torch.exp(torch.randn(1000, generator=gen) * 3)
    x[:10] = 0.0
    v = (torch.randn(1000, generator=gen) * torch.exp(torch.randn(1000, generator=gen) * 3)) ** 2
    v[256:300] = 0.0
    v[512] = 1e30                                    # a block of one large value and many that are next to nothing
    (m8, ms), (v8, vs) = encode(x, 448.0, code_m), encode(root(v), 1.9375, code_r)
    m, v2 = decode(m8, ms, v8, vs)
    steps = ms.repeat_interleave(256)[:1000]
    assert bool(((m - x).abs() <= (x.abs() / 16 + steps * 2.0 ** -10) * 1.0001).all())
    r, r2 = v.sqrt(), v2.sqrt()
    scale = vs.repeat_interleave(256)[:1000]
    assert bool(((r2 - r).abs() <= (r / 32 + scale * 2.0 ** -18) * 1.0001).all())
    assert bool(((v2 > 0) == (v > 0)).all()) and bool((m[:10] == 0).all())
    codes = torch.arange(256, dtype=torch.uint8)
    again, s = encode(decode(codes * 0, torch.ones(1), codes, torch.ones(1))[1].sqrt(), 1.9375, code_r)
    assert torch.equal(again, codes) and float(s) == 1.0


def test_entry_points_reject_bad_arguments():
    """Everything is refused before a launch, so no GPU is needed; pointers are never followed."""
    lib, inv, uns, at = _lib.load(), _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED, 4096

    def lin(x=at, w=at, y=at, ws=at, flags=at, bias=0, **kw):
        d = _lib.LinearDesc()
        d.M, d.K, d.N, d.x_stride, d.w_stride = 32, 64, 16, 64, 16
        for k, v in kw.items():
            setattr(d, k, v)
        a = ctypes.addressof(d)
        return (lib.gdn2_linear_fwd(a, x, w, bias, 0, y, 0, ws, flags, 0), lib.gdn2_linear_fwd_workspace_bytes(a),
                lib.gdn2_linear_bwd(a, x, w, 0, y, at, at, at, ws, flags, 0), lib.gdn2_linear_bwd_workspace_bytes(a, 7))

    for kw in (dict(M=-1), dict(K=0), dict(N=0), dict(dtype=2), dict(bias_dtype=7), dict(act=3), dict(x_stride=63), dict(w_stride=15)):
        assert lin(**kw) == (inv, 0, inv, 0), kw
    for kw in (dict(M=2 ** 29), dict(K=2 ** 30, x_stride=2 ** 30), dict(x_stride=2 ** 31), dict(M=2 ** 27, N=2 ** 27, w_stride=2 ** 27)):
        assert lin(**kw)[0] == uns and lin(**kw)[1] == 0, kw
    for kw in (dict(x=0), dict(w=0), dict(y=0), dict(flags=0), dict(x=at + 8), dict(w=at + 4), dict(y=at + 2), dict(bias=at + 2),
               dict(ws=0, K=2048, x_stride=2048), dict(ws=at + 64, K=2048, x_stride=2048)):
        assert lin(**kw)[0] == inv, kw
    assert lin(x=0)[1] == 0 and lin(x=0)[3] == 0 and lin(x=0, K=2048, x_stride=2048)[1] > 0     # small products need no workspace
    for kw in (dict(x=at + 8), dict(flags=0), dict(act=1), dict(ws=0, M=2048), dict(y=at + 4)):
        assert lin(**kw)[2] == inv, kw
    assert lib.gdn2_linear_fwd(0, *[at] * 9) == inv and lib.gdn2_linear_bwd(0, *[at] * 10) == inv
    assert lin(M=0)[0] == _lib.OK and lin(M=0)[2] == inv

    def gated(x=at, g=at, h0=0, idx=0, last=at, flags=at, marks=at, **kw):
        d = _lib.GatedDesc()
        d.B, d.L, d.C = 2, 8, 16
        for i in range(2):
            d.x_stride[i] = d.g_stride[i] = 16
        for k, v in kw.items():
            if k == "stride":
                d.x_stride[1] = v
            else:
                setattr(d, k, v)
        a = ctypes.addressof(d)
        return (lib.gdn2_gated_fwd(a, x, g, h0, idx, 0, 0, at, last, 0, flags, 0), lib.gdn2_gated_marks_bytes(a),
                lib.gdn2_gated_bwd(a, x, g, 0, 0, marks, at, 0, at, at, 0, flags, 0))

    for kw in (dict(B=0), dict(L=-1), dict(C=0), dict(dtype=5), dict(n_states=-1), dict(stride=-16)):
        assert gated(**kw) == (inv, 0, inv), kw
    assert gated(B=2 ** 27, C=2 ** 20)[0] == uns
    for kw in (dict(x=0), dict(g=0), dict(x=at + 2), dict(last=0), dict(flags=0), dict(idx=at), dict(h0=at), dict(h0=at, n_states=1),
               dict(h0=at, idx=at), dict(h0=at + 2, n_states=2), dict(dtype=1, x=at + 2)):
        assert gated(**kw)[0] == inv, kw
    for kw in (dict(x=0), dict(marks=0), dict(marks=at + 2), dict(flags=0), dict(L=0)):
        assert gated(**kw)[2] == inv, kw
    assert lib.gdn2_gated_fwd(0, *[at] * 11) == inv and lib.gdn2_gated_bwd(0, *[at] * 12) == inv

    def adamw(n=1, control=at, ws=at, desc=None, **kw):
        d, t = _lib.AdamwDesc(), (_lib.AdamwTensor * 2)()
        d.state_bits, d.beta1, d.beta2, d.eps = 32, 0.9, 0.95, 1e-8
        for k, v in (desc or {}).items():
            setattr(d, k, v)
        t[0].p = t[0].g = t[0].m = t[0].v = t[0].step = at
        t[0].n = 100
        for k, v in kw.items():
            setattr(t[0], k, v)
        a, b = ctypes.addressof(d), ctypes.addressof(t)
        return lib.gdn2_adamw_step(a, b, n, 0, control, ws, 0), lib.gdn2_adamw_workspace_bytes(a, b, n)

    for kw in (dict(n=-1), dict(desc=dict(state_bits=4)), dict(desc=dict(beta1=1.0)), dict(desc=dict(beta2=-0.5)),
               dict(desc=dict(eps=-1.0)), dict(desc=dict(clip=-1.0)), dict(desc=dict(spike=float("nan"))), dict(p=0), dict(g=at + 2),
               dict(m=0), dict(v=at + 1), dict(dtype=4), dict(desc=dict(state_bits=8))):
        assert adamw(**kw) == (inv, 0), kw
    for kw in (dict(step=0), dict(control=0), dict(control=at + 2), dict(ws=0), dict(ws=at + 128)):
        assert adamw(**kw)[0] == inv, kw
    assert adamw(n=0) == (_lib.OK, 0) and adamw(**{"n": 1, "p": 0, "g": 0}) == (inv, 0)
    t = (_lib.AdamwTensor * 1)()
    t[0].n = 5
    assert lib.gdn2_adamw_moments(ctypes.addressof(t), 1, 0) == inv and lib.gdn2_adamw_step(0, 0, 0, 0, at, at, 0) == inv


def test_a_descriptor_lives_as_long_as_its_call(monkeypatch):
    """Other threads may empty the descriptors' cache while a call, which has let go of the interpreter, reads its own."""
    import gc
    import importlib
    import types
    import weakref

    L = importlib.import_module("atomic_gdn2.linear")      # the package's name is the function's
    made, calls = [], []

    class Desc(_lib.LinearDesc):
        def __init__(self):
            super().__init__()
            made.append(weakref.ref(self))

    def call(at, *_):
        L._descs.clear()
        gc.collect()
        calls.append(any(r() is not None and ctypes.addressof(r()) == at for r in made))
        return 0

    lib = types.SimpleNamespace(gdn2_linear_fwd=call, gdn2_linear_bwd=call, gdn2_linear_fwd_workspace_bytes=lambda at: 0,
                                gdn2_linear_bwd_workspace_bytes=lambda at, want: 0)
    monkeypatch.setattr(L._lib, "load", lambda: lib)
    monkeypatch.setattr(L._lib, "LinearDesc", Desc)
    monkeypatch.setattr(L, "_guard", lambda dev: L.pipeline._NULL)
    monkeypatch.setattr(L, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(L, "_check_flags", lambda *a: None)
    monkeypatch.setattr(L.pipeline, "_host_flags", lambda dev: types.SimpleNamespace(ptr=0))
    L._descs.clear()
    x, w = torch.zeros(5, 3), torch.zeros(3, 4)
    x, w, y, _ = L._forward(x, w, None, None, 0, False)
    ctx = types.SimpleNamespace(saved_tensors=(x, w, None), needs_input_grad=(True, True, False, False, False), act=0, bias_dtype=None)
    L._Linear.backward(ctx, torch.zeros(5, 4))
    assert calls == [True, True]


@pytest.mark.parametrize("clip", [None, 1.0])
def test_a_closures_loss(clip, monkeypatch):
    """What a closure returns guards the step only where there is a guard, and may be anything: torch's optimizers take no
    notice of it.  A loss that is given always counts."""
    import types
    seen = []
    monkeypatch.setattr(_lib, "binding", lambda: types.SimpleNamespace(adamw_step=lambda *a: seen.append(a[8]) or 0))
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    opt = AdamW([p], clip=clip)
    losses = [torch.tensor(float("nan")), torch.zeros(2), torch.zeros(0), torch.zeros((), dtype=torch.complex64), 1.5, None, (torch.zeros(()), 2)]
    for x in losses:
        assert opt.step(lambda: x) is x
    assert opt.step(lambda: losses[1], loss=losses[0]) is losses[1]
    assert all(s is None for s in seen[1:-1]) and seen[-1] is losses[0]
    assert seen[0] is None if clip is None else bool(torch.isnan(seen[0])) and seen[0].device == p.device


def test_a_steps_clip_and_spike_are_the_optimizers():
    """TrainStep's limits hold from when they are set, with either optimizer, and an optimizer keeps those that it was given."""
    m = GDN2LM(make_cfg(), d_model=32, n_heads=1, d_head=16, n_layers=1, blr_fn=lambda *a: None)
    opt = make_optimizer(m, 1e-3, state_bits=32)
    step = TrainStep(m, opt)
    assert (step.clip, step.spike, opt.clip, opt.spike_factor) == (1.0, 5.0, 1.0, 5.0)
    step.clip, step.spike = 0.25, 7.0
    assert (step.clip, step.spike, opt.clip, opt.spike_factor) == (0.25, 7.0, 0.25, 7.0)
    opt.clip, opt.spike_factor = 0.5, None
    assert (step.clip, step.spike) == (0.5, None)
    opt = AdamW(m.parameters(), clip=0.3, spike_factor=9.0)
    step = TrainStep(m, opt)
    assert (step.clip, step.spike, opt.clip, opt.spike_factor) == (0.3, 9.0, 0.3, 9.0)
    step = TrainStep(m, opt, clip=None, spike_factor=2.0)
    assert (step.clip, step.spike, opt.clip, opt.spike_factor) == (None, 2.0, None, 2.0)
    step = TrainStep(m, make_optimizer(m, 1e-3))
    step.clip = 0.75
    assert (step.clip, step.spike) == (0.75, 5.0)


def test_rows_too_far_apart_are_copied():
    """linear reads rows of any strides; those beyond what the kernels take (2^28 elements, or 2^36 in all) are copied first."""
    import importlib
    rows = importlib.import_module("atomic_gdn2.linear")._rows
    wide = lambda n, ld: torch.empty((n - 1) * ld + 64, device="meta", dtype=torch.bfloat16).as_strided((n, 64), (ld, 1))
    for n, ld in ((2, 2 ** 28 + 8), (2, 2 ** 31), (2 ** 12 + 1, 2 ** 24)):
        t = rows(wide(n, ld))
        assert t.is_contiguous() and t.shape == (n, 64)
    for n, ld in ((2, 2 ** 28), (2 ** 12, 2 ** 24), (1, 2 ** 40), (3, 64)):
        t = wide(n, ld)
        assert rows(t) is t
