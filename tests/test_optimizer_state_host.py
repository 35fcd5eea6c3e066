"""AdamW's saved states, loaded on the CPU: memory orders, torch's load hooks, refused loads."""
import copy
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2.training import AdamW  # noqa: E402
from training_ref import BLOCK, code_m, code_r, decode, encode, root  # noqa: E402


def _order(t):
    """t's values, flat, in the order of its memory."""
    dims = sorted(range(t.ndim), key=lambda i: -t.stride(i))
    return t.permute(dims).reshape(-1)


def _as(flat, like):
    """Flat values, in memory's order, as a tensor of `like`'s shape and strides."""
    out = torch.empty_like(like, dtype=flat.dtype, requires_grad=False)
    out.as_strided((flat.numel(),), (1,)).copy_(flat)
    return out


def _weights(shape, order, dtype=torch.float32):
    """A parameter of `shape` whose memory has its dimensions in `order`, the slowest first."""
    back = [order.index(i) for i in range(len(shape))]
    return torch.nn.Parameter(torch.zeros([shape[i] for i in order], dtype=dtype).permute(back))


def _stepped(p, bits, seed=0):
    """An optimizer of p whose state stands for moments drawn here: magnitudes of neighbours in memory differ by orders."""
    gen = torch.Generator().manual_seed(seed)
    n = p.numel()
    size = torch.exp(torch.linspace(-6.0, 6.0, n))
    m, v = torch.randn(n, generator=gen) * size, (torch.randn(n, generator=gen) * size) ** 2
    opt = AdamW([p], lr=1e-2, state_bits=bits)
    st = opt.state[p]
    st["step"] = torch.tensor(3.0)
    if bits == 32:
        st["exp_avg"], st["exp_avg_sq"] = _as(m, p), _as(v, p)
    else:
        (m8, ms), (v8, vs) = encode(m, 448.0, code_m), encode(root(v), 1.9375, code_r)
        st["exp_avg"], st["exp_avg_scale"], st["exp_avg_sq"], st["exp_avg_sq_scale"] = _as(m8, p), ms, _as(v8, p), vs
    return opt


def _moments(opt, p):
    """What the state stands for: m and v in the parameter's shape."""
    st = opt.state[p]
    if opt.state_bits == 32:
        return st["exp_avg"], st["exp_avg_sq"]
    m, v = decode(_order(st["exp_avg"]), st["exp_avg_scale"], _order(st["exp_avg_sq"]), st["exp_avg_sq_scale"])
    return _as(m, p), _as(v, p)


ORDERS = [((90, 100), (0, 1), (1, 0)), ((90, 100), (1, 0), (0, 1)), ((4, 6, 10, 7), (0, 1, 2, 3), (0, 2, 3, 1)),
          ((4, 6, 10, 7), (3, 0, 2, 1), (0, 1, 2, 3)), ((1, 300), (0, 1), (1, 0)), ((3, 5), (0, 1), (1, 0)), ((4, 0, 3), (0, 1, 2), (2, 1, 0)), ((90, 100), (1, 0), (1, 0))]


@pytest.mark.parametrize("shape,saved,new", ORDERS)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_state_loads_into_another_order(shape, saved, new, bits, dtype):
    """The moments of every value, whatever order the parameters' memory has.  8 bits: where the order is the same, or one
    block holds all, bit by bit; else rounded once more into the new blocks: half a step of a code, 1/16 of m and 1/32 of
    sqrt v, or half of the new scale's smallest step (2^-10 and 2^-19), and a root above zero stays above zero, at one such
    step at most."""
    p, q = _weights(shape, saved, dtype), _weights(shape, new, dtype)
    opt, other = _stepped(p, bits), AdamW([q], state_bits=bits)
    was = _moments(opt, p)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    st = other.state[q]
    assert float(st["step"]) == 3.0 and st["exp_avg"].stride() == q.stride() == st["exp_avg_sq"].stride()
    now = _moments(other, q)
    if bits == 32 or saved == new or 1 in shape or q.numel() <= BLOCK:
        assert all(torch.equal(a, b) for a, b in zip(was, now))
        return
    far_m = _as(st["exp_avg_scale"].repeat_interleave(BLOCK)[:q.numel()], q)
    far_r = _as(st["exp_avg_sq_scale"].repeat_interleave(BLOCK)[:q.numel()], q)
    assert bool(((now[0] - was[0]).abs() <= (was[0].abs() / 16 + far_m * 2.0 ** -10) * 1.0001).all())
    r, r2 = was[1].sqrt(), now[1].sqrt()
    assert bool(((r2 - r).abs() <= (r / 32 + far_r * 2.0 ** -18) * 1.0001).all())
    assert bool(((now[1] > 0) == (was[1] > 0)).all())
    again = torch.empty_like(q, dtype=torch.float32, requires_grad=False).copy_(was[0])
    m8, ms = encode(_order(again), 448.0, code_m)
    assert torch.equal(_order(st["exp_avg"]), m8) and torch.equal(st["exp_avg_scale"], ms)


def test_codes_whose_blocks_are_unknown_are_refused():
    """Codes that do not fill their memory have no order that scales could belong to."""
    p = _weights((20, 30), (0, 1))
    opt, other = _stepped(p, 8), AdamW([_weights((20, 30), (0, 1))], state_bits=8)
    saved = copy.deepcopy(opt.state_dict())
    wide = torch.zeros(20, 60, dtype=torch.uint8)
    wide[:, ::2] = saved["state"][0]["exp_avg"]
    saved["state"][0]["exp_avg"] = wide[:, ::2]
    with pytest.raises(ValueError, match="order"):
        other.load_state_dict(saved)


@pytest.mark.parametrize("bits", [32, 8])
def test_load_hooks(bits):
    """What a pre hook returns is what is loaded, and what a post hook writes stays, as in torch's optimizers."""
    p, q = _weights((20, 30), (0, 1)), _weights((20, 30), (0, 1))
    opt, other = _stepped(p, bits), AdamW([q], state_bits=bits)
    name = "exp_avg" if bits == 32 else "exp_avg_scale"

    def before(o, d):
        assert o is other
        d = copy.deepcopy(d)
        d["state"][0][name] *= 4.0
        d["state"][0]["step"] += 2.0
        return d

    def after(o):
        st = o.state[q]
        assert torch.equal(_moments(o, q)[0], 4.0 * _moments(opt, p)[0])    # all of it is there by now
        st["exp_avg_sq"].zero_()

    handles = [other.register_load_state_dict_pre_hook(before), other.register_load_state_dict_post_hook(after)]
    saved = opt.state_dict()
    for _ in range(2):
        other.load_state_dict(saved)
        m, v = _moments(other, q)
        assert torch.equal(m, 4.0 * _moments(opt, p)[0]) and not bool(v.any()) and float(other.state[q]["step"]) == 5.0
    for h in handles:
        h.remove()
    other.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(_moments(other, q), _moments(opt, p))) and float(other.state[q]["step"]) == 3.0
    assert not other._optimizer_load_state_dict_pre_hooks and not other._optimizer_load_state_dict_post_hooks


def _everything(opt):
    return copy.deepcopy([(k, v.stride(), v) if isinstance(v, torch.Tensor) else (k, v) for p in opt.param_groups[0]["params"]
                          for k, v in sorted(opt.state[p].items())]), {k: v for k, v in opt.param_groups[0].items() if k != "params"}


def _without(d, *names):
    return {k: v for k, v in d.items() if k not in names}


BAD = {
    "width": lambda st, bits: None,                                  # the other width's state
    "no scale": lambda st, bits: _without(st, "exp_avg_sq_scale"),
    "no scales": lambda st, bits: _without(st, "exp_avg_scale", "exp_avg_sq_scale"),
    "one scale too many": lambda st, bits: {**st, "exp_avg_scale": torch.ones(1)},
    "no moment": lambda st, bits: _without(st, "exp_avg_sq"),
    "no step": lambda st, bits: _without(st, "step"),
    "two steps": lambda st, bits: {**st, "step": torch.ones(2)},
    "shape": lambda st, bits: {**st, "exp_avg": st["exp_avg"].t()},
    "one row": lambda st, bits: {**st, "exp_avg_sq": st["exp_avg_sq"][:1]},
    "type": lambda st, bits: {**st, "exp_avg": st["exp_avg"].to(torch.int32)},
    "not a tensor": lambda st, bits: {**st, "exp_avg": 0.0},
    "another optimizer's": lambda st, bits: {"momentum_buffer": torch.zeros(20, 30)},
}


@pytest.mark.parametrize("bad", sorted(BAD))
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_load_changes_nothing(bad, bits):
    """Weights, moments, scales, step counts, rates: all as before, and the optimizer goes on from there."""
    if bits == 32 and bad in ("no scale", "no scales"):
        pytest.skip("32 bits have none")
    good, p = _weights((20, 30), (0, 1)), _weights((20, 30), (0, 1))
    q = torch.nn.Parameter(torch.ones(4))
    opt = _stepped(p, bits, seed=5)
    opt.add_param_group(dict(params=[q]))
    opt.state[q] = {}
    saved = copy.deepcopy(_stepped(good, 40 - bits if bad == "width" else bits, seed=6).state_dict())
    saved["param_groups"][0]["lr"] = 0.5
    saved["param_groups"].append({**saved["param_groups"][0], "params": [1]})
    st = BAD[bad](saved["state"][0], bits)
    if st is not None:
        saved["state"][0] = st
    was = _everything(opt)
    with pytest.raises(ValueError, match="AdamW"):
        opt.load_state_dict(saved)
    now = _everything(opt)
    assert now[1] == was[1] and opt.param_groups[1]["lr"] == 1e-2
    assert [x[:2] for x in now[0]] == [x[:2] for x in was[0]] and all(torch.equal(a[2], b[2]) for a, b in zip(now[0], was[0]))
    assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks


def test_what_still_loads():
    """torch's own states, of either type; a parameter that was not stepped; a step that is a number."""
    p = torch.nn.Parameter(torch.ones(3, 4, dtype=torch.bfloat16))
    theirs = torch.optim.AdamW([p])
    p.grad = torch.ones_like(p)
    theirs.step()
    p.grad = None
    opt = AdamW([p, torch.nn.Parameter(torch.zeros(2))])
    d = theirs.state_dict()
    d["param_groups"][0]["params"].append(1)
    opt.load_state_dict(d)
    st = opt.state[p]
    assert st["exp_avg"].dtype == torch.float32 and torch.equal(st["exp_avg"], theirs.state[p]["exp_avg"].float()) and float(st["step"]) == 1.0
    d["state"][0]["step"], d["state"][1] = 7, {}
    opt.load_state_dict(d)
    assert float(opt.state[p]["step"]) == 7.0 and opt.state[p]["step"].dtype == torch.float32
    with pytest.raises(ValueError):                                   # torch's own refusal
        opt.load_state_dict(torch.optim.AdamW([p]).state_dict())


def test_a_large_state_is_encoded_in_parts():
    """More values than are encoded at a time, the last block and the last part short: as if all were encoded at once."""
    p, q = _weights((2049, 2051), (0, 1)), _weights((2049, 2051), (1, 0))
    opt, other = _stepped(p, 8), AdamW([q], state_bits=8)
    m, v = _moments(opt, p)
    other.load_state_dict(opt.state_dict())
    st, new = other.state[q], lambda t: _order(torch.empty_like(q, dtype=torch.float32, requires_grad=False).copy_(t))
    r = decode(torch.zeros(p.numel(), dtype=torch.uint8), opt.state[p]["exp_avg_scale"], _order(opt.state[p]["exp_avg_sq"]),
               opt.state[p]["exp_avg_sq_scale"])[1]
    assert torch.equal(_as(r, p), v)
    for name, x, top, code in (("exp_avg", new(m), 448.0, code_m), ("exp_avg_sq", root(new(v)), 1.9375, code_r)):
        codes, scale = encode(x, top, code)
        assert torch.equal(_order(st[name]), codes) and torch.equal(st[name + "_scale"], scale), name
