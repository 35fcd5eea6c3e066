"""AdamW's saved states on the B200: loaded into parameters of another memory order, and stepped on from there."""
import copy

import pytest
import torch

from atomic_gdn2.training import AdamW

pytestmark = pytest.mark.gpu


def _weights(transposed, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = (torch.randn(300, 170, generator=gen) * 0.1).to(dtype).cuda()
    return torch.nn.Parameter(t.t().contiguous().t() if transposed else t)


def _train(opt, p, seed, n=3):
    for k in range(n):
        gen = torch.Generator(device="cuda").manual_seed(seed + k)
        size = torch.exp(torch.randn(p.shape, generator=gen, device="cuda") * 2)
        p.grad = (torch.randn(p.shape, generator=gen, device="cuda") * size).to(p.dtype)
        opt.step()


@pytest.mark.parametrize("on", ["cuda", "cpu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("saved,new", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_into_another_order(bits, saved, new, dtype, on):
    """The moments before and after: the same, or encoded once more (half a step of a code: 1/16 of m, 1/32 of sqrt v, or half
    the scale's smallest step); and the next steps are those of an optimizer that had these moments from the start."""
    p, q, r = (_weights(t, dtype) for t in (saved, new, new))
    opt = AdamW([p], lr=1e-2, clip=1.0, state_bits=bits)
    _train(opt, p, 10)
    state = copy.deepcopy(opt.state_dict())
    for st in state["state"].values():
        for k, v in st.items():
            st[k] = v.to(on)
    a, b = (AdamW([t], lr=1e-2, clip=1.0, state_bits=bits) for t in (q, r))
    a.load_state_dict(state)
    (m, v), (m2, v2) = opt.moments()[0], a.moments()[0]
    if bits == 32 or saved == new:
        assert torch.equal(m, m2) and torch.equal(v, v2)
    else:
        st = a.state[q]
        flat = lambda t: (t.t() if new else t).reshape(-1)
        far_m, far_r = (st[n + "_scale"].repeat_interleave(256)[:q.numel()] for n in ("exp_avg", "exp_avg_sq"))
        assert bool((flat(m2 - m).abs() <= (flat(m).abs() / 16 + far_m * 2.0 ** -10) * 1.0001).all())
        assert bool((flat(v2.sqrt() - v.sqrt()).abs() <= (flat(v.sqrt()) / 32 + far_r * 2.0 ** -18) * 1.0001).all())
    b.load_state_dict(a.state_dict())
    for o, t in ((a, q), (b, r)):
        _train(o, t, 20)
    assert torch.equal(q, r) and float(a.state[q]["step"]) == 6.0
    assert all(torch.equal(x, y) for x, y in zip(a.moments()[0], b.moments()[0]))
