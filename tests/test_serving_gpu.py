"""The serving operators on the B200 against 64-bit restatements.

Tolerances, with u = 2^-24 (fp32) and before any run:
* recurrent: a token's reductions are sums of 128 products in fp32 whose chains are at most about
  20 adds long, 20 u relative; the update is a contraction (gates <= 1, b |k|^2 <= 1) with a memory
  of about 20 tokens at the tested gates, and errors of tokens are independent: 20 u sqrt(20) = 5.3e-6.
* w4: the products are exact (bf16 x) or carry 24 bits (fp32 x); at most K / 16 + 24 additions follow
  one another in fp32 (the tensor core's may truncate: 2 u each): (K / 16 + 24) 2 u sum |x| |W|,
  and half a unit of bf16 (2^-8 of the value covers it) where y is bf16; GELU's slope is below 1.2.
* beam: whole numbers are equal where no two totals of different beams are nearer than 1e-4 (the
  totals themselves are off by a few u of |score| + |logit| < 128: 1e-4 is ten times that).
"""
import math
import pathlib
import sys

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
import atomic_gdn2  # noqa: E402
from atomic_gdn2 import (beam_select, last_status, make_blr_recurrent, make_blr_trainable, make_cfg, pack_w4,  # noqa: E402
                         w4_linear)
from serving_ref import beam_ref, recurrent_ref, w4_ref  # noqa: E402

pytestmark = pytest.mark.gpu
D, U = 128, 2.0 ** -24
REC_TOL = 5.3e-6
SCALE = D ** -0.5


@pytest.fixture(autouse=True)
def _sync_checks():
    atomic_gdn2.set_checks(True)
    yield
    atomic_gdn2.set_checks("async")


def _rel(a, b):
    a, b = a.detach().double().cpu(), b.double()
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


def _inputs(B, H, L, seed, dtype=torch.float32, layout="bhld", g_scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    n = lambda: torch.randn(B, H, L, D, generator=gen)
    l2 = lambda x: x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)
    xs = [l2(n()), l2(n()), n(), l2(n()), torch.sigmoid(n()), g_scale * torch.nn.functional.logsigmoid(n() + 3.0)]
    xs = [t.to(dtype) for t in xs]
    h0 = torch.randn(B, H, D, D, generator=gen) * 0.1
    if layout == "blhd":
        flat = torch.stack([t.transpose(1, 2) for t in xs], 2).contiguous().cuda()   # (B, L, 6, H, D)
        dev = [flat[:, :, i].transpose(1, 2) for i in range(6)]
    else:
        dev = [t.cuda() for t in xs]
    return xs, dev, h0


# ---- recurrent -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["bhld", "blhd"])
@pytest.mark.parametrize("B,H,L", [(1, 1, 1), (3, 2, 1), (40, 6, 1), (160, 5, 1), (2, 3, 2), (1, 2, 3), (1, 6, 7),
                                   (2, 1, 8), (1, 1, 33), (1, 2, 130), (60, 6, 5), (33, 3, 9)])
def test_recurrent_matches_the_recurrence(B, H, L, dtype, layout):
    xs, dev, h0 = _inputs(B, H, L, B * 100 + L, dtype, layout)
    fn = make_blr_recurrent(make_cfg(), SCALE)
    o, h = fn(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    assert o.dtype == h.dtype == torch.float32 and o.shape == (B, H, L, D)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL
    o, h = fn(*dev)
    o_r, h_r = recurrent_ref(*xs, SCALE)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL


@pytest.mark.parametrize("L", [1, 6, 40])
def test_recurrent_lengths_and_index(L):
    """Ragged lengths (empty ones too), states read through an index (repeats, a fresh start)."""
    B, H = 5, 2
    xs, dev, _ = _inputs(B, H, L, 7)
    pool = torch.randn(4, H, D, D, generator=torch.Generator().manual_seed(9)) * 0.1
    lengths = torch.tensor([L, 0, 1, L // 2, L], dtype=torch.int32)
    index = torch.tensor([3, 0, -1, 0, 3], dtype=torch.int32)
    for cast in (torch.int32, torch.int64):
        keep = pool.cuda()
        o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, keep, lengths=lengths.cuda().to(cast), h_index=index.cuda().to(cast))
        o_r, h_r = recurrent_ref(*xs, SCALE, pool, lengths, index)
        assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL
        assert torch.equal(h[1].cpu(), pool[0])                       # an empty sequence keeps its state
        for i, n in enumerate(lengths.tolist()):
            assert bool((o[i, :, n:] == 0).all())
        assert torch.equal(keep.cpu(), pool)


@pytest.mark.parametrize("B,H,L", [(56, 2, 53), (19, 6, 100)])
def test_recurrent_many_heads_many_blocks(B, H, L):
    """112 and 114 heads: the state walks on from block to block, through every slot of the records' ring."""
    xs, dev, h0 = _inputs(B, H, L, L)
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,H,L,layout", [(120, 3, 173, "bhld"), (32, 3, 345, "blhd")])
def test_recurrent_records_in_several_segments(B, H, L, layout, in_place):
    """More records than are kept at a time (64 MiB: 80 tokens of 360 heads, 320 of 96): sequences that are
    empty, end inside a segment, on its border or in the last one, their states in place or through an index."""
    xs, dev, h0 = _inputs(B, H, L, 41, layout=layout)
    gen = torch.Generator().manual_seed(42)
    lengths = torch.randint(0, L + 1, (B,), generator=gen, dtype=torch.int32)
    edge = 80 if B * H == 360 else 320
    lengths[:8] = torch.tensor([L, 0, edge, edge + 1, edge - 1, 1, min(2 * edge, L), L - 1])
    index = None if in_place else torch.randint(-1, B, (B,), generator=gen, dtype=torch.int32)
    state = h0.cuda()
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, state, lengths=lengths.cuda(),
                                                 **(dict(h_out=state) if in_place else dict(h_index=index.cuda())))
    o_r, h_r = recurrent_ref(*xs, SCALE, h0, lengths, index)
    assert (h is state) == in_place and (in_place or torch.equal(state.cpu(), h0))
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL
    for i, n in enumerate(lengths.tolist()):
        assert bool((o[i, :, n:] == 0).all())


def test_recurrent_no_tokens():
    h0 = torch.randn(2, 3, D, D, generator=torch.Generator().manual_seed(1)).cuda()
    x = [torch.empty(2, 3, 0, D, device="cuda") for _ in range(6)]
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*x, h0)
    assert o.shape == (2, 3, 0, D) and torch.equal(h, h0)


def test_recurrent_in_place_and_split_calls():
    """Token by token with h_out = h0 is one call over all tokens."""
    B, H, L = 2, 2, 11
    xs, dev, h0 = _inputs(B, H, L, 4)
    fn = make_blr_recurrent(make_cfg(), SCALE)
    h = h0.cuda()
    o = torch.cat([fn(*[t[:, :, i:i + 1] for t in dev], h, h_out=h)[0] for i in range(L)], 2)
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL
    h = h0.cuda()
    o, h2 = fn(*dev, h, h_out=h)
    assert h2 is h and _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL


def test_recurrent_strides_and_types():
    """Rows that are not contiguous or not on 16 bytes, broadcast inputs, mixed types."""
    B, H, L = 2, 2, 5
    xs, dev, h0 = _inputs(B, H, L, 12)
    wide = torch.zeros(B, H, L, D + 1, device="cuda")
    wide[..., 1:] = dev[0]
    odd = [wide[..., 1:], dev[1].transpose(2, 3).contiguous().transpose(2, 3), dev[2].double(), dev[3],
           dev[4][:1, :, :1].expand(B, H, L, D), dev[5]]
    ref = list(xs)
    ref[4] = xs[4][:1, :, :1].expand(B, H, L, D)
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*odd, h0.cuda())
    o_r, h_r = recurrent_ref(*ref, SCALE, h0)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL


@pytest.mark.parametrize("g_scale", [0.0, 200.0])
def test_recurrent_extreme_gates(g_scale):
    """No decay at all, and gates that close completely (exp underflows)."""
    xs, dev, h0 = _inputs(2, 2, 20, 3, g_scale=g_scale)
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL
    xs[5][:, :, 3] = -math.inf
    dev[5][:, :, 3] = -math.inf
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL


@pytest.mark.parametrize("L", [1, 9])
def test_recurrent_sanitizes(L):
    """NaN -> 0 and clipping at cfg.clip, in o and the final state only."""
    xs, dev, h0 = _inputs(1, 1, L, 5)
    for t in (xs, dev):
        t[2][0, 0, 0, 7] = float("nan")       # poisons column 7 of the state
        t[2][0, 0, 0, 9] = 1e9
    o, h = make_blr_recurrent(make_cfg(clip=2.0), SCALE)(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0, clip=2.0)
    assert bool((h[..., 7] == 0).all()) and bool((o[..., 7] == 0).all())
    assert float(h.abs().max()) <= 2.0 and _rel(h, h_r) < REC_TOL and _rel(o, o_r) < REC_TOL


@pytest.mark.parametrize("B", [1, 40])
@pytest.mark.parametrize("which,col", [(0, None), (1, None), (2, 7), (3, 90), (4, None), (5, None)])
def test_recurrent_nan_counts_from_its_token_on(which, col, B):
    """A NaN in one token of one head: the tokens before it, the other heads and (v, w) the other columns keep
    their values; o of q's token, the column, or everything after it, becomes 0."""
    H, L, at = 3, 21, 12
    xs, dev, h0 = _inputs(B, H, L, 31)
    fn = make_blr_recurrent(make_cfg(), SCALE)
    o_w, h_w = fn(*dev, h0.cuda())
    bad = [t.clone() for t in dev]
    bad[which][0, 1, at, col if col is not None else 5] = float("nan")
    o, h = fn(*bad, h0.cuda())
    assert torch.equal(o[1:], o_w[1:]) and torch.equal(o[0, 0], o_w[0, 0]) and torch.equal(o[0, 2], o_w[0, 2])
    assert _rel(o[0, 1, :at], o_w[0, 1, :at].double().cpu()) < REC_TOL
    if which == 0:
        assert bool((o[0, 1, at] == 0).all())
        assert _rel(o[0, 1, at + 1:], o_w[0, 1, at + 1:].double().cpu()) < REC_TOL
        assert _rel(h, h_w.double().cpu()) < REC_TOL
    elif col is not None:
        keep = [c for c in range(D) if c != col]
        assert bool((o[0, 1, at:, col] == 0).all()) and bool((h[0, 1, :, col] == 0).all())
        assert _rel(o[0, 1, at:][:, keep], o_w[0, 1, at:][:, keep].double().cpu()) < REC_TOL
        assert _rel(h[0, 1][:, keep], h_w[0, 1][:, keep].double().cpu()) < REC_TOL
    else:
        assert bool((o[0, 1, at + 1:] == 0).all())
        assert bool((h[0, 1, 5] == 0).all()) if which in (1, 5) else True


def _same_with_infinities(got, ref, clip=1e4):
    """What an infinity or a NaN reaches is 0 or at the bound, exactly as in 64 bits; the rest as ever."""
    got, at = got.detach().double().cpu(), (ref == 0) | (ref.abs() == clip)
    assert torch.equal(got[at], ref[at])
    assert bool(at.all()) or float((got[~at] - ref[~at]).norm() / ref[~at].norm()) < REC_TOL


@pytest.mark.parametrize("B", [1, 40])
@pytest.mark.parametrize("L,at", [(1, 0), (2, 1), (9, 8), (16, 15), (21, 6), (21, 20)])
@pytest.mark.parametrize("which,value", [(0, math.inf), (1, math.inf), (2, math.inf), (3, -math.inf), (4, math.inf),
                                         (5, -math.inf), ("h0", math.inf), ("h0", math.nan)])
def test_recurrent_infinities(which, value, L, at, B):
    """An infinity in one token of one head, or in its state: in the token's o and in the state what the
    recurrence makes of it, the bound where it stays an infinity and 0 where it becomes a NaN."""
    xs, dev, h0 = _inputs(B, 3, L, 23)
    for t in xs[:2] + dev[:2]:
        t[0, 2] = t[0, 2].abs()                # one head whose sums of infinities keep their sign
    for head in (1, 2):
        if which == "h0":
            h0[0, head, 50, 7] = value
        else:
            for t in (xs, dev):
                t[which][0, head, at, 7] = value
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    _same_with_infinities(o, o_r)
    _same_with_infinities(h, h_r)


@pytest.mark.parametrize("B", [1, 40])
@pytest.mark.parametrize("L,at", [(1, 0), (8, 7), (19, 3)])
@pytest.mark.parametrize("which", range(6))
def test_recurrent_nan_is_the_recurrences(which, L, at, B):
    """The state and the outputs after a NaN in one token, value by value."""
    xs, dev, h0 = _inputs(B, 2, L, 37)
    for t in (xs, dev):
        t[which][0, 1, at, 99] = math.nan
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0)
    _same_with_infinities(o, o_r)
    _same_with_infinities(h, h_r)


def test_recurrent_infinities_in_several_segments():
    """The second of two segments starts from a state with an infinity, and from one that is NaN."""
    B, H, L = 120, 3, 90
    xs, dev, h0 = _inputs(B, H, L, 43, torch.bfloat16)
    for t in (xs, dev):
        t[2][3, 1, 79, 20] = math.inf
        t[2][4, 0, 50, 21] = -math.inf
        t[0][5, 2, 85, 22] = math.inf
    lengths = torch.full((B,), L, dtype=torch.int32)
    lengths[3], lengths[6] = 81, 80
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda(), lengths=lengths.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0, lengths)
    _same_with_infinities(o, o_r)
    _same_with_infinities(h, h_r)


@pytest.mark.parametrize("B", [2, 60])
def test_recurrent_infinite_state_of_short_sequences(B):
    """One token from a state with infinities in a batch of longer ones, and infinities past a sequence's end."""
    xs, dev, h0 = _inputs(B, 2, 20, 29, torch.bfloat16)
    h0[0, 1, 3, 5], h0[0, 1, 90, 100], h0[1, 0, 7, 7] = math.inf, -math.inf, math.nan
    lengths = torch.tensor([1, 0] + [17] * (B - 2), dtype=torch.int32)
    for t in xs + dev:
        t[0, :, 1:] = math.inf
        if B > 2:
            t[2, :, 17:] = math.nan
    o, h = make_blr_recurrent(make_cfg(), SCALE)(*dev, h0.cuda(), lengths=lengths.cuda())
    o_r, h_r = recurrent_ref(*xs, SCALE, h0, lengths)
    _same_with_infinities(o, o_r)
    _same_with_infinities(h, h_r)


def test_recurrent_equals_the_chunked_operator():
    """wy_eps = 0: both evaluate the same function (the chunked one to its fp32-class tolerance, 1e-4)."""
    xs, dev, h0 = _inputs(2, 2, 256, 6)
    cfg = make_cfg(wy_eps=0.0)
    o1, h1 = make_blr_trainable(cfg, SCALE)(*dev, h0.cuda())
    o2, h2 = make_blr_recurrent(cfg, SCALE)(*dev, h0.cuda())
    assert _rel(o2, o1.double().cpu()) < 1e-4 and _rel(h2, h1.double().cpu()) < 1e-4


@pytest.mark.parametrize("L", [1, 10])
def test_recurrent_reports_bad_values(L):
    """A positive gate, an index or a length out of range raise; the results stay defined."""
    xs, dev, h0 = _inputs(2, 1, L, 8)
    fn = make_blr_recurrent(make_cfg(), SCALE)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for kw in (dict(h_index=i32(0, 2)), dict(lengths=i32(L + 1, 0)), dict(lengths=i32(-1, 0)),
               dict(h_index=torch.tensor([0, 2 ** 40], device="cuda"))):
        with pytest.raises(RuntimeError, match="out of range"):
            fn(*dev, h0.cuda(), **kw)
    bad = [t.clone() for t in dev]
    bad[5][1, 0, L - 1, 3] = 0.5
    with pytest.raises(RuntimeError, match="g > 0"):
        fn(*bad, h0.cuda())
    assert last_status() == 0
    fn(*dev, h0.cuda())
    atomic_gdn2.set_checks(False)
    o, h = fn(*dev, h0.cuda(), h_index=i32(1, 9), lengths=i32(L + 5, L))
    assert last_status() == atomic_gdn2._lib.DEV_BAD_INDEX
    o_r, h_r = recurrent_ref(*xs, SCALE, h0, torch.tensor([L, L]), torch.tensor([1, -1]))
    assert _rel(o, o_r) < REC_TOL and _rel(h, h_r) < REC_TOL
    atomic_gdn2.set_checks("async")
    with pytest.raises(RuntimeError, match="later call"):
        fn(*dev, h0.cuda())
    fn(*dev, h0.cuda())
    torch.cuda.synchronize()
    assert last_status() == 0


def test_recurrent_refusals():
    _, dev, h0 = _inputs(2, 2, 4, 1)
    h0 = h0.cuda()
    fn = make_blr_recurrent(make_cfg(), SCALE)
    idx = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        fn(dev[0][:, :, :3], *dev[1:], h0)
    with pytest.raises(ValueError):
        fn(*dev[:5], dev[5].cpu(), h0)
    with pytest.raises(NotImplementedError):
        fn(*[t[..., :64] for t in dev])
    with pytest.raises(ValueError):
        fn(*[t[:0] for t in dev])
    for bad in (h0[:1], h0[:, :1], h0[..., :64], h0.cpu(), h0[0]):
        with pytest.raises(ValueError):
            fn(*dev, bad)
    for kw in (dict(h_index=idx[:1]), dict(h_index=idx.float()), dict(h_index=idx.cpu()), dict(lengths=idx[None]),
               dict(h_index=idx, h_out=h0), dict(h_out=h0[:1]), dict(h_out=h0.bfloat16()), dict(lengths=[1, 2])):
        with pytest.raises(ValueError):
            fn(*dev, h0, **kw)
    big = torch.zeros(3, 2, D, D, device="cuda")
    with pytest.raises(ValueError):
        fn(*dev, big[:2], h_out=big[1:])
    with pytest.raises(ValueError):
        fn(*dev, h_index=idx)
    with pytest.raises(RuntimeError, match="no backward"):
        fn(*dev[:5], dev[5].clone().requires_grad_(True), h0)
    with torch.no_grad():
        fn(*dev[:5], dev[5].clone().requires_grad_(True), h0)


# ---- w4 ------------------------------------------------------------------------------------------
def _w4_inputs(M, din, dout, group, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randint(-8, 8, (din, dout), generator=gen, dtype=torch.int8)
    s = ((torch.rand(-(-din // group), dout, generator=gen) + 0.5) / (4 * math.sqrt(din))).to(torch.bfloat16)
    x = torch.randn(M, din, generator=gen).to(dtype)
    return q, s, x, torch.randn(dout, generator=gen), torch.randn(M, dout, generator=gen).to(dtype)


def _w4_check(y, ref, mag, din, dtype):
    lim = (din / 16 + 24) * 2 * U * 1.2 * mag
    if dtype == torch.bfloat16:
        lim = lim + 2.0 ** -8 * ref.abs()
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,din,dout,group", [
    (1, 64, 16, 64), (1, 1, 1, 32), (1, 512, 4608, 64), (2, 768, 512, 64), (3, 100, 17, 32), (4, 130, 33, 128),
    (5, 2048, 512, 128), (7, 63, 65, 64), (8, 515, 129, 32), (9, 512, 256, 64), (16, 777, 100, 32), (17, 96, 1000, 32),
    (32, 1000, 345, 128), (33, 320, 48, 64), (70, 200, 50, 32), (1, 8192, 64, 128), (6, 4100, 40, 64)])
def test_w4_matches_64_bits(M, din, dout, group, dtype):
    q, s, x, bias, res = _w4_inputs(M, din, dout, group, dtype, M * 7 + din)
    w = pack_w4(q.cuda(), s.cuda(), group)
    assert torch.equal(w.integers().cpu(), q)
    y = w4_linear(x.cuda(), w)
    _w4_check(y, *w4_ref(x, q, s, group), din, dtype)
    y = w4_linear(x.cuda(), w, bias.cuda(), act="gelu", residual=res.cuda())
    assert y.dtype == dtype
    _w4_check(y, *w4_ref(x, q, s, group, bias, "gelu", res), din, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_w4_strides_and_shapes(dtype):
    q, s, x, bias, res = _w4_inputs(6, 200, 70, 64, dtype, 2)
    w = pack_w4(q.cuda(), s.cuda(), 64)
    want = w4_linear(x.cuda(), w, bias.cuda(), residual=res.cuda())
    wide = torch.full((6, 211), float("nan"), dtype=dtype, device="cuda")       # rows off 16 bytes, NaN around them
    wide[:, 3:203] = x.cuda()
    rwide = torch.zeros(6, 75, dtype=dtype, device="cuda")
    rwide[:, 5:] = res.cuda()
    assert torch.equal(w4_linear(wide[:, 3:203], w, bias.cuda(), residual=rwide[:, 5:]), want)
    assert torch.equal(w4_linear(x.cuda().t().contiguous().t(), w, bias.cuda(), residual=res.cuda().t().contiguous().t()), want)
    y3 = w4_linear(x.cuda().view(2, 3, 200), w, bias.double().cuda(), residual=res.cuda().view(2, 3, 70))
    assert y3.shape == (2, 3, 70) and torch.equal(y3.view(6, 70), want)
    assert torch.equal(w4_linear(x[0].cuda(), w, bias.cuda(), residual=res[0].cuda()), want[0])
    one = x[:1].cuda().expand(6, 200)
    assert torch.equal(w4_linear(one, w), w4_linear(x[:1].cuda(), w).expand(6, 70))
    assert w4_linear(x.cuda()[:0], w).shape == (0, 70)


def test_w4_rows_do_not_touch_one_another():
    """An infinity or a NaN in one row of x stays in that row's outputs."""
    q, s, x, _, _ = _w4_inputs(5, 128, 32, 64, torch.float32, 3)
    w = pack_w4(q.cuda(), s.cuda(), 64)
    want = w4_linear(x.cuda(), w)
    x[2, 5], x[4, 7] = math.inf, float("nan")
    y = w4_linear(x.cuda(), w)
    assert torch.equal(y[[0, 1, 3]], want[[0, 1, 3]])
    assert not bool(torch.isfinite(y[2]).any()) and bool(torch.isnan(y[4]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_w4_calls_one_after_the_other(dtype):
    """Calls whose rows are laid out first, back to back in the same workspace: each sees its own x."""
    q, s, x, _, _ = _w4_inputs(8, 1131, 300, 32, dtype, 9)
    w, x = pack_w4(q.cuda(), s.cuda(), 32), x.cuda()
    xs = [(x * f).contiguous() for f in (1.0, -2.0, 0.5, 4.0)]
    want = []
    for t in xs:
        want.append(w4_linear(t, w))
        torch.cuda.synchronize()
    got = [w4_linear(xs[i % 4], w) for i in range(200)]
    assert all(torch.equal(y, want[i % 4]) for i, y in enumerate(got))
    _w4_check(want[0], *w4_ref(x.cpu(), q, s, 32), 1131, dtype)


def test_w4_fp32_range():
    """Very large and very small fp32 values keep their 24 bits."""
    q, s, x, _, _ = _w4_inputs(4, 96, 40, 32, torch.float32, 4)
    w = pack_w4(q.cuda(), s.cuda(), 32)
    for f in (1e30, 1e-25):
        _w4_check(w4_linear((x * f).cuda(), w) , *w4_ref(x * f, q, s, 32), 96, torch.float32)


@pytest.mark.parametrize("M,din", [(3, 200), (3, 131), (12, 200)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_w4_huge_and_infinite_values(M, din, dtype):
    """Values near the type's end, an infinity (the sign of each weight; NaN where one is 0) and a NaN."""
    for group in (32, 64, 128):
        q, s, x, _, _ = _w4_inputs(M, din, 50, group, dtype, 8)
        w = pack_w4(q.cuda(), s.cuda(), group)
        big = (x.float() * 1e36).to(dtype)
        _w4_check(w4_linear(big.cuda(), w), *w4_ref(big, q, s, group), din, dtype)
        x[1, 77], x[2, 9] = -math.inf, float("nan")
        y = w4_linear(x.cuda(), w).float().cpu()
        want = x[1:2].double() @ (q.double() * s.double().repeat_interleave(group, 0)[:din])
        assert torch.equal(torch.isnan(y[1]), torch.isnan(want[0])) and bool(torch.isnan(y[2]).all())
        assert torch.equal(torch.nan_to_num(y[1], nan=0.0, posinf=1.0, neginf=-1.0).double(),
                           torch.nan_to_num(want[0], nan=0.0, posinf=1.0, neginf=-1.0))
        _w4_check(w4_linear(x[:1].cuda(), w), *w4_ref(x[:1], q, s, group), din, dtype)


@pytest.mark.parametrize("M", [1, 8, 9])
@pytest.mark.parametrize("far", [1e3, 1e5, 1e6, 2.0 ** 30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_w4_one_value_far_above_the_rest(M, far, dtype):
    """A value of x that a zero weight leaves out of half the columns (and the smallest weights let into the
    others) must not cost those columns their bits."""
    for group in (32, 64, 128):
        q, s, x, _, _ = _w4_inputs(M, 512, 64, group, dtype, 17)
        for k in (5, 77, 300):
            x[:, k] = far
            q[k, :32], q[k, 32:] = 0, torch.tensor([1, -1], dtype=torch.int8).repeat(16)
        w = pack_w4(q.cuda(), s.cuda(), group)
        _w4_check(w4_linear(x.cuda(), w), *w4_ref(x, q, s, group), 512, dtype)


def test_w4_refusals():
    q, s, x, bias, res = (t.cuda() for t in _w4_inputs(2, 64, 16, 64, torch.float32, 5))
    w = pack_w4(q, s, 64)
    for bad in (lambda: w4_linear(x[:, :60], w), lambda: w4_linear(x.half(), w), lambda: w4_linear(x, w, bias[:8]),
                lambda: w4_linear(x, w, bias.cpu()), lambda: w4_linear(x, w, act="relu"),
                lambda: w4_linear(x, w, residual=res[:1]), lambda: w4_linear(x, w, residual=res.bfloat16()),
                lambda: w4_linear(x, w.to("cpu")), lambda: w4_linear(x[0, 0], w)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: w4_linear(x.requires_grad_(True), w), lambda: w4_linear(x.detach(), w, bias.requires_grad_(True))):
        with pytest.raises(RuntimeError, match="no backward"):
            bad()


def test_w4_refuses_a_weight_of_another_size():
    """A weight whose size was changed after it was packed: nothing is launched."""
    q, s, x, _, _ = (t.cuda() for t in _w4_inputs(2, 128, 32, 64, torch.float32, 5))
    for name, value in (("dout", 64), ("din", 256), ("group", 32), ("group", 0), ("scales", s[:1])):
        w = pack_w4(q, s, 64)
        setattr(w, name, value)
        with pytest.raises(ValueError):
            w4_linear(torch.zeros(2, w.din, device="cuda"), w)


def test_row_counts_past_32_bits_are_refused():
    """They would have been cut to their low 32 bits on the way to the kernels."""
    q, s, x, _, _ = (t.cuda() for t in _w4_inputs(1, 64, 1, 64, torch.bfloat16, 5))
    with pytest.raises(NotImplementedError):
        w4_linear(x.expand(2 ** 32 + 1, 64), pack_w4(q, s, 64))
    with pytest.raises(NotImplementedError):
        beam_select(torch.zeros(1, 1, 8, device="cuda").expand(2 ** 32 + 1, 1, 8),
                    torch.zeros(1, 1, device="cuda").expand(2 ** 32 + 1, 1))


# ---- beam ----------------------------------------------------------------------------------------
def _beam_inputs(B, K, V, dtype, seed, masked=0.0):
    """Inputs whose totals are apart (module docstring): the first seed from `seed` on that gives them."""
    for sd in range(seed, seed + 50):
        gen = torch.Generator().manual_seed(sd)
        x = torch.randn(B, K, V, generator=gen) * 2.5
        if masked:
            x[torch.rand(B, K, V, generator=gen) < masked] = -math.inf
        x = x.to(dtype)
        sc = torch.randn(B, K, generator=gen) * 2 - 12
        fin = torch.rand(B, K, generator=gen) < 0.2
        if beam_ref(x.float(), sc, fin, 0)[4] > 1e-4 and beam_ref(x.float(), sc)[4] > 1e-4:
            return x, sc, fin
    raise AssertionError("no inputs with totals apart")


def _beam_check(got, ref, lim=1e-4):
    sc, rows, tok, done = (t.cpu() for t in got)
    fine = torch.isfinite(ref[0])
    assert torch.equal(torch.isfinite(sc), fine) and torch.equal(sc[~fine].double(), ref[0][~fine])
    assert float((sc.double() - ref[0])[fine].abs().max() if bool(fine.any()) else 0) < lim
    assert torch.equal(rows.long(), ref[1]) and torch.equal(tok.long(), ref[2]) and torch.equal(done, ref[3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,masked", [(1, 1, 1, 0), (1, 1, 300, 0), (3, 4, 256, 0), (2, 5, 33, 0.5), (1, 32, 40, 0),
                                          (2, 16, 7, 0.3), (2, 3, 5000, 0), (1, 2, 20011, 0.7), (1, 8, 4097, 0),
                                          (4, 32, 100, 0.9)])
def test_beam_matches_64_bits(B, K, V, masked, dtype):
    x, sc, fin = _beam_inputs(B, K, V, dtype, 10 * K + V, masked)
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x.float(), sc))
    _beam_check(beam_select(x.cuda(), sc.cuda(), eos=0), beam_ref(x.float(), sc, None, 0))
    _beam_check(beam_select(x.cuda(), sc.cuda(), fin.cuda(), eos=0), beam_ref(x.float(), sc, fin, 0))


def test_beam_first_step_and_dead_beams():
    x, sc, _ = _beam_inputs(2, 4, 50, torch.float32, 1)
    sc[:, 1:] = -math.inf
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))
    x[1] = -math.inf                                        # a sequence with nothing left
    x[0, 0, 3:] = -math.inf                                 # fewer live continuations than beams
    sc[0, 2] = float("nan")
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))
    fin = torch.ones(2, 4, dtype=torch.bool)                # everything finished, two of the scores -inf
    _beam_check(beam_select(x.cuda(), sc.cuda(), fin.cuda(), eos=7), beam_ref(x, sc, fin, 7))


def test_beam_special_logits():
    x, sc, _ = _beam_inputs(1, 4, 64, torch.float32, 2)
    x[0, 0, 5] = float("nan")
    x[0, 1, 9] = math.inf
    x[0, 2, 10:] = torch.finfo(torch.float32).min           # masks of the type's lowest value
    x[0, 3, :] = torch.finfo(torch.float32).min
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))


@pytest.mark.parametrize("V", [64, 9000])
def test_beam_ties(V):
    """Equal logits: the lowest token; equal totals of different beams: the lowest beam; -0 equals 0."""
    x = torch.zeros(1, 4, V)
    sc = torch.full((1, 4), -3.0)
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))
    x[0, :, 1::2] = -0.0
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))
    x[0, :, V - 1] = x[0, :, V // 2] = x[0, :, 3] = 4.0
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))


def test_beam_rising_logits():
    """Every value beats all before it (the list changes at every step), and the reverse."""
    x = torch.arange(20000, dtype=torch.float32).mul_(1e-3).repeat(1, 3, 1)
    x[0, 1] = x[0, 1].flip(0)
    sc = torch.tensor([[-1.0, -1.5, -2.25]])
    _beam_check(beam_select(x.cuda(), sc.cuda()), beam_ref(x, sc))


def test_beam_strides():
    x, sc, fin = _beam_inputs(3, 4, 77, torch.float32, 3)
    want = beam_select(x.cuda(), sc.cuda(), fin.cuda(), eos=2)
    wide = torch.full((4, 3, 80), 99.0, device="cuda")
    wide[..., 2:79] = x.transpose(0, 1).cuda()
    views = [wide[..., 2:79].transpose(0, 1), x.cuda().transpose(1, 2).contiguous().transpose(1, 2)]
    for v in views:
        got = beam_select(v, sc.t().contiguous().t().cuda(), fin.cuda(), eos=2)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_beam_refusals():
    x, sc, fin = _beam_inputs(2, 3, 20, torch.float32, 4)
    x, sc, fin = x.cuda(), sc.cuda(), fin.cuda()
    for bad in (lambda: beam_select(x[0], sc), lambda: beam_select(x.half(), sc), lambda: beam_select(x, sc[:1]),
                lambda: beam_select(x, sc.double()), lambda: beam_select(x, sc.cpu()), lambda: beam_select(x, sc, fin),
                lambda: beam_select(x, sc, fin, eos=20), lambda: beam_select(x, sc, eos=-1),
                lambda: beam_select(x, sc, fin.int(), eos=1), lambda: beam_select(x, sc, fin[:, :2], eos=1),
                lambda: beam_select(x[:, :, :0], sc)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        beam_select(torch.zeros(1, 33, 40, device="cuda"), torch.zeros(1, 33, device="cuda"))
    with pytest.raises(RuntimeError, match="no backward"):
        beam_select(x.requires_grad_(True), sc)


# ---- gradients --------------------------------------------------------------------------------------
def test_forward_mode_is_refused():
    """A dual tensor's tangent would be lost: every operator refuses it, in each of its arguments."""
    fw = torch.autograd.forward_ad
    _, dev, h0 = _inputs(2, 1, 3, 1)
    q, s, x, bias, res = (t.cuda() for t in _w4_inputs(2, 64, 16, 64, torch.float32, 5))
    lg, sc, _ = (t.cuda() for t in _beam_inputs(2, 3, 20, torch.float32, 4))
    fn, w, h0 = make_blr_recurrent(make_cfg(), SCALE), pack_w4(q, s, 64), h0.cuda()
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        for i in range(6):
            with pytest.raises(RuntimeError, match="forward-mode"):
                fn(*dev[:i], dual(dev[i]), *dev[i + 1:], h0)
        for bad in (lambda: fn(*dev, dual(h0)), lambda: w4_linear(dual(x), w), lambda: w4_linear(x, w, dual(bias)),
                    lambda: w4_linear(x, w, residual=dual(res)), lambda: beam_select(dual(lg), sc),
                    lambda: beam_select(lg, dual(sc))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                bad()
            with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                bad()
        fn(*dev, h0), w4_linear(x, w, bias, residual=res), beam_select(lg, sc)


def test_h_out_is_an_in_place_change():
    """A tensor that autograd has saved and h_out overwrites makes its backward raise; one that needs a gradient
    is refused."""
    _, dev, h0 = _inputs(2, 1, 3, 1)
    h0, fn = h0.cuda(), make_blr_recurrent(make_cfg(), SCALE)
    for xs in (dev, [t.double() for t in dev], [t[:, :, :0] for t in dev]):
        buf, p = torch.zeros_like(h0), torch.ones_like(h0).requires_grad_(True)
        y = (p * buf).sum()
        before = buf._version
        fn(*xs, h0, h_out=buf)
        assert buf._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with pytest.raises(RuntimeError, match="no backward"):
            fn(*xs, h0, h_out=p)
        with torch.no_grad():
            fn(*xs, h0, h_out=p)
        with torch.inference_mode():
            fn(*xs, h0, h_out=torch.empty_like(h0))
        assert fn(*xs, h0)[1]._version == 0


# ---- streams and graphs --------------------------------------------------------------------------
def test_other_stream_and_graph_capture():
    """On a side stream, and captured into a CUDA graph and replayed on new values."""
    xs, dev, h0 = _inputs(2, 2, 1, 9)
    q, s, x, bias, res = _w4_inputs(3, 128, 64, 64, torch.float32, 6)
    lg, sc, _ = _beam_inputs(2, 3, 64, torch.float32, 6)
    fn, w = make_blr_recurrent(make_cfg(), SCALE), pack_w4(q.cuda(), s.cuda(), 64)
    h0, x, lg, sc = h0.cuda(), x.cuda(), lg.cuda(), sc.cuda()
    run = lambda: (*fn(*dev, h0), w4_linear(x, w), *beam_select(lg, sc, eos=1))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for t in (h0, x):
        t.mul_(0.5)
    lg.copy_(lg.flip(0))
    graph.replay()
    want = run()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_dependent_launches_in_a_graph():
    """The paths of two launches (x laid out first, slices joined after, blocks of tokens) captured and
    replayed on new values, on another stream than the one they were captured on."""
    xs, dev, h0 = _inputs(2, 2, 20, 9)
    q, s, x, bias, res = _w4_inputs(3, 131, 64, 64, torch.bfloat16, 6)
    lg, sc, _ = _beam_inputs(1, 3, 20000, torch.float32, 6)
    fn, w = make_blr_recurrent(make_cfg(), SCALE), pack_w4(q.cuda(), s.cuda(), 64)
    h0, x, lg, sc = h0.cuda(), x.cuda(), lg.cuda(), sc.cuda()
    run = lambda: (*fn(*dev, h0), w4_linear(x, w), *beam_select(lg, sc, eos=1))
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for t in (h0, x):
        t.mul_(0.5)
    lg.copy_(lg.flip(-1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    want = run()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
