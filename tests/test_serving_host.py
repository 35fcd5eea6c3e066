"""Host side of the serving operators: the packed 4-bit layout, quantising, and the refusals that
need no GPU."""
import ctypes
import sys
import pathlib

import pytest
import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2 import _lib, beam_select, make_blr_recurrent, make_cfg, pack_w4, quantize_w4, w4_linear  # noqa: E402


@pytest.mark.parametrize("din,dout,group", [(64, 16, 32), (64, 16, 64), (1, 1, 32), (100, 17, 64), (130, 33, 128),
                                            (512, 48, 128), (191, 257, 32)])
def test_pack_round_trip(din, dout, group):
    gen = torch.Generator().manual_seed(din + dout)
    q = torch.randint(-8, 8, (din, dout), generator=gen, dtype=torch.int8)
    s = torch.rand(-(-din // group), dout, generator=gen).to(torch.bfloat16)
    w = pack_w4(q, s, group)
    assert w.packed.numel() == -(-dout // 32) * -(-din // 128) * 512
    assert torch.equal(w.integers(), q) and torch.equal(w.group_scales(), s)
    assert torch.equal(w.dequantize(), q.float() * s.float().repeat_interleave(group, 0)[:din])


def test_packed_layout_is_the_documented_one():
    """include/gdn2_b200.h: nibble c + 4 e + 2 f of word 4 l + s of tile (u, v) of block (i, j)."""
    din, dout, group = 320, 72, 64
    q = torch.randint(-8, 8, (din, dout), generator=torch.Generator().manual_seed(3), dtype=torch.int8)
    sc = torch.rand(5, dout, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    w = pack_w4(q, sc, group)
    words, scales = w.packed.view(-1).tolist(), w.scales.float().view(-1).tolist()
    for i, j, u, v, l, s, c, e, f in [(0, 0, 0, 0, 0, 0, 0, 0, 0), (1, 1, 1, 1, 31, 3, 1, 1, 1), (2, 2, 0, 0, 13, 2, 0, 1, 0),
                                      (2, 1, 1, 1, 9, 1, 1, 0, 1), (0, 2, 1, 0, 17, 2, 1, 1, 0)]:
        col = 32 * i + 16 * v + l // 4 + 8 * c
        row = 128 * j + 64 * u + 32 * (s // 2) + 8 * (l % 4) + 4 * (s % 2) + 2 * f + e
        nib = (words[((i * 3 + j) * 4 + u * 2 + v) * 128 + 4 * l + s] >> (4 * (c + 4 * e + 2 * f))) & 15
        assert nib == (int(q[row, col]) + 8 if col < dout and row < din else 8)
        if col < dout and row < din:  # [i][j][v][column][row half][c]
            assert scales[((((i * 3 + j) * 2 + v) * 8 + l // 4) * 2 + u) * 2 + c] == float(sc[row // 64, col])


def test_quantize_error_is_half_a_step():
    """|W - s Q| <= s / 2 inside the range of Q (and s / 2 plus the scale's own rounding at the ends:
    7 s >= (1 - 2^-8) max |W|)."""
    W = torch.randn(200, 50, generator=torch.Generator().manual_seed(1))
    W[32:64, 3] = 0.0
    w = quantize_w4(W, 32)
    step = w.group_scales().float().repeat_interleave(32, 0)[:200]
    assert bool(((w.dequantize() - W).abs() <= step * (0.5 + 7 / 256)).all())
    assert bool((w.dequantize()[32:64, 3] == 0).all())


def test_pack_refusals():
    q, s = torch.zeros(64, 16, dtype=torch.int8), torch.ones(1, 16, dtype=torch.bfloat16)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q + 8), dict(q=q - 9), dict(s=s.float()), dict(s=s[:, :8]),
                dict(group=48), dict(q=q[:0]), dict(q=q.bool())):
        with pytest.raises(ValueError):
            pack_w4(bad.get("q", q), bad.get("s", s), bad.get("group", 64))
    for bad in (torch.zeros(4, 4, dtype=torch.int8), torch.zeros(4), torch.full((4, 4), float("nan"))):
        with pytest.raises(ValueError):
            quantize_w4(bad)
    with pytest.raises(ValueError):
        quantize_w4(torch.zeros(4, 4), group=16)


def test_sizes_past_the_kernels_counters_are_refused():
    """Sizes near 2^31, where tokens and columns would be counted past the type's end."""
    lib, at, d = _lib.load(), 4096, _lib.RecDesc()
    d.B, d.H, d.L, d.D, d.n_states, d.in_dtype, d.scale, d.clip = 1, 1, 2 ** 31 - 4, 128, 1, 0, 1.0, 1e4
    assert lib.gdn2_recurrent(ctypes.addressof(d), *[at] * 6, 0, 0, 0, at, at, at, at, 0) == _lib.ERR_UNSUPPORTED
    assert lib.gdn2_recurrent_workspace_bytes(ctypes.addressof(d)) == 0
    d = _lib.W4Desc()
    d.M, d.K, d.N, d.group, d.x_stride, d.y_stride = 1, 64, 2 ** 31 - 1, 64, 64, 2 ** 31
    assert lib.gdn2_w4_linear(ctypes.addressof(d), at, at, at, 0, 0, at, 0, 0) == _lib.ERR_UNSUPPORTED


def test_weight_buffers_have_their_size():
    """The kernel reads din x dout: buffers of another size, type or order are refused when they are put together."""
    from atomic_gdn2 import W4Weight
    w = pack_w4(torch.zeros(130, 40, dtype=torch.int8), torch.ones(3, 40, dtype=torch.bfloat16), 64)
    assert torch.equal(W4Weight(w.packed, w.scales, 130, 40, 64).integers(), w.integers())
    for packed, scales, din, dout, group in (
            (w.packed[:1], w.scales, 130, 40, 64), (w.packed, w.scales[:, :1], 130, 40, 64), (w.packed, w.scales, 257, 40, 64),
            (w.packed, w.scales, 130, 65, 64), (w.packed, w.scales, 130, 40, 32), (w.packed, w.scales, 130, 40, 48),
            (w.packed.long(), w.scales, 130, 40, 64), (w.packed, w.scales.float(), 130, 40, 64), (w.packed, w.scales, 0, 40, 64),
            (w.packed.transpose(0, 1), w.scales, 130, 40, 64)):
        with pytest.raises(ValueError):
            W4Weight(packed, scales, din, dout, group)


def test_binding_is_the_running_torchs(monkeypatch):
    """A binding built against another torch is neither taken for current nor loaded."""
    from atomic_gdn2 import _build
    assert _build.ext_path().exists() and hasattr(_lib.binding(), "recurrent")
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    monkeypatch.setattr(_lib, "_ext", None)
    assert _build._stale()
    with pytest.raises(RuntimeError, match="build it with"):
        _lib.binding()


def test_binding_that_does_not_load(monkeypatch, tmp_path):
    from atomic_gdn2 import _build
    bad = tmp_path / "gdn2_torch.so"
    bad.write_bytes(b"not a library")
    monkeypatch.setattr(_build, "ext_path", lambda: bad)
    monkeypatch.setattr(_lib, "_ext", None)
    with pytest.raises(RuntimeError, match="does not load"):
        _lib.binding()


def test_operators_have_no_cpu_path():
    x = [torch.zeros(1, 1, 1, 128)] * 6
    with pytest.raises(RuntimeError):
        make_blr_recurrent(make_cfg(), 1.0)(*x)
    w = pack_w4(torch.zeros(64, 16, dtype=torch.int8), torch.ones(1, 16, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        w4_linear(torch.zeros(1, 64), w)
    with pytest.raises(RuntimeError):
        beam_select(torch.zeros(1, 1, 8), torch.zeros(1, 1))


def test_entry_points_reject_bad_arguments():
    """Everything is refused before a launch, so no GPU is needed; pointers are never followed."""
    lib, inv, uns, at = _lib.load(), _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED, 4096

    def rec(ptr=at, h0=at, idx=0, hout=at * 2, ws=at, flags=at, **kw):
        d = _lib.RecDesc()
        d.B, d.H, d.L, d.D, d.n_states, d.in_dtype, d.scale, d.clip = 2, 1, 3, 128, 2, 0, 1.0, 1e4
        for i in range(6):
            for j in range(3):
                d.stride[i][j] = 128
        for j in range(3):
            d.o_stride[j] = 128
        for k, v in kw.items():
            if k == "stride":
                d.stride[3][1] = v
            elif k == "o_stride":
                d.o_stride[2] = v
            else:
                setattr(d, k, v)
        return lib.gdn2_recurrent(ctypes.addressof(d), at, at, ptr, at, at, at, h0, idx, 0, at, hout, ws, flags, 0)

    assert lib.gdn2_recurrent(0, *[at] * 14) == inv
    for kw in (dict(B=0), dict(H=-1), dict(L=-1), dict(in_dtype=3), dict(clip=0.0), dict(ptr=0), dict(ptr=at + 4),
               dict(stride=129), dict(stride=-128), dict(o_stride=2), dict(hout=0), dict(hout=at * 2 + 8), dict(flags=0), dict(ws=0), dict(ws=at + 64),
               dict(n_states=1), dict(n_states=0), dict(h0=at * 2, idx=at), dict(h0=at + 4), dict(D=0)):
        assert rec(**kw) == inv, kw
    assert rec(D=64) == uns

    def w4(x=at, packed=at, scales=at, y=at, ws=0, **kw):
        d = _lib.W4Desc()
        d.M, d.K, d.N, d.group, d.x_stride, d.y_stride = 1, 64, 16, 64, 64, 16
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.gdn2_w4_linear(ctypes.addressof(d), x, packed, scales, 0, 0, y, ws, 0)

    for kw in (dict(M=0), dict(K=0), dict(N=-1), dict(dtype=2), dict(act=5), dict(x=0), dict(packed=0), dict(packed=at + 8),
               dict(scales=0), dict(scales=at + 2), dict(x=at + 8), dict(y=0), dict(x_stride=65),
               dict(x_stride=65, ws=at + 8), dict(x_stride=-1), dict(y_stride=15)):
        assert w4(**kw) == inv, kw
    assert w4(group=48) == uns and lib.gdn2_w4_linear(0, *[at] * 8) == inv

    def beam(logits=at, ws=at, **kw):
        d = _lib.BeamDesc()
        d.B, d.K, d.V, d.stride_b, d.stride_k, d.eos = 1, 2, 100000, 200000, 100000, -1
        for k, v in kw.items():
            setattr(d, k, v)
        return (lib.gdn2_beam_select(ctypes.addressof(d), logits, at, 0, at, at, at, at, ws, 0),
                lib.gdn2_beam_workspace_bytes(ctypes.addressof(d)))

    for kw in (dict(B=0), dict(K=0), dict(V=0), dict(dtype=9), dict(stride_b=-1)):
        assert beam(**kw) == (inv, 0), kw
    assert beam(K=33) == (uns, 0)
    assert beam(logits=at + 1)[0] == inv and beam(V=8)[1] == 0
    assert beam(logits=0)[0] == inv and beam(ws=0)[0] == inv and beam(ws=at + 16)[0] == inv
    assert lib.gdn2_beam_select(0, *[at] * 9) == inv
