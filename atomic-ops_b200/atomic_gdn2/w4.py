"""Products of a few rows with 4-bit weights: y = act(x W + bias) + residual.

W (din, dout) is Q * s: integers Q in [-8, 7] and one bf16 scale per group of 32, 64 or 128 rows of
a column.  pack_w4 lays a quantised weight out once for the kernel, quantize_w4 quantises one;
w4_linear multiplies.  x, residual and y are fp32 or bf16; the products are exact for bf16 x and
carry 24 bits of fp32 x, sums and scales are fp32.  The kernel reads the weight once per 32 rows
of x, which is what few rows cost; there is no backward.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, pipeline
from .recurrent import _raw_stream

GROUPS = (32, 64, 128)
_ACTS = {None: 0, "gelu": 1}


class W4Weight:
    """A packed 4-bit weight (layout: include/gdn2_b200.h, gdn2_w4_linear).  `packed` (int32) and
    `scales` (bf16) are its buffers, din x dout its size, `group` the rows per scale.  Buffers that
    do not have that size are refused, here and by w4_linear: the kernel trusts them."""

    __slots__ = ("packed", "scales", "din", "dout", "group", "device")

    def __init__(self, packed, scales, din, dout, group):
        self.packed, self.scales, self.din, self.dout, self.group = packed, scales, din, dout, group
        self.check()
        self.device = packed.device

    def check(self) -> None:
        """Raises ValueError where the buffers are not those of a din x dout weight."""
        if self.group not in GROUPS:
            raise ValueError(f"group={self.group} must be one of {GROUPS}")
        if self.din < 1 or self.dout < 1:
            raise ValueError(f"a weight cannot be {self.din} x {self.dout}")
        blocks = -(-self.dout // 32) * -(-self.din // 128)
        for name, t, dtype, n in (("packed", self.packed, torch.int32, blocks * 512),
                                  ("scales", self.scales, torch.bfloat16, blocks * 32 * (128 // self.group))):
            if t.dtype != dtype or t.numel() != n or not t.is_contiguous() or t.device != self.packed.device:
                raise ValueError(f"{name} of a {self.din} x {self.dout} weight must be {n} contiguous {dtype} on one "
                                 f"device; got {tuple(t.shape)} {t.dtype} on {t.device}")

    def to(self, device):
        return W4Weight(self.packed.to(device), self.scales.to(device), self.din, self.dout, self.group)

    def integers(self) -> torch.Tensor:
        """Q (din, dout) int8."""
        nb, kb = -(-self.dout // 32), -(-self.din // 128)
        w = self.packed.view(nb, kb, 2, 2, 8, 4, 2, 2, 1)       # rows' half, columns' half, column, t, quarter, step
        sh = torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)
        n = ((w >> sh) & 15).view(nb, kb, 2, 2, 8, 4, 2, 2, 2, 2, 2)    # ..., e, f, c (nibble c + 2 f + 4 e)
        n = n.permute(1, 2, 6, 5, 7, 9, 8, 0, 3, 10, 4)         # kb, half, quarter, t, step, f, e | nb, half, c, column
        return (n.reshape(kb * 128, nb * 32)[:self.din, :self.dout] - 8).to(torch.int8)

    def dequantize(self) -> torch.Tensor:
        """W (din, dout) fp32."""
        return self.integers().float() * self.group_scales().float().repeat_interleave(self.group, 0)[:self.din]

    def group_scales(self) -> torch.Tensor:
        """s (ceil(din / group), dout) bf16."""
        s = self.scales.permute(1, 4, 0, 2, 5, 3)               # batch, per | block, half, c, column
        return s.reshape(s.shape[0] * s.shape[1], -1)[:-(-self.din // self.group), :self.dout]


def pack_w4(q: torch.Tensor, scales: torch.Tensor, group: int = 64) -> W4Weight:
    """q (din, dout) integers in [-8, 7]; scales (ceil(din / group), dout) bf16.  Lays the weight out
    on q's device.  Values outside the range are refused."""
    if q.ndim != 2 or not q.numel() or q.dtype.is_floating_point or q.dtype == torch.bool:
        raise ValueError("q must be a (din, dout) tensor of integers")
    if group not in GROUPS:
        raise ValueError(f"group={group} must be one of {GROUPS}")
    din, dout = q.shape
    if scales.shape != (-(-din // group), dout) or scales.dtype != torch.bfloat16:
        raise ValueError(f"scales must be bfloat16 of shape {(-(-din // group), dout)}")
    if scales.device != q.device:
        raise ValueError(f"scales are on {scales.device}, q on {q.device}")
    lo, hi = torch.stack(torch.aminmax(q)).tolist()
    if lo < -8 or hi > 7:
        raise ValueError(f"q has values in [{lo}, {hi}], outside [-8, 7]")
    nb, kb = -(-dout // 32), -(-din // 128)
    n = torch.full((kb * 128, nb * 32), 8, dtype=torch.uint8, device=q.device)
    n[:din, :dout] = (q + 8).to(torch.uint8)
    # rows 128 kb + 64 half + 32 quarter + 8 t + 4 step + 2 f + e, columns 32 nb + 16 half + 8 c + column
    n = n.view(kb, 2, 2, 4, 2, 2, 2, nb, 2, 2, 8).permute(7, 0, 1, 8, 10, 3, 2, 4, 6, 5, 9)
    n = n.reshape(nb, kb, 4, 32, 4, 8)                          # block, batch, tile, lane, step, nibble
    packed = (n[..., 0::2] | (n[..., 1::2] << 4)).contiguous().view(torch.int32).squeeze(-1)
    per = 128 // group
    s = torch.zeros(kb * per, nb * 32, dtype=torch.bfloat16, device=q.device)
    s[:scales.shape[0], :dout] = scales
    s = s.view(kb, per, nb, 2, 2, 8).permute(2, 0, 3, 5, 1, 4).contiguous()  # block, batch, half, column, per, c
    return W4Weight(packed, s, din, dout, group)


def quantize_w4(weight: torch.Tensor, group: int = 64) -> W4Weight:
    """Rounds a (din, dout) weight to 4 bits: per group the scale is max |W| / 7 in bf16 (rounded
    first, so that the integers fit the scale that is used), Q = round(W / s) within [-8, 7]."""
    if weight.ndim != 2 or not weight.numel() or not weight.dtype.is_floating_point:
        raise ValueError("weight must be a (din, dout) floating-point tensor")
    if group not in GROUPS:
        raise ValueError(f"group={group} must be one of {GROUPS}")
    w = weight.detach().float()
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weight has values that are not finite")
    din, dout = w.shape
    n = -(-din // group)
    p = torch.zeros(n * group, dout, device=w.device)
    p[:din] = w
    p = p.view(n, group, dout)
    s = (p.abs().amax(1) / 7.0).to(torch.bfloat16)
    q = torch.round(p / torch.where(s > 0, s, torch.ones_like(s)).float()[:, None]).clamp(-8, 7)
    return pack_w4(q.view(n * group, dout)[:din].to(torch.int8), s, group)


_descs = {}
_fast = None


def w4_linear(x: torch.Tensor, weight: W4Weight, bias=None, *, act=None, residual=None) -> torch.Tensor:
    """act(x W + bias) + residual.  x (..., din) fp32 or bf16 CUDA tensor; bias (dout) or None;
    act None or "gelu" (tanh form); residual (..., dout) of x's type.  Returns (..., dout) of x's
    type, rounded once."""
    global _fast
    if x.is_cuda and act in _ACTS:                               # the common call; None: it needs more than that
        if _fast is None:
            _fast = _lib.binding().w4_linear
        y = _fast(x, weight.packed, weight.scales, bias, residual, weight.din, weight.dout, weight.group, _ACTS[act])
        if y is not None:
            return y
    dt, shape, dev = x.dtype, x.shape, x.device
    if not x.is_cuda:
        raise RuntimeError("w4_linear: x must be a CUDA tensor (the product runs only on the B200 kernels)")
    if dt != torch.float32 and dt != torch.bfloat16:
        raise ValueError(f"w4_linear: x must be float32 or bfloat16, not {dt}")
    din, dout = weight.din, weight.dout
    if not shape or shape[-1] != din:
        raise ValueError(f"w4_linear: x has shape {tuple(shape)}, the weight {din} rows")
    weight.check()
    if weight.packed.device != dev:
        raise ValueError(f"w4_linear: x is on {dev}, the weight on {weight.packed.device}")
    if act not in _ACTS:
        raise ValueError(f"w4_linear: act={act!r} is not None or 'gelu'")
    pipeline._refuse_gradients("w4_linear", (x, bias, residual))
    x2 = x if len(shape) == 2 else x.reshape(-1, din)
    M = x2.shape[0]
    if M >= 1 << 31:
        raise NotImplementedError(f"w4_linear: {M} rows of x")
    if din > 1 and x2.stride(1) != 1 or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    y = torch.empty((*shape[:-1], dout), dtype=dt, device=dev)
    bp = rp = rs = 0
    if bias is not None:
        if bias.shape != (dout,) or bias.device != dev:
            raise ValueError(f"w4_linear: bias must have shape {(dout,)} on {dev}")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
        bp = bias.data_ptr()
    if residual is not None:
        if residual.shape != y.shape or residual.dtype != dt or residual.device != dev:
            raise ValueError(f"w4_linear: residual must be {dt} of shape {tuple(y.shape)} on {dev}")
        r2 = residual if len(shape) == 2 else residual.reshape(-1, dout)
        if dout > 1 and r2.stride(1) != 1:
            r2 = r2.contiguous()
        rp, rs = r2.data_ptr(), r2.stride(0)
    if M == 0:
        return y
    xs = 0 if M == 1 else x2.stride(0)
    key = (M, din, dout, weight.group, dt, act, xs, rs)
    desc = _descs.get(key)
    if desc is None:
        d = _lib.W4Desc()
        d.M, d.K, d.N, d.group = M, din, dout, weight.group
        d.dtype = _lib.BF16 if dt == torch.bfloat16 else _lib.F32
        d.act = _ACTS[act]
        d.x_stride, d.res_stride, d.y_stride = xs, rs, dout
        at = ctypes.addressof(d)
        if len(_descs) > 1024:
            _descs.clear()
        desc = _descs[key] = (d, at, _lib.load().gdn2_w4_workspace_bytes(at))
    ws = torch.empty(desc[2], dtype=torch.uint8, device=dev) if desc[2] else None
    with torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else pipeline._NULL:
        rc = _lib.load().gdn2_w4_linear(desc[1], x2.data_ptr(), weight.packed.data_ptr(), weight.scales.data_ptr(),
                                        bp, rp, y.data_ptr(), 0 if ws is None else ws.data_ptr(),
                                        _raw_stream(dev.index))
    if rc:
        _lib.check(rc, "gdn2_w4_linear")
    return y
