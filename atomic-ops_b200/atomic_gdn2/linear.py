"""The linear product with its epilogue: linear(x, W, b, act=, residual=) -> act(x W + b) + residual.

The full-precision sibling of w4_linear, for training and for prompts: differentiable in x, W, b and the
residual, W stored (din, dout) as in the layers.  x, W and the residual are all fp32 or all bf16; sums are fp32.

* bf16: products are exact; the tensor cores add up to 1024 of them, truncating (some 4e-6 of their sum), and these
  sums meet in rounded fp32 additions, whatever the length; y is rounded once.  The backward rounds dz = dy act'(z) to
  bf16 before its two products (not in small products), and z is kept in bf16 between the passes (half a step of each, 2^-8).
* fp32: the tensor cores multiply three bf16 terms of every value (24 bits), sums leave them every 64 values and
  go on in rounded fp32 additions: errors are those of a plain fp32 product.  Magnitudes below about 2^-110 lose
  their low bits.
* small products of either type (some 256 x 256 x 256 and below): plain fp32 in one launch, their backward in one.

Up to 16 rows of fp32 x (4 of bf16) are multiplied without the tensor cores, W read once per eight rows.  Infinities
and NaN come out as the plain sums would have them.

Workspace, for the time of a call: fp32 6 bytes a value of x and W, in the backward of x, W and dz; bf16 2 bytes a value of
dz behind an activation and of operands whose rows are not on 16 bytes; up to 16 times 4 bytes a result where few results
have long sums.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, pipeline
from .recurrent import _check_flags, _raw_stream

_ACTS = {None: 0, "gelu": 1}
_descs = {}
_fast, _last = None, (None, None)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix, or a copy of it, whose rows the kernels can read: unit stride, not overlapping, 16-byte aligned, less than
    2^28 elements apart and 2^36 in all."""
    n, ld = t.shape[0], t.stride(0)
    if (t.shape[1] > 1 and t.stride(1) != 1) or (n > 1 and not (t.shape[1] <= ld <= 1 << 28 and n * ld <= 1 << 36)) \
            or t.data_ptr() % 16 or t.is_neg():
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _desc(x, w, bias_dtype, act, res_stride):
    key = (x.shape, w.shape[1], _ld(x), _ld(w), x.dtype, bias_dtype, act, res_stride)
    e = _descs.get(key)
    if e is None:
        d = _lib.LinearDesc()
        d.M, d.K, d.N = x.shape[0], x.shape[1], w.shape[1]
        d.dtype = _lib.BF16 if x.dtype == torch.bfloat16 else _lib.F32
        d.bias_dtype = _lib.BF16 if bias_dtype == torch.bfloat16 else _lib.F32
        d.act, d.x_stride, d.w_stride, d.res_stride = act, _ld(x), _ld(w), res_stride
        if len(_descs) > 1024:
            _descs.clear()
        at = ctypes.addressof(d)
        lib = _lib.load()
        e = _descs[key] = (d, at, lib.gdn2_linear_fwd_workspace_bytes(at),
                           [lib.gdn2_linear_bwd_workspace_bytes(at, want) for want in range(8)])
    return e


def _guard(dev):
    return torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else pipeline._NULL


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _forward(x, w, bias, residual, act, keep):
    """x (M, K), w (K, N), bias (N), residual (M, N) -> x and w as they were read, y, z (None unless `keep`)."""
    dev = x.device
    x, w = _rows(x), _rows(w)
    if bias is not None:
        bias = bias.resolve_neg().contiguous()
    if residual is not None:
        residual = residual.resolve_neg()
        if residual.shape[1] > 1 and residual.stride(1) != 1:
            residual = residual.contiguous()
    y = torch.empty((x.shape[0], w.shape[1]), dtype=x.dtype, device=dev)
    z = torch.empty_like(y) if keep else None
    fl = pipeline._host_flags(dev)
    if x.shape[0]:
        d, at, ws_bytes, _ = _desc(x, w, None if bias is None else bias.dtype, act,
                                   0 if residual is None else residual.stride(0))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        with _guard(dev):
            rc = _lib.load().gdn2_linear_fwd(at, _ptr(x), _ptr(w), _ptr(bias), _ptr(residual), _ptr(y), _ptr(z),
                                             _ptr(ws), fl.ptr, _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "gdn2_linear_fwd")
        _check_flags(fl, "gdn2_linear_fwd")
    return x, w, y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act):
        x, w, y, z = _forward(x, w, bias, residual, act, act != 0)
        ctx.save_for_backward(x, w, z)
        ctx.act, ctx.bias_dtype = act, None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors                   # or what their hooks made of them
        x, w = _rows(x), _rows(w)
        if z is not None:
            z = z.resolve_neg().contiguous()
        M, K, N, dev = x.shape[0], x.shape[1], w.shape[1], x.device
        want_x, want_w, want_b, want_r, _ = ctx.needs_input_grad
        dr = dy if want_r else None
        if dy.shape != (M, N) or w.shape[0] != K or (z is not None and z.shape != (M, N)) or \
                any(t is not None and (t.device != dev or t.dtype != x.dtype) for t in (w, z, dy)):
            raise RuntimeError("linear: a saved tensor came back on another device, or with another type or size")
        dx = torch.empty((M, K), dtype=x.dtype, device=dev) if want_x else None
        new = torch.empty if M else torch.zeros
        dw = new((K, N), dtype=w.dtype, device=dev) if want_w else None
        db = new((N,), dtype=ctx.bias_dtype, device=dev) if want_b else None
        if M and (want_x or want_w or want_b):
            dy = dy.resolve_neg().contiguous()
            if dy.data_ptr() % 16:
                dy = dy.clone()
            d, at, _, sizes = _desc(x, w, ctx.bias_dtype, ctx.act, 0)
            ws_bytes = sizes[want_x + 2 * want_w + 4 * want_b]
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
            fl = pipeline._host_flags(dev)
            with _guard(dev):
                rc = _lib.load().gdn2_linear_bwd(at, _ptr(x), _ptr(w), _ptr(z), _ptr(dy), _ptr(dx), _ptr(dw), _ptr(db),
                                                 _ptr(ws), fl.ptr, _raw_stream(dev.index))
            if rc:
                _lib.check(rc, "gdn2_linear_bwd")
            _check_flags(fl, "gdn2_linear_bwd")
        return *pipeline._once("linear", (dx, dw, db, dr)), None


def linear(x: torch.Tensor, weight: torch.Tensor, bias=None, *, act=None, residual=None) -> torch.Tensor:
    """act(x W + bias) + residual.  x (..., din) and weight (din, dout), both fp32 or both bf16, on one CUDA device,
    any strides; bias (dout) fp32 or bf16, or None; act None or "gelu" (tanh form); residual (..., dout) of x's
    type, or None.  Returns (..., dout) of x's type.  Differentiable (once) in all four."""
    global _fast, _last
    if isinstance(x, torch.Tensor) and x.is_cuda and act in _ACTS and pipeline._check_mode != "sync":
        if _fast is None:                                        # the common call; None: it needs more than that
            _fast = _lib.binding().linear
        dev, fl = _last
        if dev != x.device:
            _last = dev, fl = x.device, pipeline._host_flags(x.device)
        y = _fast(x, weight, bias, residual, _ACTS[act], fl.ptr)
        if y is not None:
            if any(fl.words):
                _check_flags(fl, "gdn2_linear_fwd")
            return y
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise RuntimeError("linear: x must be a CUDA tensor (the product runs only on the B200 kernels)")
    dt, shape, dev = x.dtype, x.shape, x.device
    if dt != torch.float32 and dt != torch.bfloat16:
        raise ValueError(f"linear: x must be float32 or bfloat16, not {dt}")
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2 or not weight.numel():
        raise ValueError("linear: weight must be a (din, dout) tensor and not empty")
    din, dout = weight.shape
    if weight.dtype != dt or weight.device != dev:
        raise ValueError(f"linear: weight must be {dt} on {dev}, as x is; it is {weight.dtype} on {weight.device}")
    if not shape or shape[-1] != din:
        raise ValueError(f"linear: x has shape {tuple(shape)}, the weight {din} rows")
    if act not in _ACTS:
        raise ValueError(f"linear: act={act!r} is not None or 'gelu'")
    if bias is not None and (bias.shape != (dout,) or bias.device != dev or bias.dtype not in (torch.float32, torch.bfloat16)):
        raise ValueError(f"linear: bias must be float32 or bfloat16 of shape {(dout,)} on {dev}")
    out = (*shape[:-1], dout)
    if residual is not None and (residual.shape != out or residual.dtype != dt or residual.device != dev):
        raise ValueError(f"linear: residual must be {dt} of shape {out} on {dev}")
    x2 = x if len(shape) == 2 else x.reshape(-1, din)
    r2 = residual if residual is None or len(shape) == 2 else residual.reshape(-1, dout)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        y = _Linear.apply(x2, weight, bias, r2, _ACTS[act])
    else:
        pipeline._refuse_gradients("linear", (x, weight, bias, residual))
        y = _forward(x2, weight, bias, r2, _ACTS[act], False)[2]
    return y if len(shape) == 2 else y.view(out)
