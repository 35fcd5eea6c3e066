"""The diagonal gated linear recurrence: gated_scan(x, g, h0) -> (h, last).

    h_t = exp(min(g_t, 0)) h_{t-1} + x_t            each channel by itself, over (B, L, C)

The elementwise sibling of make_blr_trainable and make_blr_recurrent in one operator: any L >= 0, long
sequences by a scan over their segments, single tokens while a model answers, differentiable.  Gates are
logarithms as there (domain I-1: g <= 0, -inf forgets everything); states are fp32, inputs and outputs fp32 or
bf16, rounded once.  x and g of two types, or of others, are copied to fp32; h and the gradients come back in the types of
their inputs.

Sequences of different lengths in one padded batch: `lengths`; past a sequence's length the state stands
still, h and the gradients are zero, and what the inputs hold there does not matter.  Several documents one
after the other in a sequence: `reset` marks the tokens that start from nothing (h_t = x_t, whatever the
state before it holds).

Gates that multiply up to less than fp32's smallest number within a stretch of tokens count as that number, 2^-149:
next to nothing, but of a state of 1e38 it is 1e-7.

Device status as with make_blr_recurrent: a positive gate, an index or a length out of range are reported in
mapped host memory, by default at a later call.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, pipeline
from .recurrent import _check_flags, _int32, _overlap, _raw_stream

_descs = {}
_fast, _last = None, (None, None)


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it that the kernels can read: unit stride along C, bf16 pairs on 4 bytes."""
    if (t.shape[2] != 1 and t.stride(2) != 1) or (t.dtype == torch.bfloat16 and t.data_ptr() % 4) or t.is_neg():
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _spans(t: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether `out`, contiguous, lies within the memory from t's first value to its last."""
    if not t.numel():
        return False
    first, a = t.data_ptr(), out.data_ptr()
    end = first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    return a < end and first < a + out.numel() * out.element_size()


def _desc(x, g, n_states):
    B, L, C = x.shape
    key = (x.shape, x.stride(), g.stride(), x.dtype, n_states)
    e = _descs.get(key)
    if e is None:
        d = _lib.GatedDesc()
        d.B, d.L, d.C, d.n_states = B, L, C, n_states
        d.dtype = _lib.BF16 if x.dtype == torch.bfloat16 else _lib.F32
        for i in range(2):
            d.x_stride[i] = x.stride(i) if x.shape[i] > 1 else 0
            d.g_stride[i] = g.stride(i) if x.shape[i] > 1 else 0
        if len(_descs) > 1024:
            _descs.clear()
        at = ctypes.addressof(d)
        e = _descs[key] = (d, at, _lib.load().gdn2_gated_marks_bytes(at))
    return e


def _guard(dev):
    return torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else pipeline._NULL


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _forward(x, g, h0, lengths, reset, h_index, last, keep):
    """Returns x and g as they were read, h, last and the marks (None unless `keep`)."""
    dt, dev = x.dtype, x.device
    if dt != g.dtype or dt not in (torch.float32, torch.bfloat16):
        x, g = x.float(), g.float()
    x, g = _readable(x), _readable(g)
    if h0 is not None:
        h0 = h0.to(torch.float32).resolve_neg().contiguous()
    d, at, mark_bytes = _desc(x, g, 0 if h0 is None else h0.shape[0])
    h = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if last is None:
        last = torch.empty((x.shape[0], x.shape[2]), dtype=torch.float32, device=dev)
    marks = torch.empty(mark_bytes, dtype=torch.uint8, device=dev) if keep else None
    fl = pipeline._host_flags(dev)
    with _guard(dev):
        rc = _lib.load().gdn2_gated_fwd(at, _ptr(x), _ptr(g), _ptr(h0), _ptr(h_index), _ptr(lengths), _ptr(reset),
                                        _ptr(h), _ptr(last), _ptr(marks), fl.ptr, _raw_stream(dev.index))
    _lib.check(rc, "gdn2_gated_fwd")
    return x, g, h, last, marks, fl


def _as_input(h: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return h.to(dtype) if dtype.is_floating_point else h


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, h0, lengths, reset):
        ctx.types = x.dtype, g.dtype, None if h0 is None else h0.dtype
        x, g, h, last, marks, fl = _forward(x, g, h0, lengths, reset, None, None, True)
        ctx.save_for_backward(x, g, marks, lengths, reset)
        ctx.set_materialize_grads(False)
        _check_flags(fl, "gdn2_gated_fwd")
        return _as_input(h, ctx.types[0]), last

    @staticmethod
    def backward(ctx, dh, dlast):
        x, g, marks, lengths, reset = ctx.saved_tensors     # or what their hooks made of them
        x, g = _readable(x), _readable(g)
        B, L, C = x.shape
        dev = x.device
        marks, lengths, reset = (None if t is None else t.contiguous() for t in (marks, lengths, reset))
        if any(t is not None and t.device != dev for t in (g, marks, lengths, reset, dh, dlast)):
            raise RuntimeError("gated_scan: a saved tensor came back on another device")
        for t, shape in ((g, x.shape), (lengths, (B,)), (reset, (B, L)), (dh, x.shape), (dlast, (B, C))):
            if t is not None and t.shape != shape or g.dtype != x.dtype or marks.numel() != _desc(x, g, 0)[2]:
                raise RuntimeError("gated_scan: a saved tensor came back with another type or size")
        tx, tg, th = ctx.types
        if dlast is not None:
            dlast = dlast.to(torch.float32).resolve_neg().contiguous()
        if L == 0:
            d0 = None
            if th is not None:
                d0 = (torch.zeros(B, C, device=dev) if dlast is None else dlast).to(th)
            empty = [torch.empty(B, L, C, dtype=t, device=dev) for t in (tx, tg)]
            return *pipeline._once("gated_scan", (*empty, d0)), None, None
        dh = torch.zeros(x.shape, dtype=x.dtype, device=dev) if dh is None else dh.to(x.dtype).resolve_neg().contiguous()
        if dh.data_ptr() % 4:
            dh = dh.clone()
        dx, dg = torch.empty_like(dh), torch.empty_like(dh)
        d0 = torch.empty((B, C), dtype=torch.float32, device=dev) if th is not None and ctx.needs_input_grad[2] else None
        d, at, _ = _desc(x, g, 0)
        fl = pipeline._host_flags(dev)
        with _guard(dev):
            rc = _lib.load().gdn2_gated_bwd(at, _ptr(x), _ptr(g), _ptr(lengths), _ptr(reset), _ptr(marks), _ptr(dh),
                                            _ptr(dlast), _ptr(dx), _ptr(dg), _ptr(d0), fl.ptr,
                                            _raw_stream(dev.index))
        _lib.check(rc, "gdn2_gated_bwd")
        _check_flags(fl, "gdn2_gated_bwd")
        return *pipeline._once("gated_scan", (dx.to(tx), dg.to(tg), None if d0 is None else d0.to(th))), None, None


def gated_scan(x: torch.Tensor, g: torch.Tensor, h0=None, *, lengths=None, reset=None, h_index=None, h_out=None):
    """x, g (B, L, C) on the GPU, both fp32 or both bf16 (copied to fp32 where they are not), rows of any strides.
      h0       (B, C), or None for zeros; with h_index any number of rows: (n, C)
      lengths  (B) int32 or int64, tokens of each sequence, 0..L
      reset    (B, L) bool: tokens that drop the state before them
      h_index  (B) the row of h0 that each sequence starts from, negative for zeros (beam_select's rows)
      h_out    (B, C) fp32 contiguous, written and returned as `last` (an in-place change to autograd); it may
               be h0 itself where there is no h_index, and otherwise lies outside the inputs' memory
    Returns h (B, L, C) of x's type (fp32 where x is of whole numbers) and last (B, C) fp32, the state after each
    sequence's last token.
    Differentiable in x, g and h0, but not with h_index or h_out: those are for answering."""
    global _fast, _last
    if isinstance(x, torch.Tensor) and x.is_cuda and pipeline._check_mode != "sync":
        if _fast is None:                                        # the common call; None: it needs more than that
            _fast = _lib.binding().gated_scan
        dev, fl = _last
        if dev != x.device:
            _last = dev, fl = x.device, pipeline._host_flags(x.device)
        r = _fast(x, g, h0, lengths, reset, h_index, h_out, fl.ptr)
        if r is not None:
            if any(fl.words):
                _check_flags(fl, "gdn2_gated_fwd")
            return r
    if not isinstance(x, torch.Tensor) or x.ndim != 3:
        raise ValueError("gated_scan: x must be a (B, L, C) tensor")
    if not isinstance(g, torch.Tensor) or g.shape != x.shape:
        raise ValueError(f"gated_scan: g must have x's shape {tuple(x.shape)}")
    dev = x.device
    if not x.is_cuda:
        raise RuntimeError("gated_scan: x must be a CUDA tensor (the operator runs only on the B200 kernels)")
    if g.device != dev:
        raise ValueError("gated_scan: x and g must be on one device")
    if x.is_complex() or g.is_complex():
        raise ValueError("gated_scan: x and g must be real")
    B, L, C = x.shape
    if B == 0 or C == 0:
        raise ValueError(f"gated_scan: empty batch or no channels: {tuple(x.shape)}")
    if h0 is not None:
        if h0.ndim != 2 or h0.shape[1] != C or (h_index is None and h0.shape[0] != B) or not h0.shape[0]:
            raise ValueError(f"gated_scan: h0 must have shape {(B if h_index is None else 'n', C)}")
        if h0.device != dev:
            raise ValueError(f"gated_scan: h0 is on {h0.device}, x on {dev}")
    elif h_index is not None:
        raise ValueError("gated_scan: h_index needs h0")
    if h_index is not None:
        h_index = _int32(h_index, "h_index", B, dev)
    if lengths is not None:
        lengths = _int32(lengths, "lengths", B, dev)
    if reset is not None:
        if not isinstance(reset, torch.Tensor) or reset.shape != (B, L) or reset.dtype != torch.bool or reset.device != dev:
            raise ValueError(f"gated_scan: reset must be bool of shape {(B, L)} on {dev}")
        reset = reset.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, g, h0)):
        if h_index is not None or h_out is not None:
            raise RuntimeError("gated_scan has no backward with h_index or h_out: call it under torch.no_grad()")
        return _Gated.apply(x, g, h0, lengths, reset)
    pipeline._refuse_gradients("gated_scan", (x, g, h0, h_out))
    if h_out is not None:
        if h_out.shape != (B, C) or h_out.dtype != torch.float32 or not h_out.is_contiguous() or h_out.device != dev \
                or h_out.is_neg():
            raise ValueError(f"gated_scan: h_out must be a contiguous fp32 tensor of shape {(B, C)} on {dev}")
        if h0 is not None and h0.dtype == torch.float32 and _overlap(h0, h_out) and \
                (h_index is not None or h0.data_ptr() != h_out.data_ptr() or not h0.is_contiguous()):
            raise ValueError("gated_scan: h_out overlaps h0: only h_out = h0 without h_index is possible")
        if any(_spans(t, h_out) for t in (x, g)):
            raise ValueError("gated_scan: h_out overlaps an input")
    _, _, h, last, _, fl = _forward(x, g, h0, lengths, reset, h_index, h_out, False)
    if h_out is not None and not h_out.is_inference():         # autograd may have saved it
        torch.autograd.graph.increment_version(h_out)
    _check_flags(fl, "gdn2_gated_fwd")
    return _as_input(h, x.dtype), last
