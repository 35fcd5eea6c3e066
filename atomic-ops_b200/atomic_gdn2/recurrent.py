"""The recurrent form of the operator: make_blr_recurrent(cfg, scale)(q, k, v, w, b, g, h0) -> (o, h).

Where make_blr_trainable evaluates whole chunks of 128 tokens and is differentiable, this one runs
the token recurrence itself (reference/ref.py:116-130): any L >= 0, single tokens while a model
answers, prompts of any length, sequences of different lengths in one padded batch, states read
through an index.  Nothing is damped (it equals the chunked operator with wy_eps = 0); o and the
final state are sanitized at cfg.clip, and the other fields of cfg do not matter here.  There is no
backward: with gradients enabled it refuses inputs that require them.

Device status: the kernels report a positive gate (outside domain I-1) and an index or a length
out of range by writing to mapped host memory, which the host reads without a copy or a wait.  As
with the chunked operator the default raises at a later call, set_checks(True) synchronises and
raises at once, set_checks(False) leaves it to last_status(); nothing is checked while a stream is
being captured (make a device's first call outside a capture: it sets that memory up).

A value that is not finite counts from its token on: in q for that token's o, in v or w for its
column, in k, b or g for the head.  What it reaches is what the recurrence makes of it, a NaN sanitized
to 0 and an infinity to the bound.  Where there are several tokens, each of such a head takes about
0.6 us.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, pipeline
from .config import BLRConfig

_D = 128
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _check_flags(fl: pipeline._HostFlags, what: str) -> None:
    mode = pipeline._check_mode
    if mode == "off" or (mode == "sync" and torch.cuda.is_current_stream_capturing()):
        return
    if mode == "sync":
        torch.cuda.current_stream(fl.index).synchronize()
    if any(fl.words):
        if torch.cuda.is_current_stream_capturing():
            return
        code = fl.take()
        raise RuntimeError(pipeline._status_message(code, what if mode == "sync" else f"{what} (reported at a later call)"))


def _strides(t: torch.Tensor):
    """t's strides, 0 for a dimension of one (never used)."""
    return [0 if m == 1 else s for m, s in zip(t.shape[:3], t.stride())] + [t.stride(3)]


def _rows_ok(t: torch.Tensor) -> bool:
    """Whether the kernels can read t's rows in place: unit stride, every row on 16 bytes, neighbouring
    tokens less than 2^27 elements apart."""
    n = 16 // t.element_size()
    st = _strides(t)
    return st[3] == 1 and st[2] < 1 << 27 and not (st[0] % n or st[1] % n or st[2] % n or t.data_ptr() % 16)


def _int32(t, name, B, dev):
    if not isinstance(t, torch.Tensor) or t.shape != (B,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor of shape {(B,)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, the inputs on {dev}")
    if t.dtype == torch.int64:  # values past 32 bits stay out of range
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    pa, pb = a.data_ptr(), b.data_ptr()
    return pa < pb + b.numel() * 4 and pb < pa + a.numel() * 4


_descs = {}


def make_blr_recurrent(cfg: BLRConfig, scale):
    """Returns call(q, k, v, w, b, g, h0=None, *, lengths=None, h_index=None, h_out=None) -> (o, h)."""
    scale, clip = float(scale), float(cfg.clip)
    fast, last = None, (None, None)

    def call(q, k, v, w, b, g, h0=None, *, lengths=None, h_index=None, h_out=None):
        """q..g (B, H, L, D) float tensors, D = 128, any strides (rows that are not contiguous or not
        on 16 bytes are copied); mixed or other types are taken as fp32.
          h0       (B, H, D, D), or None for zeros; with h_index any number of rows: (n, H, D, D)
          h_index  (B) the row of h0 that each sequence starts from, negative for zeros: the rows
                   that beam_select returns read each beam's parent without a copy of the states
          lengths  (B) tokens of each sequence, 0..L; past them o is zero and the state stands still
          h_out    (B, H, D, D) fp32 contiguous, written and returned as h (an in-place change to
                   autograd); it may be h0 itself, or without h_index overlap nothing of it
        Returns o (B, H, L, D) fp32 (token-major in memory where q is) and h (B, H, D, D) fp32."""
        nonlocal fast, last
        if isinstance(q, torch.Tensor) and q.is_cuda:           # the common call; None: it needs more than that
            if fast is None:
                fast = _lib.binding().recurrent
            dev, fl = last
            if dev != q.device:
                last = dev, fl = q.device, pipeline._host_flags(q.device)
            r = fast(q, k, v, w, b, g, h0, lengths, h_index, h_out, scale, clip, fl.ptr)
            if r is not None:
                if pipeline._check_mode != "async" or any(fl.words):
                    _check_flags(fl, "gdn2_recurrent")
                return r
        xs = (q, k, v, w, b, g)
        shape, dt, dev = q.shape, q.dtype, q.device
        if len(shape) != 4:
            raise ValueError(f"q must be (B, H, L, D); got shape {tuple(shape)}")
        same = True
        for t in xs:
            if t.shape != shape:
                raise ValueError(f"all of q, k, v, w, b, g must have shape {tuple(shape)}")
            if t.device != dev:
                raise ValueError("all of q, k, v, w, b, g must be on one device")
            same = same and t.dtype == dt
        if not q.is_cuda:
            raise RuntimeError("gdn2: inputs must be CUDA tensors (the operator runs only on the B200 kernels)")
        B, H, L, D = shape
        if D != _D:
            raise NotImplementedError(f"gdn2: head size {D}; the B200 kernels implement {_D}")
        if B == 0 or H == 0:
            raise ValueError(f"gdn2: empty batch or no heads: {tuple(shape)}")
        pipeline._refuse_gradients("make_blr_recurrent", (*xs, h0, h_out))
        if not same or dt not in (torch.float32, torch.bfloat16):
            dt = torch.float32
            xs = tuple(t.to(dt) for t in xs)
        if L and not all([_rows_ok(t) for t in xs]):
            xs = tuple(t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format) for t in xs)
        n_states, given = 0, h_out is not None
        if h0 is not None:
            if h0.ndim != 4 or h0.shape[1:] != (H, D, D) or (h_index is None and h0.shape[0] != B) or not h0.shape[0]:
                raise ValueError(f"h0 must have shape {(B if h_index is None else 'n', H, D, D)}")
            if h0.device != dev:
                raise ValueError(f"h0 is on {h0.device}, the inputs on {dev}")
            if h0.dtype != torch.float32 or not h0.is_contiguous() or h0.data_ptr() % 16:
                h0 = h0.to(torch.float32).clone(memory_format=torch.contiguous_format)
            n_states = h0.shape[0]
        elif h_index is not None:
            raise ValueError("h_index needs h0")
        if h_index is not None:
            h_index = _int32(h_index, "h_index", B, dev)
        if lengths is not None:
            lengths = _int32(lengths, "lengths", B, dev)
        if h_out is None:
            h_out = torch.empty((B, H, D, D), dtype=torch.float32, device=dev)
        else:
            if h_out.shape != (B, H, D, D) or h_out.dtype != torch.float32 or not h_out.is_contiguous() \
                    or h_out.device != dev or h_out.data_ptr() % 16:
                raise ValueError(f"h_out must be a contiguous fp32 tensor of shape {(B, H, D, D)} on {dev}")
            if h0 is not None and _overlap(h0, h_out) and (h_index is not None or h0.data_ptr() != h_out.data_ptr()):
                raise ValueError("h_out overlaps h0: only h_out = h0 without h_index is possible")
        qst = xs[0].stride()
        if qst[1] < qst[2]:                                    # token-major: so is o
            o = torch.empty((B, L, H, D), dtype=torch.float32, device=dev).transpose(1, 2)
        else:
            o = torch.empty((B, H, L, D), dtype=torch.float32, device=dev)
        key = (shape, dt, scale, clip, n_states, qst, *[t.stride() for t in xs[1:]])
        desc = _descs.get(key)
        if desc is None:
            d = _lib.RecDesc()
            d.B, d.H, d.L, d.D, d.n_states = B, H, L, D, n_states
            for i, t in enumerate(xs):
                for j, st in enumerate(_strides(t)[:3]):
                    d.stride[i][j] = st if L else 0
            for j in range(3):
                d.o_stride[j] = o.stride(j)
            d.in_dtype = _lib.BF16 if dt == torch.bfloat16 else _lib.F32
            d.scale, d.clip = scale, clip
            if len(_descs) > 1024:
                _descs.clear()
            at = ctypes.addressof(d)
            desc = _descs[key] = (d, at, _lib.load().gdn2_recurrent_workspace_bytes(at))
        ws = torch.empty(desc[2], dtype=torch.uint8, device=dev) if desc[2] else None
        fl = pipeline._host_flags(dev)
        with torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else pipeline._NULL:
            rc = _lib.load().gdn2_recurrent(
                desc[1], xs[0].data_ptr(), xs[1].data_ptr(), xs[2].data_ptr(), xs[3].data_ptr(), xs[4].data_ptr(),
                xs[5].data_ptr(), 0 if h0 is None else h0.data_ptr(), 0 if h_index is None else h_index.data_ptr(),
                0 if lengths is None else lengths.data_ptr(), o.data_ptr(), h_out.data_ptr(),
                0 if ws is None else ws.data_ptr(), fl.ptr,
                _raw_stream(dev.index))
        if rc:
            _lib.check(rc, "gdn2_recurrent")
        if given and not h_out.is_inference():                 # autograd may have saved it
            torch.autograd.graph.increment_version(h_out)
        _check_flags(fl, "gdn2_recurrent")
        return o, h_out

    return call
