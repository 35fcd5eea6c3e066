"""One step of beam search: beam_select(logits, scores, finished) -> (scores, rows, tokens, finished).

Each of B sequences has K beams.  A beam offers its continuations with the total
    score + (x - max x) - log sum exp(x - max x)
over its logits x, and the K best of all the sequence's beams become its new beams.  Inside a beam
they are ordered by logit, the lowest token first among equals; over the beams by total, the lowest
beam first among equals.  A NaN logit or score counts as -inf, a +inf logit as the largest finite
value; a beam whose logits are all -inf (and one whose score is -inf, as all but one at the first
step) offers totals of -inf.  A finished beam offers itself alone, with the end token and its score.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, pipeline
from .recurrent import _raw_stream

MAX_BEAMS = 32
_descs = {}
_fast = None


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished=None, *, eos=None):
    """logits (B, K, V) fp32 or bf16 on the GPU (K <= 32; V contiguous, other strides free); scores
    (B, K) fp32; finished (B, K) bool or None (needs eos); eos: the token that finishes a beam, or None.
    Returns, each (B, K), best first: scores fp32; rows int32, b * K + the beam that is continued
    (an index into the (B K) rows of the logits and of the states: make_blr_recurrent's h_index);
    tokens int32; finished bool."""
    global _fast
    if logits.is_cuda:                                           # the common call; None: it needs more than that
        if _fast is None:
            _fast = _lib.binding().beam_select
        r = _fast(logits, scores, finished, eos)
        if r is not None:
            return r
    else:
        raise RuntimeError("beam_select: logits must be a CUDA tensor (the selection runs only on the B200 kernels)")
    shape, dt, dev = logits.shape, logits.dtype, logits.device
    if len(shape) != 3 or not logits.numel():
        raise ValueError(f"beam_select: logits must be (B, K, V) and not empty; got shape {tuple(shape)}")
    if dt != torch.float32 and dt != torch.bfloat16:
        raise ValueError(f"beam_select: logits must be float32 or bfloat16, not {dt}")
    B, K, V = shape
    if K > MAX_BEAMS:
        raise NotImplementedError(f"beam_select: {K} beams; the B200 kernels implement up to {MAX_BEAMS}")
    if B >= 1 << 31:
        raise NotImplementedError(f"beam_select: {B} sequences")
    if scores.shape != (B, K) or scores.dtype != torch.float32 or scores.device != dev:
        raise ValueError(f"beam_select: scores must be float32 of shape {(B, K)} on {dev}")
    if eos is None:
        if finished is not None:
            raise ValueError("beam_select: finished needs eos, the token that a finished beam goes on with")
        eos = -1
    elif not 0 <= eos < V:
        raise ValueError(f"beam_select: eos={eos} is not a token of 0..{V - 1}")
    if finished is not None and (finished.shape != (B, K) or finished.dtype != torch.bool or finished.device != dev):
        raise ValueError(f"beam_select: finished must be bool of shape {(B, K)} on {dev}")
    pipeline._refuse_gradients("beam_select", (logits, scores))
    if V > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    fp = 0
    if finished is not None:
        finished = finished.contiguous()
        fp = finished.data_ptr()
    lib = _lib.load()
    st = logits.stride()
    key = (shape, dt, st, eos)
    desc = _descs.get(key)
    if desc is None:
        d = _lib.BeamDesc()
        d.B, d.K, d.V, d.eos = B, K, V, eos
        d.dtype = _lib.BF16 if dt == torch.bfloat16 else _lib.F32
        d.stride_b, d.stride_k = st[0], st[1]
        at = ctypes.addressof(d)
        if len(_descs) > 1024:
            _descs.clear()
        desc = _descs[key] = (d, at, lib.gdn2_beam_workspace_bytes(at))
    out = torch.empty((B, K), dtype=torch.float32, device=dev)
    rows = torch.empty((B, K), dtype=torch.int32, device=dev)
    tokens = torch.empty((B, K), dtype=torch.int32, device=dev)
    done = torch.empty((B, K), dtype=torch.bool, device=dev)
    ws = torch.empty(desc[2], dtype=torch.uint8, device=dev) if desc[2] else None
    with torch.cuda.device(dev) if dev.index != torch.cuda.current_device() else pipeline._NULL:
        rc = lib.gdn2_beam_select(desc[1], logits.data_ptr(), scores.data_ptr(), fp, out.data_ptr(), rows.data_ptr(),
                                  tokens.data_ptr(), done.data_ptr(), 0 if ws is None else ws.data_ptr(), _raw_stream(dev.index))
    if rc:
        _lib.check(rc, "gdn2_beam_select")
    return out, rows, tokens, done
