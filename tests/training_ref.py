"""Plain restatements, in 64 bits on the CPU, of the training operators (test-only)."""
import torch


def gated_ref(x, g, h0=None, lengths=None, reset=None):
    """The recurrence token by token; differentiable.  x, g (B, L, C) double."""
    B, L, C = x.shape
    h = torch.zeros(B, C, dtype=x.dtype) if h0 is None else h0
    out = []
    for t in range(L):
        a = torch.exp(torch.clamp(g[:, t], max=0.0))
        new = a * h + x[:, t]
        if reset is not None:
            new = torch.where(reset[:, t, None], x[:, t], new)
        if lengths is not None:
            on = (t < lengths)[:, None]
            out.append(torch.where(on, new, torch.zeros_like(new)))
            h = torch.where(on, new, h)
        else:
            out.append(new)
            h = new
    return (torch.stack(out, 1) if L else x), h
