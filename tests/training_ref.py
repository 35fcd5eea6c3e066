"""Plain restatements, in 64 bits on the CPU, of the training operators (test-only)."""
import numpy as np
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


# ---- AdamW: one rounding to fp32 for each operation, as the operator defines it ---------------------
BLOCK = 256


def decode(m, ms, v, vs):
    """The moments that codes and scales stand for, fp32 and flat."""
    n = m.numel()
    c = torch.arange(256, dtype=torch.float64)
    table = torch.where(c < 16, c, (16 + c % 16) * torch.exp2(torch.floor(c / 16) - 1)) * 2.0 ** -18
    rep = lambda s: s.repeat_interleave(BLOCK)[:n]
    r = table.float()[v.flatten().long()] * rep(vs)
    return m.flatten().view(torch.float8_e4m3fn).float() * rep(ms), r * r


def encode(x, top, code):
    """Codes and scales of flat values: code(x / scale) with the scale max |x| / top."""
    n = x.numel()
    p = torch.zeros(-(-n // BLOCK) * BLOCK)
    p[:n] = x
    b = p.view(-1, BLOCK)
    scale = b.abs().amax(1) * torch.tensor(1.0 / top, dtype=torch.float32)
    up = torch.where(scale >= 2.0 ** -126, 1.0 / scale, torch.zeros(()))
    return code(torch.clamp(b * up[:, None], -top, top), b).flatten()[:n], scale


def code_m(x, _):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def code_r(x, r):
    """The nearest of the 256 values, ties to the even code; a root above zero is at least code 1."""
    c = torch.arange(256, dtype=torch.float64)
    table = torch.where(c < 16, c, (16 + c % 16) * torch.exp2(torch.floor(c / 16) - 1)) * 2.0 ** -18
    hi = torch.searchsorted(table, x.double().contiguous()).clamp(1, 255)
    lo = hi - 1
    a, b = x.double() - table[lo], table[hi] - x.double()
    k = torch.where((a < b) | ((a == b) & (lo % 2 == 0)), lo, hi)
    return torch.where((r > 0) & (k == 0), torch.ones_like(k), k).to(torch.uint8)


def root(v):
    """The square root rounded to nearest (torch's on the CPU is not)."""
    return torch.from_numpy(np.sqrt(v.numpy()))


def adamw_ref(p, g, m, v, t, lr, wd, b1, b2, eps, coef):
    """One tensor's step on flat fp32 values -> p, m, v; t is the new step count.  numpy rounds each operation."""
    f = np.float32
    p, g, m, v = p.float().numpy(), g.float().numpy() * f(coef), m.numpy(), v.numpy()
    m = f(b1) * m + f(1 - b1) * g
    v = f(b2) * v + f(1 - b2) * (g * g)
    size, r = f(lr / (1 - b1 ** t)), f((1 - b2 ** t) ** 0.5)
    p = p * f(1 - lr * wd) - size * (m / (np.sqrt(v) / r + f(eps)))
    return torch.from_numpy(p), torch.from_numpy(m), torch.from_numpy(v)


def linear_ref(x, w, b=None, act=None, residual=None):
    """act(x W + b) + residual in 64 bits; differentiable."""
    y = x @ w
    if b is not None:
        y = y + b
    if act == "gelu":
        y = torch.nn.functional.gelu(y, approximate="tanh")
    return y if residual is None else y + residual
