"""64-bit restatements of the serving operators for the tests, on the CPU."""
import math

import torch


def recurrent_ref(q, k, v, w, b, g, scale, h0=None, lengths=None, h_index=None, clip=1e4):
    q, k, v, w, b, g = (t.detach().double().cpu() for t in (q, k, v, w, b, g))
    B, H, L, D = q.shape
    if h0 is None:
        S = torch.zeros(B, H, D, D, dtype=torch.float64)
    else:
        h0 = h0.detach().double().cpu()
        if h_index is None:
            S = h0.clone()
        else:
            S = torch.stack([h0[i] if 0 <= i < len(h0) else torch.zeros_like(h0[0]) for i in h_index.tolist()])
    o = torch.zeros(B, H, L, D, dtype=torch.float64)
    n = [L] * B if lengths is None else [min(max(int(x), 0), L) for x in lengths.tolist()]
    for i in range(B):
        for t in range(n[i]):
            S[i] *= torch.exp(g[i, :, t].clamp(max=0.0))[:, :, None]
            d = w[i, :, t] * v[i, :, t] - torch.einsum("hd,hdv->hv", b[i, :, t] * k[i, :, t], S[i])
            S[i] += k[i, :, t][:, :, None] * d[:, None, :]
            o[i, :, t] = scale * torch.einsum("hd,hdv->hv", q[i, :, t], S[i])
    fix = lambda x: torch.nan_to_num(x.clamp(-clip, clip), nan=0.0)
    return fix(o), fix(S)


def w4_ref(x, q, s, group, bias=None, act=None, residual=None):
    """(y, sum |x| |W|) in 64 bits."""
    W = q.double().cpu() * s.double().cpu().repeat_interleave(group, 0)[: q.shape[0]]
    x = x.double().cpu()
    y, mag = x @ W, x.abs() @ W.abs()
    if bias is not None:
        y, mag = y + bias.double().cpu(), mag + bias.double().cpu().abs()
    if act == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if residual is not None:
        y, mag = y + residual.double().cpu(), mag + residual.double().cpu().abs()
    return y, mag


def beam_ref(logits, scores, finished=None, eos=None):
    """Candidates one by one, sorted by the stated order: (scores, rows, tokens, finished, gap), gap
    the smallest distance between two different totals of different beams near the selection."""
    logits, scores = logits.double().cpu(), scores.double().cpu()
    B, K, V = logits.shape
    ninf, top = -math.inf, float(torch.finfo(torch.float32).max)
    out, gap = [], math.inf
    for b in range(B):
        cand = []
        for k in range(K):
            sc = float(scores[b, k])
            sc = ninf if sc != sc else sc
            if finished is not None and bool(finished[b, k]):
                cand += [(sc, k, 0, eos)] + [(ninf, k, r, eos) for r in range(1, min(K, V))]
                continue
            x = torch.nan_to_num(logits[b, k], nan=ninf, posinf=top, neginf=ninf).clamp(max=top)
            m = float(x.max())
            lse = math.log(float(torch.exp(x - m).sum())) if m > ninf else 0.0
            x = x.tolist()
            order = sorted(range(V), key=lambda t: (-x[t], t))[: min(K, V)]
            for r, t in enumerate(order):
                tot = sc + ((x[t] - m) - lse) if m > ninf and x[t] > ninf and sc > ninf else ninf
                cand.append((tot, k, r, t))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        pick = cand[:K]
        for a, c in zip(cand[:K], cand[1:K + 1]):
            if a[1] != c[1] and a[0] != c[0]:
                gap = min(gap, abs(a[0] - c[0]))
        out.append(pick)
    sc = torch.tensor([[c[0] for c in p] for p in out], dtype=torch.float64)
    rows = torch.tensor([[b * K + c[1] for c in p] for b, p in enumerate(out)])
    tok = torch.tensor([[c[3] for c in p] for p in out])
    done = torch.tensor([[bool(finished is not None and finished[b, c[1]]) or (eos is not None and c[3] == eos)
                          for c in p] for b, p in enumerate(out)])
    return sc, rows, tok, done, gap
