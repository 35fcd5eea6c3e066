"""What the training operators are measured on: the linear product with its epilogue, the gated scan and the AdamW step.

Each operator has a plain form here (elementary torch operations in 32 bits) and the framework's call; `own` says which
of the two `run` makes.  The widths 512 / 768 / 2048 / 4608, the batch of 8 sequences of 2048 tokens, the eight layers and
the 256-entry vocabulary are the language model's own; the other sizes are generic.
"""
import math

import torch

own = False

BLOCK = 256  # values that share a scale where the optimizer's moments are held in 8 bits
LR, BETAS, EPS, DECAY, CLIP = 3e-4, (0.9, 0.95), 1e-8, 0.1, 1.0


def listed():
    return [
        # the layer's input projection for one token, not quantised: the smallest call
        dict(name="linear m1 512x4608", op="linear", M=1, K=512, N=4608, dtype="fp32", bias=True, act="", residual=False,
             train=False),
        # the layer's up projection in a training step: 8 sequences of 2048 tokens, fp32 weights
        dict(name="linear m16384 512x2048 train", op="linear", M=16384, K=512, N=2048, dtype="fp32", bias=True,
             act="gelu", residual=False, train=True),
        # a prompt of odd length through odd widths: rows on no 16 bytes, tiles that are cut
        dict(name="linear m777 1001x2503", op="linear", M=777, K=1001, N=2503, dtype="bf16", bias=True, act="gelu",
             residual=True, train=False),
        # a large down projection with its residual in a bf16 training step
        dict(name="linear m8192 4096x4096 train", op="linear", M=8192, K=4096, N=4096, dtype="bf16", bias=True, act="",
             residual=True, train=True),
        # 256 beams' next token: each reads its parent's state
        dict(name="scan step b256 c768", op="scan", B=256, L=1, C=768, dtype="fp32", h0=True, ragged=False,
             packed=False, indexed=True, train=False),
        # a layer's mixer in a training step
        dict(name="scan b8 l2048 c768 train", op="scan", B=8, L=2048, C=768, dtype="fp32", h0=False, ragged=False,
             packed=False, indexed=False, train=True),
        # padded sequences of different lengths (one of them empty) with several documents in each, odd sizes
        dict(name="scan b5 l3001 c1001 train", op="scan", B=5, L=3001, C=1001, dtype="bf16", h0=True, ragged=True,
             packed=True, indexed=False, train=True),
        # one very long sequence: few channels, a long dependent chain
        dict(name="scan b1 l131072 c256 train", op="scan", B=1, L=131072, C=256, dtype="fp32", h0=True, ragged=False,
             packed=False, indexed=False, train=True),
        # a model that a test trains: 20 tensors, all latency
        dict(name="adamw 2 x 64", op="adamw", layers=2, d=64, dh=128, vocab=256, dtype="fp32", bits=32, clip=True,
             tight=False),
        # the language model's 39 M parameters in 68 tensors
        dict(name="adamw 8 x 512", op="adamw", layers=8, d=512, dh=768, vocab=256, dtype="fp32", bits=32, clip=True,
             tight=False),
        # the same with moments in 8 bits
        dict(name="adamw 8 x 512 8 bit", op="adamw", layers=8, d=512, dh=768, vocab=256, dtype="fp32", bits=8, clip=True,
             tight=False),
        # a wider model with odd sizes and bf16 weights, no clipping
        dict(name="adamw 4 x 1801 bf16", op="adamw", layers=4, d=1801, dh=1280, vocab=50001, dtype="bf16", bits=8,
             clip=False, tight=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "scan", "scan", "step", "adamw", "adamw"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "linear":
        K, N = _log_int(rng, 32, 8192), _log_int(rng, 32, 8192)
        if rng.random() < 0.5:  # widths that are multiples of 64, as most are
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        most = (1 << 35) if dtype == "fp32" else (1 << 37)
        return dict(op="linear", M=_log_int(rng, 1, max(1, min(32768, most // (K * N)))), K=K, N=N, dtype=dtype,
                    bias=rng.random() < 0.7, act=rng.choice(["", "gelu"]), residual=rng.random() < 0.5,
                    train=rng.random() < 0.5)
    if op == "step":
        return dict(op="scan", B=_log_int(rng, 1, 1024), L=1, C=_log_int(rng, 32, 4096), dtype=dtype, h0=True,
                    ragged=False, packed=False, indexed=rng.random() < 0.5, train=False)
    if op == "scan":
        L, C = _log_int(rng, 2, 131072), _log_int(rng, 16, 4096)
        return dict(op="scan", B=_log_int(rng, 1, max(1, min(64, (1 << 25) // (L * C)))), L=L,
                    C=min(C, (1 << 25) // L), dtype=dtype, h0=rng.random() < 0.5, ragged=rng.random() < 0.4,
                    packed=rng.random() < 0.4, indexed=False, train=rng.random() < 0.7)
    d, dh, vocab = _log_int(rng, 16, 1024), _log_int(rng, 16, 1024), _log_int(rng, 64, 32768)
    bits = rng.choice([32, 8])
    return dict(op="adamw", layers=_log_int(rng, 1, 8), d=d, dh=dh, vocab=vocab, dtype=dtype, bits=bits,
                clip=rng.random() < 0.7, tight=bits == 32 and rng.random() < 0.3)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def package():
    """The package's folder is on the path of a program that uses it."""
    import pathlib
    import sys
    p = str(pathlib.Path(__file__).resolve().parents[1] / "atomic-ops_b200")
    if p not in sys.path:
        sys.path.insert(0, p)


def _shapes(case):
    """The parameters of a model of the framework's layers: (shape, whether weight decay applies)."""
    d, dh = case["d"], case["dh"]
    layer = [((d, 6 * dh), True), ((6 * dh,), False), ((dh, d), True), ((d,), False), ((d, 4 * d), True),
             ((4 * d,), False), ((4 * d, d), True), ((d,), False)]
    return [((case["vocab"], d), False)] + layer * case["layers"] + [((d, case["vocab"]), True), ((case["vocab"],), False)]


def _places(case):
    """Where each parameter starts in the model's flat buffers, and how long these are."""
    at, places = 0, []
    for shape, _ in _shapes(case):
        places.append(at)
        n = math.prod(shape)
        at += n if case["tight"] else -(-n // BLOCK) * BLOCK
    return places, at


# Moments in 8 bits: blocks of 256 values share a scale.  The first moment is e4m3 of m / scale with scale max |m| / 448,
# the root r of the second an unsigned number with four bits of exponent and four of mantissa, of r / scale with scale
# max r / 1.9375: c * 2^-18 below 16 and (16 + c % 16) * 2^(c / 16 - 19) from there on; a root above zero is at least
# code 1.  A scale below the smallest normal number stores zeros (and that code 1).
def _decode_m(codes, scale):
    return (codes.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _decode_v(codes, scale):
    c = torch.arange(256, device=codes.device)
    values = torch.where(c < 16, c.double(), (16 + c % 16) * torch.exp2((torch.div(c, 16, rounding_mode="floor") - 1).double()))
    r = (values * 2.0 ** -18).float()[codes.int()].view(-1, BLOCK) * scale[:, None]
    return (r * r).view(-1)


def _scaled(x, largest):
    """x over its blocks' scales, within +-largest, and the scales."""
    b = x.view(-1, BLOCK)
    scale = b.abs().amax(1) * (1.0 / largest)
    up = torch.where(scale >= 2.0 ** -126, torch.reciprocal(scale), 0.0)
    return torch.clamp(b * up[:, None], -largest, largest), scale


def _encode_m(m):
    x, scale = _scaled(m, 448.0)
    return x.to(torch.float8_e4m3fn).view(torch.uint8).view(-1), scale


def _encode_v(v):
    r = torch.sqrt(v)
    x, scale = _scaled(r, 1.9375)
    # to nearest, ties to even: below 2^-14 in steps of 2^-18, from there on in 16 steps per power of two
    x = x.double()
    e = torch.floor(torch.log2(x)).clamp(min=-14.0)
    code = (e + 14) * 16 + torch.round(x * torch.exp2(4 - e))
    code = torch.where((r.view(-1, BLOCK) > 0) & (code < 1), 1.0, code)
    return code.to(torch.uint8).view(-1), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    dt = _dtype(case)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = normal(M, K).to(dt)
        s["w"] = (normal(K, N) / math.sqrt(K)).to(dt)
        s["b"] = (normal(N) * 0.1).to(dt) if case["bias"] else None
        s["r"] = normal(M, N).to(dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = normal(M, N).to(dt)
        if own:
            package()
            s["leaves"] = [s[n].requires_grad_(case["train"]) for n in "xwbr" if s[n] is not None]
    elif case["op"] == "scan":
        B, L, C = case["B"], case["L"], case["C"]
        s["x"] = normal(B, L, C).to(dt)
        # gates of channels that remember between a few and some thousand tokens
        s["g"] = -torch.exp(normal(B, L, C) * 0.5 - 6.0 * torch.rand(C, generator=gen, device=dev)).to(dt)
        s["h"] = normal(B, C) if case["h0"] else None
        s["lengths"] = s["reset"] = s["index"] = None
        if case["ragged"]:
            n = torch.randint(0, L + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            n[0] = L
            if B > 1:
                n[1] = 0
            s["lengths"] = n
        if case["packed"]:  # documents of about 500 tokens one after the other
            s["reset"] = torch.rand(B, L, generator=gen, device=dev) < 0.002
        if case["indexed"]:
            s["index"] = torch.randint(0, B, (B,), generator=gen, device=dev, dtype=torch.int32)
        if case["train"]:
            s["dy"] = normal(B, L, C).to(dt)
            s["dh"] = normal(B, C)
        if own:
            package()
            s["leaves"] = [s[n].requires_grad_(case["train"]) for n in "xgh" if s[n] is not None]
    else:
        places, total = _places(case)
        p, g, m, v = normal(total) * 0.02, normal(total) * 1e-3, normal(total) * 3e-4, normal(total)
        v = v * v * 1e-6 + 1e-12
        live = torch.zeros(total, dtype=torch.bool, device=dev)
        for at, (shape, _) in zip(places, _shapes(case)):
            live[at:at + math.prod(shape)] = True
        p, g, m, v = (torch.where(live, t, 0.0) for t in (p, g, m, v))
        s["p"], s["g"] = p.to(dt), g.to(dt)
        if case["bits"] == 8:
            s["m"], s["ms"] = _encode_m(m)
            s["v"], s["vs"] = _encode_v(v)
        else:
            s["m"], s["v"] = m, v
        s["step"] = torch.full((), 1000.0, device=dev)
        s["decay"] = torch.tensor([DECAY * float(w) for _, w in _shapes(case)], device=dev, dtype=torch.float64)
        s["sizes"] = torch.tensor([b - a for a, b in zip(places, places[1:] + [total])], device=dev)
        if own:
            _optimizer(s, case, places)
    return s


def _optimizer(s, case, places):
    package()
    from atomic_gdn2.training import AdamW
    params, groups = [], ([], [])
    for at, (shape, decays) in zip(places, _shapes(case)):
        p = torch.nn.Parameter(s["p"][at:at + math.prod(shape)].view(shape))
        p.grad = s["g"][at:at + math.prod(shape)].view(shape)
        params.append(p)
        groups[0 if decays else 1].append(p)
    s["opt"] = AdamW([dict(params=groups[0], weight_decay=DECAY), dict(params=groups[1], weight_decay=0.0)], lr=LR,
                     betas=BETAS, eps=EPS, clip=CLIP if case["clip"] else None, state_bits=case["bits"])
    if case["bits"] == 8:
        s["m32"], s["v32"] = torch.zeros(s["m"].numel(), device="cuda"), torch.zeros(s["m"].numel(), device="cuda")
        s["moments"] = []
    for at, p in zip(places, params):
        n, shape = p.numel(), p.shape
        st = s["opt"].state[p]
        st["step"] = s["step"].clone()
        st["exp_avg"], st["exp_avg_sq"] = s["m"][at:at + n].view(shape), s["v"][at:at + n].view(shape)
        if case["bits"] == 8:
            blocks = slice(at // BLOCK, at // BLOCK + -(-n // BLOCK))
            st["exp_avg_scale"], st["exp_avg_sq_scale"] = s["ms"][blocks], s["vs"][blocks]
            s["moments"].append((s["m32"][at:at + n].view(shape), s["v32"][at:at + n].view(shape)))
    s["params"] = params


def _gelu(z):
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _gelu_slope(z):
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _gelu(z) if s["act"] == "gelu" else z
    if s["r"] is not None:
        y = y + s["r"].float()
    out = dict(y=y.to(dt))
    if s["train"]:
        dz = s["dy"].float()
        if s["act"] == "gelu":
            dz = dz * _gelu_slope(z)
        out["dx"], out["dw"] = (dz @ w.t()).to(dt), (x.t() @ dz).to(dt)
        if s["b"] is not None:
            out["db"] = dz.sum(0, dtype=torch.float64).to(dt)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 1 from zero, by doubling."""
    d, L = 1, x.shape[1]
    while d < L:
        x = torch.cat((x[:, :d], a[:, d:] * x[:, :-d] + x[:, d:]), 1)
        a = torch.cat((a[:, :d], a[:, d:] * a[:, :-d]), 1)
        d *= 2
    return x


def _plain_scan(s):
    x, a = s["x"].float(), torch.exp(torch.clamp(s["g"].float(), max=0.0))
    dt, (B, L, C) = s["x"].dtype, x.shape
    h0 = torch.zeros(B, C, device=x.device) if s["h"] is None else s["h"]
    if s["index"] is not None:
        h0 = h0[s["index"].long()]
    live = None
    keep = a
    if s["lengths"] is not None:
        live = (torch.arange(L, device=x.device)[None] < s["lengths"][:, None])[..., None]
        x, keep = torch.where(live, x, 0.0), torch.where(live, keep, 1.0)
    if s["reset"] is not None:
        starts = s["reset"][..., None] if live is None else s["reset"][..., None] & live
        keep = torch.where(starts, 0.0, keep)
    first = torch.cat((keep[:, :1] * h0[:, None] + x[:, :1], x[:, 1:]), 1)
    h = _scan(keep, first)
    out = dict(h=(h if live is None else torch.where(live, h, 0.0)).to(dt), last=h[:, -1])
    if s["train"]:
        dy = s["dy"].float()
        if live is not None:
            dy = torch.where(live, dy, 0.0)
        dy = torch.cat((dy[:, :-1], dy[:, -1:] + s["dh"][:, None]), 1)
        back = torch.cat((keep[:, 1:], torch.zeros_like(keep[:, :1])), 1)
        d = _scan(back.flip(1), dy.flip(1)).flip(1)
        before = torch.cat((h0[:, None], h[:, :-1]), 1)
        dx, dg = d, d * keep * before
        if live is not None:
            dx, dg = torch.where(live, dx, 0.0), torch.where(live, dg, 0.0)
        out["dx"], out["dg"] = dx.to(dt), dg.to(dt)
        if s["h"] is not None:
            out["dh0"] = keep[:, 0] * d[:, 0]
    return out


def _plain_adamw(s):
    """One rounding to 32 bits for each operation: the codes of 8-bit moments depend on every bit."""
    b1, b2 = BETAS
    g = s["g"].float()
    if s["clip"]:
        n = torch.sqrt((g.double() * g.double()).sum()).float()
        g = g * (CLIP / torch.clamp(n, min=CLIP))
    eight = s["bits"] == 8
    m, v = (_decode_m(s["m"], s["ms"]), _decode_v(s["v"], s["vs"])) if eight else (s["m"], s["v"])
    s["step"] += 1
    t = s["step"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    size, root = (LR / (1 - b1 ** t)).float(), torch.sqrt(1 - b2 ** t).float()
    decay = torch.repeat_interleave((1 - LR * s["decay"]).float(), s["sizes"])
    p = s["p"].float() * decay - size * (m / (torch.sqrt(v) / root + EPS))
    s["p"].copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return dict(p=s["p"], m=s["m"], v=s["v"])
    for name, scale, (codes, new) in (("m", "ms", _encode_m(m)), ("v", "vs", _encode_v(v))):
        s[name].copy_(codes)
        s[scale].copy_(new)
    return dict(p=s["p"], m=_decode_m(s["m"], s["ms"]), v=_decode_v(s["v"], s["vs"]))


def run(s):
    if not own:
        return dict(linear=_plain_linear, scan=_plain_scan, adamw=_plain_adamw)[s["op"]](s)
    if s["op"] == "linear":
        from atomic_gdn2 import linear
        y = linear(s["x"], s["w"], s["b"], act=s["act"] or None, residual=s["r"])
        out = dict(y=y)
        if s["train"]:
            grads = torch.autograd.grad(y, s["leaves"], s["dy"])
            names = ["dx", "dw"] + ["db"] * (s["b"] is not None) + ["dr"] * (s["r"] is not None)
            out.update(zip(names, grads))
        return out
    if s["op"] == "scan":
        from atomic_gdn2 import gated_scan
        h, last = gated_scan(s["x"], s["g"], s["h"], lengths=s["lengths"], reset=s["reset"], h_index=s["index"])
        out = dict(h=h, last=last)
        if s["train"]:
            grads = torch.autograd.grad((h, last), s["leaves"], (s["dy"], s["dh"]))
            out.update(zip(["dx", "dg", "dh0"], grads))
        return out
    s["opt"].step()
    if s["bits"] == 8:
        s["opt"].moments(s["params"], out=s["moments"])
        return dict(p=s["p"], m=s["m32"], v=s["v32"])
    return dict(p=s["p"], m=s["m"], v=s["v"])


def work(case):
    el = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        b = (M * K + K * N + M * N * (1 + case["residual"]) + N * case["bias"]) * el
        if case["train"]:  # x, W and dy are read, dx, dW and db written
            b += (2 * M * K + 2 * K * N + M * N + N * case["bias"]) * el
        return dict(bytes=b, flops=2 * M * K * N * (3 if case["train"] else 1))
    if case["op"] == "scan":
        B, L, C = case["B"], case["L"], case["C"]
        n = B * L * C
        return dict(bytes=n * el * (8 if case["train"] else 3) + B * C * 4 * (1 + case["h0"]) * (2 if case["train"] else 1),
                    flops=n * (9 if case["train"] else 3))
    n = sum(math.prod(shape) for shape, _ in _shapes(case))
    b = n * (3 * el + el * case["clip"])  # p is read and written, g read, once more where its norm comes first
    b += n * 16 if case["bits"] == 32 else n * (4 + 8) + -(-n // BLOCK) * 16
    return dict(bytes=b, flops=n * 16)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["x"].detach().double(), s["w"].detach().double()
        z = torch.mm(x, w)
        if case["bias"]:
            z += s["b"].detach().double()
        slope, y = None, z
        if case["act"] == "gelu":  # z sigmoid(2 u)
            u = math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
            q = torch.sigmoid(2.0 * u)
            y = z * q
            slope = q + 2.0 * z * q * (1.0 - q) * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * z ** 2)
        out = dict(y=y + s["r"].detach().double() if case["residual"] else y)
        if case["train"]:
            dz = s["dy"].double()
            if slope is not None:
                dz = dz * slope
            out["dx"], out["dw"] = torch.mm(dz, w.T), torch.mm(x.T, dz)
            if case["bias"]:
                out["db"] = dz.sum(0)
            if case["residual"]:
                out["dr"] = s["dy"].double()
        return out
    if case["op"] == "scan":
        # token by token, one sequence's state after the other's in a (B, C) row
        x, g = s["x"].detach().double(), s["g"].detach().double()
        B, L, C = x.shape
        h = torch.zeros(B, C, dtype=torch.float64, device=x.device) if s["h"] is None else s["h"].detach().double()
        if s["index"] is not None:
            h = h.index_select(0, s["index"].long())
        on = torch.ones(B, L, 1, dtype=torch.bool, device=x.device)
        if s["lengths"] is not None:
            on = torch.arange(L, device=x.device)[None, :, None] < s["lengths"].long()[:, None, None]
        a = torch.exp(torch.minimum(g, torch.zeros_like(g)))
        if s["reset"] is not None:
            a = a.masked_fill(s["reset"][..., None], 0.0)
        a = a.masked_fill(~on, 1.0)
        x = x.masked_fill(~on, 0.0)
        hs = torch.empty(B, L + 1, C, dtype=torch.float64, device=x.device)
        hs[:, 0] = h
        for t in range(L):
            torch.addcmul(x[:, t], a[:, t], hs[:, t], out=hs[:, t + 1])
        out = dict(h=hs[:, 1:].masked_fill(~on, 0.0), last=hs[:, -1])
        if case["train"]:
            dy = s["dy"].double().masked_fill(~on, 0.0)
            d = s["dh"].double()
            ds = torch.empty_like(dy)
            for t in range(L - 1, -1, -1):
                torch.add(dy[:, t], d, out=ds[:, t])
                d = a[:, t] * ds[:, t]
            out["dx"] = ds.masked_fill(~on, 0.0)
            out["dg"] = (ds * a * hs[:, :-1]).masked_fill(~on, 0.0)
            if s["h"] is not None:
                out["dh0"] = d
        return out
    # the weights' definition in 64 bits; what 8-bit moments round to has no such value
    b1, b2 = BETAS
    g = s["g"].double()
    if case["clip"]:
        norm = float(torch.linalg.vector_norm(g))
        g = g * min(1.0, CLIP / norm)
    if case["bits"] == 8:
        m, v = _decode_m(s["m"], s["ms"]).double(), _decode_v(s["v"], s["vs"]).double()
    else:
        m, v = s["m"].double(), s["v"].double()
    t = float(s["step"]) + 1.0
    m = m + (g - m) * (1.0 - b1)
    v = v + (g * g - v) * (1.0 - b2)
    step = (m / (1.0 - math.pow(b1, t))) / ((v / (1.0 - math.pow(b2, t))).sqrt() + EPS)
    p = s["p"].detach().double()
    places, _ = _places(case)
    for at, (shape, decays) in zip(places, _shapes(case)):
        part = slice(at, at + math.prod(shape))
        p[part] -= LR * (step[part] + (DECAY * p[part] if decays else 0.0))
    return dict(p=p, m=None, v=None) if case["bits"] == 8 else dict(p=p, m=m, v=v)
