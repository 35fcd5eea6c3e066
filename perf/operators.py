"""What the serving operators are measured on: the recurrent GDN-2 step, the 4-bit linear product and the beam selection.

Each operator has a plain form here (elementary torch operations in 32 bits) and the framework's call; `own` says which
of the two `run` makes.  Head size 128, 6 heads, the layer widths 512 / 768 / 2048 / 4608 and the 256-entry byte
vocabulary are the language model's own; the larger sizes are generic.
"""
import math

import torch

own = False

D = 128
SCALE = D ** -0.5
CLIP = 1e4  # the operator's sanitize bound
EOS = 2


def listed():
    return [
        # one user's next token in one layer: the smallest call, all latency
        dict(name="step b1", op="recurrent", B=1, H=6, L=1, dtype="fp32", layout="blhd", ragged=False, indexed=False),
        # 32 users with 8 beams each: every beam reads its parent's state
        dict(name="step b256 beams", op="recurrent", B=256, H=6, L=1, dtype="bf16", layout="blhd", ragged=False,
             indexed=True),
        # the largest batch of single tokens: the states alone are 0.8 GB of traffic
        dict(name="step b1024", op="recurrent", B=1024, H=6, L=1, dtype="fp32", layout="bhld", ragged=False,
             indexed=False),
        # prompts of different lengths (one of them empty) in one padded batch
        dict(name="prompts b16 l777", op="recurrent", B=16, H=6, L=777, dtype="bf16", layout="blhd", ragged=True,
             indexed=False),
        # one long prompt: few heads, a long dependent chain
        dict(name="prompt b1 l4096", op="recurrent", B=1, H=6, L=4096, dtype="fp32", layout="bhld", ragged=False,
             indexed=False),
        # the layer's fused input projection for one token
        dict(name="w4 m1 512x4608", op="w4", M=1, din=512, dout=4608, group=64, dtype="fp32", bias=True, act="",
             residual=False),
        # the layer's down projection for a few beams, with its residual
        dict(name="w4 m8 2048x512", op="w4", M=8, din=2048, dout=512, group=64, dtype="fp32", bias=True, act="",
             residual=True),
        # a large square layer for a handful of users
        dict(name="w4 m4 8192x8192", op="w4", M=4, din=8192, dout=8192, group=128, dtype="bf16", bias=False, act="",
             residual=False),
        # odd sizes (a part group, no multiple of a tile) and the GELU epilogue at the largest row count
        dict(name="w4 m32 5000x12345", op="w4", M=32, din=5000, dout=12345, group=32, dtype="bf16", bias=True,
             act="gelu", residual=False),
        # the byte vocabulary of the language model
        dict(name="beam b8 k4 v256", op="beam", B=8, K=4, V=256, dtype="fp32", masked=True, started=True),
        # many users and a vocabulary of common size that is odd
        dict(name="beam b32 k8 v50001", op="beam", B=32, K=8, V=50001, dtype="bf16", masked=False, started=True),
        # one user's first step (one live beam) over a very large vocabulary
        dict(name="beam b1 k5 v262144", op="beam", B=1, K=5, V=262144, dtype="fp32", masked=True, started=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["step", "prompt", "w4", "w4", "beam", "beam"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "step":
        return dict(op="recurrent", B=_log_int(rng, 1, 1024), H=rng.randint(1, 6), L=1, dtype=dtype,
                    layout=rng.choice(["bhld", "blhd"]), ragged=False, indexed=rng.random() < 0.5)
    if op == "prompt":
        L = _log_int(rng, 2, 4096)
        return dict(op="recurrent", B=_log_int(rng, 1, max(1, min(64, 12288 // L))), H=rng.randint(1, 6), L=L,
                    dtype=dtype, layout=rng.choice(["bhld", "blhd"]), ragged=rng.random() < 0.5,
                    indexed=rng.random() < 0.25)
    if op == "w4":
        din, M = _log_int(rng, 64, 16384), _log_int(rng, 1, 32)
        return dict(op="w4", M=M, din=din, dout=_log_int(rng, 64, min(16384, 60_000_000 // din)),
                    group=rng.choice([32, 64, 128]), dtype=dtype, bias=rng.random() < 0.5,
                    act=rng.choice(["", "gelu"]), residual=rng.random() < 0.5)
    K, V = rng.randint(1, 16), _log_int(rng, 16, 262144)
    most = 25_600_000 // (2 if dtype == "bf16" else 4)
    return dict(op="beam", B=_log_int(rng, 1, max(1, min(64, most // (K * V)))), K=K, V=V, dtype=dtype,
                masked=rng.random() < 0.5, started=rng.random() < 0.8)


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    dt = _dtype(case)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "recurrent":
        B, H, L = case["B"], case["H"], case["L"]
        # the distributions of the operator's benchmark: unit q, k and w, gates near one
        six = normal(6, B, L, H, D)
        for i in (0, 1, 3):
            six[i] /= torch.sqrt((six[i] * six[i]).sum(-1, keepdim=True) + 1e-6)
        six[4] = torch.sigmoid(six[4])
        six[5] = torch.nn.functional.logsigmoid(six[5] + 3.0)
        if case["layout"] == "blhd":  # views of one (B, L, 6, H, D) projection output
            flat = six.permute(1, 2, 0, 3, 4).to(dt).contiguous()
            s["x"] = [flat[:, :, i].transpose(1, 2) for i in range(6)]
        else:
            s["x"] = [six[i].transpose(1, 2).to(dt).contiguous() for i in range(6)]
        s["h0"] = normal(B, H, D, D) * 0.1
        s["index"] = torch.randint(0, B, (B,), generator=gen, device=dev, dtype=torch.int32) if case["indexed"] else None
        s["lengths"] = None
        if case["ragged"]:
            n = torch.randint(0, L + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
            n[0] = L
            if B > 1:
                n[1] = 0
            s["lengths"] = n
        if own:
            package()
            from atomic_gdn2 import make_blr_recurrent, make_cfg
            s["fn"] = make_blr_recurrent(make_cfg(clip=CLIP), SCALE)
    elif case["op"] == "w4":
        M, din, dout = case["M"], case["din"], case["dout"]
        s["x"] = normal(M, din).to(dt)
        s["q"] = torch.randint(-8, 8, (din, dout), generator=gen, device=dev, dtype=torch.int8)
        groups = -(-din // case["group"])
        s["s"] = ((torch.rand(groups, dout, generator=gen, device=dev) + 0.5) / (4 * math.sqrt(din))).to(torch.bfloat16)
        s["bias"] = normal(dout) * 0.1 if case["bias"] else None
        s["res"] = normal(M, dout).to(dt) if case["residual"] else None
        if own:
            package()
            from atomic_gdn2 import pack_w4
            s["w"] = pack_w4(s["q"], s["s"], case["group"])
    else:
        B, K, V = case["B"], case["K"], case["V"]
        logits = normal(B, K, V) * 2.5
        if case["masked"]:  # a grammar's mask: most tokens are not allowed
            logits[torch.rand(B, K, V, generator=gen, device=dev) < 0.75] = -math.inf
        s["logits"] = logits.to(dt)
        s["finished"] = torch.zeros(B, K, dtype=torch.bool, device=dev)
        if case["started"]:
            s["scores"] = torch.sort(normal(B, K) * 2.0 - 12.0, descending=True)[0].contiguous()
            if K > 1:
                s["finished"][:, K // 2] = torch.rand(B, generator=gen, device=dev) < 0.5
        else:  # the first step: one live beam
            s["scores"] = torch.full((B, K), -math.inf, device=dev)
            s["scores"][:, 0] = 0.0
    return s


def package():
    """The package's folder is on the path of a program that uses it."""
    import pathlib
    import sys
    p = str(pathlib.Path(__file__).resolve().parents[1] / "atomic-ops_b200")
    if p not in sys.path:
        sys.path.insert(0, p)


def _plain_recurrent(s):
    q, k, v, w, b, g = (t.float() for t in s["x"])
    B, H, L, _ = q.shape
    h = s["h0"] if s["index"] is None else s["h0"][s["index"].long()]
    a, bk, wv = torch.exp(torch.clamp(g, max=0.0)), b * k, w * v
    o = torch.zeros(B, H, L, D, device=q.device)
    live = None
    if s["lengths"] is not None:
        live = torch.arange(L, device=q.device)[:, None] < s["lengths"][None, :]
    for t in range(L):
        decayed = a[:, :, t, :, None] * h
        delta = wv[:, :, t] - (bk[:, :, t, None, :] @ decayed)[:, :, 0]
        new = decayed + k[:, :, t, :, None] * delta[:, :, None, :]
        out = SCALE * (q[:, :, t, None, :] @ new)[:, :, 0]
        if live is None:
            o[:, :, t], h = out, new
        else:
            on = live[t][:, None, None]
            o[:, :, t] = torch.where(on, out, 0.0)
            h = torch.where(on[..., None], new, h)
    return _sane(o), _sane(h)


def _sane(x):
    return torch.nan_to_num(torch.clamp(x, -CLIP, CLIP), nan=0.0)


def _gelu(y):
    return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))


def _plain_w4(s):
    scales = s["s"].float().repeat_interleave(s["group"], 0)[: s["din"]]
    y = s["x"].float() @ (s["q"].float() * scales)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"] == "gelu":
        y = _gelu(y)
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["x"].dtype)


def _plain_beam(s):
    x, scores, finished = s["logits"].float(), s["scores"], s["finished"]
    B, K, V = x.shape
    ninf = torch.full((), -math.inf, device=x.device)
    m = x.amax(-1, keepdim=True)
    some = m > -math.inf
    base = torch.where(some, m, torch.zeros_like(m))
    logsum = torch.log(torch.exp(x - base).sum(-1, keepdim=True))
    # inside a beam: by logit, the lowest token first among equals
    top, token = torch.sort(x, dim=-1, descending=True, stable=True)
    R = min(K, V)
    top, token = top[..., :R], token[..., :R]
    total = scores[..., None] + ((top - base) - logsum)
    total = torch.where(some, total, ninf)
    # a finished beam goes on as it is
    done = finished[..., None]
    first = (torch.arange(R, device=x.device) == 0)[None, None]
    total = torch.where(done, torch.where(first, scores[..., None], ninf), total)
    token = torch.where(done, torch.full_like(token, EOS), token)
    # over the beams: by total, the lowest beam first among equals
    best, at = torch.sort(total.reshape(B, K * R), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    token = token.reshape(B, K * R).gather(1, at)
    row = at // R + K * torch.arange(B, device=x.device)[:, None]
    return best, row.int(), token.int(), finished.reshape(-1)[row] | (token == EOS)


def run(s):
    if s["op"] == "recurrent":
        if own:
            return s["fn"](*s["x"], s["h0"], lengths=s["lengths"], h_index=s["index"])
        return _plain_recurrent(s)
    if s["op"] == "w4":
        if own:
            from atomic_gdn2 import w4_linear
            return w4_linear(s["x"], s["w"], s["bias"], act=s["act"] or None, residual=s["res"])
        return _plain_w4(s)
    if own:
        from atomic_gdn2 import beam_select
        return beam_select(s["logits"], s["scores"], s["finished"], eos=EOS)
    return _plain_beam(s)


def work(case):
    el = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "recurrent":
        heads, L = case["B"] * case["H"], case["L"]
        n = heads * L  # token-heads that are computed: about half of them where lengths are uniform over 0..L
        if case["ragged"]:
            B = case["B"]
            n = case["H"] * (L + (max(0, B - 2) * L) // 2)
        return dict(bytes=n * 6 * D * el + heads * L * D * 4 + 2 * heads * D * D * 4, flops=n * 7 * D * D)
    if case["op"] == "w4":
        M, din, dout = case["M"], case["din"], case["dout"]
        b = din * dout / 2 + 2 * -(-din // case["group"]) * dout + M * (din + dout) * el
        b += dout * 4 * case["bias"] + M * dout * el * case["residual"]
        return dict(bytes=b, flops=2 * M * din * dout)
    n = case["B"] * case["K"]
    return dict(bytes=n * case["V"] * el + n * (4 + 1 + 4 + 4 + 4 + 1), flops=3 * n * case["V"])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "recurrent":
        # the definition token by token in 64 bits, the state held transposed (value rows, key columns)
        q, k, v, w, b, g = (t.double() for t in s["x"])
        B, H, L, _ = q.shape
        h = s["h0"].double()
        if s["index"] is not None:
            h = h.index_select(0, s["index"].long())
        st = h.transpose(2, 3).contiguous()
        n = s["lengths"].long() if s["lengths"] is not None else torch.full((B,), L, device=q.device)
        o = torch.zeros_like(q)
        for t in range(L):
            on = (n > t).double()[:, None, None]
            keep = torch.exp(torch.minimum(g[:, :, t], torch.zeros_like(g[:, :, t])) * on)
            st = st * keep[:, :, None, :]
            erased = torch.einsum("bhvk,bhk->bhv", st, b[:, :, t] * k[:, :, t])
            st = st + torch.einsum("bhv,bhk->bhvk", (w[:, :, t] * v[:, :, t] - erased) * on, k[:, :, t])
            o[:, :, t] = torch.einsum("bhvk,bhk->bhv", st, q[:, :, t]) * (on / math.sqrt(D))
        return o.clamp(-CLIP, CLIP), st.transpose(2, 3).clamp(-CLIP, CLIP)
    if case["op"] == "w4":
        y = torch.zeros(case["M"], case["dout"], dtype=torch.float64, device="cuda")
        x = s["x"].double()
        G = case["group"]
        for i in range(s["s"].shape[0]):
            part = x[:, i * G:(i + 1) * G] @ s["q"][i * G:(i + 1) * G].double()
            y += part * s["s"][i].double()
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["act"] == "gelu":
            u = math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)
            y = y * torch.sigmoid(2.0 * u)
        if s["res"] is not None:
            y += s["res"].double()
        return y
    logits, scores, finished = s["logits"].double(), s["scores"].double(), s["finished"]
    B, K, V = logits.shape
    R = min(K, V)
    m = logits.max(-1)[0]
    some = ~torch.isneginf(m)
    shifted = torch.where(some[..., None], logits - torch.where(some, m, 0.0)[..., None], -math.inf)
    logp = shifted - torch.log(torch.exp(shifted).sum(-1, keepdim=True))
    total = torch.where(some[..., None], scores[..., None] + logp, -math.inf)
    order = torch.argsort(total, dim=-1, descending=True, stable=True)[..., :R]
    total = total.gather(2, order)
    total[finished] = -math.inf
    total[..., 0] = torch.where(finished, scores, total[..., 0])
    order = torch.where(finished[..., None], EOS, order)
    at = torch.argsort(total.flatten(1), dim=1, descending=True, stable=True)[:, :K]
    beam = torch.div(at, R, rounding_mode="floor")
    token = order.flatten(1).gather(1, at)
    row = beam + torch.arange(B, device=at.device)[:, None] * K
    return total.flatten(1).gather(1, at), row.int(), token.int(), finished.gather(1, beam) | (token == EOS)
