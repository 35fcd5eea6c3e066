"""AdamW over all of a model's tensors at once, on hand-written kernels.

    opt = AdamW(model.parameters(), lr=3e-4, clip=1.0, state_bits=8)
    loss.backward(); opt.step(loss=loss); opt.zero_grad()

One step is two launches, whatever the number of tensors: the gradients' global norm, then the update.

    n = |g|,  g' = g clip / max(n, clip)
    m = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

`clip` bounds the gradients' global norm (as optax.clip_by_global_norm), `spike_factor` skips steps whose norm is
not below that many times the running mean of the norms of the steps that were made (0.98 / 0.02; as the
reference's training step, training/train.py:47-53).  With either of them a step whose norm is not finite, or the one
value that its closure returns, is skipped as well, and a step whose `loss` is given and not finite always is: weights,
moments and step counts stay as they are.  Nothing of that comes to the host: grad_norm and step_made are device values.

Moments take 8 bytes a parameter, or 2 with state_bits=8: 256 values that follow one another in memory share a
scale; the first moment is e4m3, the second is held as its root with four bits of exponent and four of mantissa
(half a step is 1/32 of it), and a root above zero never becomes zero.  The update itself uses the moments before
they are rounded.  Arithmetic is fp32, the norm's squares are summed in fp64 in a fixed order: the same inputs
give the same bits.  bf16 parameters are rounded to nearest; there is no fp32 copy of them.

state_dict() has torch.optim.AdamW's keys (and the scales); with state_bits=32 either loads the other's (not amsgrad's or
maximize's).  It does not hold the norms' mean: norm_mean can be read and set.  An 8-bit state whose parameter had another
order in memory (transposed, channels last) is encoded anew when it is loaded: its scales go by the saved codes' strides, so
keep these.
A step may be captured into a CUDA graph after one that was not (the first one makes the moments); give lr as a
tensor of one fp32 value on the device where it changes between replays.
"""
from __future__ import annotations

import torch
from torch.optim import optimizer as _base

from .. import _lib

BLOCK = 256


def _order(t: torch.Tensor):
    """The dimensions by their place in t's memory, the slowest first; None where its values do not fill it."""
    dims = sorted((i for i in range(t.ndim) if t.shape[i] > 1 and t.numel()), key=lambda i: -t.stride(i))
    step = 1
    for i in reversed(dims):
        if t.stride(i) != step:
            return None
        step *= t.shape[i]
    return dims


def _flat(t: torch.Tensor) -> torch.Tensor:
    """t's values in the order of its memory, which they fill."""
    return t.as_strided((t.numel(),), (1,))


def _code_values(square: bool, dev) -> torch.Tensor:
    """What the 256 codes stand for, of the first moment or of the second one's root."""
    c = torch.arange(256, dtype=torch.int32)
    if not square:
        return c.to(torch.uint8).view(torch.float8_e4m3fn).float().to(dev)
    return (torch.where(c < 16, c, 16 + c % 16) * torch.exp2(torch.clamp(c // 16 - 1, min=0).double()) * 2.0 ** -18).float().to(dev)


def _encoded(x: torch.Tensor, values: torch.Tensor, square: bool):
    """Codes and scales of blocks (n, 256) of fp32 values, the first moment's or the second one's roots, as a step makes them."""
    top = 1.9375 if square else 448.0
    scale = x.abs().amax(1) * (1.0 / top)
    y = torch.clamp(x * torch.where(scale >= 2.0 ** -126, 1.0 / scale, 0.0)[:, None], -top, top)
    if not square:
        return y.to(torch.float8_e4m3fn).view(torch.uint8), scale
    ties = (values[:-1] + values[1:]) / 2                    # exact; a tie goes to the even code
    k = torch.searchsorted(ties, y, out_int32=True)
    k += (k % 2 == 1) & (y == ties[torch.clamp(k, max=254)])
    return torch.where((x > 0) & (k == 0), 1, k).to(torch.uint8), scale


def _recoded(codes: torch.Tensor, scale: torch.Tensor, p: torch.Tensor, square: bool):
    """8-bit codes and scales of a tensor of p's shape whose memory has another order than p's, for p's order: decoded there
    and encoded here, a part at a time."""
    values = _code_values(square, codes.device)
    new = torch.empty_like(p, dtype=torch.uint8, device=codes.device, requires_grad=False)
    n, blocks = codes.numel(), scale.numel()
    if blocks == 1:                                          # the block's values are the same
        return new.copy_(codes), scale
    wide, x = torch.empty_like(codes, dtype=torch.float32), torch.empty_like(new, dtype=torch.float32)
    part, scales = BLOCK << 14, []
    for a in range(0, n, part):
        c = _flat(codes)[a:a + part]
        _flat(wide)[a:a + part] = values[c.int()] * scale[a // BLOCK:(a + part) // BLOCK].repeat_interleave(BLOCK)[:c.numel()]
    x.copy_(wide)
    for a in range(0, n, part):
        y = _flat(x)[a:a + part]
        k, s = _encoded(torch.nn.functional.pad(y, (0, -y.numel() % BLOCK)).view(-1, BLOCK), values, square)
        _flat(new)[a:a + part] = k.view(-1)[:y.numel()]
        scales.append(s)
    return new, torch.cat(scales)


class AdamW(torch.optim.Optimizer):
    """`params`: as for torch.optim.AdamW, fp32 or bf16 tensors on one CUDA device.  Groups may differ in lr and
    weight_decay.  clip and spike_factor: None for none.  state_bits: 32 or 8."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1, *, clip=None, spike_factor=None,
                 state_bits: int = 32):
        if state_bits not in (32, 8):
            raise ValueError(f"AdamW: state_bits={state_bits} must be 32 or 8")
        self.clip, self.spike_factor, self.state_bits = clip, spike_factor, state_bits
        self._control = None
        self._check_guard()
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        self._check_group(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        self._check_group({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def __getstate__(self):
        """What copies and pickles hold besides torch's: the options and the guard's mean."""
        keep = ("clip", "spike_factor", "state_bits", "_control")
        return {**super().__getstate__(), **{k: getattr(self, k) for k in keep}}

    @staticmethod
    def _check_group(g):
        if not all(0.0 <= b < 1.0 for b in g["betas"]) or len(g["betas"]) != 2:
            raise ValueError(f"AdamW: betas={g['betas']} must be two values in [0, 1)")
        if not g["eps"] >= 0.0:
            raise ValueError(f"AdamW: eps={g['eps']} must not be negative")
        if not isinstance(g["lr"], torch.Tensor) and not g["lr"] >= 0.0:
            raise ValueError(f"AdamW: lr={g['lr']} must not be negative")
        if not g["weight_decay"] >= 0.0:
            raise ValueError(f"AdamW: weight_decay={g['weight_decay']} must not be negative")
        # options of torch's that change the step
        for name in ("amsgrad", "maximize"):
            if g.get(name):
                raise ValueError(f"AdamW: {name} is not supported")
        if g["weight_decay"] and not g.get("decoupled_weight_decay", True):
            raise ValueError("AdamW: weight decay that goes through the moments (torch.optim.Adam's) is not supported")

    def _check_guard(self):
        for name in ("clip", "spike_factor"):
            x = getattr(self, name)
            if x is not None and not x > 0.0:
                raise ValueError(f"AdamW: {name}={x} must be above zero, or None for none")

    def _ready(self, p):
        """The parameter's state, made at its first step."""
        st = self.state[p]
        if not st or self._control is None:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: make a first step outside the capture: it makes the moments")
            if not p.is_cuda:
                raise RuntimeError("AdamW: the parameters must be on a CUDA device (the step runs only on the B200 kernels)")
            if self._control is None:
                self._control = torch.zeros(5, device=p.device)
        if not st:
            eight = self.state_bits == 8
            st["step"] = torch.zeros((), device=p.device)
            for name in ("exp_avg", "exp_avg_sq"):
                st[name] = torch.zeros_like(p, dtype=torch.uint8 if eight else torch.float32, requires_grad=False)
                if eight:
                    st[name + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), device=p.device)
        return st

    def step(self, closure=None, *, loss=None):
        """One step; returns what closure returns, or None.  Parameters without a gradient are passed over."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _base._global_optimizer_pre_hooks \
                or _base._global_optimizer_post_hooks:
            return _hooked_step(self, closure, loss=loss)
        return self._step(closure, loss=loss)

    # torch wraps a step for its hooks and a profiler's mark, 10 us a call: hooks are looked for above instead
    step.hooked = True

    def _step(self, closure=None, *, loss=None):
        result = None
        if closure is not None:
            with torch.enable_grad():
                result = closure()
            if loss is None and (self.clip or self.spike_factor) and isinstance(result, torch.Tensor) and result.numel() == 1 \
                    and not result.is_complex():
                loss = next((result.detach().to(p.device) for g in self.param_groups for p in g["params"]), None)
        self._check_guard()
        first = self.param_groups[0]
        for group in self.param_groups[1:]:
            if group["betas"] != first["betas"] or group["eps"] != first["eps"]:
                raise ValueError("AdamW: betas and eps must be the same in all groups")
        args = (float(first["betas"][0]), float(first["betas"][1]), float(first["eps"]), float(self.clip or 0.0),
                float(self.spike_factor or 0.0), self.state_bits, loss)
        rc = _lib.binding().adamw_step(self.param_groups, self.state, *args, self._control)
        if rc is None:                                       # a parameter's first step
            for group in self.param_groups:
                for p in group["params"]:
                    if p.grad is not None:
                        with torch.no_grad():
                            self._ready(p)
            rc = _lib.binding().adamw_step(self.param_groups, self.state, *args, self._control)
        if rc:
            _lib.check(rc, "gdn2_adamw_step")
        return result

    def _word(self, i):
        if self._control is None:
            raise RuntimeError("AdamW: no step was made yet")
        return self._control[i].clone()

    @property
    def grad_norm(self) -> torch.Tensor:
        """The last step's global gradient norm before clipping (with clip or spike_factor)."""
        return self._word(1)

    @property
    def step_made(self) -> torch.Tensor:
        """Whether the last step was made (bool, on the device)."""
        return self._word(2) != 0

    @property
    def norm_mean(self) -> torch.Tensor:
        """The running mean of the norms that spike_factor goes by; 0 before the first step."""
        if self._control is None:
            return torch.zeros((), device=self.param_groups[0]["params"][0].device)
        return self._word(0)

    @norm_mean.setter
    def norm_mean(self, value):
        if self._control is None:
            self._control = torch.zeros(5, device=self.param_groups[0]["params"][0].device)
        self._control[0] = value

    @torch.no_grad()
    def moments(self, params=None, out=None):
        """What the moments of `params` (all that have been stepped, if None) stand for: a list of (m, v), fp32 in
        the parameters' shape and order.  `out`: such a list to write into."""
        if params is None:
            params = [p for group in self.param_groups for p in group["params"] if self.state.get(p)]
        states = [self.state[p] for p in params]
        if any(not st for st in states):
            raise ValueError("AdamW: a parameter has not been stepped")
        if out is None:
            out = [tuple(torch.empty_like(p, dtype=torch.float32, requires_grad=False) for _ in range(2)) for p in params]
        if len(out) != len(params):
            raise ValueError("AdamW: params and out have different lengths")
        if self.state_bits == 32:
            for st, (m, v) in zip(states, out):
                m.copy_(st["exp_avg"])
                v.copy_(st["exp_avg_sq"])
            return out
        cols = [[st[n] for st in states] for n in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")]
        rc = _lib.binding().adamw_moments(*cols, [m for m, _ in out], [v for _, v in out])
        if rc:
            _lib.check(rc, "gdn2_adamw_moments")
        return out

    def load_state_dict(self, state_dict):
        """torch casts a state to its parameter's type: codes, scales and steps are put back as they were saved, or as the
        hooks before a load returned them, before the hooks after it run.  What cannot be taken is refused before anything
        changes."""
        taken = {}

        def check(_, d):
            for g in d["param_groups"]:
                self._check_group(g)
            for p, st in self._saved(d):
                self._check_state(p, st)
            taken.update(d)

        last = self.register_load_state_dict_pre_hook(check)
        first = self.register_load_state_dict_post_hook(lambda _: self._put_back(taken), prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            last.remove()
            first.remove()

    def _saved(self, state_dict):
        """The parameters and their saved states that are not empty."""
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        return [(p, state_dict["state"][i]) for i, p in zip(ids, mine) if state_dict["state"].get(i)]

    def _check_state(self, p, st):
        have = "exp_avg_scale" in st or "exp_avg_sq_scale" in st or getattr(st.get("exp_avg"), "dtype", None) == torch.uint8
        if have != (self.state_bits == 8):
            raise ValueError(f"AdamW: the saved moments have {8 if have else 32} bits, this optimizer {self.state_bits}")
        step = st.get("step")
        if step is None or (isinstance(step, torch.Tensor) and step.numel() != 1):
            raise ValueError(f"AdamW: the saved state of a {tuple(p.shape)} parameter needs one step count")
        for name in ("exp_avg", "exp_avg_sq"):
            x = st.get(name)
            if not isinstance(x, torch.Tensor) or x.shape != p.shape or not (x.dtype == torch.uint8 if have else x.is_floating_point()):
                raise ValueError(f"AdamW: the saved {name} of a {tuple(p.shape)} parameter must be a tensor of its shape, "
                                 + ("uint8" if have else "floating"))
            if not have:
                continue
            scale, n = st.get(name + "_scale"), -(-p.numel() // BLOCK)
            if not isinstance(scale, torch.Tensor) or scale.numel() != n or not scale.is_floating_point():
                raise ValueError(f"AdamW: the saved {name} of a {tuple(p.shape)} parameter needs {n} scales")
            if _order(x) is None:
                raise ValueError(f"AdamW: the saved {name} does not fill its memory: in which order its scales go is not "
                                 "known")

    def _put_back(self, state_dict):
        for p, st in self._saved(state_dict):
            new, moved = self.state[p], {}
            if self.state_bits == 8:                         # a scale belongs to 256 values of memory's order
                for name in ("exp_avg", "exp_avg_sq"):
                    if _order(st[name]) != _order(torch.empty_like(p)):
                        scale = st[name + "_scale"].detach().float().flatten().to(st[name].device)
                        moved[name], moved[name + "_scale"] = _recoded(st[name].detach(), scale, p, name == "exp_avg_sq")
            for name, x in {**st, **moved}.items():
                if name in ("exp_avg", "exp_avg_sq"):
                    kind = torch.uint8 if self.state_bits == 8 else torch.float32
                    new[name] = torch.empty_like(p, dtype=kind, requires_grad=False).copy_(x)
                elif isinstance(x, torch.Tensor):
                    new[name] = x.detach().to(p.device, torch.float32).clone(memory_format=torch.contiguous_format)
            if not isinstance(st["step"], torch.Tensor):
                new["step"] = torch.tensor(float(st["step"]), device=p.device)


_hooked_step = torch.optim.Optimizer.profile_hook_step(AdamW._step)
