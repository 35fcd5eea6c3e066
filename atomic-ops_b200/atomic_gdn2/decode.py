"""Beam search with a GDN2LM: the serving operators as they are used together.

    dec = BeamDecoder(model)                         # quantises and packs the weights once
    tokens, scores, lengths = dec.search(prompts, prompt_lengths, beams=4, steps=64, eos=0)

Every product of the model runs on 4-bit weights (w4_linear; GELU and the residuals in its epilogue),
the layers' operator in its recurrent form (make_blr_recurrent: the prompts, of different lengths, in
one padded batch; then a token at a time), and each step ends in beam_select, whose rows let the next
step's operator read every beam's parent state in place.  A layer's state is 64 KB per head and
sequence whatever the length; there is no cache that grows.

The recurrent form is the exact delta rule; a model trained with wy_eps > 0 damped the corrections
inside each 128-token chunk by that factor (1e-3 by default), so logits differ by about as much.
"""
from __future__ import annotations

import math

import torch

from .beam import beam_select
from .layer import lnorm, prologue
from .recurrent import make_blr_recurrent
from .w4 import quantize_w4, w4_linear


def _own(p):
    """A parameter's values in memory of their own."""
    return p.detach().clone(memory_format=torch.contiguous_format)


class _Layer:
    def __init__(self, layer, group):
        pack = lambda w, b: (quantize_w4(w, group), _own(b).float())
        self.proj, self.o = pack(layer.proj_w, layer.proj_b), pack(layer.o_w, layer.o_b)
        self.up, self.down = pack(layer.up_w, layer.up_b), pack(layer.down_w, layer.down_b)


class BeamDecoder:
    """A GDN2LM (on a CUDA device, fp32) with its weights packed to 4 bits, `group` rows per scale.  The
    model itself is not changed and not needed afterwards: biases and embedding are copies, so a model that
    is trained further leaves the decoder as it was made."""

    def __init__(self, model, group: int = 64):
        lay = model.layers[0]
        self.n_heads, self.d_head, self.l2norm_k, self.cfg = lay.n_heads, lay.d_head, model.l2norm_k, model.cfg
        self.embed = _own(model.embed)
        if not self.embed.is_cuda:
            raise RuntimeError("BeamDecoder: the model must be on a CUDA device (the operators run only on the B200 kernels)")
        self.layers = [_Layer(x, group) for x in model.layers]
        self.head = quantize_w4(model.head_w, group), _own(model.head_b).float()
        self.blr = make_blr_recurrent(model.cfg, 1.0 / math.sqrt(self.d_head))

    def _layers(self, x, states, lengths, rows):
        """x (B, L, d) -> (x, new states)."""
        B, L, _ = x.shape
        new = []
        for i, lay in enumerate(self.layers):
            y = w4_linear(lnorm(x), *lay.proj)
            q, k, v, w, b, g = prologue(y, self.n_heads, self.d_head, self.cfg.g_max, self.l2norm_k)
            o, h = self.blr(q, k, v, w, b, g, states[i] if states else None, lengths=lengths, h_index=rows)
            new.append(h)
            x = w4_linear(o.transpose(1, 2).reshape(B, L, -1), *lay.o, residual=x)
            u = w4_linear(lnorm(x), *lay.up, act="gelu")
            x = w4_linear(u, *lay.down, residual=x)
        return x, new

    @torch.no_grad()
    def prefill(self, tokens: torch.Tensor, lengths=None):
        """Prompts (B, L) padded on the right with anything, `lengths` (B) tokens of each (1..L; None: all L).
        Returns the logits after each prompt's last token (B, vocab) and the layers' states.  Tokens that no row
        of the embedding belongs to are refused (nothing looks at them while a stream is being captured)."""
        if tokens.ndim != 2 or not tokens.numel():
            raise ValueError(f"prompts must be (B, L) and not empty; got shape {tuple(tokens.shape)}")
        B, L = tokens.shape
        if lengths is not None:
            lo, hi = torch.stack(torch.aminmax(lengths)).tolist()
            if lengths.shape != (B,) or lo < 1 or hi > L:
                raise ValueError(f"lengths must be (B,) with values in 1..{L}")
            past = torch.arange(L, device=tokens.device) >= lengths.to(tokens.device)[:, None]
            tokens = tokens.masked_fill(past, 0)
            lengths = lengths.to(self.embed.device, torch.int32)
        V = self.embed.shape[0]
        if not torch.cuda.is_current_stream_capturing():
            lo, hi = torch.stack(torch.aminmax(tokens)).tolist()
            if lo < -V or hi >= V:
                raise ValueError(f"prompts have tokens in {lo}..{hi}, the embedding {V} rows")
        x, states = self._layers(self.embed[tokens], None, lengths, None)
        last = x[:, -1] if lengths is None else x[torch.arange(B, device=x.device), lengths.long() - 1]
        return w4_linear(lnorm(last), *self.head), states

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, states, rows=None):
        """One more token (N) for each of N sequences; sequence i goes on from row rows[i] of `states` (None:
        row i).  Returns logits (N, vocab) and the new states.  Tokens have to be of the vocabulary, as those of
        beam_select are: nothing looks at them here."""
        x, states = self._layers(self.embed[tokens][:, None], states, None, rows)
        return w4_linear(lnorm(x[:, 0]), *self.head), states

    @torch.no_grad()
    def search(self, tokens: torch.Tensor, lengths=None, *, beams: int = 4, steps: int = 32, eos=None):
        """The best `beams` continuations of each prompt, best first: tokens (B, beams, steps) int32 (eos from
        a finished beam's end on), the sums of their log-probabilities (B, beams), and how many tokens each
        has (the end token counted)."""
        if beams < 1 or steps < 1:
            raise ValueError("beams and steps must be at least 1")
        logits, states = self.prefill(tokens, lengths)
        B, V = logits.shape
        scores = torch.full((B, beams), -math.inf, device=logits.device)
        scores[:, 0] = 0.0                                   # one live beam: the prompt
        logits, done, trail = logits[:, None].expand(B, beams, V), None, []
        for i in range(steps):
            scores, rows, toks, done = beam_select(logits, scores, done if eos is not None else None, eos=eos)
            trail.append((rows.view(-1), toks.view(-1)))
            if i + 1 < steps:
                # after the prompt the states have a row per prompt, then one per beam
                parent = rows.view(-1) // beams if i == 0 else rows.view(-1)
                logits, states = self.step(toks.view(-1), states, parent)
                logits = logits.view(B, beams, V)
        out = torch.empty(B * beams, steps, dtype=torch.int32, device=scores.device)
        at = torch.arange(B * beams, device=scores.device)
        for i in range(steps - 1, -1, -1):                   # from the last step back through the parents
            rows, toks = trail[i]
            out[:, i] = toks[at]
            at = rows[at].long()
        out = out.view(B, beams, steps)
        n = torch.full((B, beams), steps, dtype=torch.int32, device=out.device)
        if eos is not None:
            n = (n - (out == eos).sum(-1) + 1).clamp(max=steps).to(torch.int32)
        return out, scores, n
