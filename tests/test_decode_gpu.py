"""Beam search with a small GDN2LM on the serving operators, against the same model (its dequantised
weights) evaluated in 64 bits on the CPU over the whole sequences.

Tolerance of the logits, before any run: a path of two layers has about 12 fp32 stages of relative error
some 2^-20 each (products of 24-bit terms, layer norms, the recurrence's 5.3e-6), on logits of order one:
12 * 1e-6 -> 2e-5 with the layer norms' amplification left as the rest; the sums of at most 6
log-probabilities: 6 times that."""
import math
import pathlib
import sys

import pytest
import torch
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent))
from atomic_gdn2 import last_status, make_cfg, quantize_w4  # noqa: E402
from atomic_gdn2.decode import BeamDecoder  # noqa: E402
from atomic_gdn2.training import GDN2LM  # noqa: E402
from oracle_blr import prologue_torch  # noqa: E402
from serving_ref import recurrent_ref  # noqa: E402

pytestmark = pytest.mark.gpu
TOL, V, H, D = 2e-5, 40, 2, 128


def _model(layers=2):
    m = GDN2LM(make_cfg(), d_model=96, n_heads=H, d_head=D, n_layers=layers, vocab=V, expansion=2, seed=3).cuda()
    gen = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for p in m.parameters():                       # weights that matter, unlike the initialisation's
            if p.ndim == 2:
                p.copy_(torch.randn(p.shape, generator=gen) / math.sqrt(p.shape[0]))
        m.embed.copy_(torch.randn(m.embed.shape, generator=gen))
    return m


def _ref_logits(m, tokens):
    """tokens (L) -> logits (L, V), 64 bits, with the weights as quantised."""
    dq = lambda w: quantize_w4(w.detach()).dequantize().double().cpu()
    bias = lambda b: b.detach().double().cpu()
    ln = lambda t: F.layer_norm(t, (t.shape[-1],), eps=1e-5)
    x = m.embed.detach().double().cpu()[tokens][None]
    L = x.shape[1]
    for lay in m.layers:
        y = ln(x) @ dq(lay.proj_w) + bias(lay.proj_b)
        xs = prologue_torch(y, H, D, m.cfg.g_max, True)
        o, _ = recurrent_ref(*xs, 1 / math.sqrt(D))
        x = x + o.transpose(1, 2).reshape(1, L, H * D) @ dq(lay.o_w) + bias(lay.o_b)
        x = x + F.gelu(ln(x) @ dq(lay.up_w) + bias(lay.up_b), approximate="tanh") @ dq(lay.down_w) + bias(lay.down_b)
    return (ln(x) @ dq(m.head_w) + bias(m.head_b))[0]


def test_prefill_and_steps_match_the_whole_sequence():
    m = _model()
    dec = BeamDecoder(m)
    gen = torch.Generator().manual_seed(1)
    toks = torch.randint(0, V, (3, 14), generator=gen)
    lengths = torch.tensor([11, 1, 4])
    logits, states = dec.prefill(toks[:, :11].cuda(), lengths.cuda())
    for i in range(3):
        n = int(lengths[i])
        ref = _ref_logits(m, toks[i, :n])
        assert float((logits[i].double().cpu() - ref[-1]).norm() / ref[-1].norm()) < TOL
    rows = torch.tensor([2, 0, 0, 1], dtype=torch.int32)
    logits, states = dec.step(torch.tensor([5, 6, 7, 8]).cuda(), states, rows.cuda())
    logits, states = dec.step(torch.tensor([9, 10, 11, 12]).cuda(), states)
    for i, r in enumerate(rows.tolist()):
        seq = torch.cat([toks[r, :int(lengths[r])], torch.tensor([5 + i, 9 + i])])
        ref = _ref_logits(m, seq)[-1]
        assert float((logits[i].double().cpu() - ref).norm() / ref.norm()) < TOL
    assert last_status() == 0


@pytest.mark.parametrize("eos", [None, 7])
def test_search_scores_are_the_models(eos):
    """A returned beam's score is the sum of the reference's log-probabilities of its tokens, the beams are
    in order and differ, and the first one is at least as good as going greedily."""
    m = _model()
    dec = BeamDecoder(m)
    prompts = torch.randint(0, V, (2, 5), generator=torch.Generator().manual_seed(2))
    lengths = torch.tensor([5, 3])
    K, steps = 3, 6
    out, scores, n = dec.search(prompts.cuda(), lengths.cuda(), beams=K, steps=steps, eos=eos)
    out, scores, n = out.cpu(), scores.cpu(), n.cpu()
    assert out.shape == (2, K, steps) and bool((scores[:, :-1] >= scores[:, 1:]).all())
    for b in range(2):
        pre = prompts[b, :int(lengths[b])]
        assert len({tuple(x) for x in out[b].tolist()}) == K
        for k in range(K):
            m_, seq = int(n[b, k]), out[b, k].long()
            lp = torch.log_softmax(_ref_logits(m, torch.cat([pre, seq[:m_]])), -1)
            want = sum(float(lp[len(pre) - 1 + i, seq[i]]) for i in range(m_))
            assert abs(float(scores[b, k]) - want) < steps * TOL * max(1.0, abs(want))
            if eos is not None:
                assert bool((seq[m_:] == eos).all()) and (m_ == steps or int(seq[m_ - 1]) == eos)
        # greedy (one beam) can only be as good or worse than the best of K here
        g_out, g_sc, _ = dec.search(prompts[b:b + 1, :int(lengths[b])].cuda(), beams=1, steps=1, eos=eos)
        assert int(g_out[0, 0, 0]) == int(torch.argmax(_ref_logits(m, pre)[-1]))
    assert last_status() == 0


def test_one_beam_goes_greedily():
    """Each token is the reference's best one, and the score the sum of their log-probabilities; the first of 32
    beams over two tokens is the best pair of all (the 32 best first tokens hold it)."""
    m = _model()
    dec = BeamDecoder(m)
    pre = torch.randint(0, V, (4,), generator=torch.Generator().manual_seed(6))
    out, scores, n = dec.search(pre[None].cuda(), beams=1, steps=5)
    seq, want = pre, 0.0
    for tok in out[0, 0].tolist():
        lp = torch.log_softmax(_ref_logits(m, seq)[-1], -1)
        assert tok == int(torch.argmax(lp))
        want += float(lp[tok])
        seq = torch.cat([seq, torch.tensor([tok])])
    assert int(n[0, 0]) == 5 and abs(float(scores[0, 0]) - want) < 5 * TOL * max(1.0, abs(want))
    out, scores, _ = dec.search(pre[None].cuda(), beams=32, steps=2)
    first = torch.log_softmax(_ref_logits(m, pre)[-1], -1)
    second = torch.stack([torch.log_softmax(_ref_logits(m, torch.cat([pre, torch.tensor([t])]))[-1], -1) for t in range(V)])
    total = (first[:, None] + second).flatten()
    assert float(first.topk(33)[0][-1]) < float(total.max())
    assert out[0, 0].tolist() == [int(total.argmax()) // V, int(total.argmax()) % V]
    assert abs(float(scores[0, 0]) - float(total.max())) < 2 * TOL * max(1.0, abs(float(total.max())))


def test_prompts_of_another_vocabulary_are_refused():
    """On the host, before anything is gathered with them; what a prompt is padded with does not matter."""
    dec = BeamDecoder(_model(1))
    toks = torch.randint(0, V, (2, 4), generator=torch.Generator().manual_seed(3)).cuda()
    lengths = torch.tensor([4, 2])
    want = dec.prefill(toks, lengths)[0]
    for bad in (V, -V - 1, 2 ** 31 - 1):
        for t in (toks, toks.cpu(), toks.int()):
            t = t.clone()
            t[1, 2] = bad
            assert torch.equal(dec.prefill(t, lengths)[0], want)
            with pytest.raises(ValueError, match="embedding"):
                dec.prefill(t)
            with pytest.raises(ValueError, match="embedding"):
                dec.search(t, torch.tensor([4, 3]))


def test_decoder_keeps_its_own_weights():
    """Training the model further changes nothing of a decoder that was made before."""
    m = _model()
    dec = BeamDecoder(m)
    toks = torch.randint(0, V, (2, 6), generator=torch.Generator().manual_seed(8)).cuda()
    want, _ = dec.prefill(toks)
    best = dec.search(toks, beams=2, steps=3, eos=1)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(-0.5).add_(0.25)
    got, _ = dec.prefill(toks)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(dec.search(toks, beams=2, steps=3, eos=1), best))


def test_decoder_refusals():
    m = _model(1)
    with pytest.raises(RuntimeError):
        BeamDecoder(GDN2LM(make_cfg(), d_model=32, n_heads=1, d_head=128, n_layers=1, blr_fn=lambda *a: None))
    dec = BeamDecoder(m)
    toks = torch.zeros(2, 4, dtype=torch.long, device="cuda")
    for bad in (lambda: dec.prefill(toks[0]), lambda: dec.prefill(toks[:, :0]),
                lambda: dec.prefill(toks, torch.tensor([0, 4])), lambda: dec.prefill(toks, torch.tensor([1, 5])),
                lambda: dec.prefill(toks, torch.tensor([1])), lambda: dec.search(toks, beams=0),
                lambda: dec.search(toks, steps=0), lambda: dec.search(toks, eos=V)):
        with pytest.raises(ValueError):
            bad()
