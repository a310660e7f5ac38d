"""Beam search with the decoder LM: its forward against the training step's, the search against
a plain one over the same logits, and the command.

Tolerances.  The decoder in bf16 runs the training forward's products and norms; its EFLA steps
keep the state in fp32 where the chunked forward rounds it and its operands to bf16 (2^-8 of
each of a few operands per layer), so logits agree to a few roundings of bf16 per layer and the
logits' own: 16 * 2^-8 relative in the 2-norm for two layers.  With 8-bit products each
operand's steps are 1/127 of its row's largest value, 0.3 of one on average: a relative
error of 0.29 / 127 * (largest / rms, at most 5 for these) * sqrt(2) = 1.6 % per product, five
products deep on either path of a block: 0.016 * sqrt(9), 5 %, and a third more for the
nonlinear parts."""
import itertools
import math

import numpy as np
import pytest
import torch

from helpers import announce, rel_l2

pytestmark = pytest.mark.gpu


def _model(seed, vocab=101, heads=2, scale=4.0):
    from ceo_amd.lm_step import EflaLM, LMConfig

    model = EflaLM(LMConfig(vocab=vocab, d_model=64 * heads, n_layers=2, n_heads=heads, head_dim=64,
                            mlp=256), seed=seed)
    model.master.mul_(scale)
    model.weights.copy_(model.master)
    return model


def _prompts(model, batch, seq, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, model.cfg.vocab, (batch, seq), generator=g, device="cuda",
                         dtype=torch.int32)


@pytest.mark.parametrize("int8,tol", [(False, 16 * 2.0 ** -8), (True, 0.07)])
@pytest.mark.parametrize("heads", [2, 8])
def test_decoder_follows_the_training_forward(heads, int8, tol):
    """heads 8: q, k, v are read in place from the fused rows."""
    from ceo_amd.generate import Decoder

    announce(f"decoder: {heads} heads, int8 {int8}")
    model = _model(1, heads=heads)
    tokens = _prompts(model, 3, 70, 5)
    want, _ = model.logits(tokens, train=False)
    want = want.view(3, 70, -1).float().cpu().numpy()
    dec = Decoder(model, int8)
    logits, states = dec.prefill(tokens[:, :66])
    assert rel_l2(logits, want[:, 65]) <= tol
    for t in range(66, 70):
        logits = dec.step(tokens[:, t].contiguous(), states)
        assert rel_l2(logits, want[:, t]) <= tol


def _plain_search(dec, prompts, beams, new_tokens, end_token):
    """One text at a time, beams in order of their scores, states copied."""
    out = []
    for b in range(prompts.shape[0]):
        logits, states = dec.prefill(prompts[b:b + 1])
        live = [(0.0, [], False)]
        states = [s.clone() for s in states]
        for t in range(new_tokens):
            logp = torch.log_softmax(logits.double().cpu(), 1).numpy()
            cand = []
            for k, (score, text, done) in enumerate(live):
                if done:
                    cand.append((score, k, end_token))
                    continue
                for v in range(logp.shape[1]):
                    cand.append((score + logp[k, v], k, v))
            cand.sort(key=lambda c: (-c[0], c[1], c[2]))
            cand = cand[:beams]
            live = [(s, live[k][1] + [v], live[k][2] or v == end_token) for s, k, v in cand]
            rows = torch.tensor([k for _, k, _ in cand], device="cuda")
            states = [s[rows].contiguous() for s in states]
            if t + 1 < new_tokens:
                tok = torch.tensor([v for _, _, v in cand], dtype=torch.int32, device="cuda")
                logits = dec.step(tok, states)
        out.append(live)
    return out


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("beams,end", [(1, None), (4, None), (5, 3), (16, 7)])
def test_search_against_a_plain_one(beams, end, int8):
    """The same logits (a row's bits depend on no other row), so the same texts."""
    from ceo_amd.generate import Decoder, beam_search

    announce(f"search: {beams} beams, end {end}, int8 {int8}")
    model = _model(2, scale=6.0)
    dec = Decoder(model, int8)
    prompts = _prompts(model, 3, 9, 7)
    text, scores = beam_search(dec, prompts, beams, 8, end)
    want = _plain_search(dec, prompts, beams, 8, end)
    for b in range(3):
        got = scores[b].cpu().numpy()
        assert (np.diff(got) <= 0).all()
        ref = np.array([s for s, _, _ in want[b]])
        # eight selections' fp32 scores and sums of exponentials
        assert np.abs(got - ref).max() <= 8 * (64 + abs(ref).max()) * 2.0 ** -24
        assert text[b].tolist() == [t for _, t, _ in want[b]]


@pytest.mark.parametrize("beams,end", [(1, None), (4, 7), (8, None)])
def test_search_from_a_graph(beams, end):
    """The same bits as without, from searches one after another, other work in between, and on
    another stream."""
    from ceo_amd.generate import GRAPH_TOKENS, Decoder, beam_search

    model = _model(6, scale=6.0)
    dec = Decoder(model)
    n = GRAPH_TOKENS + 9
    side = torch.cuda.Stream()
    for seed in (1, 2):
        prompts = _prompts(model, 3, 9, seed)
        want = beam_search(dec, prompts, beams, n, end, graph=False)
        got = beam_search(dec, prompts, beams, n, end)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = beam_search(dec, prompts, beams, n, end)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.isfinite(got[1]).all()


def test_search_finds_the_best_of_all():
    """As many beams as there are prefixes: the search is exhaustive."""
    from ceo_amd.generate import Decoder, beam_search

    model = _model(3, vocab=6, scale=6.0)
    dec = Decoder(model, int8=False)
    prompts = _prompts(model, 1, 5, 1)
    text, scores = beam_search(dec, prompts, 36, 3)
    best = []
    for seq in itertools.product(range(6), repeat=2):
        logits, states = dec.prefill(prompts)
        score = 0.0
        for v in seq:
            score += torch.log_softmax(logits.double(), 1)[0, v].item()
            logits = dec.step(torch.tensor([v], dtype=torch.int32, device="cuda"), states)
        last = torch.log_softmax(logits.double(), 1)[0].tolist()
        best += [(score + x, list(seq) + [v]) for v, x in enumerate(last)]
    best.sort(key=lambda c: -c[0])
    assert text[0, :5].tolist() == [t for _, t in best[:5]]
    assert abs(scores[0, 0].item() - best[0][0]) <= 1e-4


def test_states_in_place_are_the_same_bits():
    from ceo_amd import efla

    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(6, 2, 4, 64, generator=g, device="cuda").bfloat16() for _ in range(3))
    beta = torch.rand(6, 2, 4, generator=g, device="cuda").bfloat16()
    s0 = torch.randn(6, 4, 64, 64, generator=g, device="cuda")
    o, st = efla.chunk_efla_fwd(q, k, v, beta, s0, True)
    mine = s0.clone()
    o2, st2 = efla.chunk_efla_fwd(q, k, v, beta, mine, out_state=mine)
    assert st2 is mine and torch.equal(mine, st) and torch.equal(o, o2)
    other = torch.empty_like(s0)
    o3, _ = efla.chunk_efla_fwd(q, k, v, beta, s0, out_state=other)
    assert torch.equal(other, st) and torch.equal(o, o3)
    long = [torch.cat([t] * 4, 1) for t in (q, k, v, beta)]
    with pytest.raises(ValueError):
        efla.chunk_efla_fwd(*long, mine, out_state=mine)
    with pytest.raises(ValueError):
        efla.chunk_efla_fwd(q, k, v, beta, mine, out_state=mine[:3])


def test_states_in_place_without_a_token_and_overlapping():
    from ceo_amd import efla

    q = torch.zeros(3, 0, 2, 64, device="cuda").bfloat16()
    flat = torch.randn(4 * 2 * 64 * 64, device="cuda")
    st = flat[:3 * 2 * 64 * 64].view(3, 2, 64, 64)
    was = st.clone()
    o, got = efla.chunk_efla_fwd(q, q, q, q[..., 0], st, out_state=st)
    assert got is st and o.shape == q.shape and torch.equal(st, was)
    other = flat[2 * 64 * 64:].view(3, 2, 64, 64)
    with pytest.raises(ValueError):
        efla.chunk_efla_fwd(q, q, q, q[..., 0], st, out_state=other)
    one = torch.zeros(3, 1, 2, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError):
        efla.chunk_efla_fwd(one, one, one, one[..., 0].contiguous(), st, out_state=other)


def test_prompts_are_refused_empty():
    from ceo_amd.generate import Decoder, beam_search

    model = _model(5)
    for shape in ((0, 4), (2, 0)):
        with pytest.raises(ValueError):
            beam_search(Decoder(model), torch.zeros(shape, dtype=torch.int32, device="cuda"))
    text, scores = beam_search(Decoder(model), _prompts(model, 2, 3, 1), 4, 0)
    assert text.shape == (2, 4, 0) and scores[:, 0].tolist() == [0.0, 0.0]


def test_command_counts_on():
    """The command's model: its gradients are those of the training step, tested there; here that
    it runs and that both forms of the products give finite scores."""
    from ceo_amd.generate import Decoder, beam_search, train_counting

    model = _model(4, vocab=256, scale=1.0)
    losses = train_counting(model, steps=5)
    assert all(math.isfinite(x) for x in losses)
    for int8 in (False, True):
        text, scores = beam_search(Decoder(model, int8), _prompts(model, 2, 4, 2), 3, 6, 0)
        assert text.shape == (2, 3, 6) and torch.isfinite(scores).all()
    with pytest.raises(ValueError):
        Decoder(model).prefill(torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
