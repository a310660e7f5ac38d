"""Generating text with the decoder LM of lm_step: beam search over its logits.

The reference trains only; its state carried between calls (src/model/efla.zig:13-86) is what
a generated token costs here, whatever the text's length: there is no cache that grows.  A
prompt goes through the chunked forward once; then a token is one EFLA step per layer,
the products in 8-bit integers (``nn.linear_int8``, the weights quantised once) or in bf16, a
selection over beams and vocabulary (``nn.beam_select``) and the reordering of the beams'
states in place (``state.reorder``), all of it replayed from a graph in longer searches.

``python -m ceo_amd.generate`` trains a small model to count and lets it go on.
"""
from __future__ import annotations

import torch

from . import efla, nn
from .lm_step import EflaLM, LMConfig
from .state import StateList, reorder


class Decoder:
    """A model's forward for generation.  With ``int8`` the products' weights are quantised when
    the decoder is made (a later update of the model does not reach it); embedding, norms,
    biases and the states keep their types.  That pays where a token comes from a graph (24 layers,
    1 x 4 beams 0.88 ms, in bf16 1.22) and for long prompts (16 of 1024 tokens 11.4 and 14.0 ms), not for
    33 to some hundred rows launched one by one (16 x 4 beams 2.7 and 2.5 ms a token)."""

    def __init__(self, model: EflaLM, int8: bool = True):
        self.model = model
        names = [f"l{i}.{w}" for i in range(model.cfg.n_layers)
                 for w in ("w_in", "w_o", "w_up", "w_down")] + ["head"]
        self.weights = {n: nn.Int8Weight(model.w(n)) for n in names} if int8 else None

    def _linear(self, x, name, bias=None, residual=None, gelu=False):
        bias = None if bias is None else self.model.w(bias)
        if self.weights is not None:
            return nn.linear_int8(x, self.weights[name], bias, residual, gelu)
        w = self.model.w(name)
        if gelu:
            return nn.gemm_gelu_forward(x, w, bias)[1]
        if residual is None:
            return nn.gemm_forward(x, w, bias)
        return nn.gemm_ex(x, w, torch.empty_like(residual), bias=bias, c=residual, beta=1.0)

    def _forward(self, tokens: torch.Tensor, states):
        """(activations (B * T, d_model), final states) of (B, T) int32 tokens.  ``states``: the
        layers' states, updated in place (up to ``efla.STEP_TOKENS`` tokens), or None: from
        zero, new ones."""
        model, cfg = self.model, self.model.cfg
        B, T = tokens.shape
        H, dh = cfg.n_heads, cfg.head_dim
        HD = H * dh
        new = []
        x = nn.embedding_forward(tokens.reshape(-1), model.w("embed"))
        for i in range(cfg.n_layers):
            L = f"l{i}."
            a = nn.layernorm_forward(x, model.w(L + "ln1.w"), model.w(L + "ln1.b"), cfg.ln_eps)
            p = self._linear(a, L + "w_in")
            q, k, v = (model._io(p[:, j * HD:(j + 1) * HD]).view(B, T, H, dh) for j in range(3))
            beta = nn.sigmoid_gate_forward(p[:, 3 * HD:]).view(B, T, H)
            if states is None:
                o, st = efla.chunk_efla_fwd(q, k, v, beta, output_final_state=True)
                new.append(st)
            else:
                o, _ = efla.chunk_efla_fwd(q, k, v, beta, initial_state=states[i],
                                           out_state=states[i])
            x = self._linear(o.view(B * T, HD), L + "w_o", residual=x)
            a = nn.layernorm_forward(x, model.w(L + "ln2.w"), model.w(L + "ln2.b"), cfg.ln_eps)
            u = self._linear(a, L + "w_up", L + "b_up", gelu=True)
            x = self._linear(u, L + "w_down", L + "b_down", residual=x)
        return x, (new if states is None else states)

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        model = self.model
        x = nn.layernorm_forward(x, model.w("lnf.w"), model.w("lnf.b"), model.cfg.ln_eps)
        return self._linear(x, "head")

    def prefill(self, tokens: torch.Tensor):
        """(logits (B, vocab) behind the last token, states) of (B, T) int32 prompts."""
        B, T = tokens.shape
        if B == 0 or T == 0:
            raise ValueError("prompts: at least one, of at least one token")
        x, states = self._forward(tokens, None)
        return self._logits(x.view(B, T, -1)[:, -1].contiguous()), states

    def step(self, tokens: torch.Tensor, states) -> torch.Tensor:
        """Logits (rows, vocab) behind one more token (rows,) of each text; its states are
        updated in place."""
        x, _ = self._forward(tokens.reshape(-1, 1), states)
        return self._logits(x)


# From this many tokens on a search captures one, whatever its rows.  The decoder LM of 24 layers, a token's launches /
# from a graph, ms: 1 x 4 beams 2.2 / 0.9, 16 x 4 2.7 / 1.55, 64 x 8 3.1 / 3.1; the capture takes 3 to 7 ms, so that 64 x 8
# beams lose by it (64 tokens 235 / 242 ms, 10 tokens 39 / 44) and ``graph=False`` is the faster call there.
GRAPH_TOKENS = 8


def beam_search(decoder: Decoder, prompts: torch.Tensor, beams: int = 4, new_tokens: int = 32,
                end_token=None, graph: bool = True):
    """(tokens (B, beams, new_tokens) int32, scores (B, beams) fp32) of (B, T) int32 prompts,
    best first: the continuations with the largest sums of log-probabilities that a search of
    ``beams`` beams finds.  A text that has reached ``end_token`` keeps its score and is
    filled up with it.

    With 8-bit products, whose launches need nothing of the library's own, a longer search
    captures a token's launches and replays them (``graph``); the results are the same bits.  All
    ``new_tokens`` are computed, also behind the last beam's end."""
    with torch.cuda.device(prompts.device):
        return _beam_search(decoder, prompts, beams, new_tokens, end_token,
                            graph and decoder.weights is not None)


def _beam_search(decoder, prompts, beams, new_tokens, end_token, graph):
    B, dev = prompts.shape[0], prompts.device
    logits, states = decoder.prefill(prompts)
    logits = logits.repeat_interleave(beams, 0)
    states = [s.repeat_interleave(beams, 0) for s in states]
    text = torch.zeros(B * beams, new_tokens, dtype=torch.int32, device=dev)
    carried = StateList(states + [text], beams)
    # every beam holds the prompt: one of them counts
    scores = torch.full((B, beams), float("-inf"), device=dev)
    scores[:, 0] = 0.0
    tokens = torch.zeros(B, beams, dtype=torch.int32, device=dev)
    finished = None if end_token is None else torch.zeros(B, beams, dtype=torch.bool, device=dev)

    def choose(logits):
        new = nn.beam_select(logits, scores, finished=finished, end_token=end_token,
                             keep_slots=True)
        reorder(carried, new[1])
        scores.copy_(new[0])
        tokens.copy_(new[2])
        if finished is not None:
            finished.copy_(new[3])

    def go_on():  # everything in place: the same launches for every token
        choose(decoder.step(tokens, states))

    replay = go_on
    for t in range(new_tokens):
        if t == 0:
            choose(logits)
        else:
            if graph and t == 2 and new_tokens - t >= GRAPH_TOKENS:  # the first ran as it is
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, capture_error_mode="thread_local"):
                    go_on()
                replay = captured.replay
            replay()
        text[:, t] = tokens.view(-1)
    if replay is not go_on:
        torch.cuda.current_stream().synchronize()  # the graph and its memory go with this call
    order = scores.argsort(dim=1, descending=True, stable=True)
    text = text.view(B, beams, new_tokens)
    return text.gather(1, order[:, :, None].expand_as(text)), scores.gather(1, order)


def train_counting(model: EflaLM, steps: int = 150, batch: int = 16, seq: int = 64, seed: int = 0):
    """Next-token training on texts that count up from a random token.  Returns the losses."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    up = torch.arange(seq + 1, device="cuda", dtype=torch.int32)
    losses = []
    for _ in range(steps):
        first = torch.randint(0, model.cfg.vocab, (batch, 1), generator=g, device="cuda",
                              dtype=torch.int32)
        text = (first + up) % model.cfg.vocab
        losses.append(model.train_step(text[:, :-1].contiguous(), text[:, 1:].contiguous()))
    return torch.stack(losses).tolist()


def main() -> None:
    cfg = LMConfig(vocab=256, d_model=128, n_layers=2, n_heads=2, head_dim=64, mlp=512, lr=3e-3)
    model = EflaLM(cfg, seed=1)
    losses = train_counting(model)
    print(f"counting: loss {losses[0]:.2f} to {losses[-1]:.2f}", flush=True)
    prompts = torch.tensor([[7, 8, 9, 10], [200, 201, 202, 203]], dtype=torch.int32, device="cuda")
    for int8 in (False, True):
        text, scores = beam_search(Decoder(model, int8), prompts, beams=4, new_tokens=12)
        print("8-bit products:" if int8 else "bf16 products:")
        for p, t, s in zip(prompts.tolist(), text[:, 0].tolist(), scores[:, 0].tolist()):
            print(" ", *p, "|", *t, f"({s:.3f})", flush=True)


if __name__ == "__main__":
    main()
