"""Training the decoder LM of lm_step on rewards and on preferences.

The reference trains on next tokens only (``Trainer.run``,
src/runtime/trainer.zig:152-185); these steps keep its order -- forward, backward,
update -- with other losses on the same logits: the clipped policy loss with a KL term
against a frozen model, and the preference loss over pairs of sequences.  Both write their
gradient over the logits, and the update clips the gradients' norm without a round
trip to the host.

``python -m ceo_amd.post_train`` trains a small model both ways and prints what it learns.
"""
from __future__ import annotations

import torch

from . import nn
from .lm_step import EflaLM, LMConfig


def logprobs(model: EflaLM, tokens: torch.Tensor, targets: torch.Tensor,
             weights=None) -> torch.Tensor:
    """log p(targets) under the model, fp32 (B * T,), nothing kept for a backward pass: the
    sampling policy's or the frozen model's side of the losses.  Positions whose weight is
    0 are not scored and give 0."""
    logits, _ = model.logits(tokens, train=False)
    return nn.token_logprob_forward(logits, targets.reshape(-1), weights)


def policy_step(model: EflaLM, tokens, targets, advantages, old_logp=None, ref_logp=None,
                weights=None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, max_norm: float = 1.0):
    """One step of the clipped policy loss.  tokens, targets: (B, T) int32; the rest per
    position, fp32 (B * T,), as ``nn.policy_loss_forward_backward`` takes them.  Returns
    (loss, log-probabilities, KL or None, gradient norm), device values."""
    logits, saved = model.logits(tokens)
    loss, logp, kl, saved["dlogits"] = nn.policy_loss_forward_backward(
        logits, targets.reshape(-1), advantages, old_logp, ref_logp, weights, clip_low,
        clip_high, kl_coef, in_place=True)
    del logits
    model.backward(saved)
    return loss.sum(), logp, kl, model.update(max_norm)


def preference_step(model: EflaLM, tokens, targets, ref_logp, weights=None, beta: float = 0.1,
                    label_smoothing: float = 0.0, max_norm: float = 1.0):
    """One step of the preference loss.  tokens, targets: (2 pairs, T) int32, chosen and
    rejected in turn; ``weights`` (fp32, per position) leaves prompts and padding out.  Returns
    (loss, rewards (2 pairs,), gradient norm), device values."""
    B, T = tokens.shape
    cu = torch.arange(0, (B + 1) * T, T, dtype=torch.int32, device=tokens.device)
    logits, saved = model.logits(tokens)
    loss, rewards, _, saved["dlogits"] = nn.preference_loss_forward_backward(
        logits, targets.reshape(-1), cu, ref_logp, weights, beta, label_smoothing, in_place=True)
    del logits
    model.backward(saved)
    return loss.sum(), rewards, model.update(max_norm)


def _batch(cfg: LMConfig, batch: int, seq: int, g):
    return torch.randint(0, cfg.vocab, (batch, seq), generator=g, device="cuda",
                         dtype=torch.int32)


def train_policy(model: EflaLM, steps: int = 20, batch: int = 8, seq: int = 128, seed: int = 0,
                 kl_coef: float = 0.01):
    """Each position's prompt is the text before it, its action the token the model samples
    there, and the reward 1 for a token of the vocabulary's lower half.  Two updates for
    each sampling.  Returns the mean reward of each sampling."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    frozen = EflaLM(model.cfg)
    frozen.weights.copy_(model.weights)
    rewards = []
    for _ in range(steps):
        tokens = _batch(model.cfg, batch, seq, g)
        logits, _ = model.logits(tokens, train=False)
        p = torch.softmax(logits.float(), 1)
        actions = torch.multinomial(p, 1, generator=g)[:, 0].int()
        old = nn.token_logprob_forward(logits, actions)
        ref = logprobs(frozen, tokens, actions)
        reward = (actions < model.cfg.vocab // 2).float()
        rewards.append(reward.mean())
        for _ in range(2):
            policy_step(model, tokens, actions, reward - reward.mean(), old, ref,
                        kl_coef=kl_coef)
    return torch.stack(rewards).tolist()


def train_preference(model: EflaLM, steps: int = 20, pairs: int = 4, seq: int = 128,
                     seed: int = 0):
    """Pairs that share their first half (the prompt, without weight) and differ in the
    second: the chosen one counts up, the rejected one is random.  Returns the mean margin
    of the rewards at each step."""
    cfg = model.cfg
    g = torch.Generator(device="cuda").manual_seed(seed)
    frozen = EflaLM(cfg)
    frozen.weights.copy_(model.weights)
    weights = torch.zeros(2 * pairs, seq, device="cuda")
    weights[:, seq // 2:] = 1.0
    weights = weights.reshape(-1)
    margins = []
    for _ in range(steps):
        text = _batch(cfg, 2 * pairs, seq + 1, g)
        text[0::2, :seq // 2 + 1] = text[1::2, :seq // 2 + 1]
        up = torch.arange(1, seq - seq // 2 + 1, device="cuda", dtype=torch.int32)
        text[0::2, seq // 2 + 1:] = (text[0::2, seq // 2, None] + up) % cfg.vocab
        tokens, targets = text[:, :-1].contiguous(), text[:, 1:].contiguous()
        ref = logprobs(frozen, tokens, targets, weights)
        _, rewards, _ = preference_step(model, tokens, targets, ref, weights)
        margins.append((rewards[0::2] - rewards[1::2]).mean())
    return torch.stack(margins).tolist()


def main() -> None:
    cfg = LMConfig(vocab=256, d_model=128, n_layers=2, n_heads=2, head_dim=64, mlp=512, lr=3e-3)
    r = train_policy(EflaLM(cfg, seed=1))
    print("policy: mean reward", " ".join(f"{x:.2f}" for x in r), flush=True)
    m = train_preference(EflaLM(cfg, seed=1))
    print("preference: mean margin", " ".join(f"{x:.2f}" for x in m), flush=True)


if __name__ == "__main__":
    main()
