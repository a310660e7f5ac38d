"""The steps of training on rewards and preferences, on a small model: their gradients
against the next-token step's where the losses agree and against differences of the loss,
the clipped update, and that both train."""
import numpy as np
import pytest
import torch

from helpers import announce, rel_l2

pytestmark = pytest.mark.gpu


def _model(seed, vocab=256, scale=4.0):
    from ceo_amd.lm_step import EflaLM, LMConfig

    model = EflaLM(LMConfig(vocab=vocab, d_model=128, n_layers=2, n_heads=2, head_dim=64, mlp=512,
                            lr=3e-3), seed=seed)
    model.master.mul_(scale)
    model.weights.copy_(model.master)
    return model


def test_policy_gradient_is_cross_entropys():
    """With advantage 1, no clipping and weights 1 / rows the policy loss's gradient is the
    mean cross-entropy's: the parameters' gradients agree but for the roundings of dlogits
    to bf16 (2^-9 each way), carried through the same backward."""
    from ceo_amd import nn
    from ceo_amd.lm_step import synthetic_batch

    announce("post-training: policy gradient against cross-entropy's")
    model = _model(1)
    tokens, targets = synthetic_batch(model.cfg, 2, 128, seed=3)
    _, saved = model.forward(tokens, targets)
    model.backward(saved)
    want = model.grads.float().clone()
    logits, saved = model.logits(tokens)
    loss, _, _, saved["dlogits"] = nn.policy_loss_forward_backward(
        logits, targets.reshape(-1), torch.ones(256, device="cuda"), in_place=True)
    model.backward(saved)
    assert abs(loss.sum().item() + 1.0) <= 1e-5  # -mean(r A)
    assert rel_l2(model.grads, want.cpu().numpy()) <= 2 * 2.0 ** -8


def test_update_on_clipped_gradients():
    """update(max_norm) is update() on gradients scaled by the factor: exactly where that is
    a power of two, and without a bound."""
    announce("post-training: clipped update")
    for factor in (0.25, 1.0):
        res = []
        for fused in (True, False):
            model = _model(2)
            model.grads.zero_()
            model.grads[:1024] = 1.0 / 32  # norm 1
            if fused:
                # the formula's 1e-6 taken back: the factor is a power of two
                norm = model.update(max_norm=factor * (1.0 + 1e-6) if factor < 1 else 1e9)
                assert abs(norm.item() - 1.0) <= 2.0 ** -23
            else:
                model.grads.mul_(factor)
                assert model.update() is None
            res.append([t.clone() for t in (model.master, model.exp_avg, model.exp_avg_sq,
                                            model.weights)])
        for a, b in zip(*res):
            # the factor is off by its rounding, 2^-24, and by max_norm's; the step's
            # quotient m / sqrt(v) does not move
            assert rel_l2(a, b.float().cpu().numpy()) <= 2.0 ** -22


def test_preference_step_gradient_against_differences():
    """The loss along the gradient in the logits: (L(z + h u) - L(z - h u)) / 2h against
    <g, u> for the step's own logits, in 64 bits."""
    from ceo_amd import nn, post_train
    from ceo_amd.lm_step import synthetic_batch
    from oracle import preference_loss

    announce("post-training: preference gradient of the model's logits")
    model = _model(3)
    tokens, targets = synthetic_batch(model.cfg, 4, 32, seed=5)
    w = torch.ones(128, device="cuda")
    w.view(4, 32)[:, :10] = 0.0
    ref = post_train.logprobs(model, tokens, targets, w) - 0.3 * torch.rand(128, device="cuda")
    assert not ref[w == 0].add(0.3).lt(0).any()
    logits, _ = model.logits(tokens, train=False)
    z = logits.double().cpu().numpy()
    t, cu = targets.reshape(-1).cpu().numpy(), [0, 32, 64, 96, 128]
    loss, rewards, _, g = nn.preference_loss_forward_backward(
        logits, targets.reshape(-1), torch.tensor(cu, dtype=torch.int32, device="cuda"), ref, w)
    args = (t, cu, ref.cpu().numpy(), w.cpu().numpy(), 0.1, 0.0)
    rl, rr, _, _, rg = preference_loss(z, *args)
    assert np.allclose(loss.cpu().numpy(), rl, rtol=1e-5) and np.allclose(
        rewards.cpu().numpy(), rr, rtol=1e-4, atol=1e-5)
    u, h = np.random.default_rng(0).standard_normal(z.shape), 1e-5
    num = (preference_loss(z + h * u, *args)[0].sum()
           - preference_loss(z - h * u, *args)[0].sum()) / (2 * h)
    gd = g.double().cpu().numpy()
    # each element is off by its rounding to bf16
    assert abs(num - (gd * u).sum()) <= np.abs(gd * u).sum() * 2.0 ** -8 + 1e-7


def test_steps_train():
    from ceo_amd import post_train

    announce("post-training: both losses train")
    r = post_train.train_policy(_model(4, scale=1.0), steps=15)
    print("  rewards", [f"{x:.2f}" for x in r], flush=True)
    # 1024 actions a sampling: the first is a coin's mean (0.5, deviation 0.016)
    assert abs(r[0] - 0.5) <= 0.1 and r[-1] >= 0.8
    m = post_train.train_preference(_model(4, scale=1.0), steps=15)
    print("  margins", [f"{x:.2f}" for x in m], flush=True)
    assert abs(m[0]) <= 1e-2 and m[-1] >= 0.5


def test_a_copy_of_a_model_clips_its_own_gradients():
    """copy.deepcopy between two clipped updates: the copy's norm is of its own gradients."""
    import copy

    announce("post-training: a model's copy")
    model = _model(3)
    model.grads.zero_()
    model.grads[:1024] = 1.0 / 32  # norm 1
    assert abs(model.update(max_norm=0.5).item() - 1.0) <= 2.0 ** -23
    other = copy.deepcopy(model)
    assert torch.equal(other.master, model.master) and other.grads is not model.grads
    other.grads.mul_(2.0)
    assert abs(other.update(max_norm=0.5).item() - 2.0) <= 2.0 ** -22
    del model
    assert abs(other.update(max_norm=0.5).item() - 2.0) <= 2.0 ** -22
