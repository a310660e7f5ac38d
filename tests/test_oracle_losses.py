"""Pins for the oracle's policy and preference losses and gradient clipping (CPU
only): torch fp64 autograd of the losses written with torch's own functions, central
differences, closed forms and torch's clip_grad_norm_."""
import numpy as np
import pytest
import torch


def _inputs(seed, N, V):
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((N, V)) * 2
    t = rng.integers(0, V, N).astype(np.int32)
    lp = torch.log_softmax(torch.from_numpy(z), 1).numpy()[np.arange(N), t]
    w = np.where(rng.random(N) < 0.3, 0.0, rng.random(N) + 0.2)
    return dict(z=z, t=t, w=w, old=lp + 0.3 * rng.standard_normal(N),
                ref=lp + 0.5 * rng.standard_normal(N), adv=rng.standard_normal(N))


def _torch_policy(x, z, lo, hi, kl_coef):
    lp = torch.log_softmax(z, 1).gather(1, torch.from_numpy(x["t"]).long()[:, None])[:, 0]
    r = torch.exp(lp - torch.from_numpy(x["old"]))
    a = torch.from_numpy(x["adv"])
    k = torch.from_numpy(x["ref"]) - lp
    kl = torch.exp(k) - k - 1
    pg = -torch.minimum(r * a, torch.clamp(r, 1 - lo, 1 + hi) * a)
    return torch.from_numpy(x["w"]) * (pg + kl_coef * kl), kl


def _torch_preference(x, z, cu, beta, eps):
    lp = torch.log_softmax(z, 1).gather(1, torch.from_numpy(x["t"]).long()[:, None])[:, 0]
    term = torch.from_numpy(x["w"]) * (lp - torch.from_numpy(x["ref"]))
    r = beta * torch.stack([term[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    d = r[0::2] - r[1::2]
    ls = torch.nn.functional.logsigmoid
    return (-(1 - eps) * ls(d) - eps * ls(-d)) / len(d), r


@pytest.mark.parametrize("N,V", [(40, 17), (7, 300), (1, 1)])
def test_policy_loss_against_autograd_and_differences(oracle, N, V):
    x = _inputs(N + V, N, V)
    lo, hi, kc = 0.2, 0.3, 0.07
    z = torch.from_numpy(x["z"]).requires_grad_()
    loss, kl = _torch_policy(x, z, lo, hi, kc)
    g, = torch.autograd.grad(loss.sum(), z)
    got = oracle.policy_loss(x["z"], x["t"], x["adv"], x["old"], x["ref"], x["w"], lo, hi, kc)
    on = x["w"] != 0
    # fp64: sums of V terms and a handful of roundings
    assert np.allclose(got[0], loss.detach().numpy(), rtol=1e-12, atol=1e-13)
    assert np.allclose(got[2][on], kl.detach().numpy()[on], rtol=1e-9, atol=1e-13)
    assert np.allclose(got[4], g.numpy(), rtol=1e-10, atol=1e-13)
    # both sides of the clipping occur, except where there is one row
    if N > 1:
        assert 0 < np.count_nonzero(got[3][on]) and np.any(
            np.abs(got[0] - x["w"] * kc * got[2]) > 0)
    u = np.random.default_rng(5).standard_normal((N, V))
    h = 1e-6

    def total(zz):
        return oracle.policy_loss(zz, x["t"], x["adv"], x["old"], x["ref"], x["w"], lo, hi,
                                  kc)[0].sum()
    num = (total(x["z"] + h * u) - total(x["z"] - h * u)) / (2 * h)
    # error h^2 times a third derivative, and 1e-16 / h of rounding
    assert abs(num - (got[4] * u).sum()) <= 1e-8 * (1 + np.abs(got[4]).sum())


def test_policy_loss_without_old_is_its_gradient(oracle):
    """old None: the loss is -w A, its gradient that of -w A logp."""
    x = _inputs(3, 12, 29)
    loss, _, kl, d, _ = oracle.policy_loss(x["z"], x["t"], x["adv"], weights=x["w"], clip_low=0.0,
                                           clip_high=0.0)
    assert np.allclose(loss, -x["w"] * x["adv"]) and np.allclose(d, -x["w"] * x["adv"])
    assert not kl.any()


@pytest.mark.parametrize("cu", [[0, 9, 20, 20, 31], [0, 0, 0, 13, 31], [0, 31, 31]])
def test_preference_loss_against_autograd_and_differences(oracle, cu):
    x = _inputs(8, 31, 23)
    beta, eps = 0.4, 0.1
    z = torch.from_numpy(x["z"]).requires_grad_()
    loss, r = _torch_preference(x, z, cu, beta, eps)
    g, = torch.autograd.grad(loss.sum(), z)
    got = oracle.preference_loss(x["z"], x["t"], cu, x["ref"], x["w"], beta, eps)
    assert np.allclose(got[0], loss.detach().numpy(), rtol=1e-12)
    assert np.allclose(got[1], r.detach().numpy(), rtol=1e-11, atol=1e-13)
    assert np.allclose(got[4], g.numpy(), rtol=1e-10, atol=1e-14)
    u = np.random.default_rng(6).standard_normal(x["z"].shape)
    h = 1e-6

    def total(zz):
        return oracle.preference_loss(zz, x["t"], cu, x["ref"], x["w"], beta, eps)[0].sum()
    num = (total(x["z"] + h * u) - total(x["z"] - h * u)) / (2 * h)
    assert abs(num - (got[4] * u).sum()) <= 1e-8 * (1 + np.abs(got[4]).sum())


def test_preference_loss_of_equal_rewards(oracle):
    """No evidence: log 2 per pair, and a gradient of beta / 2 per chosen token."""
    z = np.zeros((4, 5))
    t = np.zeros(4, np.int32)
    loss, r, lp, d, _ = oracle.preference_loss(z, t, [0, 2, 4], beta=0.2)
    assert np.allclose(loss, np.log(2)) and np.allclose(lp, -np.log(5))
    assert np.allclose(d, [-0.1, -0.1, 0.1, 0.1])


def test_masked_rows_and_targets(oracle):
    z = np.random.default_rng(1).standard_normal((4, 6))
    z[1] = np.nan
    z[3, 2] = -np.inf
    t = np.array([2, 99, -1, 0], np.int32)
    w = np.array([1.0, 0.0, 1.0, 1.0])
    lp = oracle.token_logprob(z, t, w)
    assert lp[1] == 0 and np.isnan(lp[2]) and np.isfinite(lp[[0, 3]]).all()
    loss, _, _, _, g = oracle.policy_loss(z, t, np.ones(4), weights=w)
    assert loss[1] == 0 and np.isnan(loss[2]) and not g[1:3].any() and g[3, 2] == 0


@pytest.mark.parametrize("max_norm", [0.5, 100.0, 0.0])
def test_clip_coef_against_torch(oracle, max_norm):
    g = torch.Generator().manual_seed(2)
    ps = [torch.zeros(s, dtype=torch.float64, requires_grad=True) for s in ((5, 7), (3,), (1, 1))]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g, dtype=torch.float64)
    before = [p.grad.numpy().copy() for p in ps]
    norm, c = oracle.clip_coef(before, max_norm)
    n = torch.nn.utils.clip_grad_norm_(ps, max_norm)
    assert abs(n.item() - norm) <= 1e-12 * norm
    for p, b in zip(ps, before):
        assert np.allclose(p.grad.numpy(), c * b, rtol=1e-12)


def test_rows_outside_of_every_sequence(oracle):
    """Their gradient is 0 and the pair's what it is alone, whatever their logits are."""
    x = _inputs(4, 12, 6)
    x["w"][:] = 1.0
    cu = [2, 5, 9]
    alone = oracle.preference_loss(x["z"][2:9], x["t"][2:9], [0, 3, 7], x["ref"][2:9])
    x["z"][0], x["z"][1, 3], x["z"][9, 0], x["z"][10] = np.nan, np.inf, np.nan, -np.inf
    for w in (None, x["w"]):
        loss, r, _, d, g = oracle.preference_loss(x["z"], x["t"], cu, x["ref"], w)
        assert np.array_equal(loss, alone[0]) and np.array_equal(r, alone[1])
        assert not d[[0, 1, 9, 10, 11]].any() and not g[[0, 1, 9, 10, 11]].any()
        assert np.array_equal(g[2:9], alone[4])


def test_nan_advantages(oracle):
    """Loss and gradient are NaN whichever side of the clipping the ratio is on."""
    x = _inputs(7, 3, 9)
    lp = oracle.token_logprob(x["z"], x["t"])
    for kc in (0.0, 0.1):
        loss, _, _, d, g = oracle.policy_loss(x["z"], x["t"], np.full(3, np.nan),
                                              lp + np.array([1.0, 0.0, -1.0]), x["ref"],
                                              np.ones(3), kl_coef=kc)
        assert np.isnan(loss).all() and np.isnan(d).all() and np.isnan(g).all()


def test_kl_of_tokens_that_cannot_occur(oracle):
    """e^x - 1 - x for x = +inf is +inf, and for x = -inf too."""
    z = np.array([[0.0, -np.inf, 1.0], [0.0, 2.0, 1.0]])
    t = np.array([1, 0], np.int32)
    ref = np.array([-2.0, -np.inf])
    for kc in (0.0, 0.1):
        loss, lp, kl, _, _ = oracle.policy_loss(z, t, np.ones(2), np.full(2, -2.0), ref, np.ones(2),
                                                kl_coef=kc)
        assert lp[0] == -np.inf and (kl == np.inf).all()
        assert (loss == np.inf).all() if kc else np.isfinite(loss).all()
