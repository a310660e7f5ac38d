"""Rows at the edges of the losses on rewards and preferences: rows outside of every
sequence, and beside a NaN, advantages that are NaN, tokens that cannot occur, policies
that are nearly the reference."""
import numpy as np
import pytest
import torch

from helpers import announce
from test_losses_gpu import POLICY, U, make

pytestmark = pytest.mark.gpu


# the launch that draws rows and the three launches, for a few rows, for more, for pairs in
# groups and for logits of over 256 MiB in short and in long rows
OUTSIDE = {
    "few rows, one launch": (100, 70, torch.bfloat16, [3, 20, 50, 70, 90]),
    "three launches": (300, 70, torch.bfloat16, [5, 100, 290]),
    "rows in registers": (200, 20000, torch.float16, [1, 60, 120, 121, 180]),
    "pairs in groups": (5000, 64, torch.float32, [*range(7, 4994, 2)]),
    "short rows past the cache": (4400, 32000, torch.bfloat16, [9, 1000, 2000, 3000, 4391]),
    "long rows past the cache, one launch": (2700, 50257, torch.bfloat16,
                                             [9, 700, 1500, 2000, 2600]),
    "long rows past the cache, one pair": (2700, 50257, torch.bfloat16, [9, 1300, 2692]),
}


@pytest.mark.parametrize("weighted", [False, True], ids=["all count", "weights"])
@pytest.mark.parametrize("which", OUTSIDE)
def test_rows_outside_of_every_sequence(which, weighted):
    """Before the first offset and behind the last the gradient is 0 whatever the logits
    are, NaN, +inf and nothing but -inf among them; the pairs' bits are those that they
    have beside ordinary rows."""
    from ceo_amd import nn

    N, V, dtype, cu = OUTSIDE[which]
    cu = cu if len(cu) % 2 else cu[:-1]
    announce(f"rows outside of every sequence: {which}, weights {weighted}")
    g = torch.Generator(device="cuda").manual_seed(N)
    z = torch.empty(N, V, dtype=dtype, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    ref = torch.full((N,), -float(np.log(V)) - 2.0, device="cuda")
    w = torch.rand(N, generator=g, device="cuda") + 0.5 if weighted else None
    offsets = torch.tensor(cu, dtype=torch.int32, device="cuda")
    out = torch.ones(N, dtype=torch.bool, device="cuda")
    out[cu[0]:cu[-1]] = False
    rows = out.nonzero()[:, 0]

    def call(logits, **kw):
        return nn.preference_loss_forward_backward(logits, t, offsets, ref, w, beta=0.01, **kw)
    want = call(z)
    assert not want[3][out].any() and bool(want[3][~out].any(1).all())
    # each side has all four kinds of rows, or as many as it has rows
    z[rows[0::4], V // 2] = float("nan")
    z[rows[1::4], V - 1] = float("inf")
    z[rows[2::4]] = float("-inf")
    got = call(z)
    assert all(torch.equal(p, q) for p, q in zip(want[:2], got[:2]))
    assert torch.equal(want[2][~out], got[2][~out])
    bad = torch.cat([rows[0::4], rows[1::4], rows[2::4]])
    assert bool(got[2][bad].isnan().all())
    assert not got[3][out].any()  # a NaN counts as any
    assert torch.equal(want[3], got[3])
    place = z.clone()
    again = call(place, in_place=True)
    assert again[3] is place and torch.equal(want[3], place)


@pytest.mark.parametrize("which", OUTSIDE)
def test_rows_without_weight_in_a_pair_that_is_nan(which):
    """One row of the first pair is NaN: the pair's other rows that count are, those without
    weight have gradient 0, and the other pairs keep their bits."""
    from ceo_amd import nn

    N, V, dtype, cu = OUTSIDE[which]
    cu = cu if len(cu) % 2 else cu[:-1]
    announce(f"a pair that is NaN: {which}")
    g = torch.Generator(device="cuda").manual_seed(N + 1)
    z = torch.empty(N, V, dtype=dtype, device="cuda").normal_(0, 2, generator=g)
    t = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    w = torch.ones(N, device="cuda")
    w[cu[0] + 1:cu[2]:2] = 0.0
    offsets = torch.tensor(cu, dtype=torch.int32, device="cuda")

    def call():
        return nn.preference_loss_forward_backward(z, t, offsets, None, w, beta=0.001)
    want = call()
    z[cu[0], 0] = float("nan")
    got = call()
    assert bool(got[0][0].isnan()) and torch.equal(got[0][1:], want[0][1:])
    pair = got[3][cu[0]:cu[2]]
    assert bool(pair[0::2].isnan().all()) and not pair[1::2].any()
    assert torch.equal(got[3][cu[2]:], want[3][cu[2]:])


@pytest.mark.parametrize("kl_coef", [0.0, 0.05])
@pytest.mark.parametrize("V", [70, 5000, 140000])
def test_nan_advantages_reach_loss_and_gradient(oracle, V, kl_coef):
    """Whichever side of the clipping the ratio is on: below it, inside, above it."""
    announce(f"NaN advantages V={V} kl_coef={kl_coef}")
    from ceo_amd import nn

    N = 6
    x, d, _ = make(V + 3, N, V, torch.bfloat16, masked=0.0)
    x["w"][:] = 1.0
    lp = oracle.token_logprob(x["z"], x["t"])
    x["old"] = (lp + np.array([1.0, 1.0, 0.0, 0.0, -1.0, -1.0])).astype(np.float32)
    x["adv"][0::2] = np.nan
    x["adv"][1::2] = [-1.5, 1.5, 1.5]  # clipped, free and clipped
    for k in ("w", "old", "adv"):
        d[k].copy_(torch.from_numpy(x[k]))
    a = {**POLICY, "kl_coef": kl_coef}
    rl, _, _, rd, rg = oracle.policy_loss(x["z"], x["t"], x["adv"], x["old"], x["ref"], x["w"],
                                          **a)
    assert np.isnan(rl[0::2]).all() and np.isnan(rd[0::2]).all() and np.isnan(rg[0::2]).all()
    if kl_coef == 0:
        assert rd[1] == 0 and rd[3] != 0 and rd[5] == 0
    loss, logp, kl, grad = nn.policy_loss_forward_backward(
        d["z"], d["t"], d["adv"], d["old"], d["ref"], d["w"], **a)
    assert bool(loss[0::2].isnan().all()) and bool(grad[0::2].isnan().all())
    assert bool(loss[1::2].isfinite().all()) and bool(grad[1::2].isfinite().all())
    assert bool(logp.isfinite().all()) and bool(kl.isfinite().all())
    if kl_coef == 0:
        assert not grad[1].any() and bool(grad[3].any()) and not grad[5].any()


@pytest.mark.parametrize("V", [70, 5000, 140000])
def test_kl_of_tokens_that_cannot_occur(oracle, V):
    """A target at -inf that the reference model gives a chance: the KL estimate e^x - 1 - x
    is +inf, and so is a loss that it enters; without its factor the loss is the policy's own."""
    announce(f"KL of impossible tokens V={V}")
    from ceo_amd import nn

    N = 6
    x, d, _ = make(V + 4, N, V, torch.float32, masked=0.0)
    x["w"][:] = 0.5
    x["adv"][:] = [1.0, -1.0, 0.5, 2.0, -2.0, 1.0]
    bad = [0, 1, 4]
    x["z"][bad, x["t"][bad]] = -np.inf
    x["ref"][4] = np.float32(3e38)  # the largest there is, still finite
    x["ref"][5] = np.float32(-3e38)  # and its opposite: kl is large, not infinite
    d["z"].copy_(torch.from_numpy(x["z"]))
    for k in ("w", "adv", "ref"):
        d[k].copy_(torch.from_numpy(x[k]))
    for kl_coef in (0.0, 0.05):
        a = {**POLICY, "kl_coef": kl_coef}
        rl, rlp, rkl, _, rg = oracle.policy_loss(x["z"], x["t"], x["adv"], x["old"], x["ref"],
                                                 x["w"], **a)
        assert (rlp[bad] == -np.inf).all() and (rkl[bad] == np.inf).all()
        for need in (True, False):
            loss, logp, kl, grad = nn.policy_loss_forward_backward(
                d["z"], d["t"], d["adv"], d["old"], d["ref"], d["w"], need_grad=need, **a)
            assert bool((logp[bad] == -np.inf).all()) and bool((kl[bad] == np.inf).all())
            assert bool(kl[[2, 3, 5]].isfinite().all())
            loss = loss.cpu().numpy()
            if kl_coef:
                assert (rl[bad] == np.inf).all() and (loss[bad] == np.inf).all()
                assert np.isfinite(loss[[2, 3, 5]]).all()
            else:
                # r = 0: nothing to gain, and (1 - clip_low) |A| where A is negative; each
                # within the roundings of the border and of two products
                assert np.isfinite(rl[bad]).all()
                assert (np.abs(loss[bad] - rl[bad]) <= 4 * U * np.abs(rl[bad])).all()
                if need:
                    assert not rg[bad].any() and not grad[bad].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [1, 70, 5000, 140000])
def test_kl_of_a_policy_near_its_reference(V, dtype):
    """Only the target's logit is finite, so that logp is 0 and x = ref - logp the given
    reference's: e^x - 1 - x, about x^2 / 2, has to keep its digits.

    Tolerance: below 1/2 a sum of terms x^2 x^k / (k + 2)!, each at most a third of the one
    before: roundings of x^2, the product and the last additions, under 8 in all; above it
    e^x - 1, within two roundings of at most 4.4 times the result, and the difference's, under 10."""
    announce(f"KL near the reference V={V} {dtype}")
    from ceo_amd import nn

    mags = [1e-12, 1e-9, 1e-7, 3e-7, 1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 0.1, 0.3, 0.499, 0.501, 0.7, 1.0,
            3.0, 10.0]
    y = np.array([s * m for m in mags for s in (1, -1)] + [0.0, -40.0], dtype=np.float32)
    N = len(y)
    t = torch.from_numpy((np.arange(N) * 7919 % V).astype(np.int32)).cuda()
    z = torch.full((N, V), float("-inf"), dtype=dtype, device="cuda")
    z[torch.arange(N, device="cuda"), t.long()] = 0.5
    x = y.astype(np.float64)
    # the series to x^11 / 11!, 1e-13 of the sum at 0.3, and the formula beyond
    series, term = np.zeros(N), x * x / 2
    for k in range(3, 13):
        series, term = series + term, term * x / k
    want = np.where(np.abs(x) < 0.3, series, np.expm1(x) - x)
    _, logp, kl, _ = nn.policy_loss_forward_backward(
        z, t, torch.ones(N, device="cuda"), ref_logp=torch.from_numpy(y).cuda())
    assert not logp.any()
    off = np.abs(kl.double().cpu().numpy() - want)
    print(f"  worst {np.max(off[x != 0] / want[x != 0]) / U:.2f} roundings", flush=True)
    assert (off <= 16 * U * want).all()
