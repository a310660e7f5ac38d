"""Log-probabilities, policy loss and preference loss on the GPU against the oracle's 64
bits: every type, sizes around the 16-byte accesses and the forms for short and long
rows, strides and alignments, masks, in place, refusals of what can only be seen on the
device, streams and graphs.

Tolerances, derived: a sum of e^(z - m) over V terms is off, relatively, by one
rounding per addition in a thread (at most max(64, V / 256) additions of 8), the
joining of threads (under 64) and each exponential (|z - m| <= 64 or the term vanishes:
64 roundings of 2^-24), so REL(V) = (V / 256 + 256) 2^-24; log-probabilities add the roundings of
z_t - m and of the result.  A gradient adds its own rounding to the logits' type, half
of finfo.eps relative to the value (for fp16 also half of its smallest step)."""
import numpy as np
import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-37}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def rel(V):
    return (V / 256 + 256) * U


def make(seed, N, V, dtype, pad=0, skew=0, masked=0.3, std=2.5):
    """Logits (N, V) with row stride V + pad, `skew` elements into their storage, and the
    rest, on the host as fp64 and on the device."""
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((N, V)) * std
    store = torch.full((skew + N * (V + pad) + 64,), float("nan"), dtype=dtype)
    view = store[skew:skew + N * (V + pad)].view(N, V + pad)[:, :V]
    view.copy_(torch.from_numpy(z))
    dev = store.cuda()
    zd = dev[skew:skew + N * (V + pad)].view(N, V + pad)[:, :V]
    z = view.double().numpy().copy()
    t = rng.integers(0, V, N).astype(np.int32)
    w = (rng.random(N) + 0.1).astype(np.float32)
    w[rng.random(N) < masked] = 0.0
    from oracle import token_logprob

    lp = token_logprob(z, t)
    f = lambda a: a.astype(np.float32)  # noqa: E731
    x = dict(z=z, t=t, w=w, old=f(lp + 0.2 * rng.standard_normal(N)),
             ref=f(lp + 0.4 * rng.standard_normal(N)), adv=f(rng.standard_normal(N)))
    d = {k: torch.from_numpy(v).cuda() for k, v in x.items() if k != "z"}
    d["z"] = zd
    return x, d, dev


def logp_tol(x, lp, V):
    m = np.nanmax(np.where(np.isfinite(x["z"]), x["z"], -1e30), axis=1)
    zt = x["z"][np.arange(len(m)), x["t"]]
    return U * np.abs(lp) + U * np.abs(zt - m) + rel(V)


def within(got, ref, tol, what):
    got = got.detach().double().cpu().numpy()
    assert got.shape == ref.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what
    ok = ~np.isnan(ref)
    off = np.abs(got - ref)[ok] / np.broadcast_to(tol, ref.shape)[ok]
    worst = float(off.max()) if off.size else 0.0
    print(f"  {what}: {worst:.2f} of its tolerance", flush=True)
    assert worst <= 1.0, what


def grad_tol(ref, dlogp, dlogp_err, x, dtype, V):
    """ref the fp64 gradient; dlogp its per-row factor, off by dlogp_err."""
    m = x["z"].max(axis=1, keepdims=True)
    p = np.exp(x["z"] - m)
    p /= p.sum(axis=1, keepdims=True)
    p[np.arange(len(p)), x["t"]] += 1.0
    err = np.abs(dlogp)[:, None] * rel(V) + dlogp_err[:, None]
    return np.abs(ref) * torch.finfo(dtype).eps / 2 + TINY[dtype] + p * err * 1.01


POLICY = dict(clip_low=0.2, clip_high=0.28, kl_coef=0.05)


def check_policy(x, d, dtype, V, in_place=False, **kw):
    from ceo_amd import nn
    from oracle import policy_loss

    a = {**POLICY, **kw}
    loss, logp, kl, g = nn.policy_loss_forward_backward(
        d["z"], d["t"], d["adv"], old_logp=d["old"], ref_logp=d["ref"], weights=d["w"],
        in_place=in_place, **a)
    rl, rlp, rkl, rd, rg = policy_loss(x["z"], x["t"], x["adv"], x["old"], x["ref"], x["w"],
                                       a["clip_low"], a["clip_high"], a["kl_coef"])
    dl = logp_tol(x, rlp, V)
    on = x["w"] != 0
    with np.errstate(over="ignore"):
        r = np.where(on, np.exp(rlp - x["old"]), 0)
        e = np.where(on, np.exp(x["ref"] - rlp), 0)
    # a rounding of ratio, products and e^x - 1: 8 of them on each term
    slope = np.abs(x["adv"]) * r + a["kl_coef"] * e
    size = np.abs(x["adv"]) * np.maximum(r, 1.5) + a["kl_coef"] * (e + 1 + np.abs(x["ref"] - rlp))
    aw = np.abs(x["w"])
    within(logp, rlp, dl, "logp")
    within(kl, rkl, (e + 1) * dl + 8 * U * (e + 1 + np.abs(x["ref"] - rlp)) + 1e-30, "kl")
    within(loss, rl, aw * (slope + a["kl_coef"]) * dl + 8 * U * aw * size + 1e-30, "loss")
    de = aw * slope * dl + 8 * U * aw * size
    within(g, rg, grad_tol(rg, rd, de, x, dtype, V), "grad")
    return loss, logp, kl, g


def check_preference(x, d, cu, dtype, V, beta=0.3, eps=0.1, in_place=False):
    from ceo_amd import nn
    from oracle import preference_loss

    loss, rew, logp, g = nn.preference_loss_forward_backward(
        d["z"], d["t"], torch.tensor(cu, dtype=torch.int32, device="cuda"), ref_logp=d["ref"],
        weights=d["w"], beta=beta, label_smoothing=eps, in_place=in_place)
    rl, rr, rlp, rd, rg = preference_loss(x["z"], x["t"], cu, x["ref"], x["w"], beta, eps)
    P = len(cu) // 2
    dl = logp_tol(x, rlp, V)
    aw = np.abs(x["w"])
    dr = np.array([beta * (aw * dl)[a:b].sum() for a, b in zip(cu[:-1], cu[1:])]) + 1e-30
    dx = dr[0::2] + dr[1::2]
    within(logp, rlp, dl, "logp")
    within(rew, rr, dr + U * np.abs(rr), "rewards")
    within(loss, rl, dx / P + 2 * U * np.abs(rl), "loss")
    de = np.zeros(len(rlp))
    for i in range(P):
        de[cu[2 * i]:cu[2 * i + 2]] = beta * (0.25 * dx[i] / P)
    de = de * aw + 4 * U * np.abs(rd)
    within(g, rg, grad_tol(rg, rd, de, x, dtype, V), "grad")
    return loss, rew, logp, g


# around the 16-byte access of each type, one wave, one workgroup and the long rows
SIZES = [(3, 1), (5, 2), (4, 7), (6, 8), (5, 9), (7, 63), (9, 64), (6, 257), (5, 1000), (4, 2048),
         (5, 2053), (3, 4099), (2, 8192), (3, 16387), (7, 32000), (2, 50257), (2, 65536),
         (1, 100003), (2, 131075)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V", SIZES)
def test_token_logprob(oracle, N, V, dtype):
    from ceo_amd import nn

    announce(f"token_logprob {N} x {V} {dtype}")
    x, d, _ = make(N * V, N, V, dtype, pad=V % 3, skew=V % 5)
    ref = oracle.token_logprob(x["z"], x["t"], x["w"])
    within(nn.token_logprob_forward(d["z"], d["t"], d["w"]), ref, logp_tol(x, ref, V), "weights")
    ref = oracle.token_logprob(x["z"], x["t"])
    within(nn.token_logprob_forward(d["z"], d["t"]), ref, logp_tol(x, ref, V), "all")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V", SIZES)
def test_policy_loss(oracle, N, V, dtype):
    announce(f"policy {N} x {V} {dtype}")
    x, d, _ = make(N * V + 1, N, V, dtype, pad=(V + 1) % 3, skew=V % 7)
    check_policy(x, d, dtype, V)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("N,V", SIZES)
def test_preference_loss(oracle, N, V, dtype):
    announce(f"preference {N} x {V} {dtype}")
    x, d, _ = make(N * V + 2, N, V, dtype, pad=(V + 2) % 3, skew=V % 9)
    half = (N + 1) // 2
    check_preference(x, d, [0, half, N], dtype, V)


# more rows than compute units, and than workgroups in flight
@pytest.mark.parametrize("N,V,dtype", [(300, 2053, torch.bfloat16), (1500, 640, torch.float32),
                                       (2600, 1003, torch.float16), (700, 9000, torch.bfloat16)])
def test_many_rows(oracle, N, V, dtype):
    announce(f"many rows {N} x {V} {dtype}")
    x, d, _ = make(N, N, V, dtype)
    check_policy(x, d, dtype, V)
    cut = np.sort(np.random.default_rng(N).integers(0, N + 1, 11))
    check_preference(x, d, [0, *cut.tolist(), N], dtype, V)


@pytest.mark.parametrize("pairs,longest", [(1024, 3), (1025, 3), (2500, 2), (6001, 1)])
def test_preference_of_many_pairs(oracle, pairs, longest):
    """More pairs than workgroups: empty sequences, short ones, some of over a wave's 64 rows
    next to each other, some of exactly 64 and 65; offsets behind their predecessors."""
    from ceo_amd import nn

    announce(f"preference of {pairs} pairs")
    rng = np.random.default_rng(pairs)
    lengths = rng.integers(0, longest + 1, 2 * pairs)
    for at in (0, 40, 41, 42, pairs // 2, pairs - 1):
        lengths[2 * at:2 * at + 2] = rng.integers(20, 300, 2)
    lengths[20:24] = [64, 0, 30, 35]
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    N, V = int(cu[-1]), 37
    x, d, _ = make(pairs, N, V, torch.bfloat16)
    check_preference(x, d, cu.tolist(), torch.bfloat16, V)
    # the same offsets after clamping
    odd = cu.copy()
    back = np.flatnonzero(np.diff(cu) == 0) + 1
    odd[back] -= rng.integers(0, 50, len(back)).astype(np.int32)
    odd[-1] = N + 5
    f = lambda c, need: nn.preference_loss_forward_backward(  # noqa: E731
        d["z"], d["t"], torch.from_numpy(c).cuda(), d["ref"], d["w"], need_grad=need)
    want, got, only = f(cu, True), f(odd, True), f(odd, False)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert all(torch.equal(p, q) for p, q in zip(want[:3], only[:3]))


@pytest.mark.parametrize("lengths", [[0, 5, 3, 0], [1, 1], [0, 0, 0, 8], [2, 1, 0, 0, 3, 2]])
def test_preference_short_and_empty_sequences(oracle, lengths):
    announce(f"preference lengths {lengths}")
    cu = [0, *np.cumsum(lengths).tolist()]
    x, d, _ = make(11, cu[-1], 777, torch.bfloat16, masked=0.2)
    check_preference(x, d, cu, torch.bfloat16, 777, beta=0.7, eps=0.0)


def test_preference_without_rows_and_pairs():
    from ceo_amd import nn

    z = torch.empty(0, 50, dtype=torch.bfloat16, device="cuda")
    t = torch.empty(0, dtype=torch.int32, device="cuda")
    cu = torch.zeros(5, dtype=torch.int32, device="cuda")
    loss, rew, logp, g = nn.preference_loss_forward_backward(z, t, cu)
    assert np.allclose(loss.cpu().numpy(), np.log(2) / 2, rtol=2 * U) and not rew.any()
    assert logp.shape == (0,) and g.shape == (0, 50)
    x, d, _ = make(5, 4, 50, torch.bfloat16)
    loss, _, _, g = nn.preference_loss_forward_backward(d["z"], d["t"], cu[:1])
    assert loss.shape == (0,) and not g.any()
    p = nn.policy_loss_forward_backward(z, t, torch.empty(0, device="cuda"))
    assert p[0].shape == (0,) and p[3].shape == (0, 50)


def test_preference_offsets_are_clamped(oracle):
    """Offsets past the rows or behind their predecessors: clamped, and rows that no
    sequence holds get no gradient."""
    from ceo_amd import nn

    announce("preference: offsets clamped")
    x, d, _ = make(6, 12, 300, torch.bfloat16, masked=0.0)

    def call(cu):
        return nn.preference_loss_forward_backward(
            d["z"], d["t"], torch.tensor(cu, dtype=torch.int32, device="cuda"),
            ref_logp=d["ref"], weights=d["w"])
    a, b = call([-5, 4, 900]), call([0, 4, 12])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a, b = call([2, 7, 5]), call([2, 7, 7])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert not a[3][:2].any() and not a[3][7:].any() and a[3][2:7].any()
    a = call([3, 3, 3])
    assert abs(a[0].item() - np.log(2)) <= 2 * U and not a[3].any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [500, 32001, 131072])
def test_in_place_and_padding(oracle, V, dtype):
    """In place gives the same bits, touches no column past the vocabulary, and the
    gradient of a padded view is packed."""
    from ceo_amd import nn

    announce(f"in place V={V} {dtype}")
    N = 6
    cu = torch.tensor([0, 2, N], dtype=torch.int32, device="cuda")

    def both(f):
        for pad, skew in ((0, 0), (13, 3)):
            x, d, store = make(V + pad, N, V, dtype, pad=pad, skew=skew)
            kept = store.clone()
            want = f(d, False)
            assert want[3].is_contiguous() and torch.equal(store.nan_to_num(7.0),
                                                           kept.nan_to_num(7.0))
            got = f(d, True)
            assert got[3].data_ptr() == d["z"].data_ptr()
            for p, q in zip(want, got):
                assert torch.equal(p, q)
            outside = torch.ones_like(store, dtype=torch.bool)
            outside[skew:skew + N * (V + pad)].view(N, V + pad)[:, :V] = False
            assert bool(store[outside].isnan().all())
    both(lambda d, ip: nn.policy_loss_forward_backward(
        d["z"], d["t"], d["adv"], d["old"], d["ref"], d["w"], kl_coef=0.1, in_place=ip))
    both(lambda d, ip: nn.preference_loss_forward_backward(
        d["z"], d["t"], cu, d["ref"], d["w"], in_place=ip))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [70, 5000, 140000])
def test_masked_rows_and_special_logits(oracle, V, dtype):
    """Rows without weight hold NaN, targets out of range and infinite statistics; masked
    logits are -inf or the type's lowest value; rows with +inf, NaN or nothing but
    -inf give NaN, a row all of the lowest value is uniform."""
    announce(f"special logits V={V} {dtype}")
    N = 12
    x, d, _ = make(V, N, V, dtype, masked=0.0)
    x["w"][:] = 1.0
    x["w"][[1, 4]] = 0.0
    low = float(torch.finfo(dtype).min)
    z = x["z"]
    z[1] = np.nan
    z[2, V // 2:] = -np.inf
    z[2, x["t"][2]] = 1.0
    z[3, : V // 2] = low
    z[3, x["t"][3]] = 1.0
    z[4] = np.inf
    z[5, 3] = np.nan
    z[6, V - 1] = np.inf
    z[7] = -np.inf
    z[8] = low
    z[9, x["t"][9]] = -np.inf
    x["t"][1], x["t"][4] = -7, V + 5
    x["t"][10], x["t"][11] = V, -1
    for k in ("old", "ref", "adv"):
        x[k][[1, 4]] = np.nan
    x["old"][8] = x["ref"][8] = -np.log(V) + 0.1
    x["ref"][9] = -np.inf
    d["z"].copy_(torch.from_numpy(z))
    for k in ("t", "w", "old", "ref", "adv"):
        d[k].copy_(torch.from_numpy(x[k]))
    from ceo_amd import nn

    ref = oracle.token_logprob(z, x["t"], x["w"])
    got = nn.token_logprob_forward(d["z"], d["t"], d["w"])
    g = got.cpu().numpy()
    assert np.isnan(ref[[5, 6, 7, 10, 11]]).all() and ref[9] == -np.inf == g[9]
    assert (ref[[1, 4]] == 0).all() and np.isfinite(ref[[0, 2, 3, 8]]).all()
    ok = np.isfinite(ref)
    tol = U * np.abs(ref) + 64 * U + rel(V)
    assert np.array_equal(np.isnan(g), np.isnan(ref))
    assert (np.abs(g - ref)[ok] <= tol[ok]).all()
    loss, logp, kl, grad = nn.policy_loss_forward_backward(
        d["z"], d["t"], d["adv"], d["old"], d["ref"], d["w"], **POLICY)
    assert torch.equal(logp.nan_to_num(9.0), got.nan_to_num(9.0))
    loss, kl = loss.cpu().numpy(), kl.cpu().numpy()
    assert (loss[[1, 4]] == 0).all() and (kl[[1, 4]] == 0).all()
    assert np.isnan(loss[[5, 6, 7, 10, 11]]).all() and np.isfinite(loss[[0, 2, 3, 8]]).all()
    gr = grad.float()
    assert not gr[[1, 4, 10, 11]].any()
    assert bool(gr[[5, 6, 7]].isnan().all())
    assert bool(gr[[0, 2, 3, 8]].isfinite().all())
    # without their masked logits the gradient of a row is that of the row without them
    sel = [0, 2, 3, 8]
    xs = {k: v[sel] for k, v in x.items()}
    xs["z"] = np.maximum(xs["z"], -1e30 if dtype != torch.float16 else -65504.0)
    _, _, _, rd, rg = oracle.policy_loss(xs["z"], xs["t"], xs["adv"], xs["old"], xs["ref"],
                                         xs["w"], **POLICY)
    lp = oracle.token_logprob(xs["z"], xs["t"])
    r, e = np.exp(lp - xs["old"]), np.exp(xs["ref"] - lp)
    de = (np.abs(xs["adv"]) * r + 0.05 * e) * (rel(V) + 128 * U) + 8 * U * (np.abs(xs["adv"]) * np.maximum(r, 1.5) + 0.05 * (e + 1))
    within(grad[sel], rg, grad_tol(rg, rd, de, xs, dtype, V), "grad of masked logits")


@pytest.mark.parametrize("old", [True, False], ids=["old", "itself"])
@pytest.mark.parametrize("V", [70, 5000, 140000])
def test_nan_reaches_the_policy_loss(oracle, V, old):
    """Without a KL term to carry it: a row with NaN, +inf or nothing but -inf, and a NaN
    or infinite statistic of the sampling policy."""
    announce(f"nan in the policy loss V={V} old={old}")
    from ceo_amd import nn

    N = 10
    x, d, _ = make(V, N, V, torch.bfloat16, masked=0.0)
    x["w"][:] = 1.0
    x["adv"][:] = [1, -1, 2, -2, 1, -1, 0, 0.5, -0.5, 1]
    z = x["z"]
    z[1, V // 3] = np.nan
    z[2, V - 1] = np.inf
    z[3] = -np.inf
    z[4, 0] = np.nan
    x["old"][5] = np.nan
    x["old"][6] = -np.inf
    x["adv"][8] = np.nan
    d["z"].copy_(torch.from_numpy(z))
    for k in ("w", "old", "adv"):
        d[k].copy_(torch.from_numpy(x[k]))
    rl, rlp, _, _, rg = oracle.policy_loss(z, x["t"], x["adv"], x["old"] if old else None, None,
                                           x["w"])
    bad = [1, 2, 3, 4, 8] + ([5, 6] if old else [])
    assert sorted(np.flatnonzero(np.isnan(rl))) == sorted(bad)
    for need in (True, False):
        loss, logp, _, grad = nn.policy_loss_forward_backward(
            d["z"], d["t"], d["adv"], d["old"] if old else None, None, d["w"], need_grad=need)
        assert np.array_equal(np.isnan(loss.cpu().numpy()), np.isnan(rl))
        assert np.array_equal(np.isnan(logp.cpu().numpy()), np.isnan(rlp))
    grad = nn.policy_loss_forward_backward(d["z"], d["t"], d["adv"], d["old"] if old else None,
                                           None, d["w"])[3]
    assert np.array_equal(grad.isnan().all(1).cpu().numpy(), np.isnan(rg).all(1))
    assert np.array_equal(grad.isnan().any(1).cpu().numpy(), np.isnan(rg).any(1))


@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("N", [24, 400])
def test_preference_of_impossible_tokens(oracle, N, smoothing):
    """A target at -inf in the chosen, the rejected or both sequences: an infinite margin
    costs nothing on its right side, where no smoothing asks for the other."""
    announce(f"impossible tokens N={N} smoothing={smoothing}")
    from ceo_amd import nn

    V, P = 70, 4
    x, d, _ = make(N, N, V, torch.float32, masked=0.0)
    x["w"][:] = 1.0
    cu = np.linspace(0, N, 2 * P + 1).astype(np.int32)
    z = x["z"]
    for s in (0, 3, 4, 5):  # chosen, rejected, both; the last pair as it is
        z[cu[s], x["t"][cu[s]]] = -np.inf
    d["z"].copy_(torch.from_numpy(z))
    d["w"].copy_(torch.from_numpy(x["w"]))
    with np.errstate(invalid="ignore"):
        rl, rr, _, rd, rg = oracle.preference_loss(z, x["t"], cu, x["ref"], x["w"],
                                                   label_smoothing=smoothing)
    assert rl[0] == np.inf and np.isnan(rl[2]) and np.isfinite(rl[3])
    assert rl[1] == (0.0 if smoothing == 0 else np.inf)
    for need in (True, False):
        loss, rewards, _, grad = nn.preference_loss_forward_backward(
            d["z"], d["t"], torch.from_numpy(cu).cuda(), d["ref"], d["w"],
            label_smoothing=smoothing, need_grad=need)
        assert np.array_equal(loss[:3].cpu().numpy(), rl[:3].astype(np.float32), equal_nan=True)
        assert np.array_equal(np.isinf(rewards.cpu().numpy()), np.isinf(rr))
        if need:
            g = grad[:cu[4]].cpu().numpy().astype(np.float64)
            # an infinite margin's factor is exact, the softmax as good as its sum
            assert (np.abs(g - rg[:cu[4]]) <= np.abs(rd[:cu[4], None]) * (rel(V) + 64 * U)).all()
            assert bool(grad[cu[4]:cu[6]].isnan().any(1).all())
            assert bool(grad[cu[6]:].isfinite().all())


def test_everything_masked():
    from ceo_amd import nn

    x, d, _ = make(1, 5, 1234, torch.bfloat16)
    d["z"].fill_(float("nan"))
    d["t"].fill_(-1)
    w = torch.zeros(5, device="cuda")
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    assert not nn.token_logprob_forward(d["z"], d["t"], w).any()
    for t in nn.policy_loss_forward_backward(d["z"], d["t"], d["adv"], d["old"], d["ref"], w,
                                             kl_coef=0.1):
        assert not t.any()
    loss, rew, logp, g = nn.preference_loss_forward_backward(d["z"], d["t"], cu, d["ref"], w)
    assert abs(loss.item() - np.log(2)) <= 2 * U
    assert not rew.any() and not logp.any() and not g.any()


def test_preference_nan_stays_in_its_pair():
    from ceo_amd import nn

    x, d, _ = make(2, 20, 640, torch.bfloat16, masked=0.0)
    cu = torch.tensor([0, 4, 9, 15, 20], dtype=torch.int32, device="cuda")
    clean = nn.preference_loss_forward_backward(d["z"], d["t"], cu, d["ref"], d["w"])
    for row, value in ((5, float("nan")), (2, float("inf"))):
        z = d["z"].clone()
        z[row, 7] = value
        got = nn.preference_loss_forward_backward(z, d["t"], cu, d["ref"], d["w"])
        assert bool(got[0][0].isnan()) and torch.equal(got[0][1:], clean[0][1:])
        assert bool(got[3][:9].isnan().all()) and torch.equal(got[3][9:], clean[3][9:])
    t = d["t"].clone()
    t[17] = 640  # no token: its own row has gradient 0
    got = nn.preference_loss_forward_backward(d["z"], t, cu, d["ref"], d["w"])
    assert bool(got[0][1].isnan()) and not got[3][17].any()
    assert bool(got[3][9:17].isnan().all()) and torch.equal(got[3][:9], clean[3][:9])


def test_policy_borders_and_absent_operands(oracle):
    """r = 1 exactly (no old log-probabilities) at a border of the clipping keeps its
    gradient; without weights every row has 1 / rows; without a reference there is no kl; no
    upper border; the loss alone."""
    from ceo_amd import nn

    announce("policy: borders, absent operands")
    N, V = 9, 800
    x, d, _ = make(4, N, V, torch.float32, masked=0.0)
    loss, logp, kl, g = nn.policy_loss_forward_backward(d["z"], d["t"], d["adv"], clip_low=0.0,
                                                        clip_high=0.0)
    assert kl is None
    rl, rlp, _, rd, rg = oracle.policy_loss(x["z"], x["t"], x["adv"], clip_low=0.0, clip_high=0.0)
    within(loss, rl, 4 * U * np.abs(rl), "loss")
    within(g, rg, grad_tol(rg, rd, 4 * U * np.abs(rd), x, torch.float32, V), "grad")
    far = d["old"] - 5.0  # ratios around e^5: clipped where A > 0, unless there is no border
    args = (d["z"], d["t"], d["adv"], far, d["ref"], d["w"])
    clipped = nn.policy_loss_forward_backward(*args)[3]
    free = nn.policy_loss_forward_backward(*args, clip_high=float("inf"))[3]
    up = torch.from_numpy(x["adv"] > 0)
    assert not clipped.cpu()[up].any() and bool((free.abs().amax(1) > 0).all())
    only = nn.policy_loss_forward_backward(*args, need_grad=False)
    assert only[3] is None
    for p, q in zip(only[:3], nn.policy_loss_forward_backward(*args)[:3]):
        assert torch.equal(p, q)
    pl = nn.preference_loss_forward_backward
    cu = torch.tensor([0, 4, N], dtype=torch.int32, device="cuda")
    a, b = pl(d["z"], d["t"], cu, need_grad=False), pl(d["z"], d["t"], cu)
    assert a[3] is None and all(torch.equal(p, q) for p, q in zip(a[:3], b[:3]))
    rl, rr, rlp, rd, rg = oracle.preference_loss(x["z"], x["t"], [0, 4, N])
    tol = logp_tol(x, rlp, V).sum() * 0.1
    within(b[0], rl, tol + 2 * U * np.abs(rl), "loss")
    within(b[3], rg, grad_tol(rg, rd, 0.1 * 0.25 * tol + 4 * U * np.abs(rd), x, torch.float32, V),
           "grad")


@pytest.mark.parametrize("what", ["policy", "preference"])
def test_gradient_against_differences(oracle, what):
    """The kernel's gradient along a direction against central differences of the loss in
    64 bits.  fp32 logits: the sum of |g u| (REL(V) + 8 roundings each), the differences'
    own h^2."""
    from ceo_amd import nn

    N, V, h = 14, 333, 1e-5
    x, d, _ = make(21, N, V, torch.float32)
    cu = [0, 3, 7, 10, N]
    if what == "policy":
        g = nn.policy_loss_forward_backward(d["z"], d["t"], d["adv"], d["old"], d["ref"], d["w"],
                                            **POLICY)[3]

        def total(z):
            return oracle.policy_loss(z, x["t"], x["adv"], x["old"], x["ref"], x["w"],
                                      **POLICY)[0].sum()
    else:
        g = nn.preference_loss_forward_backward(
            d["z"], d["t"], torch.tensor(cu, dtype=torch.int32, device="cuda"), d["ref"], d["w"],
            beta=0.5, label_smoothing=0.2)[3]

        def total(z):
            return oracle.preference_loss(z, x["t"], cu, x["ref"], x["w"], 0.5, 0.2)[0].sum()
    g = g.double().cpu().numpy()
    for k in range(4):
        u = np.random.default_rng(k).standard_normal((N, V))
        num = (total(x["z"] + h * u) - total(x["z"] - h * u)) / (2 * h)
        scale = np.abs(g * u).sum()
        assert abs(num - (g * u).sum()) <= scale * (2 * rel(V) + 16 * U) + 1e-7 * (1 + scale)


def test_streams_repeats_and_graphs():
    """The same bits again, on another stream, and from a graph replayed between the
    program's own work."""
    from ceo_amd import nn

    announce("losses: streams, graph")
    x, d, _ = make(31, 40, 5001, torch.bfloat16)
    cu = torch.tensor([0, 9, 18, 30, 40], dtype=torch.int32, device="cuda")

    def call():
        return [*nn.policy_loss_forward_backward(d["z"], d["t"], d["adv"], d["old"], d["ref"],
                                                 d["w"], kl_coef=0.1),
                *nn.preference_loss_forward_backward(d["z"], d["t"], cu, d["ref"], d["w"]),
                nn.token_logprob_forward(d["z"], d["t"], d["w"])]
    want = call()
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        got = call()
    stream.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    for k in range(4):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, out)), k
        call()
    # new values in the same buffers
    d["z"].copy_(torch.randn(40, 5001, device="cuda"))
    want = call()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, out))


def test_cached_workspace_through_the_c_abi():
    """preference_loss_forward_backward_hip with no workspace takes the stream's, and
    gives the same bits."""
    from ceo_amd import _lib, nn, runtime

    x, d, _ = make(41, 33, 900, torch.bfloat16)
    cu = torch.tensor([0, 20, 33], dtype=torch.int32, device="cuda")
    want = nn.preference_loss_forward_backward(d["z"], d["t"], cu, d["ref"], d["w"], beta=0.2)
    loss, rew = torch.empty(1, device="cuda"), torch.empty(2, device="cuda")
    logp, g = torch.empty(33, device="cuda"), torch.empty_like(want[3])
    st = torch.cuda.current_stream().cuda_stream
    rc = _lib.lib().preference_loss_forward_backward_hip(
        d["z"].data_ptr(), d["t"].data_ptr(), d["ref"].data_ptr(), d["w"].data_ptr(),
        cu.data_ptr(), loss.data_ptr(), rew.data_ptr(), logp.data_ptr(), g.data_ptr(), 1, 33, 900,
        900, 900, 0.2, 0.0, 14, None, 0, st)
    assert rc == 0 and runtime.workspace_bytes() > 0
    for p, q in zip(want, (loss, rew, logp, g)):
        assert torch.equal(p, q)


def test_offsets_past_32_bits():
    """Rows whose elements lie past 2^32 of the logits' start."""
    from ceo_amd import nn

    announce("losses: 2^32 elements apart")
    N, V = 33, 1000
    ld = 1 << 27
    store = torch.empty((N - 1) * ld + V, dtype=torch.bfloat16, device="cuda")
    z = torch.as_strided(store, (N, V), (ld, 1))
    x, d, _ = make(51, N, V, torch.bfloat16)
    z.copy_(d["z"])
    args = (d["t"], d["adv"], d["old"], d["ref"], d["w"])
    cu = torch.tensor([0, 15, N], dtype=torch.int32, device="cuda")
    a = nn.policy_loss_forward_backward(z, *args)
    b = nn.policy_loss_forward_backward(d["z"], *args)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    a = nn.preference_loss_forward_backward(z, d["t"], cu, in_place=True)
    b = nn.preference_loss_forward_backward(d["z"], d["t"], cu)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def large_rows(d, cu, beta, eps, rows=500):
    """The preference loss in 64 bits on the GPU, some rows of the logits at a time:
    (loss, rewards, logp, each row's factor)."""
    z, t = d["z"], d["t"].long()
    N, V = z.shape
    on = d["w"] != 0
    logp = torch.zeros(N, dtype=torch.float64, device="cuda")
    for a in range(0, N, rows):
        zi = z[a:a + rows].double()
        lp = zi.gather(1, t[a:a + rows, None])[:, 0] - torch.logsumexp(zi, 1)
        logp[a:a + rows] = torch.where(on[a:a + rows], lp, 0.0)
    term = torch.where(on, d["w"].double() * (logp - d["ref"].double()), 0.0).cpu().numpy()
    r = beta * np.array([term[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    x, P = r[0::2] - r[1::2], len(cu) // 2
    loss = ((1 - eps) * np.logaddexp(0, -x) + eps * np.logaddexp(0, x)) / P
    dx = (eps * np.exp(-np.logaddexp(0, -x)) - (1 - eps) * np.exp(-np.logaddexp(0, x))) / P
    f = np.zeros(N)
    for i in range(P):
        f[cu[2 * i]:cu[2 * i + 1]] = beta * dx[i]
        f[cu[2 * i + 1]:cu[2 * i + 2]] = -beta * dx[i]
    return loss, r, logp, torch.from_numpy(f).cuda() * d["w"].double()


# logits of over 256 MiB in rows of at least 96 KiB: statistics and gradients in one launch
LARGE = [(2700, 50257, torch.bfloat16), (1101, 61003, torch.float32), (2111, 65537, torch.float16),
         (700, 100001, torch.float32)]
LARGE_CU = {
    "short pairs": lambda N: [0, 3, 3, 3, 3, *range(10, N - 37, 29)],
    "ragged, rows outside": lambda N: [5, 40, 41, 500, 500, 500, 500, 650, N - 9],
    "one pair": lambda N: [0, N // 3, N],
    # more than a workgroup's threads, one row to a sequence, some without
    "many pairs": lambda N: [*range(0, N - 99), *[N - 99] * 5, *range(N - 99, N - 2, 3)],
}


@pytest.mark.parametrize("shape", LARGE, ids=["bf16", "fp32", "fp16", "fp32 long"])
@pytest.mark.parametrize("which", LARGE_CU)
def test_preference_of_more_logits_than_the_cache(shape, which):
    from ceo_amd import nn

    N, V, dtype = shape
    announce(f"preference {N} x {V} {dtype}, {which}")
    g = torch.Generator(device="cuda").manual_seed(N)
    z = torch.empty(N, V, dtype=dtype, device="cuda")
    for a in range(0, N, 256):
        z[a:a + 256] = torch.randn(min(256, N - a), V, generator=g, device="cuda") * 2.5
    d = dict(z=z, t=torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32),
             w=torch.rand(N, generator=g, device="cuda") + 0.1,
             ref=torch.randn(N, generator=g, device="cuda") * 0.3 - 13.0)
    d["w"][torch.rand(N, generator=g, device="cuda") < 0.3] = 0.0
    z[d["w"] == 0, :64] = float("nan")  # not read
    cu = LARGE_CU[which](N)
    cu = cu if len(cu) % 2 else cu[:-1]
    beta, eps = 0.02, 0.1
    args = (d["t"], torch.tensor(cu, dtype=torch.int32, device="cuda"), d["ref"], d["w"], beta, eps)
    got = nn.preference_loss_forward_backward(z, *args)
    rl, rr, rlp, f = large_rows(d, cu, beta, eps)
    U64 = rel(V)
    dl = U * rlp.abs().cpu().numpy() + 64 * U + U64
    aw = d["w"].cpu().numpy()
    dr = np.array([beta * (aw * dl)[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    dx = dr[0::2] + dr[1::2]
    within(got[2], rlp.cpu().numpy(), dl, "logp")
    within(got[1], rr, dr + U * np.abs(rr) + 1e-30, "rewards")
    within(got[0], rl, dx / len(rl) + 2 * U * np.abs(rl), "loss")
    de = np.zeros(N)
    for i in range(len(rl)):
        de[cu[2 * i]:cu[2 * i + 2]] = beta * (0.25 * dx[i] / len(rl))
    de = torch.from_numpy(de).cuda() * d["w"].double() + 4 * U * f.abs()
    for a in range(0, N, 300):
        on = f[a:a + 300, None] != 0
        p = torch.softmax(torch.where(on, z[a:a + 300].double(), 0.0), 1)
        want = torch.where(on, -f[a:a + 300, None] * p, 0.0)
        i = torch.arange(len(p), device="cuda")
        want[i, d["t"][a:a + 300].long()] += f[a:a + 300]
        p[i, d["t"][a:a + 300].long()] += 1.0
        tol = (want.abs() * torch.finfo(dtype).eps / 2 + TINY[dtype]
               + p * (f[a:a + 300, None].abs() * U64 + de[a:a + 300, None]) * 1.01)
        assert bool(((got[3][a:a + 300].double() - want).abs() <= tol).all())
    # the same bits again, without the gradient, on a stream of its own, and in place
    again = nn.preference_loss_forward_backward(z, *args)
    only = nn.preference_loss_forward_backward(z, *args, need_grad=False)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        other = nn.preference_loss_forward_backward(z, *args)
    stream.synchronize()
    place = nn.preference_loss_forward_backward(z, *args, in_place=True)
    for p in (again, other, place):
        assert all(torch.equal(a, b) for a, b in zip(got, p))
    assert all(torch.equal(a, b) for a, b in zip(got[:3], only[:3]))


def test_large_preference_offsets_graph_and_bad_rows():
    """Of more logits than the cache: offsets that fall are those before them, a NaN stays
    in its pair, targets that are no tokens; and a graph gives the eager bits."""
    from ceo_amd import nn

    N, V = 2700, 50257
    announce("large preference: offsets, graph, NaN")
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.empty(N, V, dtype=torch.bfloat16, device="cuda")
    z.normal_(0, 2, generator=g)
    t = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    ref = torch.full((N,), -12.5, device="cuda")

    def call(cu, **kw):
        return nn.preference_loss_forward_backward(
            z, t, torch.tensor(cu, dtype=torch.int32, device="cuda"), ref, beta=0.01, **kw)
    want = call([0, 700, 1500, 1500, 2600])
    got = call([-9, 700, 1500, 1200, 2600])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert not want[3][2600:].any() and bool(want[3][:2600].any(1).all())
    got = call([0, 700, 1500, 1500, 2600, 2600, 1 << 30])  # one more pair: its only row set [2600, N)
    assert bool(got[3][2600:].any(1).all())
    none = call([0])
    assert none[0].shape == (0,) and not none[3].any() and torch.equal(none[2], want[2])
    keep = t[1000].item()
    t[1000] = V
    got = call([0, 700, 1500, 1500, 2600])
    assert bool(got[0][0].isnan()) and not got[3][1000].any() and bool(got[3][999].isnan().all())
    assert torch.equal(got[3][1500:], want[3][1500:]) and torch.equal(got[0][1:], want[0][1:])
    t[1000] = keep
    cu = torch.tensor([0, 700, 1500, 1500, 2600], dtype=torch.int32, device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = nn.preference_loss_forward_backward(z, t, cu, ref, beta=0.01)
    for k in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), k
        call([0, 100, 200])


def test_small_offsets_that_fall():
    """Offsets that fall are taken as those before them: pairs never share rows."""
    from ceo_amd import nn

    x, d, _ = make(61, 12, 300, torch.bfloat16, masked=0.0)

    def call(cu):
        return nn.preference_loss_forward_backward(
            d["z"], d["t"], torch.tensor(cu, dtype=torch.int32, device="cuda"),
            ref_logp=d["ref"], weights=d["w"])
    a, b = call([0, 8, 10, 9, 7, 6, 12]), call([0, 8, 10, 10, 10, 10, 12])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_more_rows_than_one_grid_dimension(dtype):
    """Rows past 2^20, which a grid's second dimension holds."""
    from ceo_amd import nn

    N, V = (1 << 20) + 4099, 5
    announce(f"{N} rows {dtype}")
    g = torch.Generator(device="cuda").manual_seed(5)
    z = torch.randn(N, V, generator=g, device="cuda").to(dtype)
    t = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    adv = torch.randn(N, generator=g, device="cuda")
    lp = torch.log_softmax(z.double(), 1)
    ref = lp.gather(1, t[:, None].long())[:, 0]
    tol = U * ref.abs() + U * 32 + rel(V)
    got = nn.token_logprob_forward(z, t)
    assert bool(((got.double() - ref).abs() <= tol).all())
    w = torch.ones(N, device="cuda")
    loss, logp, _, grad = nn.policy_loss_forward_backward(z, t, adv, weights=w)
    one = torch.nn.functional.one_hot(t.long(), V).double()
    want = -adv.double()[:, None] * (one - lp.exp())
    eps = torch.finfo(dtype).eps
    room = want.abs() * eps / 2 + TINY[dtype] + adv.double().abs()[:, None] * (one + lp.exp()) * (
        rel(V) + 12 * U)
    assert bool(((grad.double() - want).abs() <= room).all())
    assert torch.equal(logp, got)
    cu = torch.tensor([0, N // 2, N], dtype=torch.int32, device="cuda")
    _, _, plp, pg = nn.preference_loss_forward_backward(z, t, cu, ref_logp=got, beta=0.5)
    assert torch.equal(plp, got)
    want = -0.25 * (one - lp.exp())  # x = 0: half of beta, minus for the chosen
    want[N // 2:] *= -1
    room = want.abs() * (eps / 2 + 8 * U) + TINY[dtype] + (one + lp.exp()) * rel(V)
    assert bool(((pg.double() - want).abs() <= room).all())


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 4101), (torch.float16, 8197),
                                     (torch.float32, 4099), (torch.bfloat16, 33)], ids=str)
def test_every_alignment(oracle, dtype, V):
    """Rows that start at each multiple of the type's size within a cache line, logits and
    gradient at different ones; in place the same bits."""
    from ceo_amd import nn

    N = 130
    announce(f"every alignment {dtype} V={V}")
    x, d, store = make(V, N, V, dtype, pad=2, skew=1)  # the gradient is packed
    check_policy(x, d, dtype, V)
    check_preference(x, d, [0, 40, 65, 65, N], dtype, V)
    cu = torch.tensor([0, 40, 65, 65, N], dtype=torch.int32, device="cuda")
    for f in (lambda ip: nn.preference_loss_forward_backward(d["z"], d["t"], cu, d["ref"], d["w"],
                                                             in_place=ip),
              lambda ip: nn.policy_loss_forward_backward(d["z"], d["t"], d["adv"], d["old"],
                                                         d["ref"], d["w"], in_place=ip)):
        kept = store.clone()
        want = f(False)
        got = f(True)
        assert all(torch.equal(p, q) for p, q in zip(want[:2], got[:2]))
        assert torch.equal(want[3], got[3])
        outside = torch.ones_like(store, dtype=torch.bool)
        outside[1:1 + N * (V + 2)].view(N, V + 2)[:, :V] = False
        assert bool(store[outside].isnan().all())
        store.copy_(kept)


def test_no_rows_with_a_gradient_pointer():
    """Pairs without rows through the C ABI, a gradient and a workspace given all the same."""
    from ceo_amd import _lib

    cu = torch.zeros(5, dtype=torch.int32, device="cuda")
    loss, rew = torch.full((2,), 7.0, device="cuda"), torch.full((4,), 7.0, device="cuda")
    buf = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    rc = _lib.lib().preference_loss_forward_backward_hip(
        None, None, None, None, cu.data_ptr(), loss.data_ptr(), rew.data_ptr(), None,
        buf.data_ptr(), 2, 0, 100, 100, 100, 0.1, 0.0, 14, buf.data_ptr(), 4096, st)
    assert rc == 0
    assert np.allclose(loss.cpu().numpy(), np.log(2) / 2, rtol=2 * U) and not rew.any()
    assert not buf[2048:].any()


def test_large_preferences_on_two_streams():
    """Two of the launches whose workgroups wait for each other, at once: each waits only
    for its own."""
    from ceo_amd import nn

    N, V = 2800, 50257
    announce("large preference losses on two streams")
    cu = torch.tensor([0, 90, 200, 900, 1000, 1300, 2000, 2400, N], dtype=torch.int32,
                      device="cuda")
    t = torch.arange(N, device="cuda", dtype=torch.int32)
    zs = [torch.empty(N, V, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(2)]
    want = [nn.preference_loss_forward_backward(z, t, cu, beta=0.01) for z in zs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in zs]
    got = [[], []]
    for _ in range(3):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(nn.preference_loss_forward_backward(zs[k], t, cu, beta=0.01))
    for st in streams:
        st.synchronize()
    for w, g in zip(want, got):
        for r in g:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [20483, 24571, 37001, 45003, 53249, 81001, 95003, 114699])
def test_policy_rows_of_every_form(oracle, V, dtype):
    """Row lengths for each number of vectors that a thread holds."""
    announce(f"policy forms V={V} {dtype}")
    x, d, _ = make(V, 3, V, dtype, pad=3, skew=5, masked=0.0)
    check_policy(x, d, dtype, V)
    check_policy(x, d, dtype, V, in_place=True)
