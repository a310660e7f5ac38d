"""What the operators of a post-training step are measured on: the log-probabilities of given tokens, the
clipped policy loss and the preference loss with their gradients in the logits, and the norm of many gradients with
their clipping.  `own` selects the side: False the plain forms (torch operations in 32 bits), True the calls a
user makes of `ceo_amd.nn`.
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.05
BETA, SMOOTHING = 0.1, 0.05
MAX_NORM = 1.0

# vocabulary, width, layers, heads, head size, MLP width of the models whose gradients are clipped
MODELS = {
    # the training step of this repository's benchmark (368 million parameters)
    "step": (32000, 1024, 24, 16, 64, 4096),
    # a mid-size one with an odd vocabulary
    "mid": (5003, 384, 6, 6, 64, 1536),
    # the two-layer model of a test
    "tiny": (257, 64, 2, 2, 64, 128),
}


def listed():
    def tok(op, name, rows, vocab, dtype="bf16", pad=0, prompt=0.0, seqs=1):
        return {"name": name, "op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "pad": pad,
                "prompt": prompt, "seqs": seqs}

    return [
        # a few answers' last tokens, scored while a sampler waits for them: latency
        tok("logprob", "logprob 32x32000", 32, 32000),
        # the frozen model's log-probabilities over the benchmark's batch of 16,384 tokens, 40 % of them prompts
        tok("logprob", "logprob 16384x32000 masked", 16384, 32000, prompt=0.4, seqs=16),
        # one short answer: latency
        tok("policy", "policy 64x32000", 64, 32000),
        # an odd vocabulary, so that rows start at any multiple of two bytes, and an odd count of tokens
        tok("policy", "policy 4095x50257", 4095, 50257, prompt=0.25, seqs=9),
        # the benchmark's batch, every token an answer's
        tok("policy", "policy 16384x32000", 16384, 32000),
        # a large vocabulary in half precision, rows padded to whole tiles of the product that made them
        tok("policy", "policy 2048x128003 fp16", 2048, 128003, dtype="fp16", pad=61, prompt=0.2, seqs=4),
        # two pairs of short answers
        tok("preference", "preference 2 pairs 45x32000", 45, 32000, prompt=0.3, seqs=4),
        # eight pairs of ragged answers behind prompts that carry no weight
        tok("preference", "preference 8 pairs 8191x32000", 8191, 32000, prompt=0.3, seqs=16),
        # logits kept in fp32, odd vocabulary, many pairs
        tok("preference", "preference 32 pairs 4100x50257 fp32", 4100, 50257, dtype="fp32", prompt=0.1, seqs=64),
        # a small model's 23 gradients, one buffer each: latency
        {"name": "clip tiny fp32", "op": "clip", "model": "tiny", "dtype": "fp32", "align": 64, "layers": 0},
        # a mid-size model's, packed without gaps, so that most start unaligned
        {"name": "clip mid bf16 packed", "op": "clip", "model": "mid", "dtype": "bf16", "align": 1, "layers": 0},
        # every gradient of the benchmark's training step
        {"name": "clip step bf16", "op": "clip", "model": "step", "dtype": "bf16", "align": 64, "layers": 0},
    ]


def draw(rng):
    op = rng.choice(["logprob", "policy", "policy", "preference", "preference", "clip"])
    if op == "clip":
        model = rng.choice(["tiny", "mid", "step"])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        most = {"tiny": 40, "mid": 48, "step": 24 if SIZE[dtype] == 2 else 10}[model]
        return {"op": op, "model": model, "dtype": dtype, "align": rng.choice([1, 2, 8, 64]),
                "layers": rng.randint(1, most)}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = int(math.exp(rng.uniform(math.log(500), math.log(131072))))
    if rng.random() < 0.5:
        vocab = max(64, vocab // 64 * 64)
    most = min(16384, int(1.0e9 / (vocab * SIZE[dtype])))
    least = 2 if op == "preference" else 1
    rows = max(least, int(math.exp(rng.uniform(math.log(least), math.log(most)))))
    seqs = max(1, min(rows // 2, int(math.exp(rng.uniform(0, math.log(128))))))
    if op == "preference":
        seqs = max(2, seqs // 2 * 2)
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "pad": rng.choice([0, 0, 1, 47]),
            "prompt": round(rng.choice([0.0, rng.uniform(0.0, 0.6)]), 3), "seqs": seqs}


def _layout(case):
    """(sequence starts (seqs + 1,), weight-carrying rows as truth values): of the case alone."""
    rows, seqs = case["rows"], case["seqs"]
    r = np.random.RandomState((rows * 31 + seqs * 7 + case["vocab"]) % (2 ** 31))
    # ragged lengths, some of them short, an occasional empty one
    share = r.gamma(2.0, 1.0, seqs)
    cu = np.concatenate([[0], np.round(np.cumsum(share) / share.sum() * rows)]).astype(np.int64)
    cu[-1] = rows
    on = np.ones(rows, bool)
    for a, b in zip(cu[:-1], cu[1:]):
        on[a:a + int((b - a) * case["prompt"])] = False
    return cu, on


def _shapes(case):
    V, D, L, H, dh, F = MODELS[case["model"]]
    L = case["layers"] or L
    got = [(V, D)]
    for _ in range(L):
        got += [(D,), (D,), (D, 3 * H * dh + H), (H * dh, D), (D,), (D,), (D, F), (F,), (F, D), (D,)]
    return got + [(D,), (D,), (D, V)]


def _offsets(case):
    off, at = 0, []
    for s in _shapes(case):
        at.append(off)
        n = math.prod(s)
        off += -(-n // case["align"]) * case["align"]
    return at, off


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    dt = DT[case["dtype"]]
    if case["op"] == "clip":
        at, total = _offsets(case)
        flat = torch.zeros(total, dtype=dt, device="cuda")
        out = torch.zeros(total, dtype=dt, device="cuda")
        grads, outs = [], []
        for s, o in zip(_shapes(case), at):
            n = math.prod(s)
            v = flat[o:o + n]
            # gradients of a mean loss: small, another scale in each tensor
            scale = 10.0 ** float(torch.empty((), device="cpu").uniform_(-3.5, -2.0, generator=torch.Generator().manual_seed(seed + o)))
            for a in range(0, n, 1 << 26):
                b = min(n, a + (1 << 26))
                v[a:b] = (torch.randn(b - a, generator=g, device="cuda") * scale).to(dt)
            grads.append(v.view(s))
            outs.append(out[o:o + n].view(s))
        state = {"case": case, "grads": grads, "outs": outs, "out": out}
        if own:
            from ceo_amd import nn

            # the list of a model's gradients, laid out once as its training loop would
            state["list"] = nn.GradList(grads, outs)
        return state
    N, V = case["rows"], case["vocab"]
    cu, on = _layout(case)
    ld = V + case["pad"]
    logits = torch.empty(N, ld, dtype=dt, device="cuda")[:, :V]
    targets = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    step = max(1, (1 << 27) // ld)
    sd, logp = 2.5, torch.empty(N, dtype=torch.float32, device="cuda")
    for a in range(0, N, step):
        b = min(N, a + step)
        z = torch.randn(b - a, V, generator=g, device="cuda") * sd
        # the token that was sampled: a likely one, log-probability around -1.5
        likely = math.log(V) + sd * sd / 2 - 0.5 + 1.5 * torch.randn(b - a, 1, generator=g, device="cuda")
        z.scatter_(1, targets[a:b, None].long(), likely)
        z = z.to(dt)
        logits[a:b] = z
        logp[a:b] = _logp(z, targets[a:b])
        del z
    mask = torch.from_numpy(on).cuda()
    state = {"case": case, "logits": logits, "targets": targets, "mask": mask,
             "cu": torch.from_numpy(cu.astype(np.int32)).cuda()}
    # another state of the same policy, and the frozen model
    old = logp + 0.15 * torch.randn(N, generator=g, device="cuda")
    state["ref"] = logp + 0.3 * torch.randn(N, generator=g, device="cuda") - 0.05
    if case["op"] == "policy":
        adv = torch.randn(N, generator=g, device="cuda")
        # the gradient jumps where the ratio meets a border of the clipping; a token so near to one that
        # rounding decides says nothing about either side
        for border in (1.0 - CLIP_LOW, 1.0 + CLIP_HIGH):
            near = ((logp - old) - math.log(border)).abs() < 1e-4
            old = torch.where(near, old - 4e-4, old)
        state["old"], state["adv"] = old, adv
        # the mean over the tokens that count
        state["weights"] = mask.float() / max(1, int(on.sum()))
    else:
        state["weights"] = mask.float()
    return state


def _logp(z, t):
    """Plain log-probabilities of tokens t: (rows, V) logits in any type, fp32 out."""
    z = z.float()
    m = z.amax(1, keepdim=True)
    s = (z - m).exp_().sum(1)
    return z.gather(1, t[:, None].long())[:, 0] - m[:, 0] - s.log()


def _dlogits(z, t, mask, coef):
    """coef_i ([j = t_i] - softmax_ij), 0 in rows without weight, in the logits' type."""
    f = z.float()
    e = (f - f.amax(1, keepdim=True)).exp_()
    p = e / e.sum(1, keepdim=True)
    d = p.mul_(-coef[:, None])
    d.scatter_add_(1, t[:, None].long(), coef[:, None])
    return torch.where(mask[:, None], d, torch.zeros((), device=d.device)).to(z.dtype)


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    if op == "clip":
        # long sums: 64 bits
        norm = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt()
        coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        for g, o in zip(state["grads"], state["outs"]):
            o.copy_(g.float() * coef.float())
        return {"norm": norm.float(), "grads": state["out"]}
    z, t, mask, w = state["logits"], state["targets"], state["mask"], state["weights"]
    zero = torch.zeros((), device=z.device)
    logp = torch.where(mask, _logp(z, t), zero)
    if op == "logprob":
        return {"logp": logp}
    if op == "policy":
        ratio = (logp - state["old"]).exp()
        adv = state["adv"]
        low, high = 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH
        gain = torch.minimum(ratio * adv, ratio.clamp(low, high) * adv)
        x = state["ref"] - logp
        kl = torch.where(mask, torch.expm1(x) - x, zero)
        loss = torch.where(mask, w * (KL_COEF * kl - gain), zero)
        free = torch.where(adv >= 0, ratio <= high, ratio >= low)
        d = -adv * ratio * free - KL_COEF * torch.expm1(x)
        return {"loss": loss, "logp": logp, "kl": kl, "grad": _dlogits(z, t, mask, w * d)}
    seqs = state["cu"].numel() - 1
    seq = torch.searchsorted(state["cu"][1:], torch.arange(z.shape[0], device=z.device, dtype=torch.int32), right=True)
    # long sums: 64 bits
    d = torch.zeros(seqs, dtype=torch.float64, device=z.device)
    d.scatter_add_(0, seq, torch.where(mask, w * (logp - state["ref"]), zero).double())
    reward = BETA * d
    x = reward[0::2] - reward[1::2]
    P = seqs // 2
    plus, minus = torch.log1p(torch.exp(-x.abs())) + (-x).clamp(min=0), torch.log1p(torch.exp(-x.abs())) + x.clamp(min=0)
    loss = ((1.0 - SMOOTHING) * plus + SMOOTHING * minus) / P
    dx = (SMOOTHING / (1.0 + torch.exp(-x)) - (1.0 - SMOOTHING) / (1.0 + torch.exp(x))) / P
    coef = BETA * torch.stack([dx, -dx], 1).reshape(-1).float()[seq] * w
    return {"loss": loss.float(), "rewards": reward.float(), "logp": logp, "grad": _dlogits(z, t, mask, coef)}


def _run_own(op, state):
    from ceo_amd import nn

    if op == "clip":
        return {"norm": nn.clip_grad_norm(state["list"], MAX_NORM), "grads": state["out"]}
    z, t, w = state["logits"], state["targets"], state["weights"]
    if op == "logprob":
        return {"logp": nn.token_logprob_forward(z, t, w)}
    if op == "policy":
        loss, logp, kl, grad = nn.policy_loss_forward_backward(
            z, t, state["adv"], old_logp=state["old"], ref_logp=state["ref"], weights=w,
            clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF)
        return {"loss": loss, "logp": logp, "kl": kl, "grad": grad}
    loss, rewards, logp, grad = nn.preference_loss_forward_backward(
        z, t, state["cu"], ref_logp=state["ref"], weights=w, beta=BETA, label_smoothing=SMOOTHING)
    return {"loss": loss, "rewards": rewards, "logp": logp, "grad": grad}


def work(case):
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 4, "flops": 3 * n}
    N, V, size = case["rows"], case["vocab"], SIZE[case["dtype"]]
    on = int(_layout(case)[1].sum())
    # rows without weight are not read; their gradient is zeros that have to be written
    read = on * V * size
    if case["op"] == "logprob":
        return {"bytes": read + N * 12, "flops": 4 * on * V}
    per_row = {"policy": 9, "preference": 4}[case["op"]]
    return {"bytes": read + N * V * size + N * 4 * per_row, "flops": 7 * on * V}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for g in state["grads"]:
            total = total + torch.linalg.vector_norm(g.double()) ** 2
        norm = torch.sqrt(total)
        f = min(1.0, MAX_NORM / (float(norm) + 1e-6))
        out = torch.zeros(state["out"].numel(), dtype=torch.float64, device="cuda")
        for s, o, g in zip(_shapes(case), _offsets(case)[0], state["grads"]):
            out[o:o + math.prod(s)] = g.double().reshape(-1) * f
        return {"norm": norm, "grads": out}
    N, V = case["rows"], case["vocab"]
    cu, on = _layout(case)
    rows = torch.from_numpy(np.flatnonzero(on)).cuda()
    z, t = state["logits"], state["targets"].long()
    step = max(1, (1 << 26) // V)
    logp = torch.zeros(N, dtype=torch.float64, device="cuda")
    for i in rows.split(step):
        zi = z[i].double()
        logp[i] = zi[torch.arange(len(i), device="cuda"), t[i]] - torch.logsumexp(zi, 1)
    if case["op"] == "logprob":
        return {"logp": logp}
    w, ref = state["weights"].double(), state["ref"].double()
    leaf = logp.clone().requires_grad_()
    with torch.enable_grad():
        if case["op"] == "policy":
            adv, ratio = state["adv"].double(), torch.exp(leaf - state["old"].double())
            bound = torch.where(adv >= 0, torch.clamp(ratio, max=1.0 + CLIP_HIGH), torch.clamp(ratio, min=1.0 - CLIP_LOW))
            kl = torch.exp(ref - leaf) - (ref - leaf) - 1.0
            loss = (w * (KL_COEF * kl - bound * adv))[rows]
        else:
            sums = [(w[a:b] * (leaf[a:b] - ref[a:b])).sum() for a, b in zip(cu[:-1], cu[1:])]
            rewards = BETA * torch.stack(sums)
            x = rewards[0::2] - rewards[1::2]
            loss = -((1.0 - SMOOTHING) * torch.nn.functional.logsigmoid(x)
                     + SMOOTHING * torch.nn.functional.logsigmoid(-x)) / len(x)
        dlogp, = torch.autograd.grad(loss.sum(), leaf)
    grad = torch.zeros(N, V, dtype=torch.float64, device="cuda")
    for i in rows.split(step):
        one = torch.zeros(len(i), V, dtype=torch.float64, device="cuda")
        one[torch.arange(len(i), device="cuda"), t[i]] = 1.0
        grad[i] = dlogp[i, None] * (one - torch.softmax(z[i].double(), 1))
    if case["op"] == "policy":
        full, klf = torch.zeros_like(logp), torch.zeros_like(logp)
        full[rows], klf[rows] = loss.detach(), kl.detach()[rows]
        return {"loss": full, "logp": logp, "kl": klf, "grad": grad}
    return {"loss": loss.detach(), "rewards": rewards.detach(), "logp": logp, "grad": grad}
