"""What the operators of text generation are measured on: beam search's selection over beams and vocabulary, the
reordering of the states that its beams carry, and products in 8-bit integers with a scale for each token and
channel.  `own` selects the side: False the plain forms (torch operations in 32 bits, 64 where 32 would decide
between neighbours), True the calls a user makes of `ceo_amd.nn` and `ceo_amd.state`.
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

END = 2  # the token that finishes a text


def listed():
    def sel(name, batch, beams, vocab, dtype="bf16", pad=0, select=0, finished=False, keep=False):
        return {"name": name, "op": "select", "batch": batch, "beams": beams, "vocab": vocab, "dtype": dtype, "pad": pad,
                "select": select or beams, "finished": finished, "keep": keep}

    def mov(name, batch, beams, layers, heads, dk, dv, history, place, odd=False):
        return {"name": name, "op": "reorder", "batch": batch, "beams": beams, "layers": layers, "heads": heads, "dk": dk,
                "dv": dv, "history": history, "place": place, "odd": odd}

    def lin(name, m, k, n, dtype="bf16", bias=False, residual=False, gelu=False):
        return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias, "residual": residual,
                "gelu": gelu}

    return [
        # one text, four beams, the benchmark's vocabulary: the latency of each generated token
        sel("select 1x4 of 32000", 1, 4, 32000, keep=True),
        # sixteen texts, some beams finished, twice the beams selected, an odd vocabulary in padded rows
        sel("select 16x4 of 50257", 16, 4, 50257, pad=47, select=8, finished=True),
        # logits kept in fp32, a batch job
        sel("select 64x8 of 32000 fp32", 64, 8, 32000, dtype="fp32", finished=True, keep=True),
        # a large vocabulary, many texts
        sel("select 64x8 of 128003 fp16", 64, 8, 128003, dtype="fp16", select=16),
        # a small model's states and the texts so far, one sequence: latency
        mov("reorder 1x4 tiny", 1, 4, 2, 2, 64, 64, 40, "in"),
        # the benchmark's decoder, eight texts of four beams, in place
        mov("reorder 8x4 step", 8, 4, 24, 16, 64, 64, 512, "in"),
        # wide beams into a second set of buffers, with a tensor of odd rows
        mov("reorder 3x13 mid to outs", 3, 13, 6, 6, 64, 128, 201, "out", odd=True),
        # one generated token of four beams through a square projection that adds the residual: latency
        lin("linear 4x1024x1024", 4, 1024, 1024, residual=True),
        # the benchmark's vocabulary head for 32 beams
        lin("linear 32x1024x32000", 32, 1024, 32000),
        # a ragged prompt, odd sizes, half precision
        lin("linear 517x1001x3088 fp16", 517, 1001, 3088, dtype="fp16", bias=True),
        # prompts of the benchmark's batch through the MLP's two products
        lin("linear 16384x1024x4096 gelu", 16384, 1024, 4096, bias=True, gelu=True),
        lin("linear 16384x4096x1024", 16384, 4096, 1024, bias=True, residual=True),
    ]


def _log(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 0.999))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "linear", "linear", "linear"])
    if op == "select":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        beams = _log(rng, 1, 16)
        vocab = _log(rng, 300, 131072)
        if rng.random() < 0.5:
            vocab = max(64, vocab // 64 * 64)
        batch = _log(rng, 1, max(1, min(256, int(1.3e8 / (beams * vocab * SIZE[dtype])))))
        keep = rng.random() < 0.5
        select = beams if keep else rng.choice([beams, 2 * beams])
        return {"op": op, "batch": batch, "beams": beams, "vocab": vocab, "dtype": dtype, "pad": rng.choice([0, 0, 1, 47]),
                "select": select, "finished": rng.random() < 0.5, "keep": keep}
    if op == "reorder":
        beams, layers = _log(rng, 2, 16), _log(rng, 1, 24)
        heads, dk, dv = rng.randint(1, 16), rng.choice([64, 64, 128]), rng.choice([64, 64, 128])
        batch = _log(rng, 1, max(1, min(64, int(2.0e8 / (beams * layers * heads * dk * dv * 4)))))
        return {"op": op, "batch": batch, "beams": beams, "layers": layers, "heads": heads, "dk": dk, "dv": dv,
                "history": _log(rng, 1, 2048), "place": rng.choice(["in", "out"]), "odd": rng.random() < 0.3}
    k, n = _log(rng, 64, 4096), _log(rng, 64, 32000)
    if rng.random() < 0.6:
        k, n = max(64, k // 64 * 64), max(64, n // 16 * 16)
    m = _log(rng, 1, max(1, min(16384, int(6.5e10 / (k * n)))))
    return {"op": op, "m": m, "k": k, "n": n, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "bias": rng.random() < 0.5, "residual": rng.random() < 0.4, "gelu": rng.random() < 0.3}


def _parents(case):
    """(batch, beams) int64: the beam that each one continues, of the case alone."""
    batch, beams = case["batch"], case["beams"]
    r = np.random.RandomState((batch * 131 + beams * 17 + case["history"]) % (2 ** 31))
    got = np.zeros((batch, beams), np.int64)
    for b in range(batch):
        # a few good beams have most of the children
        p = r.dirichlet(np.full(beams, 0.7))
        child = np.sort(r.choice(beams, beams, p=p))
        if case["place"] == "out":
            got[b] = r.permutation(child)
            continue
        # in place: the first child of a beam stays where that beam was, the others take what is free
        first = np.concatenate([[True], child[1:] != child[:-1]])
        free = np.setdiff1d(np.arange(beams), child)
        got[b, child[first]] = child[first]
        got[b, free] = child[~first]
    return got


def _state_shapes(case):
    rows = case["batch"] * case["beams"]
    shapes = [((rows, case["heads"], case["dk"], case["dv"]), torch.float32)] * case["layers"]
    shapes += [((rows, case["history"]), torch.int32)]
    if case["odd"]:
        # the last inputs of a short convolution over an odd width
        shapes += [((rows, 3, 385), torch.bfloat16)]
    return shapes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = {"case": case}
    if case["op"] == "reorder":
        tensors = []
        for shape, dt in _state_shapes(case):
            if dt == torch.int32:
                t = torch.randint(0, 32000, shape, generator=g, device="cuda", dtype=dt)
            else:
                t = rnd(*shape).to(dt)
            tensors.append(t)
        state["states"] = tensors
        state["outs"] = [torch.zeros_like(t) for t in tensors] if case["place"] == "out" else None
        state["parents"] = torch.from_numpy(_parents(case).astype(np.int32)).cuda()
        if own:
            from ceo_amd.state import StateList

            # the list of a decoder's states, laid out once as its generation loop would
            state["list"] = StateList(tensors, case["beams"], state["outs"])
        return state
    dt = DT[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        # normalised activations, a few channels of them large
        x = rnd(m, k) * torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        state["x"] = x.to(dt)
        weight = (rnd(k, n) * 0.02).to(dt)
        state["bias"] = (rnd(n) * 0.1).to(dt) if case["bias"] else None
        state["residual"] = rnd(m, n).to(dt) if case["residual"] else None
        if own:
            from ceo_amd import nn

            state["weight"] = nn.Int8Weight(weight)
        else:
            q, s = _quantized(weight.t())
            state["weight"], state["scale"] = q.t().contiguous().to(torch.int8), s
        return state
    B, K, V = case["batch"], case["beams"], case["vocab"]
    ld = V + case["pad"]
    logits = torch.empty(B * K, ld, dtype=dt, device="cuda")[:, :V]
    step = max(1, (1 << 26) // ld)
    for a in range(0, B * K, step):
        logits[a:a + step] = (rnd(min(step, B * K - a), V) * 2.5).to(dt)
    finished = None
    if case["finished"]:
        # a text whose beams have all finished is taken out of the batch
        finished = (torch.rand(B, K, generator=g, device="cuda") < 0.2) & (torch.arange(K, device="cuda") > 0)
    top, tok, lse = _row_best(logits, case["select"] + 1)
    scores = -6.0 - 2.0 * rnd(B, K).abs()
    # two beams' candidates that rounding alone orders say nothing about either side: such texts get other scores
    for _ in range(20):
        value = (scores.double().view(B, K, 1) + top.view(B, K, -1) - lse.view(B, K, 1))
        if finished is not None:
            alone = torch.full_like(value, -math.inf)
            alone[:, :, 0] = scores.double()
            value = torch.where(finished[:, :, None], alone, value)
        row = torch.arange(K, device="cuda")[None, :, None].expand_as(value).reshape(B, -1)
        value, at = value.reshape(B, -1).sort(1, descending=True)
        row = row.gather(1, at)
        close = ((value[:, :-1] - value[:, 1:] < 2e-5) & (row[:, :-1] != row[:, 1:]))[:, :case["select"] + 1].any(1)
        scores = torch.where(close[:, None], -6.0 - 2.0 * rnd(B, K).abs(), scores)
    state.update(logits=logits, scores=scores, finished=finished)
    return state


def _quantized(x):
    """(whole numbers in -127 .. 127, scales fp32): one scale for each row; 64 bits where a quotient meets a border."""
    scale = x.float().abs().amax(1) / 127.0
    q = torch.round(x.double() / scale.double()[:, None]) if x.numel() < (1 << 25) else torch.cat(
        [torch.round(a.double() / s.double()[:, None]) for a, s in zip(x.split(4096), scale.split(4096))])
    return torch.where(scale[:, None] > 0, q, torch.zeros((), dtype=q.dtype, device=q.device)).float(), scale


def _row_best(z, n):
    """Of each row: its n best logits (64 bits) and their tokens, ties to the lowest, and log sum exp."""
    V = z.shape[1]
    n = min(n, V)
    best, token, lse = [], [], []
    step = max(1, (1 << 27) // V)
    for zi in z.split(step):
        f = zi.float() + 0.0  # -0 is 0
        m = f.amax(1, keepdim=True)
        lse.append(m[:, 0].double() + (f - m).exp_().sum(1, dtype=torch.float64).log())
        # order-preserving whole numbers with the token below them, so that no two are alike
        bits = f.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7fffffff) - 1, bits) * (1 << 20) + (V - 1 - torch.arange(V, device=z.device))
        i = (V - 1 - (key.topk(n, 1).values & ((1 << 20) - 1)))
        token.append(i)
        best.append(f.gather(1, i).double())
    return torch.cat(best), torch.cat(token), torch.cat(lse)


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "reorder":
        parents = state["parents"].long()
        first = torch.arange(case["batch"], device=parents.device)[:, None] * case["beams"]
        rows = (first + parents).reshape(-1)
        outs = state["outs"] or state["states"]
        for s, o in zip(state["states"], outs):
            o.copy_(s[rows])
        return outs
    if case["op"] == "linear":
        q, s = _quantized(state["x"])
        y = (q @ state["weight"].float()) * (s[:, None] * state["scale"][None, :])
        if state["bias"] is not None:
            y = y + state["bias"].float()
        if case["gelu"]:
            y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(DT[case["dtype"]])
    B, K, V, n = case["batch"], case["beams"], case["vocab"], case["select"]
    scores, finished = state["scores"].double(), state["finished"]
    top, tok, lse = _row_best(state["logits"], n)
    value = scores[:, :, None] + (top - lse[:, None]).view(B, K, -1)
    tok = tok.view(B, K, -1)
    if finished is not None:
        alone = torch.full_like(value, -math.inf)
        alone[:, :, 0] = scores
        value = torch.where(finished[:, :, None], alone, value)
        others = torch.arange(tok.shape[2], device=tok.device) - 1
        others = torch.where(others >= END, others + 1, others)
        others[0] = END
        tok = torch.where(finished[:, :, None], others, tok)
    flat = (torch.arange(K, device=tok.device)[None, :, None] * V + tok).reshape(B, -1)
    flat, at = flat.sort(1)
    value, to = value.reshape(B, -1).gather(1, at).sort(dim=1, descending=True, stable=True)
    value, flat = value[:, :n], flat.gather(1, to)[:, :n]
    parent, token = flat // V, flat % V
    if case["keep"]:
        earlier = torch.ones(n, n, dtype=torch.bool, device=flat.device).tril(-1)
        first = ~((parent[:, :, None] == parent[:, None, :]) & earlier).any(2)
        taken = torch.zeros(B, K, dtype=torch.int64, device=flat.device).scatter_add_(1, parent, first.long())
        free = taken.sort(dim=1, stable=True).indices
        slot = torch.where(first, parent, free.gather(1, ((~first).cumsum(1) - 1).clamp(min=0)))
        value, parent, token = (torch.empty_like(t).scatter_(1, slot, t) for t in (value, parent, token))
    got = {"scores": value.float(), "parents": parent.int(), "tokens": token.int()}
    if finished is not None:
        got["finished"] = finished.gather(1, parent) | (token == END)
    return got


def _run_own(case, state):
    from ceo_amd import nn
    from ceo_amd.state import reorder

    if case["op"] == "reorder":
        reorder(state["list"], state["parents"])
        return state["outs"] or state["states"]
    if case["op"] == "linear":
        return nn.linear_int8(state["x"], state["weight"], bias=state["bias"], residual=state["residual"], gelu=case["gelu"])
    finished = state["finished"]
    scores, parents, tokens, ended = nn.beam_select(
        state["logits"], state["scores"], select=case["select"], finished=finished,
        end_token=None if finished is None else END, keep_slots=case["keep"])
    got = {"scores": scores, "parents": parents, "tokens": tokens}
    if finished is not None:
        got["finished"] = ended
    return got


def work(case):
    if case["op"] == "reorder":
        p = _parents(case)
        if case["place"] == "out":
            moved = sum(len(np.unique(r)) + len(r) for r in p)
        else:
            change = p != np.arange(p.shape[1])
            moved = sum(len(np.unique(r[c])) + int(c.sum()) for r, c in zip(p, change))
        row = sum(math.prod(s[1:]) * torch.empty(0, dtype=dt).element_size() for s, dt in _state_shapes(case))
        return {"bytes": moved * row + p.size * 4, "flops": 0}
    size = SIZE[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        b = m * k * size + k * n + n * 4 + m * n * size * (2 if case["residual"] else 1) + (n * size if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * m * k * n}
    rows = case["batch"] * case["beams"]
    # a fifth of the beams but the first have finished where some have: their logits are not read
    live = rows - (case["batch"] * (case["beams"] - 1) // 5 if case["finished"] else 0)
    return {"bytes": live * case["vocab"] * size + rows * 4 + case["batch"] * case["select"] * 12,
            "flops": 4 * live * case["vocab"]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "reorder":
        # the beams' rows, gathered one by one on the host
        p = _parents(case)
        got = []
        for t in state["states"]:
            h = t.cpu()
            r = torch.stack([h[b * p.shape[1] + int(p[b, j])] for b in range(p.shape[0]) for j in range(p.shape[1])])
            got.append(r if t.dtype == torch.int32 else r.double())
        return got
    if case["op"] == "linear":
        x = state["x"].double()
        sx = (x.abs().max(dim=1).values / 127.0).float().double()
        w = state["weight"].double()
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for a in range(0, case["m"], 4096):
            q = torch.floor(x[a:a + 4096] / sx[a:a + 4096, None] + 0.5)
            # the nearest whole number, the even one where two are as near
            tie = (q - x[a:a + 4096] / sx[a:a + 4096, None] == 0.5) & (torch.remainder(q, 2.0) == 1.0)
            out[a:a + 4096] = torch.mm(q - tie.double(), w)
        y = sx[:, None] * out * state["scale"].double()
        if state["bias"] is not None:
            y = y + state["bias"].double()
        if case["gelu"]:
            y = torch.nn.functional.gelu(y, approximate="tanh")
        return y if state["residual"] is None else y + state["residual"].double()
    B, K, V, n = case["batch"], case["beams"], case["vocab"], case["select"]
    fin = state["finished"].cpu().numpy() if state["finished"] is not None else np.zeros((B, K), bool)
    scores = state["scores"].double()
    found = {"scores": [], "parents": [], "tokens": [], "finished": []}
    for b in range(B):
        v = torch.log_softmax(state["logits"][b * K:(b + 1) * K].double(), 1) + scores[b][:, None]
        for k in np.flatnonzero(fin[b]):
            v[k] = -math.inf
            v[k, END] = scores[b, k]
        v = v.reshape(-1)
        least = torch.topk(v, n).values[-1]
        i = torch.nonzero(v >= least)[:, 0]
        i, x = i.cpu().numpy(), v[i].cpu().numpy()
        order = np.lexsort((i, -x))[:n]
        i, x = i[order], x[order]
        if case["keep"]:
            slots, rest = [None] * K, []
            for c in range(n):
                if slots[i[c] // V] is None:
                    slots[i[c] // V] = c
                else:
                    rest.append(c)
            for s in range(K):
                if slots[s] is None:
                    slots[s] = rest.pop(0)
            i, x = i[slots], x[slots]
        found["scores"].append(x)
        found["parents"].append(i // V)
        found["tokens"].append(i % V)
        found["finished"].append(fin[b][i // V] | (i % V == END))
    got = {"scores": torch.from_numpy(np.array(found["scores"])),
           "parents": torch.from_numpy(np.array(found["parents"]).astype(np.int32)),
           "tokens": torch.from_numpy(np.array(found["tokens"]).astype(np.int32))}
    if case["finished"]:
        got["finished"] = torch.from_numpy(np.array(found["finished"]))
    return got
