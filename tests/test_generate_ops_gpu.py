"""Beam selection, state reordering and 8-bit integer products on the GPU.

Tolerances.  Selection: sums of exponentials are fp32 (a thread's up to 32 terms one by one, then
6 + 2 pairwise steps, each term's exponential off by 2 units and its argument d by 3 roundings, and
|d| e^d <= 0.37), so log sum exp is off by at most 64 * 2^-24; a score is that and its own
rounding.  Candidates whose values are nearer than twice that may change places.  Reordering is
exact.  Products: the whole numbers are exact, so what is left is 5 fp32 roundings of
each summand, the GELU's (its argument's and its own, 40 * 2^-24 of the value before it) and the type's
half step."""
import math

import numpy as np
import pytest
import torch

from helpers import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
LSE = 64 * U


def dev_rows(host, dtype, ld=None, offset=0):
    """Rows on the device with a stride, `offset` elements behind an allocation's start; what
    is around them is NaN."""
    rows, cols = host.shape
    ld = ld or cols
    flat = torch.full((offset + rows * ld + 64,), float("nan"), dtype=dtype, device="cuda")
    v = flat[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    v.copy_(host)
    return v


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------
def ref_values(z, scores, finished, end):
    """(batch, beams * vocab) float64."""
    B, K = scores.shape
    z = z.double()
    with np.errstate(all="ignore"):
        m = z.max(1, keepdim=True).values
        lse = m[:, 0] + (z - m).exp().sum(1).log()
    v = scores.double().reshape(-1, 1) + z - lse[:, None]
    dead = ~torch.isfinite(lse) | ~torch.isfinite(scores.reshape(-1)) | torch.isnan(z).any(1)
    if finished is not None:
        f = finished.reshape(-1)
        v[f] = -math.inf
        v[f, end] = scores.double().reshape(-1)[f]
        dead &= ~f | ~torch.isfinite(scores.reshape(-1))
    v[dead] = -math.inf
    return v.reshape(B, -1)


def ref_order(v, n):
    """The n best (value, flat index), ties to the lowest index."""
    out = []
    for row in v.numpy():
        at = np.lexsort((np.arange(row.size), -row))[:n]
        out.append(at)
    return np.stack(out)


def keep_slots(parents, beams):
    """rank -> slot"""
    to = []
    for p in parents:
        used, rest, t = set(), [], {}
        for r, k in enumerate(p):
            if k in used:
                rest.append(r)
            else:
                used.add(k)
                t[r] = k
        free = [k for k in range(beams) if k not in used]
        t.update(zip(rest, free))
        to.append([t[r] for r in range(len(p))])
    return np.array(to)


def check_select(z, scores, n, finished=None, end=None, keep=False, ld=None, offset=0, exact=False):
    from ceo_amd import nn

    B, K = scores.shape
    V = z.shape[1]
    dz = dev_rows(z, z.dtype, ld, offset)
    got = nn.beam_select(dz, scores.cuda(), n, None if finished is None else finished.cuda(), end,
                         keep)
    torch.cuda.synchronize()
    s, p, t = (x.cpu().numpy() for x in got[:3])
    v = ref_values(z, scores, finished, end).numpy()
    order = ref_order(torch.from_numpy(v), n)
    flat = p.astype(np.int64) * V + t
    if keep:
        # back into their order: by score, ties by place
        ranks = np.stack([np.lexsort((flat[b], -s[b])) for b in range(B)])
        to = keep_slots(np.take_along_axis(p, ranks, 1), K)
        assert (to == ranks).all()
        s, p, t, flat = (np.take_along_axis(x, ranks, 1) for x in (s, p, t, flat))
    for b in range(B):
        assert len(set(flat[b])) == n
        want, have = v[b, order[b]], v[b, flat[b]]
        same = order[b] == flat[b]
        if exact:
            assert same.all(), (order[b], flat[b])
        inf = np.isneginf(want)
        assert (np.isneginf(s[b]) == inf).all() and (same | ~inf).all()
        w, h = want[~inf], have[~inf]
        tol = LSE + U * np.abs(w)
        assert (np.abs(s[b][~inf] - h) <= tol).all()
        assert (np.abs(w - h) <= 2 * LSE + 2 * U * np.abs(w)).all()
        assert (same[~inf] | (np.abs(w - h) <= 2 * LSE)).all()
    if end is None:
        assert got[3] is None
    else:
        f = np.zeros((B, K), bool) if finished is None else finished.numpy()
        want = np.take_along_axis(f, got[1].cpu().numpy().astype(np.int64), 1) | \
            (got[2].cpu().numpy() == end)
        assert (got[3].cpu().numpy() == want).all()


def texts(B, K, V, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(B * K, V, generator=g) * scale).to(dtype)
    return z, -6.0 - 2.0 * torch.randn(B, K, generator=g).abs(), g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,n", [
    (1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 1, 3), (1, 4, 7, 8), (3, 2, 63, 4), (2, 5, 257, 5),
    (1, 4, 4099, 4), (2, 8, 5003, 16), (5, 16, 1000, 32), (1, 64, 300, 64), (2, 64, 129, 64),
    (1, 2, 50257, 64), (40, 4, 2048, 4), (300, 4, 9000, 8), (1, 1, 131072, 1), (2, 3, 128003, 6),
    # a text is one workgroup's up to 49152 logits, 16 beams and 32 selected
    (2, 4, 12288, 4), (2, 4, 12289, 4), (3, 16, 3071, 32), (3, 17, 500, 17), (3, 16, 500, 33),
    (2, 7, 7001, 14), (2, 1, 49153, 2), (600, 2, 300, 2),
])
def test_select(dtype, B, K, V, n):
    announce(f"select {dtype} {B} {K} {V} {n}")
    z, s, _ = texts(B, K, V, dtype, seed=B + K + V)
    check_select(z, s, n)
    check_select(z, s, n, ld=V + 13, offset=3)
    if n == K:
        check_select(z, s, n, keep=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 5, 8, 33, 64])
def test_select_alignments(dtype, offset):
    announce(f"select {dtype} offset {offset}")
    z, s, _ = texts(2, 3, 4321, dtype, seed=offset)
    check_select(z, s, 6, ld=4321 + offset % 7, offset=offset)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("V,end", [(11, 10), (5003, 2), (5003, 0)])
def test_select_finished(V, end, keep):
    z, s, g = texts(6, 4, V, torch.bfloat16, seed=V + end)
    fin = torch.rand(6, 4, generator=g) < 0.4
    fin[0] = True                        # nothing but the ends: -inf behind them
    fin[1] = False
    z[12:16] = float("nan")              # text 3: what finished beams hold is not read
    fin[3] = True
    check_select(z, s, 4, fin, end, keep)
    check_select(z, s, 4, None, end, keep)


def test_select_at_the_start():
    """All beams hold the prompt, one counts."""
    z, s, _ = texts(3, 5, 700, torch.float32)
    s[:, 1:] = -math.inf
    check_select(z, s, 5)
    check_select(z, s, 5, keep=True)
    check_select(z, s, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_select_masks(dtype):
    """Tokens that are ruled out, fewer of them left than are selected, and rows that have none."""
    z, s, _ = texts(4, 3, 5000, dtype, seed=5)
    ninf = -math.inf
    z[0:3] = ninf
    z[1, [17, 4000]] = torch.tensor([1.0, 2.0], dtype=dtype)  # text 0: two tokens of one beam
    z[3, 1:] = ninf                                           # one token: certain
    z[4, 100:] = ninf
    z[6:9] = ninf                                             # text 2: nothing at all
    z[9, 7] = float("nan")                                    # text 3: beams that offer nothing
    z[10, 4999] = math.inf
    check_select(z, s, 8)
    lowest = torch.finfo(dtype).min
    z[torch.isneginf(z)] = lowest
    z[0] = lowest                                             # all the same: uniform
    s[2] = ninf
    check_select(z, s, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 4, 64])
def test_select_ties(dtype, n):
    """Equal logits, in whole rows and in places, and -0 beside 0: the lowest token first."""
    s = torch.tensor([[-1.0, -1.0, -2.0, -1.5], [-3.0, -math.inf, -2.5, -2.5]])
    check_select(torch.zeros(2 * 4, 20480, dtype=dtype), s, n, exact=True)
    z = torch.zeros(2 * 4, 8192, dtype=dtype)
    check_select(z, s, n, exact=True)
    z[:, 5::2] = -0.0
    check_select(z, s, n, exact=True)
    z[:, 3000:] = 1.0
    check_select(z, s, n, exact=True)
    z[:, ::5] = -math.inf
    check_select(z, s, n, exact=True)


def test_select_sorted_rows():
    """Rising and falling logits: many pass a lane's bound."""
    V = 40000
    up = torch.arange(V).float().div(V) * 20
    z = torch.stack([up, up.flip(0), up, up])
    s = torch.tensor([[-1.0, -1.2, -1.7, -9.0]])
    for n in (4, 17, 64):
        check_select(z, s, n)
        check_select(z.bfloat16(), s, n)


def test_select_extreme_scores():
    z, s, _ = texts(2, 4, 999, torch.float32)
    s[0] = torch.tensor([math.nan, math.inf, -1e30, -3.0])
    z *= 30
    check_select(z, s, 7)


def test_select_repeats_and_streams():
    """The same bits each time, also beside itself on another stream, and the inputs stay."""
    from ceo_amd import nn

    z, s, _ = texts(7, 4, 30011, torch.bfloat16)
    z, s = z.cuda(), s.cuda()
    z0, s0 = z.clone(), s.clone()
    want = nn.beam_select(z, s, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = nn.beam_select(z, s, 8)
        b = nn.beam_select(z, s, 8)
        torch.cuda.synchronize()
        for x in (a, b):
            assert all(torch.equal(p, q) for p, q in zip(x[:3], want[:3]))
    assert torch.equal(z, z0) and torch.equal(s, s0)


def test_select_refusals():
    from ceo_amd import nn

    z, s, _ = texts(2, 3, 50, torch.bfloat16)
    z, s = z.cuda(), s.cuda()
    fin = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for bad in (lambda: nn.beam_select(z.cpu(), s), lambda: nn.beam_select(z.double(), s),
                lambda: nn.beam_select(z, s.double()), lambda: nn.beam_select(z, s[:1]),
                lambda: nn.beam_select(z, s.reshape(-1)), lambda: nn.beam_select(z[None], s),
                lambda: nn.beam_select(z.t(), s), lambda: nn.beam_select(z, s, 0),
                lambda: nn.beam_select(z, s, 65), lambda: nn.beam_select(z[:, :1], s, 4),
                lambda: nn.beam_select(z, s, 4, keep_slots=True),
                lambda: nn.beam_select(z, s, finished=fin),
                lambda: nn.beam_select(z, s, finished=fin.byte(), end_token=1),
                lambda: nn.beam_select(z, s, finished=fin[:1], end_token=1),
                lambda: nn.beam_select(z, s, end_token=50),
                lambda: nn.beam_select(z, s, end_token=-1),
                lambda: nn.beam_select(z[:1].expand(6, 50), s)):
        with pytest.raises(ValueError):
            bad()
    assert nn.beam_select(z[:0], s[:0])[0].shape == (0, 3)


# ---------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------
def states_of(rows, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return [r(rows, 2, 64, 64), r(rows, 5, 13).bfloat16(), r(rows, 1000),
            torch.randint(0, 9, (rows, 37), generator=g, device="cuda", dtype=torch.int32),
            torch.randint(0, 9, (rows, 7), generator=g, device="cuda").to(torch.uint8),
            r(rows) > 0, r(rows, 0)]


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("batch", [1, 3])
def test_reorder(beams, batch):
    from ceo_amd.state import StateList, reorder

    announce(f"reorder {batch} {beams}")
    g = torch.Generator().manual_seed(beams)
    rows = batch * beams
    for kind in ("any", "cycle", "same", "one", "outside"):
        p = {"any": torch.randint(0, beams, (batch, beams), generator=g),
             "cycle": ((torch.arange(beams) + 1) % beams).expand(batch, beams),
             "same": torch.arange(beams).expand(batch, beams),
             "one": torch.full((batch, beams), beams - 1),
             "outside": torch.randint(-3, beams + 3, (batch, beams), generator=g)}[kind]
        p = p.to(torch.int32).contiguous()
        p[:, 0] = p[:, 0] if kind != "outside" else 2 ** 31 - 1
        src = torch.where((p >= 0) & (p < beams), p, torch.arange(beams, dtype=torch.int32))
        src = (src + beams * torch.arange(batch)[:, None]).reshape(-1).cuda()
        st = states_of(rows)
        want = [t[src] for t in st]
        outs = [torch.full_like(t, 1) for t in st]
        old = [t.clone() for t in st]
        reorder(StateList(st, beams, outs), p.cuda())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(torch.equal(a, b) for a, b in zip(st, old))
        reorder(StateList(st, beams), p.cuda())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(st, want))


def test_reorder_writes_nothing_else():
    from ceo_amd.state import StateList, reorder

    flat = torch.arange(3 + 12 * 31 + 9, device="cuda", dtype=torch.int16)
    keep = flat.clone()
    t = flat[3:3 + 12 * 31].view(12, 31)  # rows of 62 bytes from byte 6 on
    p = torch.tensor([[1, 1, 0], [2, 0, 1], [0, 1, 2], [2, 2, 2]], dtype=torch.int32, device="cuda")
    rows = (p + 3 * torch.arange(4, device="cuda")[:, None]).reshape(-1).long()
    want = t[rows]
    reorder(StateList([t], 3), p)
    torch.cuda.synchronize()
    assert torch.equal(t, want)
    assert torch.equal(flat[:3], keep[:3]) and torch.equal(flat[-9:], keep[-9:])


def test_reorder_refusals():
    import copy

    from ceo_amd import HipError
    from ceo_amd.state import StateList, reorder

    a, b = torch.zeros(6, 4, device="cuda"), torch.zeros(6, 8, device="cuda")
    p = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for bad in (lambda: StateList([], 3), lambda: StateList([a], 4), lambda: StateList([a], 0),
                lambda: StateList([a.cpu()], 3), lambda: StateList([a, b[:3]], 3),
                lambda: StateList([a.t()], 2), lambda: StateList([a], 3, [b]),
                lambda: StateList([a], 3, [a.int()]), lambda: StateList([a, b], 3, [a]),
                lambda: StateList([torch.zeros(130, 1, device="cuda")], 65)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(HipError):
        StateList([a, a], 3)                       # the same memory twice
    with pytest.raises(HipError):
        StateList([a], 3, [a])                     # an output over its state
    flat = torch.zeros(60, device="cuda")
    with pytest.raises(HipError):
        StateList([flat[:24].view(6, 4), flat[20:44].view(6, 4)], 3)
    sl = StateList([a, b], 3)
    for bad in (p.long(), p[:1], p.cpu(), p.reshape(-1)):
        with pytest.raises(ValueError):
            reorder(sl, bad)
    with pytest.raises(TypeError):
        reorder([a], p)
    other = copy.copy(sl)
    assert other._handle.value != sl._handle.value
    reorder(other, p)
    reorder(StateList([a[:0]], 3), p[:0])


# ---------------------------------------------------------------------------
# 8-bit integer products
# ---------------------------------------------------------------------------
def quantized(x):
    """(whole numbers, scales) of the rows, float64."""
    x = x.double()
    s = (x.abs().amax(1).float() * (torch.ones(()) / 127.0)).double()
    s = torch.where(torch.isfinite(s), s, torch.full_like(s, math.nan))
    q = torch.where(s[:, None] > 0, (x / s[:, None]).round().clamp(-127, 127), torch.zeros_like(x))
    return torch.nan_to_num(q), s


def gelu64(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))


def check_linear(x, w, bias=None, residual=None, gelu=False, ldx=None, offset=0, ldr=None):
    from ceo_amd import nn

    dt = x.dtype
    qx, sx = quantized(x)
    qw, sw = quantized(w.t())
    prod = (qx @ qw.t()) * sx[:, None] * sw[None, :]
    size = prod.abs()
    y = prod
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    tol = 5 * U * size
    if gelu:
        tol = 1.2 * tol + 40 * U * y.abs()
        y = gelu64(y)
    if residual is not None:
        y = y + residual.double()
        tol = tol + U * (y.abs() + residual.double().abs())
    tol = tol + torch.finfo(dt).eps / 2 * (y.abs() + tol) + \
        {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40, torch.float32: 1e-44}[dt]
    dx = dev_rows(x, dt, ldx, offset)
    r = None if residual is None else dev_rows(residual, dt, ldr, offset)
    got = nn.linear_int8(dx, nn.Int8Weight(w.cuda()), None if bias is None else bias.cuda(), r,
                         gelu)
    torch.cuda.synchronize()
    assert got.dtype == dt and got.shape == y.shape
    got = got.double().cpu()
    nan = torch.isnan(y)
    assert torch.equal(torch.isnan(got), nan)
    off = (got - y).abs()
    assert bool((off <= tol)[~nan].all()), float((off / tol)[~nan].max())
    return got


def operands(m, k, n, dtype, seed=0, wdtype=None):
    g = torch.Generator().manual_seed(seed + m + k + n)
    x = torch.randn(m, k, generator=g) * torch.where(torch.rand(k, generator=g) < 0.02, 8.0, 1.0)
    w = torch.randn(k, n, generator=g) * 0.05
    return (x.to(dtype), w.to(wdtype or dtype), torch.randn(n, generator=g).to(dtype),
            torch.randn(m, n, generator=g).to(dtype))


SIZES = [(1, 1, 1), (1, 64, 64), (3, 17, 5), (4, 1024, 1024), (16, 128, 16), (17, 129, 33),
         (33, 500, 100), (64, 1000, 257), (5, 5000, 48), (16, 4096, 1024), (48, 4096, 130),
         (65, 1, 3), (65, 128, 128), (100, 1001, 300), (257, 640, 511), (1000, 130, 1030),
         (300, 2048, 8), (129, 8200, 136)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(dtype, m, k, n):
    announce(f"linear {dtype} {m} {k} {n}")
    x, w, b, r = operands(m, k, n, dtype)
    check_linear(x, w)
    check_linear(x, w, b, r, gelu=True)
    check_linear(x, w, b, ldx=k + 3, offset=1)
    check_linear(x, w, None, r, ldr=n + 5, offset=3)


@pytest.mark.parametrize("m", [2, 70])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_weight_types_and_strides(m, dtype):
    for wdt in TYPES:
        x, w, b, _ = operands(m, 200, 72, dtype, wdtype=wdt)
        check_linear(x, w, b)
    from ceo_amd import nn

    big = torch.randn(200, 100, device="cuda").bfloat16()
    a, c = nn.Int8Weight(big[:, 20:92]), nn.Int8Weight(big[:, 20:92].contiguous())
    assert torch.equal(a.packed[:72 * 4], c.packed[:72 * 4])
    x = torch.randn(m, 200, device="cuda").to(dtype)
    assert torch.equal(nn.linear_int8(x, a), nn.linear_int8(x, c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(500, 1100, 4000), (520, 1024, 4096), (33, 3000, 1000),
                                   (1000, 136, 2040), (64, 200, 16385), (512, 4096, 1024)])
def test_linear_in_between(m, k, n, dtype):
    """Outputs of few tiles: one or two of 64 x 64 to a compute unit, or one of 128 x 128."""
    x, w, b, r = operands(m, k, n, dtype)
    check_linear(x, w, b, r, gelu=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_large(dtype):
    x, w, b, r = operands(2100, 1024, 3088, dtype)
    check_linear(x, w, b, r, gelu=True)


@pytest.mark.parametrize("m", [3, 40, 100])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_special_rows(m, dtype):
    """Rows and channels of zeros, of one value, with NaN and infinities, tiny and huge ones."""
    x, w, b, r = operands(m, 300, 40, dtype)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 7] = float("-inf")
    w[:, 3] = 0
    w[9, 4] = float("nan")
    w[9, 6] = float("inf")
    check_linear(x, w, b, r)
    if m > 3:
        x[3] = torch.finfo(dtype).tiny
        x[4] = torch.finfo(dtype).max / 4
        x[5] = 0
        x[5, 299] = -2.0
        w[:, 4] = 0.5
        w[:, 6] = 0
        w[:, 7] = -torch.finfo(dtype).tiny
        if dtype is torch.float16:  # what leaves its range
            x[4] = 16.0
        else:
            x[4] = 1e30
        check_linear(x, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(3, 300, 40), (40, 2000, 40), (100, 300, 40), (2100, 256, 3088)])
def test_linear_large_tokens_small_weights(m, k, n, dtype):
    """A sum times its token's scale is past fp32's range, the result is not."""
    x, w, b, r = operands(m, k, n, dtype)
    x, w = (x.float() * 4e36).to(dtype), (w.float() * 1e-36).to(dtype)
    x[0] = 0
    check_linear(x, w)
    check_linear(x, w, b, r)


@pytest.mark.parametrize("m", [1, 80])
def test_linear_quotients_on_halves(m):
    """Values on and next to half a step: to the even one, as the exact quotient decides.  The
    weight is one 127 a channel, so an output is 127 times the whole number times the scales."""
    k = 2048
    for scale in (1.0, 0.37, 3.1e-5):
        s = torch.tensor(127.0 * scale) * (torch.ones(()) / 127.0)
        steps = torch.arange(k).sub(k // 2).remainder(254).sub(127).double() + 0.5
        x = (steps * s.double()).float()
        i = torch.arange(k)
        up, down = torch.nextafter(x, x.abs() * 2 + 1), torch.nextafter(x, -x.abs() * 2 - 1)
        x = torch.where(i % 3 == 0, x, torch.where(i % 3 == 1, up, down)).clamp(-127 * s, 127 * s)
        x[0] = 127.0 * scale
        x = x[None].repeat(m, 1)
        q, sx = quantized(x)
        # each k in a channel of its own
        from ceo_amd import nn

        for c0 in range(0, k, 512):
            w = torch.zeros(k, 512)
            w[torch.arange(c0, c0 + 512), torch.arange(512)] = 127.0
            y = nn.linear_int8(x.cuda(), nn.Int8Weight(w.cuda())).double().cpu()
            got = (y / (127.0 * sx[:, None])).round()
            assert torch.equal(got, q[:, c0:c0 + 512])


def test_linear_long_sums():
    """The longest contraction, every product of the same sign: sums near 2^31."""
    k = 131072
    x = torch.ones(2, k, dtype=torch.bfloat16)
    w = torch.ones(k, 16, dtype=torch.bfloat16)
    w[:, 1] = -1.0
    check_linear(x, w)
    check_linear(x.repeat(33, 1), w)


def test_linear_rows_do_not_depend_on_each_other():
    """A row's bits are the same alone, among a few and among many."""
    from ceo_amd import nn

    x, w, b, r = (t.cuda() for t in operands(700, 1000, 300, torch.bfloat16))
    wt = nn.Int8Weight(w)
    full = nn.linear_int8(x, wt, b, r, gelu=True)
    for m in (1, 2, 16, 31, 64, 65, 300):
        assert torch.equal(nn.linear_int8(x[:m], wt, b, r[:m], gelu=True), full[:m])


def test_linear_refusals():
    from ceo_amd import nn

    x, w, b, r = (t.cuda() for t in operands(4, 32, 16, torch.bfloat16))
    wt = nn.Int8Weight(w)
    for bad in (lambda: nn.Int8Weight(w.cpu()), lambda: nn.Int8Weight(w.double()),
                lambda: nn.Int8Weight(w.t()), lambda: nn.Int8Weight(w[:0]),
                lambda: nn.Int8Weight(w[:, :0]), lambda: nn.Int8Weight(w[0]),
                lambda: nn.Int8Weight(torch.zeros(131073, 1, device="cuda")),
                lambda: nn.linear_int8(x.cpu(), wt), lambda: nn.linear_int8(x.double(), wt),
                lambda: nn.linear_int8(x[:, :31], wt), lambda: nn.linear_int8(x[0], wt),
                lambda: nn.linear_int8(x, wt, b.float()), lambda: nn.linear_int8(x, wt, b[:15]),
                lambda: nn.linear_int8(x, wt, None, r.float()),
                lambda: nn.linear_int8(x, wt, None, r[:3]),
                lambda: nn.linear_int8(x[:1].expand(4, 32), wt)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        nn.linear_int8(x, w)
    assert nn.linear_int8(x[:0], wt).shape == (0, 16)
    assert torch.equal(nn.linear_int8(x, wt, None, r[:1].expand(4, 16)),
                       nn.linear_int8(x, wt, None, r[:1].repeat(4, 1)))


def test_library_workspace_on_two_streams():
    """The C entries without a workspace: the library's, one for each stream, calls of both kinds
    sharing it in turn."""
    from ceo_amd import _lib, nn

    L = _lib.lib()
    B, K, V, n = 5, 4, 50257, 7
    g = torch.Generator(device="cuda").manual_seed(4)
    z = torch.randn(B * K, V, generator=g, device="cuda").half()
    scores = -torch.rand(B, K, generator=g, device="cuda")
    x = torch.randn(300, 1000, generator=g, device="cuda").bfloat16()
    wt = nn.Int8Weight(torch.randn(1000, 520, generator=g, device="cuda").bfloat16())
    want = nn.beam_select(z, scores, n)
    want_y = nn.linear_int8(x, wt)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                s = torch.empty(B, n, device="cuda")
                p, t = (torch.empty(B, n, dtype=torch.int32, device="cuda") for _ in range(2))
                y = torch.empty_like(want_y)
            h = st.cuda_stream
            assert L.beam_select_hip(z.data_ptr(), scores.data_ptr(), None, s.data_ptr(),
                                     p.data_ptr(), t.data_ptr(), None, B, K, V, V, n, -1, 0, 2, None,
                                     0, h) == 0
            assert L.linear_int8_hip(x.data_ptr(), 1000, wt.packed.data_ptr(), None, None, 0,
                                     y.data_ptr(), 520, 300, 1000, 520, 0, 14, None, 0, h) == 0
            outs.append((s, p, t, y))
    torch.cuda.synchronize()
    for s, p, t, y in outs:
        assert torch.equal(s, want[0]) and torch.equal(p, want[1]) and torch.equal(t, want[2])
        assert torch.equal(y, want_y)


# ---------------------------------------------------------------------------
# offsets past 32 bits
# ---------------------------------------------------------------------------
def test_select_past_32_bits():
    """5 GB of logits: texts at the end as when they are alone."""
    from ceo_amd import nn

    B, K, V = 2500, 8, 128003
    z = torch.empty(B * K, V, dtype=torch.float16, device="cuda").normal_(0, 2)
    scores = -torch.rand(B, K, device="cuda")
    got = nn.beam_select(z, scores)
    for b in (0, 2095, 2097, B - 1):  # 2^31 elements are 2097.1 texts
        alone = nn.beam_select(z[b * K:(b + 1) * K].clone(), scores[b:b + 1])
        # another cut into slices: sums in another order
        assert (got[0][b] - alone[0][0]).abs().max().item() <= 2 * LSE + 2 * U * 40
        assert torch.equal(got[1][b], alone[1][0]) and torch.equal(got[2][b], alone[2][0])


@pytest.mark.parametrize("outs", [False, True])
def test_reorder_past_32_bits(outs):
    """A state of 5 GB, rows of 640 MB."""
    from ceo_amd.state import StateList, reorder

    x = torch.arange(8 * 160_000_001, device="cuda", dtype=torch.int32).view(8, -1)
    y = torch.empty_like(x) if outs else x
    p = torch.tensor([[1, 0, 3, 3], [2, 9, 0, 1]], dtype=torch.int32, device="cuda")
    reorder(StateList([x], 4, [y] if outs else None), p)
    n = x.shape[1]
    for row, src in enumerate((1, 0, 3, 3, 6, 5, 4, 5)):
        for at in (0, 1, n // 2, n - 2, n - 1):
            v = (src * n + at) & 0xFFFFFFFF
            assert y[row, at].item() == (v - (1 << 32) if v >> 31 else v)
        d = y[row, 1:] - y[row, :-1]
        assert bool((d == 1).all())


@pytest.mark.parametrize("m,k,n", [(70001, 65536, 24), (600001, 128, 4096)])
def test_linear_past_32_bits(m, k, n):
    """4.6 GB of quantised tokens, 4.9 GB of output: rows as when they are alone."""
    from ceo_amd import nn

    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda").normal_()
    wt = nn.Int8Weight(torch.randn(k, n, device="cuda").bfloat16())
    y = nn.linear_int8(x, wt)
    for r in (0, 32767, 32769, 65535, 65537, m // 2, m - 300, m - 1):
        assert torch.equal(y[r:r + 1], nn.linear_int8(x[r:r + 1], wt))
    assert torch.equal(y[m - 300:], nn.linear_int8(x[m - 300:], wt))


def test_weight_past_32_bits():
    """A packed weight of 4.4 GB."""
    from ceo_amd import nn

    k, n = 131072, 33600
    w = torch.empty(k, n, dtype=torch.bfloat16, device="cuda").normal_()
    x = torch.randn(40, k, device="cuda").bfloat16()
    y = nn.linear_int8(x, nn.Int8Weight(w))
    for c in (0, 16384, n - 8):
        assert torch.equal(y[:, c:c + 8], nn.linear_int8(x, nn.Int8Weight(w[:, c:c + 8])))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_captured_and_replayed():
    """Head, selection and reordering in one graph, replayed on new inputs with eager work
    between, each replay against the eager calls."""
    from ceo_amd import nn
    from ceo_amd.state import StateList, reorder

    B, K, D, V = 3, 4, 96, 1003
    g = torch.Generator(device="cuda").manual_seed(3)
    wt = nn.Int8Weight(torch.randn(D, V, generator=g, device="cuda").bfloat16())
    h = torch.zeros(B * K, D, dtype=torch.bfloat16, device="cuda")
    big = torch.zeros(100, D, dtype=torch.bfloat16, device="cuda")
    scores = torch.zeros(B, K, device="cuda")
    fin = torch.zeros(B, K, dtype=torch.bool, device="cuda")
    st = [torch.randn(B * K, 2, 16, 16, generator=g, device="cuda"),
          torch.zeros(B * K, 9, dtype=torch.int32, device="cuda")]
    sl = StateList(st, K)

    def step():
        z = nn.linear_int8(h, wt)
        y = nn.linear_int8(big, wt)
        got = nn.beam_select(z, scores, finished=fin, end_token=5, keep_slots=True)
        reorder(sl, got[1])
        return got + (z, y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        h.copy_(torch.randn(B * K, D, generator=g, device="cuda"))
        big.copy_(torch.randn(100, D, generator=g, device="cuda"))
        scores.copy_(torch.randn(B, K, generator=g, device="cuda"))
        fin.copy_(torch.rand(B, K, generator=g, device="cuda") < 0.3)
        old = [t.clone() for t in st]
        graph.replay()
        torch.cuda.synchronize()
        got, moved = [t.clone() for t in out], [t.clone() for t in st]
        for t, o in zip(st, old):
            t.copy_(o)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(moved, st))
