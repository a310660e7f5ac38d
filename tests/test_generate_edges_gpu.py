"""Beam selection where it can go wrong: logits far from zero, scores far below.

Tolerance of a selection's scores, in units of 2^-24: a sum of exponentials has at most 64 terms added one by one
in a thread (8 vectors of 8; in the one-launch form at most 32 between two rescalings of 5 units, 4 of
them, or 16 and 7), 6 + 3 steps of a wave and a workgroup, and four exponentials on a term's way (its
own and three rescalings) of 1 each, 3 roundings of an argument d that e^d weighs (|d| e^d <= 0.37)
and a product's 1: 63 + 9 + 4 * 3.2 < 128.  The score's own rounding is half a unit of it.  Within a
beam the order is that of the logits, whatever the sum."""
import math

import numpy as np
import pytest
import torch

from helpers import announce
from test_generate_ops_gpu import dev_rows

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
LSE = 128 * U


def values(z, scores):
    """(beams * vocab,) float64 of one text: score + ((z - max z) - log sum exp(z - max z)); a beam without a
    finite sum or score: -inf."""
    z = z.double()
    m = z.max(1, keepdim=True).values
    d = z - m
    v = (d - d.exp().sum(1, keepdim=True).log()) + scores.double()[:, None]
    v[~torch.isfinite(scores) | ~torch.isfinite(m[:, 0]) | torch.isnan(z).any(1)] = -math.inf
    return v.reshape(-1).numpy()


def check(z, scores, n):
    """Against `values`, text by text; each beam's tokens are the first of its order by logit and token."""
    from ceo_amd import nn

    B, K = scores.shape
    V = z.shape[1]
    s, p, t = (x.cpu().numpy() for x in nn.beam_select(dev_rows(z, z.dtype), scores.cuda(), n)[:3])
    for b in range(B):
        zb = z[b * K:(b + 1) * K]
        v = values(zb, scores[b])
        flat = p[b].astype(np.int64) * V + t[b]
        want = -np.sort(-v)[:n]
        have = v[flat]
        assert len(set(flat)) == n
        inf = np.isneginf(want)
        assert (np.isneginf(have) == inf).all() and (np.isneginf(s[b]) == inf).all()
        off = np.abs(s[b][~inf] - have[~inf])
        assert (off <= LSE + U * np.abs(have[~inf])).all(), off.max()
        assert (np.abs(want - have)[~inf] <= 2 * LSE + 4e-16 * np.abs(want[~inf])).all()
        rest = np.setdiff1d(np.flatnonzero(np.isneginf(v)), flat[~inf])
        assert (flat[inf] == rest[:inf.sum()]).all()
        for k in range(K):
            mine = t[b][~inf][p[b][~inf] == k]
            row = zb[k].double().numpy() + 0.0
            order = np.lexsort((np.arange(V), -row))
            assert (mine == order[:len(mine)]).all(), (k, mine, order[:len(mine)])


def text(B, K, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(B * K, V, generator=g) * 2.5).to(dtype)
    return z, -6.0 - 2.0 * torch.randn(B, K, generator=g).abs()


# one workgroup a text, and slices: many logits, many beams, many selected
SHAPES = [(2, 3, 5000, 4), (2, 3, 30011, 4), (1, 17, 700, 17), (1, 4, 9000, 40), (40, 8, 60000, 8)]


def masks(dtype):
    if dtype is torch.float16:
        return [-6e4, torch.finfo(dtype).min]
    return [-1e6, -3e7, -1e9, -5e9, -1e10, -1e20, -1e30, -1e32, -1e37, torch.finfo(dtype).min]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,n", SHAPES)
def test_masked_runs(dtype, B, K, V, n):
    """Finite masks over runs of tokens and over all but a few."""
    for mask in masks(dtype):
        announce(f"masked runs {dtype} {B} {K} {V} {mask}")
        z, s = text(min(B, 2), K, V, dtype, K + V)
        z[:, V // 5:V // 2] = mask
        z[0, 7:] = mask
        z[1, ::2] = mask
        z = z.repeat(-(-B * K // z.shape[0]), 1)[:B * K]
        s = s.repeat(-(-B // s.shape[0]), 1)[:B]
        check(z, s, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,n", SHAPES[:4])
def test_masked_rows(dtype, B, K, V, n):
    """Beams that a finite mask leaves nothing are uniform, at their own score: behind the live ones."""
    for mask in masks(dtype) + [-m for m in masks(dtype)]:
        announce(f"masked rows {dtype} {B} {K} {V} {mask}")
        z, s = text(B, K, V, dtype, K * V)
        z[0] = mask
        z[K - 1] = mask
        check(z, s, n)
        z[:] = mask
        check(z, s, n)
        z[:, 3] = 0.0  # one token far above the rest, or far below
        check(z, s, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V,n", SHAPES[:4])
def test_logits_far_from_zero(dtype, B, K, V, n):
    """Around one large value, and spread over many magnitudes."""
    for far in (1e3, 1e6, 2e7, 3e8, 1e10, 1e14, 1e16, 1e30):
        announce(f"far {dtype} {B} {K} {V} {far}")
        z, s = text(B, K, V, torch.float32, K + n)
        check((z + far).to(dtype), s, n)
        check((z - far).to(dtype), s, n)
        check((z * far).to(dtype), s, n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,V,n", SHAPES[:4])
def test_beams_far_below(dtype, B, K, V, n):
    """Scores and logits beside which 64 bits do not hold a token's part: the beam's own order stays."""
    announce(f"far below {dtype} {B} {K} {V}")
    z, s = text(B, K, V, dtype, 3 * K + n)
    s[:, 1:] = -1e30
    check(z, s, n)
    s[:] = -1e9
    check(z, s, n)
    if dtype is not torch.float16:
        z[:, 11] = 1e30
        check(z, s, n)


@pytest.mark.parametrize("B,K,V,n", SHAPES[:4])
def test_first_of_more(B, K, V, n):
    """A selection is the start of a larger one, also where 64 bits do not tell a beam's values apart."""
    from ceo_amd import nn

    z, s = text(B, K, V, torch.float32, n)
    z[:, V // 3:] *= 1e-20
    s[:, 0] = -1e20
    z, s = z.cuda(), s.cuda()
    more = nn.beam_select(z, s, 64)
    for m in (1, 2, n, 31, 33):
        few = nn.beam_select(z, s, m)
        assert all(torch.equal(a, b[:, :m]) for a, b in zip(few[1:3], more[1:3])), m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,n", [(4, 4), (17, 3), (8, 64)])
def test_workspace_of_the_size_asked_for(dtype, K, n):
    """Rows and vocabularies on both sides of where a thread takes 1, 2, 4 or 8 vectors: the same results, and nothing
    is written behind the workspace."""
    from ceo_amd import _lib, nn

    L = _lib.lib()
    code = {torch.bfloat16: 14, torch.float16: 2, torch.float32: 0}[dtype]
    size = 4 if dtype is torch.float32 else 2
    g = torch.Generator(device="cuda").manual_seed(n)
    for rows in (K, 12 * K, 30 * K, 150 * K, 600 * K):
        for v in (1, 2, 4, 8):
            slices = max(1, 1024 // rows)
            for V in {max(slices * 4096 * v // size + d, 50) for d in (-64, -1, 0, 1, 2050)}:
                if rows * V * size > 1 << 30:
                    continue
                announce(f"workspace {dtype} {rows} {K} {V} {n}")
                z = torch.empty(rows * V + 3, dtype=dtype, device="cuda").normal_(generator=g)[3:].view(rows, V)
                s = -torch.rand(rows // K, K, generator=g, device="cuda")
                need = L.beam_select_workspace_size(rows // K, K, V, n)
                ws = torch.full((need + 4096,), 171, dtype=torch.uint8, device="cuda")
                want = nn.beam_select(z, s, n)
                a = torch.empty(rows // K, n, device="cuda")
                p, t = (torch.empty(rows // K, n, dtype=torch.int32, device="cuda") for _ in range(2))
                assert L.beam_select_hip(z.data_ptr(), s.data_ptr(), None, a.data_ptr(), p.data_ptr(), t.data_ptr(), None,
                                         rows // K, K, V, V, n, -1, 0, code, ws.data_ptr(), need,
                                         torch.cuda.current_stream().cuda_stream) == 0
                assert all(torch.equal(x, y) for x, y in zip((a, p, t), want))
                assert bool((ws[need:] == 171).all())


@pytest.mark.parametrize("B,K,V", [(300, 4, 1000), (300, 5, 20000), (3, 64, 3000)])
@pytest.mark.parametrize("keep", [False, True])
def test_marks_in_place(B, K, V, keep):
    from ceo_amd import _lib, nn

    announce(f"marks in place {B} {K} {V}")
    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randn(B * K, V, generator=g, device="cuda").bfloat16()
    scores = -torch.rand(B, K, generator=g, device="cuda") * 12
    for _ in range(3):
        fin = torch.rand(B, K, generator=g, device="cuda") < 0.4
        want = nn.beam_select(z, scores, finished=fin, end_token=3, keep_slots=keep)
        s, p, t = (torch.empty_like(x) for x in want[:3])
        assert _lib.lib().beam_select_hip(z.data_ptr(), scores.data_ptr(), fin.data_ptr(), s.data_ptr(), p.data_ptr(),
                                          t.data_ptr(), fin.data_ptr(), B, K, V, V, K, 3, int(keep), 14, None, 0,
                                          torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((s, p, t, fin), want))


@pytest.mark.parametrize("K,V,dtype", [(64, 64, torch.float32), (64, 64, torch.bfloat16), (128, 256, torch.bfloat16)])
def test_states_in_place_up_to_the_last_step(K, V, dtype):
    from ceo_amd import efla

    g = torch.Generator(device="cuda").manual_seed(K + V)
    for T in (1, efla.STEP_TOKENS, efla.STEP_TOKENS + 1):
        q, k = (torch.randn(3, T, 2, K, generator=g, device="cuda").to(dtype) for _ in range(2))
        v = torch.randn(3, T, 2, V, generator=g, device="cuda").to(dtype)
        beta = torch.rand(3, T, 2, generator=g, device="cuda").to(dtype)
        s0 = torch.randn(3, 2, K, V, generator=g, device="cuda")
        o, st = efla.chunk_efla_fwd(q, k, v, beta, s0, True)
        mine = s0.clone()
        if T > efla.STEP_TOKENS:
            with pytest.raises(ValueError):
                efla.chunk_efla_fwd(q, k, v, beta, mine, out_state=mine)
            continue
        o2, _ = efla.chunk_efla_fwd(q, k, v, beta, mine, out_state=mine)
        assert torch.equal(mine, st) and torch.equal(o, o2)
