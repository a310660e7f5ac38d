"""What the entry points for generating text refuse, through the C ABI, without a GPU: the
checks come before anything is launched."""
import ctypes

import pytest

from ceo_amd import _lib

NULL = None
P = ctypes.c_void_p(1 << 12)
Q = ctypes.c_void_p(1 << 20)
BIG = 1 << 62


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _select(L, z=P, s=P, fin=NULL, os=P, op=P, ot=P, of=NULL, batch=2, beams=3, vocab=100, ld=100,
            n=3, end=-1, keep=0, dt=14, ws=P, wsb=1 << 20):
    return L.beam_select_hip(z, s, fin, os, op, ot, of, batch, beams, vocab, ld, n, end, keep, dt,
                             ws, wsb, NULL)


def test_select_refusals(L):
    for name in ("z", "s", "os", "op", "ot"):
        assert _select(L, **{name: NULL}) == 1
    for dt in (1, 3, 99, -1):
        assert _select(L, dt=dt) == 1
    assert _select(L, z=ctypes.c_void_p(4097)) == 1
    assert _select(L, z=ctypes.c_void_p(4098), dt=0) == 1
    assert _select(L, beams=0) == 1 and _select(L, beams=65, n=3) == 1
    assert _select(L, n=0) == 1 and _select(L, n=65) == 1
    assert _select(L, vocab=0) == 1 and _select(L, ld=99) == 1
    assert _select(L, vocab=1, ld=1, n=4) == 1                   # fewer continuations than asked for
    assert _select(L, keep=1, n=4) == 1                          # slots are the beams'
    assert _select(L, fin=P) == 1 and _select(L, of=P) == 1      # without an end token
    assert _select(L, fin=P, end=100) == 1 and _select(L, of=P, end=-2) == 1
    big = dict(vocab=50000, ld=50000)
    need = L.beam_select_workspace_size(2, 3, 50000, 3)
    assert need > 0 and _select(L, wsb=need - 1, **big) == 1
    assert _select(L, ws=ctypes.c_void_p(4100), **big) == 1
    assert _select(L, vocab=1 << 30, ld=1 << 30) == 9
    assert _select(L, batch=BIG) == 9
    assert _select(L, ld=BIG) == 9
    assert _select(L, batch=0, z=NULL, s=NULL, os=NULL, op=NULL, ot=NULL, ws=NULL) == 0
    assert _select(L, batch=0, n=65) == 1


def test_select_workspace_holds_every_cut(L):
    """Monotonic in the vocabulary and the rows, 0 where a text is one workgroup's and out of
    range."""
    size = L.beam_select_workspace_size
    last = 0
    for v in (6145, 50257, 128003, 1 << 20):
        got = size(4, 8, v, 8)
        assert got >= max(last, 4 * 8 * (8 + 8 * 8))
        last = got
    assert size(4, 8, 6144, 8) == 0 and size(4, 8, 1, 8) == 0
    assert size(4, 17, 100, 8) > 0 and size(4, 8, 100, 33) > 0
    assert size(1, 65, 100, 3) == 0 and size(1, 3, 100, 65) == 0 and size(1, 3, 1 << 30, 3) == 0
    assert size(BIG, 3, 100, 3) == 0


def test_more_threads_than_a_launch_has(L):
    """A launch has fewer than 2^32 threads in a dimension: refused before any of them."""
    size = L.beam_select_workspace_size
    assert _select(L, batch=1 << 22, beams=1, n=1) == 9
    assert _select(L, batch=1 << 22, beams=1, n=1, vocab=60000, ld=60000) == 9
    assert size((1 << 22) - 1, 1, 60000, 1) > 0 and size(1 << 22, 1, 60000, 1) == 0
    assert _create(L, states=(4096,), rows=(4,), batch=1 << 24, beams=1) == 9
    assert _create(L, states=(4096, 1 << 40), rows=(1, 1), batch=1 << 23, beams=3) == 9
    assert _linear(L, m=1 << 24) == 9 and _linear(L, n=1 << 29, ldy=1 << 29) == 9
    assert L.linear_int8_workspace_size((1 << 24) - 1, 32, 16, 14) > 0
    assert L.linear_int8_workspace_size(1 << 24, 32, 16, 14) == 0
    assert L.int8_weight_size(1, 1 << 29) == 0 and L.int8_weight_size(1, (1 << 29) - 1) > 0
    assert _pack(L, n=1 << 29, ld=1 << 29) == 9


def _create(L, states=(4096, 1 << 20), outs=None, rows=(64, 8), batch=2, beams=3, count=None):
    h = ctypes.c_void_p(7)
    n = len(states)
    arr = (ctypes.c_void_p * n)(*states)
    out = None if outs is None else (ctypes.c_void_p * n)(*outs)
    rc = L.state_list_create_hip(ctypes.byref(h), arr, out, (ctypes.c_size_t * n)(*rows),
                                 n if count is None else count, batch, beams)
    assert rc == 0 or h.value is None
    return rc


def test_state_list_refusals(L):
    assert L.state_list_create_hip(NULL, NULL, NULL, NULL, 0, 1, 1) == 1
    h = ctypes.c_void_p()
    one = (ctypes.c_size_t * 1)(4)
    assert L.state_list_create_hip(ctypes.byref(h), NULL, NULL, one, 1, 1, 1) == 1
    assert L.state_list_create_hip(ctypes.byref(h), (ctypes.c_void_p * 1)(64), NULL, NULL, 1, 1,
                                   1) == 1
    assert _create(L, beams=0) == 1 and _create(L, beams=65) == 1
    assert _create(L, states=(4096, None)) == 1
    assert _create(L, outs=(1 << 22, None)) == 1
    assert _create(L, states=(4096, 4096 + 6 * 64 - 1)) == 1     # one byte shared
    assert _create(L, outs=(4096, 1 << 22)) == 1                 # an output over its state
    assert _create(L, outs=(1 << 22, 4096 + 8)) == 1             # over another's
    assert _create(L, batch=BIG) == 9 and _create(L, rows=(BIG, 8)) == 9
    assert _create(L, rows=(1 << 45, 8)) == 9
    assert _create(L, count=1 << 30) == 9
    assert L.state_list_destroy_hip(NULL) == 0
    assert L.state_reorder_hip(NULL, P, NULL) == 1


def _pack(L, w=P, ld=16, p=Q, k=32, n=16, dt=14):
    return L.int8_weight_pack_hip(w, ld, p, k, n, dt, NULL)


def _linear(L, x=P, ldx=32, p=Q, b=NULL, r=NULL, ldr=0, y=P, ldy=16, m=100, k=32, n=16, dt=14,
            ws=P, wsb=1 << 30):
    return L.linear_int8_hip(x, ldx, p, b, r, ldr, y, ldy, m, k, n, 0, dt, ws, wsb, NULL)


def test_weight_refusals(L):
    assert L.int8_weight_size(0, 4) == 0 and L.int8_weight_size(4, 0) == 0
    assert L.int8_weight_size(131073, 4) == 0 and L.int8_weight_size(4, 1 << 30) == 0
    assert L.int8_weight_size(1, 1) == 128 + 16 * 128            # a line of scales, 16 channels
    assert L.int8_weight_size(129, 33) == 256 + 48 * 256
    assert _pack(L, w=NULL) == 1 and _pack(L, p=NULL) == 1
    assert _pack(L, k=0) == 1 and _pack(L, n=0) == 1 and _pack(L, ld=15) == 1
    assert _pack(L, w=ctypes.c_void_p(4097)) == 1 and _pack(L, p=ctypes.c_void_p(4096 + 64)) == 1
    for dt in (1, 3, 99, -1):
        assert _pack(L, dt=dt) == 1
    assert _pack(L, k=131073) == 9 and _pack(L, n=1 << 30, ld=1 << 30) == 9
    assert _pack(L, ld=BIG) == 9


def test_linear_refusals(L):
    assert _linear(L, x=NULL) == 1 and _linear(L, p=NULL) == 1 and _linear(L, y=NULL) == 1
    assert _linear(L, ldx=31) == 1 and _linear(L, ldy=15) == 1
    assert _linear(L, r=P, ldr=15) == 1
    assert _linear(L, k=0) == 1 and _linear(L, n=0) == 1
    for dt in (1, 3, 99, -1):
        assert _linear(L, dt=dt) == 1
    odd = ctypes.c_void_p(4097)
    for name in ("x", "y", "b"):
        assert _linear(L, **{name: odd}) == 1
    assert _linear(L, r=odd, ldr=16) == 1
    assert _linear(L, p=ctypes.c_void_p(4096 + 64)) == 1
    need = L.linear_int8_workspace_size(100, 32, 16, 14)
    assert need > 0 and _linear(L, wsb=need - 1) == 1
    assert _linear(L, ws=ctypes.c_void_p(4104)) == 1
    assert _linear(L, k=131073, ldx=131073) == 9
    assert _linear(L, m=1 << 30) == 9 and _linear(L, n=1 << 30, ldy=1 << 30) == 9
    assert _linear(L, ldx=BIG) == 9
    assert _linear(L, m=0, x=NULL, p=NULL, y=NULL, ws=NULL) == 0
    assert L.linear_int8_workspace_size(1, 64, 64, 14) == 0      # quantised by the kernel itself
    assert L.linear_int8_workspace_size(100, 131073, 64, 14) == 0
    assert L.linear_int8_workspace_size(100, 64, 64, 5) == 0
