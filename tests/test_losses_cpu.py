"""Refusals of the policy and preference losses and of gradient lists, without a
GPU: they come before any HIP call, with the library's codes (0 success, 1 invalid
value, 9 invalid configuration)."""
import contextlib
import copy
import ctypes

import pytest
import torch

from ceo_amd import _lib, nn

NULL = None
P = ctypes.c_void_p(64)
BIG = 1 << 31


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _logprob(L, z=P, t=P, w=NULL, lp=P, rows=4, vocab=100, ld=100, dt=14):
    return L.token_logprob_forward_hip(z, t, w, lp, rows, vocab, ld, dt, NULL)


def _policy(L, z=P, t=P, a=P, old=P, ref=P, w=NULL, loss=P, lp=P, kl=P, g=P, rows=4, vocab=100,
            ld=100, ldg=100, lo=0.2, hi=0.2, kc=0.1, dt=14):
    if g is P:
        g = ctypes.c_void_p(4096)
    return L.policy_loss_forward_backward_hip(z, t, a, old, ref, w, loss, lp, kl, g, rows, vocab,
                                              ld, ldg, lo, hi, kc, dt, NULL)


def _preference(L, z=P, t=P, ref=P, w=NULL, cu=P, loss=P, r=P, lp=P, g=P, pairs=2, rows=4,
                vocab=100, ld=100, ldg=100, beta=0.1, eps=0.0, dt=14, ws=P, wsb=1 << 20):
    if g is P:
        g = ctypes.c_void_p(4096)
    return L.preference_loss_forward_backward_hip(z, t, ref, w, cu, loss, r, lp, g, pairs, rows,
                                                  vocab, ld, ldg, beta, eps, dt, ws, wsb, NULL)


@pytest.mark.parametrize("call", [_logprob, _policy, _preference])
def test_logits_refusals(L, call):
    assert call(L, z=NULL) == 1
    assert call(L, t=NULL) == 1
    assert call(L, lp=NULL) == 1
    assert call(L, vocab=0) == 1
    assert call(L, ld=99) == 1
    assert call(L, z=ctypes.c_void_p(65)) == 1          # half an element
    assert call(L, z=ctypes.c_void_p(66), dt=0) == 1
    for dt in (1, 3, 99, -1):
        assert call(L, dt=dt) == 1
    assert call(L, rows=BIG) == 9
    assert call(L, vocab=BIG, ld=BIG, **({} if call is _logprob else {"ldg": BIG})) == 9


def test_no_rows(L):
    assert _logprob(L, z=NULL, t=NULL, lp=NULL, rows=0) == 0
    assert _policy(L, z=NULL, t=NULL, a=NULL, loss=NULL, lp=NULL, rows=0) == 0
    assert _preference(L, z=NULL, t=NULL, lp=NULL, cu=NULL, loss=NULL, r=NULL, rows=0,
                       pairs=0) == 0


def test_policy_refusals(L):
    nan, inf = float("nan"), float("inf")
    assert _policy(L, a=NULL) == 1
    assert _policy(L, loss=NULL) == 1
    assert _policy(L, ref=NULL) == 1                     # a KL term without its reference
    assert _policy(L, ref=NULL, kc=0.0) == 1             # kl asked for without it
    assert _policy(L, lo=-0.1) == 1 and _policy(L, lo=1.5) == 1 and _policy(L, lo=nan) == 1
    assert _policy(L, hi=-0.1) == 1 and _policy(L, hi=nan) == 1
    assert _policy(L, kc=-1.0) == 1 and _policy(L, kc=nan) == 1 and _policy(L, kc=inf) == 1
    assert _policy(L, ldg=99) == 1
    assert _policy(L, g=P, z=ctypes.c_void_p(4096), ldg=104) == 1  # in place, another stride
    assert _policy(L, g=ctypes.c_void_p(4097)) == 1


def test_preference_refusals(L):
    nan, inf = float("nan"), float("inf")
    assert _preference(L, cu=NULL) == 1
    assert _preference(L, loss=NULL) == 1
    assert _preference(L, r=NULL) == 1
    for b in (0.0, -0.1, nan, inf):
        assert _preference(L, beta=b) == 1
    for e in (-0.1, 1.0, nan):
        assert _preference(L, eps=e) == 1
    assert _preference(L, pairs=1 << 30) == 9
    need = L.preference_loss_workspace_size(4)
    assert need > 0 and _preference(L, wsb=need - 1) == 1
    assert _preference(L, ws=ctypes.c_void_p(68)) == 1   # unaligned workspace
    assert L.preference_loss_workspace_size(BIG) == 0


def test_preference_without_rows_refuses_an_unknown_type(L):
    for dt in (1, 3, 99, -1):
        assert _preference(L, z=NULL, t=NULL, lp=NULL, g=NULL, rows=0, dt=dt) == 1


def test_grad_list_refusals(L):
    h = ctypes.c_void_p()
    ptrs = (ctypes.c_void_p * 2)(64, 128)
    nums, dts = (ctypes.c_size_t * 2)(8, 8), (ctypes.c_int * 2)(14, 0)
    make = L.grad_list_create_hip
    assert make(NULL, ptrs, NULL, nums, dts, 2) == 1
    assert make(ctypes.byref(h), NULL, NULL, nums, dts, 2) == 1
    assert make(ctypes.byref(h), ptrs, NULL, NULL, dts, 2) == 1
    assert make(ctypes.byref(h), ptrs, NULL, nums, NULL, 2) == 1
    assert make(ctypes.byref(h), ptrs, NULL, nums, (ctypes.c_int * 2)(14, 5), 2) == 1
    assert make(ctypes.byref(h), (ctypes.c_void_p * 2)(64, None), NULL, nums, dts, 2) == 1
    assert make(ctypes.byref(h), ptrs, (ctypes.c_void_p * 2)(64, None), nums, dts, 2) == 1
    assert make(ctypes.byref(h), (ctypes.c_void_p * 2)(65, 128), NULL, nums, dts, 2) == 1
    assert make(ctypes.byref(h), (ctypes.c_void_p * 2)(64, 130), NULL, nums, dts, 2) == 1
    assert make(ctypes.byref(h), ptrs, NULL, (ctypes.c_size_t * 2)(8, 1 << 47), dts, 2) == 9
    assert make(ctypes.byref(h), ptrs, NULL, (ctypes.c_size_t * 2)(1 << 45, 1 << 45), dts, 2) == 9
    assert h.value is None
    assert L.grad_list_destroy_hip(NULL) == 0
    assert L.grad_norm_hip(NULL, 1.0, P, P, NULL) == 1
    assert L.grad_clip_hip(NULL, 1.0, P, NULL) == 1


def test_copies_of_a_grad_list_have_their_own_table(monkeypatch):
    """A copy (of a model that keeps a list, say) makes and frees a table of its own; a deep
    copy holds the copied gradients.  The library is a stand-in that counts."""
    made, freed = [], []

    class Counts:
        def grad_list_create_hip(self, handle, ptrs, *rest):
            made.append(64 * (len(made) + 1))
            handle._obj.value = made[-1]
            return 0

        def grad_list_destroy_hip(self, handle):
            freed.append(handle.value)
            return 0

    counts = Counts()
    monkeypatch.setattr(nn, "lib", lambda: counts)
    monkeypatch.setattr(nn, "_require", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    flat = torch.ones(6)
    lists = [nn.GradList([flat], [flat])]
    try:
        lists.append(copy.copy(lists[0]))
        assert lists[1].grads[0] is flat and lists[1].outs[0] is flat
        deep = copy.deepcopy({"flat": flat, "list": lists[0]})
        lists.append(deep["list"])
        assert deep["list"].grads[0] is deep["flat"] is deep["list"].outs[0] is not flat
    finally:
        for gl in lists:
            gl.__del__()
    assert len(made) == 3 and sorted(freed) == made


def test_adamw_scaled_refusals(L):
    ok = (3e-4, 0.9, 0.999, 1e-8, 0.1, 1)
    f = L.adamw_step_master_scaled_hip
    assert f(NULL, NULL, NULL, NULL, NULL, NULL, 0, *ok, NULL) == 0
    assert f(P, P, NULL, P, P, NULL, 8, *ok, NULL) == 1
    assert f(P, NULL, P, P, P, NULL, 8, *ok, NULL) == 1
    assert f(P, P, P, P, P, NULL, 8, 3e-4, 1.0, 0.999, 1e-8, 0.1, 1, NULL) == 1


def test_python_refusals():
    """Wrong tensors are refused before the library is called."""
    z, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32)
    for f in (lambda: nn.token_logprob_forward(z, t),
              lambda: nn.policy_loss_forward_backward(z, t, z[:, 0]),
              lambda: nn.preference_loss_forward_backward(z, t, t),
              lambda: nn.GradList([z]), lambda: nn.GradList([])):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        nn.token_logprob_forward(None, t)
