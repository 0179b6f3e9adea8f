"""The losses' entry points without a GPU: what they refuse, they refuse before anything is launched."""
import ctypes as C
import math

import pytest
import torch

from molla_b200 import capi, losses

P = C.c_void_p(4096)   # an aligned address that nothing may touch: every call below ends before a launch
FAR = C.c_void_p(1 << 40)
NULL = C.c_void_p(None)


def block(logits=P, kind=0, stride=8, B=2, V=8, tokens=P, temperature=NULL):
    return [logits, kind, stride, B, V, tokens, temperature]


def score(L, *a, logprob=P, status=P, **k):
    return L.molla_sample_token_logprobs(*block(*a, **k), NULL, logprob, NULL, NULL, status)


def backward(L, stats=P, entropy=P, g=P, h=P, grad=FAR, grad_stride=8, **k):
    return L.molla_sample_token_logprobs_backward(*block(**k), stats, entropy, g, h, NULL, grad, grad_stride)


def policy(L, old=P, adv=P, ref=P, low=0.2, high=0.2, kl=0.1, ent=0.0, scale=1.0, grad_scale=1.0, loss=P, row=P, logprob=P,
           kl_out=NULL, grad=FAR, grad_stride=8, status=P, **k):
    return L.molla_sample_policy_loss(*block(**k), old, adv, NULL, ref, low, high, kl, ent, scale, grad_scale, NULL, loss, row,
                                      logprob, NULL, kl_out, NULL, grad, grad_stride, status)


def preference(L, off=P, pairs=1, beta=0.1, smoothing=0.0, scale=1.0, grad_scale=1.0, ws=P, ws_bytes=1 << 20, loss=P, pair=P,
               margin=P, ratio=P, logprob=P, grad=FAR, grad_stride=8, status=P, pair_status=P, **k):
    return L.molla_sample_preference_loss(*block(**k), off, pairs, NULL, NULL, beta, smoothing, scale, grad_scale, ws, ws_bytes, NULL,
                                          loss, pair, margin, ratio, logprob, grad, grad_stride, status, pair_status)


@pytest.mark.parametrize("call", [score, backward, policy, preference])
@pytest.mark.parametrize("bad,code", [
    (dict(logits=NULL), capi.ERR_ARGUMENT), (dict(tokens=NULL), capi.ERR_ARGUMENT), (dict(kind=3), capi.ERR_ARGUMENT),
    (dict(kind=-1), capi.ERR_ARGUMENT), (dict(B=-1), capi.ERR_ARGUMENT), (dict(B=2**30 + 1), capi.ERR_ARGUMENT), (dict(V=0), capi.ERR_ARGUMENT),
    (dict(stride=7), capi.ERR_ARGUMENT), (dict(V=720897, stride=720897), capi.ERR_VOCAB),
    (dict(logits=C.c_void_p(4098)), capi.ERR_ARGUMENT), (dict(kind=1, logits=C.c_void_p(4097)), capi.ERR_ARGUMENT)])
def test_blocks_against_the_rules(lib, call, bad, code):
    assert call(lib, **bad) == code
    assert capi.last_error()


@pytest.mark.parametrize("call,names", [
    (score, ["logprob", "status"]), (backward, ["stats", "g", "grad", "entropy"]),
    (policy, ["old", "adv", "loss", "row", "logprob", "status", "ref"]),
    (preference, ["off", "loss", "pair", "margin", "ratio", "logprob", "status", "pair_status"])])
def test_missing_arrays(lib, call, names):
    for n in names:
        assert call(lib, **{n: NULL}) == capi.ERR_ARGUMENT, n
        assert capi.last_error()


def test_a_kl_output_needs_reference_logprobs(lib):
    assert policy(lib, kl=0.0, ref=NULL, kl_out=P) == capi.ERR_ARGUMENT


@pytest.mark.parametrize("call,bad", [
    (policy, dict(low=-0.1)), (policy, dict(high=-0.1)), (policy, dict(low=math.nan)), (policy, dict(kl=math.inf)),
    (policy, dict(ent=math.nan)), (policy, dict(scale=math.inf)), (policy, dict(grad_scale=math.nan)),
    (preference, dict(beta=0.0)), (preference, dict(beta=-1.0)), (preference, dict(beta=math.inf)), (preference, dict(beta=math.nan)),
    (preference, dict(smoothing=-0.01)), (preference, dict(smoothing=0.51)), (preference, dict(smoothing=math.nan)),
    (preference, dict(scale=math.nan)), (preference, dict(grad_scale=math.inf))])
def test_settings_against_the_rules(lib, call, bad):
    assert call(lib, **bad) == capi.ERR_CONFIG
    assert capi.last_error()


def test_the_preference_workspace(lib):
    need = lib.molla_sample_preference_workspace_bytes(2)
    assert need > 0 and lib.molla_sample_preference_workspace_bytes(-1) == capi.ERR_ARGUMENT
    assert preference(lib, ws=NULL) == capi.ERR_WORKSPACE
    assert preference(lib, ws_bytes=need - 1) == capi.ERR_WORKSPACE
    assert preference(lib, ws=C.c_void_p(4100)) == capi.ERR_ARGUMENT
    assert preference(lib, pairs=-1) == capi.ERR_ARGUMENT
    assert lib.molla_sample_preference_workspace_bytes(2**31 - 1) > 2**34


@pytest.mark.parametrize("call", [backward, policy, preference])
def test_the_gradient_takes_the_logits_place_or_stays_clear_of_them(lib, call):
    at = lambda n: C.c_void_p(4096 + 4 * n)
    for grad, stride in ((at(8), 8), (at(-8), 8), (at(1), 8), (at(0), 9), (at(15), 8)):   # two rows of eight fp32 logits
        assert call(lib, grad=grad, grad_stride=stride) == capi.ERR_ARGUMENT
        assert "overlaps" in capi.last_error()
    # rows that interleave: a step of twenty, eight logits and eight of the gradient, but for one that they share
    assert call(lib, stride=20, grad=at(7), grad_stride=20) == capi.ERR_ARGUMENT
    assert call(lib, stride=20, grad=at(13), grad_stride=20) == capi.ERR_ARGUMENT
    assert call(lib, stride=20, grad=at(8), grad_stride=21) == capi.ERR_ARGUMENT
    assert call(lib, grad_stride=7) == capi.ERR_ARGUMENT
    assert call(lib, grad=C.c_void_p((1 << 40) + 2)) == capi.ERR_ARGUMENT


def test_the_python_side_refuses_tensors_that_do_not_fit():
    f = lambda *s: torch.zeros(s)
    tok = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        losses.token_logprobs(f(2, 8), tok)
    with pytest.raises(ValueError, match="CUDA"):
        losses.policy_loss(f(2, 8), tok, f(2), f(2))
    with pytest.raises(ValueError, match="CUDA"):
        losses.preference_loss(f(2, 8), tok, torch.zeros(3, dtype=torch.int32))


def test_the_forms_with_a_depth_refuse_what_the_others_do(lib):
    def score_depth(logprob=P, status=P, depth=P, **k):
        return lib.molla_sample_token_logprobs_with_depth(*block(**k), NULL, logprob, NULL, depth, NULL, status)

    def backward_depth(stats=P, depth=P, g=P, h=P, grad=FAR, grad_stride=8, **k):
        return lib.molla_sample_token_logprobs_backward_with_depth(*block(**k), stats, depth, g, h, NULL, grad, grad_stride)

    for call, names in ((score_depth, ["logits", "tokens", "logprob", "status"]), (backward_depth, ["logits", "tokens", "stats", "depth", "g", "grad"])):
        for n in names:
            assert call(**{n: NULL}) == capi.ERR_ARGUMENT, n
            assert capi.last_error()
        assert call(stride=7) == capi.ERR_ARGUMENT and call(V=720897, stride=720897) == capi.ERR_VOCAB
    assert backward_depth(grad=C.c_void_p(4096 + 4)) == capi.ERR_ARGUMENT and "overlaps" in capi.last_error()
