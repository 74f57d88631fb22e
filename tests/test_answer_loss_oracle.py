"""The policy and preference losses on the CPU: the float64 oracle's gradients
against differences, and the refusals of the host side (no kernel is launched)."""
import ctypes

import numpy as np
import pytest
import torch

import femtochat_amd as F
import femtochat_amd._lib as L
from oracle import answer_loss as O


def _case(seed, B=4, T=3, V=7):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((B, T, V)) * 2
    tok = rng.integers(0, V, (B, T))
    tok[0, 0] = tok[2, 1] = -1
    lp, _ = O.log_probs(x, tok)
    old = lp + rng.choice([-0.5, -0.1, 0.0, 0.1, 0.5], (B, T))  # no ratio within 0.04 of a clip of 0.2
    return x, tok, old, rng.standard_normal((B, T)), lp + 0.3 * rng.standard_normal((B, T))


def _difference(f, x, at, h=1e-6):
    up, down = x.copy(), x.copy()
    up[at] += h
    down[at] -= h
    return (f(up) - f(down)) / (2 * h)


@pytest.mark.parametrize("kl", [0.0, 0.3])
def test_policy_gradient_against_differences(kl):
    x, tok, old, adv, ref = _case(1)
    loss, g, _ = O.policy(x, tok, old, adv, ref, kl=kl, dy=0.7)
    f = lambda z: 0.7 * O.policy(z, tok, old, adv, ref, kl=kl)[0].sum()  # noqa: E731
    for at in np.ndindex(*x.shape):
        # differences of h = 1e-6: truncation below 1e-11, rounding below 1e-9
        assert abs(_difference(f, x, at) - g[at]) < 1e-8
    assert loss[0, 0] == 0 and not g[0, 0].any()


@pytest.mark.parametrize("smoothing", [0.0, 0.2])
def test_preference_gradient_against_differences(smoothing):
    x, tok, _, _, _ = _case(2)
    ref = O.log_probs(x, tok)[0].sum(-1) + np.array([1.0, -2.0, 0.5, 3.0])
    dy = np.array([0.7, -1.3])
    g = O.preference(x, tok, ref, 0.3, smoothing, dy=dy)[2]
    f = lambda z: (dy * O.preference(z, tok, ref, 0.3, smoothing)[0]).sum()  # noqa: E731
    for at in np.ndindex(*x.shape):
        assert abs(_difference(f, x, at) - g[at]) < 1e-8


def test_python_refusals():
    x, t = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
    o = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="HIP device"):
        F.policy_loss(x, t, o, o)
    with pytest.raises(ValueError, match="HIP device"):
        F.preference_loss(x, t, torch.zeros(2))
    with pytest.raises(ValueError, match="reduction"):
        F.policy_loss(x, t, o, o, reduction="max")
    with pytest.raises(ValueError, match="answers, T, V"):
        F.policy_loss(x[0], t[0], o[0], o[0])


def _desc(**kw):
    d = dict(V=8, answers=2, T=3, index_base=0, ignore_index=-1, index_type=L.FC_INDEX_I64, dtype=L.FC_F32, reduction=L.FC_REDUCE_SUM,
             flags=0)
    d.update(kw)
    return L.AnswerDesc(**d)


ROOM = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(ROOM) + 255) & ~255  # host memory: only checks look at it


def _policy(desc=None, options=None, entry="fwd", **swap):
    """The status of a call whose arguments pass every check but the one swapped in."""
    d, o = desc or _desc(), options or L.PolicyOptions(0.2, 0.2, 0.0, 0)
    p = dict(logits=AT, tokens=AT, old=AT, adv=AT, ref=None, losses=AT, logprobs=None, stats=None, weights=None, reduced=None,
             count=None, dlogits=AT + 2048, dy=None)
    p.update(swap)
    a = [p[k] for k in ("logits", "tokens", "old", "adv", "ref", "losses", "logprobs", "stats", "weights", "reduced")]
    lib = L.lib()
    if entry == "fwd":
        return lib.fc_policy_loss_fwd(ctypes.byref(d), ctypes.byref(o), *a, p["count"], None)
    if entry == "fused":
        return lib.fc_policy_loss_fused(ctypes.byref(d), ctypes.byref(o), *a, p["count"], p["dlogits"], p["dy"], None)
    return lib.fc_policy_loss_bwd(ctypes.byref(d), p["dlogits"], p["logits"], p["tokens"], p["stats"], p["weights"], p["dy"],
                                  p["count"], None)


@pytest.mark.parametrize("kw", [dict(V=0), dict(answers=0), dict(T=-1), dict(index_base=2), dict(index_type=7), dict(dtype=5),
                                dict(reduction=9), dict(flags=4)])
@pytest.mark.parametrize("entry", ["fwd", "fused", "bwd"])
def test_bad_descriptors(kw, entry):
    assert _policy(_desc(**kw), entry=entry) == L.FC_ERR_INVALID_ARGUMENT


def test_too_many():
    assert _policy(_desc(answers=1 << 16, T=1 << 15)) == L.FC_ERR_UNSUPPORTED
    assert _policy(_desc(V=1 << 30, answers=1 << 10, T=1)) == L.FC_ERR_UNSUPPORTED
    assert _policy(_desc(V=2, answers=1 << 11, T=1 << 11)) == L.FC_ERR_UNSUPPORTED
    assert _policy(_desc(V=1 << 13, answers=(1 << 20) + 1, T=1)) == L.FC_ERR_UNSUPPORTED
    assert _policy(_desc(V=1 << 17), entry="fused", dlogits=AT + (1 << 30)) == L.FC_ERR_UNSUPPORTED  # 512 KB columns


@pytest.mark.parametrize("o", [(-0.1, 0.2, 0.0), (1.5, 0.2, 0.0), (0.2, -1.0, 0.0), (0.2, 0.2, -1.0), (0.2, 0.2, 0.5),
                               (float("nan"), 0.2, 0.0), (0.2, 0.2, float("nan")), (0.2, 0.2, float("inf"))])
def test_bad_policy_options(o):
    assert _policy(options=L.PolicyOptions(*o, 0)) == L.FC_ERR_INVALID_ARGUMENT  # kl 0.5: no ref_logprobs


@pytest.mark.parametrize("entry,swap", [
    ("fwd", dict(logits=None)), ("fwd", dict(tokens=None)), ("fwd", dict(losses=None)), ("fwd", dict(old=None)), ("fwd", dict(adv=None)),
    ("fwd", dict(tokens=AT + 4)), ("fwd", dict(logits=AT + 2)), ("fwd", dict(stats=AT + 4)), ("fwd", dict(losses=AT + 1)),
    ("fused", dict(dlogits=None)), ("fused", dict(dlogits=AT)), ("fused", dict(dlogits=AT + 64)), ("fused", dict(dlogits=AT + 2052)),
    ("bwd", dict(stats=None, weights=AT)), ("bwd", dict(stats=AT, weights=None)), ("bwd", dict(stats=AT, weights=AT, dlogits=AT + 64)),
])
def test_bad_pointers(entry, swap):
    assert _policy(entry=entry, **swap) == L.FC_ERR_INVALID_ARGUMENT
    assert L.lib().fc_last_error()


@pytest.mark.parametrize("entry", ["fused", "bwd"])
def test_mean_gradient_needs_the_count(entry):
    assert _policy(_desc(reduction=L.FC_REDUCE_MEAN), entry=entry, stats=AT, weights=AT) == L.FC_ERR_INVALID_ARGUMENT


def test_preference_refusals():
    lib = L.lib()

    def call(desc=None, beta=0.1, smoothing=0.0, ref=AT, losses=AT, ws=AT, ws_bytes=2048):
        d, o = desc or _desc(), L.PreferenceOptions(beta, smoothing)
        return lib.fc_preference_loss_fwd(ctypes.byref(d), ctypes.byref(o), AT, AT, ref, losses, None, None, None, None, None, ws,
                                          ws_bytes, None)

    assert call(_desc(answers=3)) == L.FC_ERR_INVALID_ARGUMENT
    for bad in (dict(beta=0.0), dict(beta=float("nan")), dict(smoothing=-0.1), dict(smoothing=1.1), dict(ref=None), dict(losses=None)):
        assert call(**bad) == L.FC_ERR_INVALID_ARGUMENT, bad
    for bad in (dict(ws=None), dict(ws_bytes=47), dict(ws=AT + 4)):
        assert call(**bad) == L.FC_ERR_WORKSPACE, bad
    d = _desc(answers=3)
    assert lib.fc_preference_loss_bwd(ctypes.byref(d), AT + 2048, AT, AT, AT, AT, None, None) == L.FC_ERR_INVALID_ARGUMENT
    n = ctypes.c_size_t(0)
    d = _desc()
    assert lib.fc_preference_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == L.FC_OK and n.value == 48


def test_scale_refusals():
    lib = L.lib()
    for args in ((None, L.FC_F32, 4, AT), (AT, L.FC_F32, 4, None), (AT, L.FC_F32, 0, AT), (AT, 9, 4, AT), (AT + 2, L.FC_F32, 4, AT),
                 (AT, L.FC_F32, 4, AT + 1)):
        assert lib.fc_scale_gradient(*args, None) == L.FC_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("kw,swap", [
    (dict(flags=L.FC_FLAG_FORMED), {}), (dict(reduction=L.FC_REDUCE_NONE), {}), ({}, dict(dy=None)), ({}, dict(dlogits=AT)),
])
def test_a_formed_gradient_refusals(kw, swap):
    """It is overwritten, of a sum or a mean, under a dy, in an array of its own."""
    d = dict(flags=L.FC_FLAG_OVERWRITE | L.FC_FLAG_FORMED)
    d.update(kw)
    s = dict(stats=AT, weights=AT, dy=AT)
    s.update(swap)
    assert _policy(_desc(**d), entry="bwd", **s) == L.FC_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("entry", ["fwd", "fused"])
def test_only_the_gradient_takes_a_formed_one(entry):
    assert _policy(_desc(flags=L.FC_FLAG_FORMED | L.FC_FLAG_OVERWRITE), entry=entry) == L.FC_ERR_INVALID_ARGUMENT


def test_inputs_without_a_gradient_are_refused_one():
    """What the losses take as constants is not silently left without a gradient."""
    x, t, o = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    asks = o.clone().requires_grad_()
    for old, adv, ref in ((asks, o, None), (o, asks, None), (o, o, asks), (o, o[:, 0].clone().requires_grad_(), o)):
        with pytest.raises(ValueError, match="no gradient"):
            F.PolicyLossFunction.apply(x, t, old, adv, ref, (0.2, 0.2), 0.1, -1, "mean")
    with pytest.raises(ValueError, match="no gradient"):
        F.PreferenceLossFunction.apply(x, t, asks[:, 0], 0.1, 0.0, -1, "mean")
    with pytest.raises(ValueError, match="HIP device"):  # detached: the next check speaks
        F.PolicyLossFunction.apply(x, t, asks.detach(), o, None, (0.2, 0.2), 0.0, -1, "mean")
