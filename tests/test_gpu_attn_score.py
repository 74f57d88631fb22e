"""GPU parity of attention with capped, biased and prefix-masked scores.

Tolerances are the fast mode's own (tests/helpers.py: 2e-2 of the largest value,
P and dS being rounded to bf16), and besides 1e-2 in the 2-norm, where those
roundings (2^-9 each, at most three of them) average out.  The log-sum-exp is
within 1e-5, for a cap c plus c 2^-21, and for a bias plus 2^-22 of the largest
one, which is added in float32."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from femtochat_amd import workloads as W
from oracle import attention_score as S

from tests.helpers import TOL, TOL_LSE, lse_err, rel_err

pytestmark = pytest.mark.gpu
A = F.MFMAFast()
KINDS = ["cap", "bias", "cap+bias", "prefix", "cap+prefix", "bias+prefix", "all"]


def _inputs(seed, B, T, H, Hkv, D, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * f).bfloat16() for s, f in
            (((B, T, H, D), scale), ((B, T, Hkv, D), 1.0), ((B, T, Hkv, D), 1.0), ((B, T, H, D), 0.1))]


def _options(kind, seed, B, T, H, per_token=False):
    rng = np.random.default_rng(seed)
    cap, bias, prefix = ("cap" in kind, "bias" in kind, "prefix" in kind) if kind != "all" else (True,) * 3
    return dict(softcap=5.0 if cap else 0.0,
                slopes=(2.0 ** (-8.0 * (np.arange(H) + 1) / H)).astype(np.float32) if bias else None,
                prefix=rng.integers(0, T + 1, (B, T) if per_token else B).astype(np.int32) if prefix else None)


def _dev(gpu, how):
    return {k: torch.from_numpy(v).to(gpu) if isinstance(v, np.ndarray) else v for k, v in how.items()}


def _run(gpu, host, window, pos, how, out=torch.bfloat16, grad=torch.bfloat16, init=None):
    """(O, l, m, dQ, dK, dV); the gradients added to `init` if given, else written over NaN."""
    Q, K, V, dO = (x.to(gpu) for x in host)
    B, T, H, D = Q.shape
    d = _dev(gpu, how)
    p = None if pos is None else torch.from_numpy(pos).to(gpu)
    O = torch.full(Q.shape, float("nan"), dtype=out, device=gpu)
    l, m = torch.empty(B, H, T, device=gpu), torch.empty(B, H, T, device=gpu)
    F.attention_(A, O, l, m, Q, K, V, window, positions=p, **d)
    grads = [torch.full(x.shape, float("nan") if init is None else init, dtype=grad, device=gpu) for x in (Q, K, V)]
    F.delta_attention_(A, *grads, dO.to(out), Q, K, V, O, l, m, window, positions=p, accumulate=init is not None, **d)
    return [O, l, m] + grads


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(x, ref, name, norm=1e-2):
    x = _np(x)
    assert np.isfinite(x).all(), name
    assert rel_err(x, ref) <= TOL["fast"], (name, rel_err(x, ref))
    n = np.linalg.norm(ref)
    if n > 1e-3:
        assert np.linalg.norm(x - ref) <= norm * n, (name, np.linalg.norm(x - ref) / n)


def _check(got, host, window, pos, how, norm=1e-2):
    Q, K, V, dO = (x.double().numpy() for x in host)
    O, l, m = S.forward(Q, K, V, window, pos, **how)
    _close(got[0], O, "O", norm)
    room = TOL_LSE + how["softcap"] * 2.0 ** -21 + (0.0 if how["slopes"] is None else np.abs(how["slopes"]).max() * Q.shape[1] * 2.0 ** -22)
    assert lse_err(_np(got[1]), _np(got[2]), l, m) <= room
    assert ((_np(got[1]) == 0) == (l == 0)).all()
    for x, ref, name in zip(got[3:], S.backward(dO, Q, K, V, window, pos, **how), ("dQ", "dK", "dV")):
        _close(x, ref, name, norm)


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_kinds_and_head_dims(gpu, kind, D):
    B, T, H, Hkv = 2, 201, 4, 2
    host = _inputs(D, B, T, H, Hkv, D)
    how = _options(kind, D, B, T, H)
    _check(_run(gpu, host, (-1, 0), None, how), host, (-1, 0), None, how)


@pytest.mark.parametrize("window", [(37, 0), (20, 15), (300, 300), (10, -3), (-4, 9), (0, 0)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
def test_windows(gpu, window, kind, D):
    """Windows on either side, past the sequence, that leave rows without keys, and of one key."""
    B, T, H, Hkv = 1, 170, 2, 1
    host = _inputs(7, B, T, H, Hkv, D)
    how = _options(kind, 8, B, T, H)
    _check(_run(gpu, host, window, None, how), host, window, None, how)


@pytest.mark.parametrize("T", [1, 2, 31, 64, 65, 127, 129, 400, 777, 1100])
@pytest.mark.parametrize("kind", KINDS)
def test_lengths_and_documents(gpu, T, kind):
    """Packed documents with a prefix per token, from one token to several tiles (the
    longer ones in two parts of the key tiles)."""
    B, H, Hkv, D = 2, 2, 1, 64
    host = _inputs(T, B, T, H, Hkv, D)
    pos = W.document_positions(T, B, T, mean=120, sigma=1.0, cap=500)
    how = _options(kind, T, B, T, H, per_token=True)
    if how["prefix"] is not None:
        how["prefix"] = (how["prefix"] % 90).astype(np.int32)
    norm = 1e-2 if T >= 100 else 2e-2
    _check(_run(gpu, host, (-1, 0), pos, how), host, (-1, 0), pos, how, norm)
    _check(_run(gpu, host, (60, 0), pos, how), host, (60, 0), pos, how, norm)
    if T > 600:
        how = _options(kind, T, B, T, H)
        _check(_run(gpu, host, (-1, 0), None, how), host, (-1, 0), None, how)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 96])
def test_many_workgroups(gpu, kind, D):
    """Grids of more than two workgroups per CU, GQA groups of 5."""
    B, T, H, Hkv = 9, 300, 20, 4
    host = _inputs(5, B, T, H, Hkv, D)
    how = _options(kind, 6, B, T, H)
    _check(_run(gpu, host, (-1, 0), None, how), host, (-1, 0), None, how)


@pytest.mark.parametrize("B,T,H,Hkv,D", [(1, 1300, 8, 1, 128), (1, 1300, 8, 2, 48), (2, 700, 4, 1, 64), (1, 2100, 2, 2, 32), (3, 140, 10, 2, 96)])
@pytest.mark.parametrize("kind", ["cap", "all", "prefix"])
@pytest.mark.parametrize("documents", [False, True])
def test_few_key_tiles(gpu, B, T, H, Hkv, D, kind, documents):
    """Problems whose dK/dV items are split over heads and query tiles and joined, with
    gradients overwritten and added to, in both types."""
    host = _inputs(24, B, T, H, Hkv, D)
    pos = W.document_positions(T, B, 25, mean=400) if documents else None
    how = _options(kind, 26, B, T, H, per_token=documents)
    if documents and how["prefix"] is not None:
        how["prefix"] = (how["prefix"] % 300).astype(np.int32)
    for window in ((-1, 0), (200, 0)):
        got = _run(gpu, host, window, pos, how)
        _check(got, host, window, pos, how)
    for x, y in zip(got, _run(gpu, host, window, pos, how)):
        assert torch.equal(x, y)
    for grad in (torch.bfloat16, torch.float32):
        added = _run(gpu, host, window, pos, how, grad=grad, init=-0.5)
        for x, y in zip(got[3:], added[3:]):
            # got is rounded to bf16 once, added once in its own type
            room = 2.0 ** -8 * x.float().abs() + (2.0 ** -8 * y.float().abs() if grad == torch.bfloat16 else 1e-6)
            assert ((y.float() - x.float() + 0.5).abs() <= room + 1e-6).all()


def test_prefixes_of_any_value(gpu):
    """Below 0, past T, and of each token its own: nothing monotone."""
    B, T, H, Hkv, D = 3, 290, 2, 2, 64
    host = _inputs(9, B, T, H, Hkv, D)
    rng = np.random.default_rng(10)
    wild = rng.integers(-50, T + 50, (B, T)).astype(np.int32)
    wild[rng.random((B, T)) < 0.5] = 0
    wild[0, :5] = [-2 ** 31, 2 ** 31 - 1, -1, T, T + 1]
    for prefix in (wild, np.array([-7, 2 ** 31 - 1, 100], np.int32), np.zeros(B, np.int32)):
        how = dict(softcap=0.0, slopes=None, prefix=prefix)
        _check(_run(gpu, host, (-1, 0), None, how), host, (-1, 0), None, how)
    pos = W.document_positions(T, B, 3, mean=80)
    how["prefix"] = wild
    _check(_run(gpu, host, (50, 0), pos, how), host, (50, 0), pos, how)
    # without a prefix that matters, the plain kernels' results
    how = dict(softcap=0.0, slopes=None, prefix=np.zeros(B, np.int32))
    for x, y in zip(_run(gpu, host, (-1, 0), None, how), _run(gpu, host, (-1, 0), None, dict(softcap=0.0, slopes=None, prefix=None))):
        _close(x, _np(y), "against plain")


@pytest.mark.parametrize("slopes", [[0.9, 3.0, 0.0, 0.01], [-0.05, -0.5, 0.5, 40.0]])
@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_steep_and_rising_biases(gpu, slopes, prefix, D):
    """Biases that move a row's scores by far more than 2^64 along the keys, in both
    directions, also from keys behind a prompt's query."""
    B, T, H, Hkv = 1, 900, 4, 4
    host = _inputs(11, B, T, H, Hkv, D)
    how = dict(softcap=0.0, slopes=np.array(slopes, np.float32), prefix=np.array([600], np.int32) if prefix else None)
    _check(_run(gpu, host, (-1, 0), None, how), host, (-1, 0), None, how)


@pytest.mark.parametrize("softcap,scale", [(2.0 ** -10, 3.0), (0.5, 3.0), (30.0, 300.0), (50.0, 8.0), (4096.0, 2.0)])
@pytest.mark.parametrize("D", [32, 128])
def test_saturated_and_loose_caps(gpu, softcap, scale, D):
    B, T, H, Hkv = 1, 333, 2, 1
    host = _inputs(12, B, T, H, Hkv, D, scale=scale)
    how = dict(softcap=softcap, slopes=None, prefix=None)
    _check(_run(gpu, host, (-1, 0), None, how), host, (-1, 0), None, how)


def test_infinite_scores_meet_the_cap(gpu):
    """q.k beyond float32 caps at +-c; a NaN in a query stays in its row."""
    B, T, H, Hkv, D = 1, 70, 1, 1, 64
    Q, K, V, dO = _inputs(13, B, T, H, Hkv, D)
    Q[0, 5], K[0, 3] = 1e30, 1e30
    how = _dev(gpu, dict(softcap=20.0))
    O = F.attention(Q.to(gpu), K.to(gpu), V.to(gpu), (-1, 0), **how)
    assert torch.isfinite(O).all()
    ref = S.forward(*(x.double().numpy() for x in (Q, K, V)), (-1, 0), softcap=20.0)[0]
    assert rel_err(_np(O), ref) <= TOL["fast"]
    Q[0, 40, 0, 7] = float("nan")
    O = F.attention(Q.to(gpu), K.to(gpu), V.to(gpu), (-1, 0), **how)
    bad = torch.isnan(O).any(-1)[0, :, 0]
    assert bad.nonzero().flatten().tolist() == [40]


@pytest.mark.parametrize("window", [(1, 0), (2, 1), (64, 0), (-1, 0)])
@pytest.mark.parametrize("T", [16, 200, 1500])
@pytest.mark.parametrize("kind", ["cap", "prefix"])
def test_few_keys_keep_their_gradients(gpu, T, window, kind):
    """The 2-norm of the gradients' errors where O's rounding weighs most: sharp scores,
    few rows or few keys.  dS and the gradient are rounded once each (2^-9 / sqrt(3) on
    average over their values' places, 2.3e-3 together); Delta from the rounded O alone
    brought it to 6e-3 with two keys."""
    B, H, Hkv, D = 1, 2, 1, 64
    host = _inputs(27, B, T, H, Hkv, D, scale=3.0)
    how = dict(softcap=30.0 if kind == "cap" else 0.0, slopes=None,
               prefix=np.array([T // 8], np.int32) if kind == "prefix" else None)
    got = _run(gpu, host, window, None, how)
    Q, K, V, dO = (x.double().numpy() for x in host)
    for x, ref in zip(got[3:], S.backward(dO, Q, K, V, window, None, **how)):
        assert np.linalg.norm(_np(x) - ref) <= (4e-3 if T > 256 and window == (-1, 0) else 3.5e-3) * np.linalg.norm(ref)


@pytest.mark.parametrize("out,grad", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("kind", ["all", "cap", "bias"])
def test_storage_types_and_accumulation(gpu, out, grad, kind):
    B, T, H, Hkv, D = 2, 150, 4, 1, 80
    host = _inputs(14, B, T, H, Hkv, D)
    how = _options(kind, 15, B, T, H)
    plain = _run(gpu, host, (-1, 0), None, how, out, grad)
    _check(plain, host, (-1, 0), None, how)
    added = _run(gpu, host, (-1, 0), None, how, out, grad, init=0.25)
    for x, y in zip(plain[3:], added[3:]):  # each rounded once
        room = 0.0 if grad == torch.float32 else 2.0 ** -8
        assert ((y.float() - x.float() - 0.25).abs() <= 1e-5 + room * (x.float().abs() + y.float().abs())).all()


def test_a_long_row_of_documents(gpu):
    """More query tiles than the dK/dV kernel tabulates: each document by itself."""
    T, H, D = 33100, 1, 16
    host = _inputs(16, 1, T, H, H, D)
    pos = W.document_positions(T, 1, 17, mean=300, sigma=0.8, cap=700, mid_document_start=False)
    pre = np.zeros((1, T), np.int32)
    starts = np.flatnonzero(pos[0] == 0).tolist() + [T]
    rng = np.random.default_rng(18)
    for s, e in zip(starts, starts[1:]):
        pre[0, s:e] = rng.integers(0, e - s + 1)
    how = dict(softcap=6.0, slopes=np.array([0.02], np.float32), prefix=pre)
    got = _run(gpu, host, (-1, 0), pos, how)
    want = [np.zeros(tuple(x.shape)) for x in host]
    for s, e in zip(starts, starts[1:]):
        Q, K, V, dO = (x[:, s:e].double().numpy() for x in host)
        h2 = dict(how, prefix=pre[:, s])
        want[0][:, s:e] = S.forward(Q, K, V, (-1, 0), **h2)[0]
        for i, g in enumerate(S.backward(dO, Q, K, V, (-1, 0), **h2)):
            want[1 + i][:, s:e] = g
    for x, ref, name in zip([got[0]] + got[3:], want, ("O", "dQ", "dK", "dV")):
        _close(x, ref, name)


@pytest.mark.parametrize("D", [64, 96])
def test_autograd_views_and_instructions(gpu, D):
    """Through autograd: fp32 leaves, and views off a 16-byte boundary (D 96 copies them)."""
    B, T, H, Hkv = 2, 140, 4, 2
    host = _inputs(19, B, T, H, Hkv, D)
    how = _options("all", 20, B, T, H)
    d = _dev(gpu, how)
    want = S.backward(host[3].double().numpy(), *(x.double().numpy() for x in host[:3]), (-1, 0), **how)
    for dtype, off in ((torch.float32, 0), (torch.bfloat16, 0), (torch.bfloat16, 1)):
        leaves = []
        for x in host[:3]:
            room = torch.empty(x.numel() + off, dtype=dtype, device=gpu)
            leaves.append(room[off:].view(x.shape).copy_(x).requires_grad_())
        if off and D == 64:
            continue  # the powers of two take tensors on 16-byte boundaries
        O = F.AttentionFunction.apply(*leaves, (-1, 0), None, None, d["softcap"], d["slopes"], d["prefix"])
        assert O.dtype == dtype
        for g, ref, name in zip(torch.autograd.grad(O, leaves, host[3].to(gpu, dtype)), want, ("dQ", "dK", "dV")):
            assert g.dtype == dtype
            _close(g, ref, name)


def test_the_same_bits_again_and_captured(gpu):
    """Repeats, dirty workspaces, another stream and graph replays give the same bits."""
    B, T, H, Hkv, D = 2, 500, 4, 2, 128
    hosts = [_inputs(30 + i, B, T, H, Hkv, D) for i in range(2)]
    how = _options("all", 21, B, T, H)
    want = [_run(gpu, h, (-1, 0), None, how) for h in hosts]
    Q, K, V, dO = (x.to(gpu) for x in hosts[0])
    d = _dev(gpu, how)
    O, l, m = torch.empty_like(Q), torch.empty(B, H, T, device=gpu), torch.empty(B, H, T, device=gpu)
    grads = [torch.empty_like(x) for x in (Q, K, V)]
    n = F.backward_workspace_bytes(A, Q, K, **d)
    ws = torch.full((n,), 255, dtype=torch.uint8, device=gpu)

    def step():
        F.attention_(A, O, l, m, Q, K, V, (-1, 0), **d)
        F.delta_attention_(A, *grads, dO, Q, K, V, O, l, m, (-1, 0), accumulate=False, workspace=ws, **d)

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(gpu).wait_stream(side)
    for x, y in zip([O, l, m] + grads, want[0]):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (1, 0, 1):
        for x, h in zip((Q, K, V, dO), hosts[i]):
            x.copy_(h)
        ws.fill_(255 - i)
        graph.replay()
        again = _run(gpu, hosts[i], (-1, 0), None, how)
        torch.cuda.synchronize()
        for x, y, z in zip([O, l, m] + grads, want[i], again):
            assert torch.equal(x, y) and torch.equal(y, z)


def test_a_layer_then_its_losses(gpu):
    """A run as it is used: prompt-prefix attention with a cap and a bias, a projection
    to a vocabulary, and both losses on the answers, with gradients for the weights."""
    g = torch.Generator().manual_seed(22)
    B, T, H, D, V = 4, 48, 2, 16, 300
    x = torch.randn(B, T, H * D, generator=g).to(gpu)
    prompt = torch.tensor([10, 20, 5, 30], dtype=torch.int32, device=gpu)
    tokens = torch.randint(0, V, (B, T), generator=g).to(gpu)
    tokens[torch.arange(T, device=gpu)[None] < prompt[:, None]] = -1
    w = {n: (torch.randn(H * D, o, generator=g) / 6).to(gpu).requires_grad_() for n, o in (("q", H * D), ("k", H * D), ("v", H * D), ("o", V))}
    slopes = torch.tensor([0.25, 0.0625], device=gpu)

    def logits():
        q, k, v = ((x @ w[n]).view(B, T, H, D) for n in "qkv")
        O = F.AttentionFunction.apply(q, k, v, (-1, 0), None, None, 10.0, slopes, prompt)
        return O.reshape(B, T, H * D) @ w["o"]

    z = logits()
    lp = torch.log_softmax(z.detach(), -1).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    old = (lp + 0.05).contiguous()
    adv = torch.tensor([1.0, -1.0, 0.5, 2.0], device=gpu)
    a = F.PolicyLossFunction.apply(z, tokens, old, adv, old, (0.2, 0.2), 0.1, -1, "mean")
    b, rewards = F.PreferenceLossFunction.apply(z, tokens, torch.zeros(B, device=gpu) - 250, 0.1, 0.0, -1, "mean")
    grads = torch.autograd.grad(a + b, list(w.values()))
    on = tokens != -1
    zr = z.detach().double().requires_grad_()
    lpr = torch.log_softmax(zr, -1).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    r = torch.exp(lpr - old)
    k3 = torch.exp(old - lpr) - (old - lpr) - 1
    ar = ((-torch.minimum(r * adv[:, None], r.clamp(0.8, 1.2) * adv[:, None]) + 0.1 * k3) * on).sum() / on.sum()
    h = 0.1 * ((lpr * on).sum(-1) + 250)
    br = -torch.nn.functional.logsigmoid(h[:2] - h[2:]).mean()
    assert abs(float(a.detach()) - float(ar)) < 1e-5 and abs(float(b.detach()) - float(br)) < 1e-4
    gz = torch.autograd.grad(ar + br, zr)[0].float()
    want = torch.autograd.grad(logits(), list(w.values()), gz)
    for x1, x2 in zip(grads, want):
        assert (x1 - x2).abs().max() <= 1e-3 * x2.abs().max()


def test_gpu_refusals(gpu):
    Q, K, V, _ = (x.to(gpu) for x in _inputs(23, 2, 8, 4, 2, 16))
    ok = torch.zeros(4, device=gpu)
    for how in (dict(slopes=ok[:3]), dict(slopes=ok.double()), dict(slopes=ok.cpu()), dict(prefix=torch.zeros(2, device=gpu)),
                dict(prefix=torch.zeros(3, dtype=torch.int32, device=gpu)), dict(prefix=torch.zeros(2, 7, dtype=torch.int32, device=gpu)),
                dict(slopes=[0.1] * 4)):
        with pytest.raises((ValueError, TypeError)):
            F.attention(Q, K, V, (-1, 0), **how)
    for how in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf"))):
        with pytest.raises(F._lib.AttentionError):
            F.attention(Q, K, V, (-1, 0), **how)
    f = [x.float() for x in (Q, K, V)]
    with pytest.raises(F._lib.AttentionError, match="fast mode"):
        F.attention(F.MFMAExact(), *f, (-1, 0), softcap=3.0)
    assert torch.equal(F.attention(F.MFMAExact(), *f, (-1, 0), softcap=0.0), F.attention(F.MFMAExact(), *f, (-1, 0)))


def test_slopes_that_ask_for_a_gradient_are_refused(gpu):
    Q, K, V, _ = (x.to(gpu) for x in _inputs(25, 1, 40, 4, 2, 32))
    slopes = torch.full((4,), 0.1, device=gpu, requires_grad=True)
    with pytest.raises(ValueError, match="slopes"):
        F.AttentionFunction.apply(Q, K, V, (-1, 0), None, None, 0.0, slopes)
    F.AttentionFunction.apply(Q, K, V, (-1, 0), None, None, 0.0, slopes.detach())


def test_workspaces_that_repeat_their_memory_are_refused(gpu):
    """A broadcast tensor has the values but not the bytes."""
    Q, K, V, dO = (x.to(gpu) for x in _inputs(26, 1, 300, 4, 2, 32))
    n = F.backward_workspace_bytes(A, Q, K, softcap=5.0)
    O, l, m = torch.empty_like(Q), torch.empty(1, 4, 300, device=gpu), torch.empty(1, 4, 300, device=gpu)
    F.attention_(A, O, l, m, Q, K, V, (-1, 0), softcap=5.0)
    grads = [torch.empty_like(x) for x in (Q, K, V)]
    ws = torch.empty(1, dtype=torch.uint8, device=gpu).expand(n)
    with pytest.raises(ValueError, match="contiguous"):
        F.delta_attention_(A, *grads, dO, Q, K, V, O, l, m, (-1, 0), softcap=5.0, workspace=ws)
    x, t, r = torch.zeros(2, 3, 5, device=gpu), torch.zeros(2, 3, dtype=torch.int64, device=gpu), torch.zeros(2, device=gpu)
    with pytest.raises(ValueError, match="contiguous"):
        F.preference_loss(x, t, r, workspace=torch.empty(1, 1, dtype=torch.float64, device=gpu).expand(2, 3))


def test_two_streams_at_once(gpu):
    """Scored steps and losses on two streams at a time, the same bits as alone."""
    def step(seed):
        Q, K, V, dO = (x.to(gpu).requires_grad_(i < 3) for i, x in enumerate(_inputs(seed, 2, 700, 4, 2, 64)))
        prefix = torch.tensor([40, 650], dtype=torch.int32, device=gpu)
        x = torch.randn(4, 33, 1000, device=gpu, generator=torch.Generator(device=gpu).manual_seed(seed)).requires_grad_()
        t = torch.randint(0, 1000, (4, 33), device=gpu, generator=torch.Generator(device=gpu).manual_seed(seed))
        r = torch.zeros(4, device=gpu)
        torch.cuda.current_stream(gpu).synchronize()

        def run():
            out = F.AttentionFunction.apply(Q, K, V, (-1, 0), None, None, 5.0, None, prefix)
            loss = F.PreferenceLossFunction.apply(x, t, r, 0.1, 0.0, -1, "mean")[0]
            return torch.autograd.grad([out, loss], [Q, K, V, x], [dO, torch.ones_like(loss)])
        return run

    runs = [step(27), step(28)]
    want = [[g.clone() for g in run()] for run in runs]
    streams = [torch.cuda.Stream(gpu), torch.cuda.Stream(gpu)]
    torch.cuda.synchronize(gpu)
    got = [None, None]
    for _ in range(3):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = runs[i]()
    torch.cuda.synchronize(gpu)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
