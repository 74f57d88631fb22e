"""GPU parity of the policy and preference losses against the float64 oracle.

Tolerances.  A log-probability is max, a float32 sum over the vocabulary and a
float64 logarithm: each exponential is within (2 + 1.5 |x - max|) 2^-23 of its
value and a sum of V terms in rounds of 2048 adds under 200 2^-24, so with the
mean of |x - max| under the softmax below 20 here, lp is within 2e-5.  Losses move
by at most |w| + |w'| times that; gradients are w (onehot - p) with p within 1e-5
of itself, and in bf16 half a step (2^-8) of the result is added."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import answer_loss as O

pytestmark = pytest.mark.gpu
LP = 2e-5
CLIP = (0.2, 0.3)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _logits(gpu, seed, B, T, V, dtype, scale=2.5, shift=0.0, off=0):
    """(float64 values, the device tensor `off` elements into its buffer)."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, T, V, generator=g) * scale + shift).to(DTYPES[dtype])
    room = torch.empty(x.numel() + off, dtype=x.dtype, device=gpu)[off:].view(B, T, V)
    room.copy_(x)
    return x.double().numpy(), room


def _tokens(seed, B, T, V, ignored):
    rng = np.random.default_rng(seed)
    t = rng.integers(0, V, (B, T))
    if ignored == "some":
        t[rng.random((B, T)) < 0.3] = -1
    elif ignored == "all":
        t[:] = -1
    return t


def _policy_inputs(seed, x, tok, per_answer):
    rng = np.random.default_rng(seed + 1)
    lp, _ = O.log_probs(x, tok)
    # ratios of exp(-0.5), exp(-0.1), 1, exp(0.1), exp(0.5): none within 0.06 of a clip
    old = (lp + rng.choice([-0.5, -0.1, 0.0, 0.1, 0.5], lp.shape)).astype(np.float32)
    ref = (lp + 0.3 * rng.standard_normal(lp.shape)).astype(np.float32)
    adv = rng.standard_normal(lp.shape[0] if per_answer else lp.shape).astype(np.float32)
    return old, ref, adv


def _dev(gpu, *arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(gpu) for a in arrays]


def _check_gradient(got, ref, w, dtype):
    """got within half a step of its type plus 2e-5 |w| of ref."""
    g = got.double().cpu().numpy()
    room = (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) * np.abs(ref) + 2 * LP * np.abs(w)[..., None]
    worst = np.max(np.abs(g - ref) - room)
    assert worst <= 0, (worst, np.abs(g - ref).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 3, 8, 259, 1000, 2049, 4097, 8191, 16400, 50257])
@pytest.mark.parametrize("kl", [0.0, 0.25])
def test_policy(gpu, V, dtype, kl):
    B, T = 3, 5
    x, xd = _logits(gpu, V, B, T, V, dtype)
    tok = _tokens(V, B, T, V, "some")
    old, ref, adv = _policy_inputs(V, x, tok, per_answer=True)
    td, od, rd, ad = _dev(gpu, tok, old, ref if kl else None, adv)
    n = max(1, (tok != -1).sum())
    loss, g, w = O.policy(x, tok, old, adv, ref, CLIP, kl, dy=0.5 / n)
    how = dict(ref_logprobs=rd, clip=CLIP, kl=kl)
    losses, lps, stats = torch.full((B, T), 9.0, device=gpu), torch.empty(B, T, device=gpu), torch.empty(B, T, 2, device=gpu)
    weights, reduced, count = torch.empty(B, T, device=gpu), torch.empty(1, device=gpu), torch.empty(1, device=gpu)
    F.policy_loss_(losses, xd, td, od, ad, logprobs=lps, stats=stats, weights=weights, reduced=reduced, count=count, **how)
    room = LP * (1 + np.abs(w).max() * 2 + 2 * kl)
    assert np.abs(losses.double().cpu().numpy() - loss).max() <= room
    assert np.abs(lps.double().cpu().numpy() - O.log_probs(x, tok)[0]).max() <= LP
    assert np.abs(weights.double().cpu().numpy() - w).max() <= room
    assert float(count) == (tok != -1).sum() and abs(float(reduced) - loss.sum() / n) <= room
    for accumulate in (False, True):
        delta = torch.full_like(xd, 2.0)
        F.policy_loss_gradient_(delta, xd, td, 0.5, stats, weights, count=count, accumulate=accumulate)
        if accumulate:  # 2 + g, rounded once
            want = 2.0 + g
            err = np.abs(delta.double().cpu().numpy() - want) - (2.0 ** -8 if dtype == "bf16" else 2.0 ** -23) * np.abs(want)
            assert (err <= 2 * LP * np.abs(w)[..., None]).all()
            assert bool((delta[td == -1] == 2.0).all())
        else:
            _check_gradient(delta, g, w * 0.5 / n, dtype)
    delta = torch.full_like(xd, float("nan"))
    losses2 = torch.full((B, T), 9.0, device=gpu)
    F.policy_loss_fused_(losses2, delta, xd, td, od, ad, 0.5, reduced=reduced, **how)
    _check_gradient(delta, g, w * 0.5 / n, dtype)
    assert np.abs(losses2.double().cpu().numpy() - loss).max() <= room and abs(float(reduced) - loss.sum() / n) <= room


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_policy_autograd_and_views(gpu, dtype, reduction, off):
    """Leaves off a 16-byte boundary, advantages per token, each reduction, a
    second backward through the same graph."""
    B, T, V = 4, 7, 1003
    x, xd = _logits(gpu, 3 + off, B, T, V, dtype, off=off)
    tok = _tokens(5, B, T, V, "some")
    old, ref, adv = _policy_inputs(6, x, tok, per_answer=False)
    td, od, rd, ad = _dev(gpu, tok, old, ref, adv)
    xd.requires_grad_()
    assert xd.data_ptr() % 16 == (off * xd.element_size()) % 16
    out = F.PolicyLossFunction.apply(xd, td, od, ad, rd, CLIP, 0.1, -1, reduction)
    n = (tok != -1).sum()
    dy = np.random.default_rng(1).standard_normal((B, T)) if reduction == "none" else 1.0
    scale = 1.0 / n if reduction == "mean" else 1.0
    loss, g, w = O.policy(x, tok, old, adv, ref, CLIP, 0.1, dy=dy * scale)
    dyd = torch.from_numpy(dy).float().to(gpu) if reduction == "none" else torch.ones((), device=gpu)
    g1 = torch.autograd.grad(out, xd, dyd, retain_graph=True)[0]
    g2 = torch.autograd.grad(out, xd, dyd * 3)[0]
    wd = np.abs(w * dy * scale)
    _check_gradient(g1, g, wd, dtype)
    _check_gradient(g2, 3 * g, 3 * wd, dtype)
    # the first backward with a factor scales what the forward left, rounding twice in bf16
    out = F.PolicyLossFunction.apply(xd, td, od, ad, rd, CLIP, 0.1, -1, reduction)
    g3 = torch.autograd.grad(out, xd, dyd * 3)[0].double().cpu().numpy()
    step = 2.0 ** -7 if dtype == "bf16" else 2.0 ** -22
    assert (np.abs(g3 - 3 * g) <= step * 1.01 * np.abs(3 * g) + 6 * LP * wd[..., None]).all()


@pytest.mark.parametrize("base,dtype", [(0, torch.int32), (1, torch.int32), (1, torch.int64)])
def test_index_types_and_bases(gpu, base, dtype):
    B, T, V = 2, 6, 300
    x, xd = _logits(gpu, 8, B, T, V, "f32")
    tok = _tokens(9, B, T, V, "some")
    old, ref, adv = _policy_inputs(10, x, tok, True)
    od, ad = _dev(gpu, old, adv)
    shifted = torch.from_numpy(np.where(tok == -1, -1, tok + base)).to(gpu, dtype)
    got = F.policy_loss(xd, shifted, od, ad, clip=CLIP, index_base=base, reduction="none")
    want, _, w = O.policy(x, tok, old, adv, None, CLIP)
    assert np.abs(got.double().cpu().numpy() - want).max() <= LP * (1 + 2 * np.abs(w).max())


def test_no_answers_and_bad_tokens(gpu):
    B, T, V = 2, 4, 5000
    _, xd = _logits(gpu, 11, B, T, V, "f32")
    o = torch.zeros(B, T, device=gpu)
    none = torch.full((B, T), -1, dtype=torch.int64, device=gpu)
    xn = torch.full_like(xd, float("nan"))  # not read
    delta = torch.full_like(xd, 7.0)
    losses = torch.full((B, T), 9.0, device=gpu)
    F.policy_loss_fused_(losses, delta, xn, none, o, o, reduction="sum")
    assert not losses.any() and not delta.any()
    xl = xn.clone().requires_grad_()
    loss = F.PolicyLossFunction.apply(xl, none, o, o, None, CLIP, 0.0, -1, "none")
    assert not loss.any() and not torch.autograd.grad(loss.sum(), xl)[0].any()
    bad = torch.zeros(B, T, dtype=torch.int64, device=gpu)
    bad[1, 2], bad[0, 3] = V, -5
    got = F.policy_loss(xd, bad, o, o + 1, reduction="none")
    assert torch.isnan(got).tolist() == (bad != 0).tolist()
    F.policy_loss_fused_(losses, delta, xd, bad, o, o + 1, reduction="sum")
    assert torch.isnan(delta).any(-1).tolist() == (bad != 0).tolist()


@pytest.mark.parametrize("V", [100, 3001, 20000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_vocabulary_and_large_logits(gpu, V, dtype):
    """-inf logits take no part; logits of 1e4 keep their differences."""
    B, T = 2, 3
    x, xd = _logits(gpu, 12, B, T, V, dtype, scale=2.0, shift=1e4 if dtype == "f32" else 0.0)
    x[:, :, ::3] = -np.inf
    xd[:, :, ::3] = -float("inf")
    tok = np.full((B, T), 1)
    lp, _ = O.log_probs(x, tok)
    old, adv = lp.astype(np.float32), np.ones((B, T), np.float32)
    td, od, ad = _dev(gpu, tok, old, adv)
    loss, g, w = O.policy(x, tok, old, adv)
    losses, delta = torch.empty(B, T, device=gpu), torch.empty_like(xd)
    F.policy_loss_fused_(losses, delta, xd, td, od, ad, reduction="sum")
    assert np.abs(losses.double().cpu().numpy() - loss).max() <= 3 * LP
    _check_gradient(delta, g, w, dtype)
    xl = xd.clone().requires_grad_()
    out = F.PolicyLossFunction.apply(xl, td, od, ad, None, (0.2, 0.2), 0.0, -1, "none")
    _check_gradient(torch.autograd.grad(out, xl, torch.ones_like(out))[0], g, w, dtype)


@pytest.mark.parametrize("V", [4 * 1024 * 16 + 9, 140000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_columns_longer_than_the_fused_kernel_holds(gpu, V, dtype):
    B, T = 1, 2
    x, xd = _logits(gpu, 13, B, T, V, dtype)
    tok = _tokens(14, B, T, V, "none")
    old, _, adv = _policy_inputs(15, x, tok, True)
    td, od, ad = _dev(gpu, tok, old, adv)
    loss, g, w = O.policy(x, tok, old, adv, None, CLIP, dy=0.5)
    xd.requires_grad_()
    out = F.PolicyLossFunction.apply(xd, td, od, ad, None, CLIP, 0.0, -1, "mean")
    assert abs(float(out.detach()) - loss.mean()) <= LP * (1 + 2 * np.abs(w).max())
    _check_gradient(torch.autograd.grad(out, xd)[0], g, w * 0.5, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("P,T,V", [(1, 1, 2), (2, 33, 1000), (3, 17, 4099), (1, 1500, 64), (5, 4, 50257), (9, 6, 200), (40, 3, 33), (1, 5000, 16)])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference(gpu, P, T, V, dtype, smoothing):
    x, xd = _logits(gpu, 20 + V, 2 * P, T, V, dtype)
    tok = _tokens(21, 2 * P, T, V, "some" if T > 1 else "none")
    rng = np.random.default_rng(22)
    ref = (O.log_probs(x, tok)[0].sum(-1) + 5 * rng.standard_normal(2 * P)).astype(np.float32)
    beta = 0.1
    td, rd = _dev(gpu, tok, ref)
    xd.requires_grad_()
    loss, rewards, g, w = O.preference(x, tok, ref, beta, smoothing, dy=1.0 / P)
    out, got = F.PreferenceLossFunction.apply(xd, td, rd, beta, smoothing, -1, "mean")
    room = beta * T * LP + 2.0 ** -23 * np.abs(rewards).max()  # T log-probabilities in a sum
    assert np.abs(got.double().cpu().numpy() - rewards).max() <= room
    assert abs(float(out) - loss.mean()) <= 2 * room + 2.0 ** -23 * loss.mean()
    wt = np.broadcast_to(np.abs(w)[:, None] * (1 + 2 * room / LP) / P, tok.shape)  # w moves by up to beta * 2 room
    _check_gradient(torch.autograd.grad(out, xd)[0], g, wt, dtype)
    # one value per pair, one gradient per pair
    out, _ = F.PreferenceLossFunction.apply(xd, td, rd, beta, smoothing, -1, "none")
    dy = rng.standard_normal(P)
    g = O.preference(x, tok, ref, beta, smoothing, dy=dy)[2]
    assert np.abs(out.detach().double().cpu().numpy() - loss).max() <= 2 * room + 2.0 ** -23 * loss.max()
    wt = wt * P * np.abs(np.concatenate([dy, dy]))[:, None]
    _check_gradient(torch.autograd.grad(out, xd, torch.from_numpy(dy).float().to(gpu))[0], g, wt, dtype)


def test_preference_far_apart(gpu):
    """Pairs whose margins are far beyond where exp overflows."""
    P, T, V = 3, 2, 10
    x, xd = _logits(gpu, 30, 2 * P, T, V, "f32")
    tok = _tokens(31, 2 * P, T, V, "none")
    lp = O.log_probs(x, tok)[0].sum(-1)
    ref = (lp + np.array([2e4, -2e4, 0, -2e4, 2e4, 0])).astype(np.float32)
    td, rd = _dev(gpu, tok, ref)
    xd.requires_grad_()
    loss, rewards, g, w = O.preference(x, tok, ref, 0.5, 0.0)
    out, got = F.PreferenceLossFunction.apply(xd, td, rd, 0.5, 0.0, -1, "none")
    # A reward is beta times a sum of T log-probabilities, each within LP (a reference that equals
    # that sum leaves the difference of their errors alone), then half a float32 step of it; a
    # loss moves by at most both rewards' differences.
    room = 0.5 * T * LP + 2.0 ** -23 * np.abs(rewards)
    assert (np.abs(got.double().cpu().numpy() - rewards) <= room).all()
    assert (np.abs(out.detach().double().cpu().numpy() - loss) <= room[:P] + room[P:] + 2.0 ** -23 * loss).all()
    gd = torch.autograd.grad(out, xd, torch.ones_like(out))[0]
    assert torch.isfinite(gd).all()
    assert not gd[1].any() and not gd[1 + P].any()  # h = 2e4: nothing left to learn
    _check_gradient(gd, g, np.broadcast_to(np.abs(w)[:, None], tok.shape) + 1e-4, "f32")


def test_captured_and_replayed(gpu):
    """A step of both losses in a graph, replayed on new inputs with eager work
    between, the same bits as the eager step on another stream."""
    B, T, V = 4, 9, 6007
    xs = [_logits(gpu, 40 + i, B, T, V, "bf16")[1] for i in range(3)]
    tok = torch.from_numpy(_tokens(41, B, T, V, "some")).to(gpu)
    old, adv, ref = torch.full((B, T), -8.0, device=gpu), torch.ones(B, device=gpu), torch.full((B,), -50.0, device=gpu)

    def step(x):
        x = x.detach().requires_grad_()
        a = F.PolicyLossFunction.apply(x, tok, old, adv, None, CLIP, 0.0, -1, "mean")
        b, rewards = F.PreferenceLossFunction.apply(x, tok, ref, 0.1, 0.0, -1, "mean")
        return [a.detach(), b.detach(), rewards] + [torch.autograd.grad(a, x)[0], torch.autograd.grad(b, x)[0]]

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        want = [[t.clone() for t in step(x)] for x in xs]
    torch.cuda.current_stream(gpu).wait_stream(side)
    buf = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for i in (1, 2, 0, 2):
        buf.copy_(xs[i])
        graph.replay()
        eager = step(xs[i])
        torch.cuda.synchronize()
        for a, b, c in zip(out, want[i], eager):
            assert torch.equal(a, b) and torch.equal(b, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,off", [(1, 0), (7, 1), (4096, 3), (1 << 20, 0), ((1 << 22) + 5, 1)])
def test_scale_gradient(gpu, n, off, dtype):
    from femtochat_amd.answer_loss import _scale

    x = torch.randn(n + off, device=gpu).to(DTYPES[dtype])
    for f in (1.0, -0.37):
        y = x.clone()
        _scale(y[off:], torch.tensor(f, device=gpu))
        assert torch.equal(y[off:], (x[off:].float() * torch.tensor(f, device=gpu)).to(x.dtype)) and torch.equal(y[:off], x[:off])


@pytest.mark.parametrize("V", [32768, 50257])
def test_beyond_32_bit_offsets(gpu, V):
    """More than 2^31 bf16 logits (and 2^32 bytes): the last answers give the bits that
    they give by themselves, in both losses."""
    T, B = 1024, 2 * (-(-(1 << 31) // (2 * 1024 * V)) + 1)
    g = torch.Generator(device=gpu).manual_seed(50)
    x = torch.empty(B, T, V, dtype=torch.bfloat16, device=gpu)
    for i in range(B):
        x[i].normal_(0.0, 2.0, generator=g)
    tok = torch.randint(0, V, (B, T), device=gpu, generator=g)
    tok[:, ::3] = -1
    old, adv = torch.full((B, T), -9.0, device=gpu), torch.randn(B, device=gpu, generator=g)

    def policy(x, tok, old, adv):
        losses, delta = torch.empty(tok.shape, device=gpu), torch.empty_like(x)
        F.policy_loss_fused_(losses, delta, x, tok, old, adv, reduction="sum")
        return losses, delta

    losses, delta = policy(x, tok, old, adv)
    l2, d2 = policy(x[-2:].contiguous(), tok[-2:].contiguous(), old[-2:].contiguous(), adv[-2:].contiguous())
    assert torch.equal(losses[-2:], l2) and torch.equal(delta[-2:], d2)
    del delta, d2
    ref = torch.full((B,), -6000.0, device=gpu)
    pair = torch.tensor([B // 2 - 1, B - 1], device=gpu)
    xs = x[pair].requires_grad_()
    small, _ = F.PreferenceLossFunction.apply(xs, tok[pair], ref[:2], 0.1, 0.0, -1, "sum")
    want = torch.autograd.grad(small, xs)[0]
    x.requires_grad_()
    loss, rewards = F.PreferenceLossFunction.apply(x, tok, ref, 0.1, 0.0, -1, "sum")
    got = torch.autograd.grad(loss, x)[0]
    assert torch.equal(got[pair], want)


def test_gpu_refusals(gpu):
    x = torch.zeros(2, 3, 5, device=gpu)
    t = torch.zeros(2, 3, dtype=torch.int64, device=gpu)
    o = torch.zeros(2, 3, device=gpu)
    for bad in (dict(old_logprobs=o[:1]), dict(advantages=torch.zeros(3, device=gpu)), dict(tokens=t.cpu()), dict(logits=x.half()),
                dict(old_logprobs=o.double()), dict(logits=x.transpose(0, 1))):
        args = dict(logits=x, tokens=t, old_logprobs=o, advantages=o)
        args.update(bad)
        with pytest.raises((ValueError, TypeError)):
            F.policy_loss(**args)
    with pytest.raises(ValueError, match="pairs"):
        F.preference_loss(x[:1], t[:1], o[0, :1])
    with pytest.raises(F._lib.AttentionError):
        F.policy_loss(x, t, o, o, kl=0.1)
    with pytest.raises(F._lib.AttentionError):
        F.preference_loss(x, t, o[:, 0].contiguous(), beta=-1.0)


@pytest.mark.parametrize("V", [1003, 4 * 1024 * 16 + 9])
def test_saved_tensors_that_move(gpu, V):
    """Saved-tensor hooks may hand the backward copies: what lay where the forward
    left it is overwritten here."""
    B, T = 2, 5
    x, xd = _logits(gpu, 41, B, T, V, "f32")
    tok = _tokens(42, B, T, V, "some")
    old, ref, adv = _policy_inputs(43, x, tok, per_answer=True)
    td, od, rd, ad = _dev(gpu, tok, old, ref, adv)
    xd.requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t.clone()):
        out = F.PolicyLossFunction.apply(xd, td, od, ad, rd, CLIP, 0.1, -1, "mean")
        pref, _ = F.PreferenceLossFunction.apply(xd, td, ad, 0.1, 0.0, -1, "mean")
    dirt = [torch.full((4 * B * T + k,), float("nan"), device=gpu) for k in (1, 1, B + 1, B + 1)]
    _, g, w = O.policy(x, tok, old, adv, ref, CLIP, 0.1, dy=1.0 / (tok != -1).sum())
    wd = np.abs(w) / (tok != -1).sum()
    one = torch.ones((), device=gpu)
    _check_gradient(torch.autograd.grad(out, xd, one, retain_graph=True)[0], g, wd, "f32")
    _check_gradient(torch.autograd.grad(out, xd, one)[0], g, wd, "f32")
    again, _ = F.PreferenceLossFunction.apply(xd, td, ad, 0.1, 0.0, -1, "mean")
    assert torch.equal(torch.autograd.grad(pref, xd)[0], torch.autograd.grad(again, xd)[0])
    assert all(d.isnan().all() for d in dirt)


@pytest.mark.parametrize("B,T", [(1, 1), (3, 21), (1, 64), (1, 513), (4, 256), (5, 205), (3, 700)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_the_mean_of_any_number_of_tokens(gpu, B, T, index):
    """The divisor, also where only the gradient asks for it, and the count."""
    V = 50
    x, xd = _logits(gpu, 51, B, T, V, "f32")
    tok = _tokens(52, B, T, V, "some")
    tok[0, 0] = 3
    old, ref, adv = _policy_inputs(53, x, tok, per_answer=True)
    td, od, rd, ad = _dev(gpu, tok, old, ref, adv)
    n = int((tok != -1).sum())
    loss, g, w = O.policy(x, tok, old, adv, ref, CLIP, 0.1, dy=1.0 / n)
    # A token whose two terms cancel has a small w and moves with lp all the same:
    # w = -A r + kl (1 - exp(d)), so |dw / dlp| <= |A| r + kl exp(d).
    lp, _ = O.log_probs(x, tok)
    slope = np.where(tok != -1, np.abs(adv)[:, None] * np.exp(lp - old) + 0.1 * np.exp(ref - lp), 0.0)
    for wants in (True, False):
        losses, delta = torch.full((B, T), float("nan"), device=gpu), torch.full_like(xd, float("nan"))
        reduced, count = (torch.full((1,), float("nan"), device=gpu) for _ in range(2))
        F.policy_loss_fused_(losses, delta, xd, td.to(index), od, ad, ref_logprobs=rd, clip=CLIP, kl=0.1,
                             reduced=reduced if wants else None, count=count)
        assert float(count) == n
        _check_gradient(delta, g, (np.abs(w) + slope) / n, "f32")
        if wants:
            total = losses.double().sum().item() / n
            assert abs(float(reduced) - total) <= 2.0 ** -24 * abs(total) + 1e-30
