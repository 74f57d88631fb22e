"""The policy loss's gradient under an incoming gradient other than 1 (a loss divided by
its micro-batches, or added to another one with a factor): rounded once, and the same
bits in the first and in any further backward through a node."""
import numpy as np
import pytest
import torch

import femtochat_amd as F
from oracle import answer_loss as O

from tests.test_gpu_answer_loss import CLIP, LP, _check_gradient, _dev, _logits, _policy_inputs, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("V,off", [(5, 0), (259, 1), (1003, 3), (8192, 0), (50257, 0), (70001, 0)])
@pytest.mark.parametrize("factor", [1.0, 0.125, 3.0, -0.37, 0.0])
def test_rounded_once(gpu, dtype, reduction, V, off, factor):
    B, T = 3, 4
    x, xd = _logits(gpu, 3 + V, B, T, V, dtype, off=off)
    tok = _tokens(5, B, T, V, "some")
    old, ref, adv = _policy_inputs(6, x, tok, per_answer=True)
    td, od, rd, ad = _dev(gpu, tok, old, ref, adv)
    xd.requires_grad_()
    f = np.float32(factor)
    scale = float(f) / (max(1, (tok != -1).sum()) if reduction == "mean" else 1)
    _, g, w = O.policy(x, tok, old, adv, ref, CLIP, 0.1, dy=scale)
    # a token's w = -A r + kl (1 - exp(d)) moves with lp by at most |A| r + kl exp(d)
    lp, _ = O.log_probs(x, tok)
    slope = np.where(tok != -1, np.abs(adv)[:, None] * np.exp(lp - old) + 0.1 * np.exp(ref - lp), 0.0)
    out = F.PolicyLossFunction.apply(xd, td, od, ad, rd, CLIP, 0.1, -1, reduction)
    dy = torch.tensor(f, device=gpu)
    first = torch.autograd.grad(out, xd, dy, retain_graph=True)[0].clone()
    second = torch.autograd.grad(out, xd, dy, retain_graph=True)[0]
    _check_gradient(first, g, (np.abs(w) + slope) * abs(scale), dtype)
    assert torch.equal(first, second)
    assert not first[td == -1].any()
    # divided behind the node, as a step of micro-batches does
    out = F.PolicyLossFunction.apply(xd, td, od, ad, rd, CLIP, 0.1, -1, reduction)
    assert torch.equal(torch.autograd.grad(out * float(f), xd)[0], first)


def test_masked_and_spoilt_columns(gpu):
    """-inf logits, a token outside the vocabulary, a NaN column and columns outside the
    answers, whose NaN logits are not read."""
    B, T, V = 2, 3, 1000
    _, xd = _logits(gpu, 1, B, T, V, "bf16")
    xd[..., ::3] = -float("inf")
    xd[0, 0], xd[1, 2, 5] = float("nan"), float("nan")
    tok = torch.tensor([[-1, 1, V], [4, 7, 2]], device=gpu)
    old, adv = torch.full((B, T), -7.0, device=gpu), torch.ones(B, device=gpu)
    xd.requires_grad_()
    out = F.PolicyLossFunction.apply(xd, tok, old, adv, None, CLIP, 0.0, -1, "sum")
    g = torch.autograd.grad(out, xd, torch.tensor(2.0, device=gpu))[0]
    assert not g[0, 0].any()
    assert torch.isnan(g[0, 2]).all() and torch.isnan(g[1, 2]).all()
    assert torch.isfinite(g[0, 1]).all() and torch.isfinite(g[1, :2]).all() and not g[0, 1, ::3].any()


def test_captured(gpu):
    """A factor that changes between the replays of a captured step, through 1 and back."""
    B, T, V = 4, 9, 6007
    xs = [_logits(gpu, 40 + i, B, T, V, "bf16")[1] for i in range(2)]
    tok = torch.from_numpy(_tokens(41, B, T, V, "some")).to(gpu)
    old, adv, dy = torch.full((B, T), -8.0, device=gpu), torch.ones(B, device=gpu), torch.ones((), device=gpu)

    def step(x):
        x = x.detach().requires_grad_()
        a = F.PolicyLossFunction.apply(x, tok, old, adv, None, CLIP, 0.0, -1, "mean")
        return [a.detach(), torch.autograd.grad(a, x, dy)[0]]

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step(xs[0])
    torch.cuda.current_stream(gpu).wait_stream(side)
    buf = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for i, f in ((1, 0.25), (0, 1.0), (1, 1.0), (1, -3.0), (0, 0.25)):
        buf.copy_(xs[i])
        dy.fill_(f)
        graph.replay()
        eager = step(xs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_hooks_that_change_the_alignment(gpu):
    """The copy of the logits that a hook hands back lies one value off a 16-byte boundary."""
    B, T, V = 2, 5, 1003
    _, xd = _logits(gpu, 9, B, T, V, "bf16")
    tok = torch.from_numpy(_tokens(42, B, T, V, "some")).to(gpu)
    old, adv = torch.full((B, T), -7.0, device=gpu), torch.ones(B, device=gpu)
    xd.requires_grad_()

    def shifted(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        return room[1:].view(t.shape).copy_(t) if t.dtype == torch.bfloat16 else t

    for f in (1.0, 0.125):
        dy = torch.tensor(f, device=gpu)
        got = []
        for unpack in (lambda t: t, shifted):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
                out = F.PolicyLossFunction.apply(xd, tok, old, adv, None, CLIP, 0.0, -1, "mean")
            got.append(torch.autograd.grad(out, xd, dy)[0])
        assert torch.equal(*got)
