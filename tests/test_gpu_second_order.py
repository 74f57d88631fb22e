"""create_graph through the answer losses and scored attention: the first gradients are
as without it, and differentiating them raises instead of leaving the term out."""
import pytest
import torch

import femtochat_amd as F

pytestmark = pytest.mark.gpu


def _losses(gpu):
    B, T, V = 4, 6, 300
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, T, V, generator=g).to(gpu).requires_grad_()
    tok = torch.randint(0, V, (B, T), generator=g).to(gpu)
    old, adv, ref = torch.full((B, T), -6.0, device=gpu), torch.ones(B, device=gpu), torch.full((B,), -30.0, device=gpu)
    return x, {"policy": lambda: F.PolicyLossFunction.apply(x, tok, old, adv, None, (0.2, 0.2), 0.0, -1, "mean"),
               "preference": lambda: F.PreferenceLossFunction.apply(x, tok, ref, 0.1, 0.0, -1, "mean")[0]}


@pytest.mark.parametrize("which", ["policy", "preference"])
@pytest.mark.parametrize("factor", [1.0, 0.5])
def test_losses(gpu, which, factor):
    x, runs = _losses(gpu)
    run = runs[which]
    dy = torch.tensor(factor, device=gpu)
    want = torch.autograd.grad(run(), x, dy)[0].clone()
    loss = run()
    got = torch.autograd.grad(loss, x, dy, create_graph=True)[0]
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        (loss + got.square().sum()).backward()
    # a graph that is built but not used stays a first-order step
    loss = run()
    loss.backward(dy, create_graph=True)
    assert torch.equal(x.grad, want)
    x.grad = None
    # and by the incoming gradient alone
    dy.requires_grad_()
    x0 = x
    got = torch.autograd.grad(run(), x0, dy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(got.sum(), dy)


def test_attention(gpu):
    g = torch.Generator().manual_seed(2)
    Q, K, V = (torch.randn(1, 40, 2, 32, generator=g).bfloat16().to(gpu).requires_grad_() for _ in range(3))

    def run(softcap):
        return F.AttentionFunction.apply(Q, K, V, (-1, 0), None, None, softcap)

    for leaves in ((Q, K, V), (Q,), (V,)):
        want = torch.autograd.grad(run(5.0).sum(), leaves)
        got = torch.autograd.grad(run(5.0).sum(), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            torch.autograd.grad(got[0].float().sum(), leaves)
    # plain scores are as they were
    assert not torch.autograd.grad(run(0.0).sum(), Q, create_graph=True)[0].requires_grad


@pytest.mark.parametrize("which", ["policy", "preference"])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_copies_of_the_leaves(gpu, which, reduction):
    """Logits that the node copies (not contiguous), with gradients of gradients by the
    leaf they came from."""
    B, T, V = 4, 6, 300
    g = torch.Generator().manual_seed(1)
    leaf = torch.randn(B, T + 1, V, generator=g).to(gpu).requires_grad_()
    tok = torch.randint(0, V, (B, T), generator=g).to(gpu)
    old, adv, ref = torch.full((B, T), -6.0, device=gpu), torch.ones(B, device=gpu), torch.full((B,), -30.0, device=gpu)

    def run():
        x = leaf[:, :-1]
        if which == "policy":
            return F.PolicyLossFunction.apply(x, tok, old, adv, None, (0.2, 0.2), 0.0, -1, reduction)
        return F.PreferenceLossFunction.apply(x, tok, ref, 0.1, 0.0, -1, reduction)[0]

    want = torch.autograd.grad(run().sum(), leaf)[0]
    got = torch.autograd.grad(run().sum(), leaf, create_graph=True)[0]
    assert torch.equal(got, want) and not got[:, -1].any()
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        torch.autograd.grad(got.square().sum(), leaf)


def test_attention_of_float32_leaves(gpu):
    g = torch.Generator().manual_seed(2)
    Q, K, V = (torch.randn(1, 40, 2, 32, generator=g).to(gpu).requires_grad_() for _ in range(3))
    slopes = torch.tensor([0.5, 0.25], device=gpu)
    dO = torch.randn(1, 40, 2, 32, generator=g).to(gpu)

    def run():
        return F.AttentionFunction.apply(Q, K, V, (-1, 0), None, None, 0.0, slopes)

    want = torch.autograd.grad(run(), (Q, K, V), dO)
    got = torch.autograd.grad(run(), (Q, K, V), dO, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for x in got:
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            torch.autograd.grad(x.sum(), Q, retain_graph=True)


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_losses_changed_in_place(gpu, which):
    """loss /= n behind the node, on contiguous logits and on views."""
    B, T, V = 4, 6, 300
    g = torch.Generator().manual_seed(1)
    leaf = torch.randn(B, T + 1, V, generator=g).to(gpu).requires_grad_()
    tok = torch.randint(0, V, (B, T + 1), generator=g).to(gpu)
    old, adv, ref = torch.full((B, T + 1), -6.0, device=gpu), torch.ones(B, device=gpu), torch.full((B,), -30.0, device=gpu)
    for n in (T + 1, T):
        grads = []
        for in_place in (False, True):
            t, o, x = tok[:, :n].contiguous(), old[:, :n].contiguous(), leaf[:, :n]
            if which == "policy":
                loss = F.PolicyLossFunction.apply(x, t, o, adv, None, (0.2, 0.2), 0.0, -1, "mean")
            else:
                loss = F.PreferenceLossFunction.apply(x, t, ref, 0.1, 0.0, -1, "mean")[0]
            if in_place:
                loss /= 4
            else:
                loss = loss / 4
            grads.append(torch.autograd.grad(loss, leaf)[0])
        assert torch.equal(*grads)
