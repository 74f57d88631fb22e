"""Gradients under saved-tensor hooks that change strides or keep tensors on the host:
the same bits as without hooks."""
import pytest
import torch

import femtochat_amd as F

pytestmark = pytest.mark.gpu

HOOKS = {
    "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.detach() if t.dim() < 2 else t.detach().transpose(1, -1).contiguous(), lambda t: t if t.dim() < 2 else t.transpose(1, -1)),
    "host": lambda: torch.autograd.graph.save_on_cpu(),
}


def _grads(run, leaves, dy, hooks):
    with hooks:
        out = run()
    return torch.autograd.grad(out, leaves, dy)


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("kind", ["plain", "documents", "scored"])
@pytest.mark.parametrize("D", [64, 96])
def test_attention(gpu, hooks, kind, D):
    B, T, H, Hkv = 2, 150, 4, 2
    g = torch.Generator().manual_seed(1)
    Q, K, V = (torch.randn(B, T, h, D, generator=g).bfloat16().to(gpu).requires_grad_() for h in (H, Hkv, Hkv))
    dO = torch.randn(B, T, H, D, generator=g).bfloat16().to(gpu)
    pos = (torch.arange(T, dtype=torch.int32) % 40).repeat(B, 1).to(gpu) if kind != "plain" else None
    how = (5.0, torch.full((H,), 0.05, device=gpu), torch.full((B, T), 17, dtype=torch.int32, device=gpu)) if kind == "scored" else ()

    def run():
        return F.AttentionFunction.apply(Q, K, V, (-1, 0), None, pos, *how)

    want = _grads(run, (Q, K, V), dO, torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    got = _grads(run, (Q, K, V), dO, HOOKS[hooks]())
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("hooks", HOOKS)
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_losses(gpu, hooks, reduction):
    B, T, V = 4, 9, 1003
    g = torch.Generator().manual_seed(2)
    x = torch.randn(B, T, V, generator=g).bfloat16().to(gpu).requires_grad_()
    tok = torch.randint(0, V, (B, T), generator=g).to(gpu)
    tok[:, ::4] = -1
    old, adv, ref = torch.full((B, T), -7.0, device=gpu), torch.ones(B, device=gpu), torch.full((B,), -40.0, device=gpu)
    for run, n in ((lambda: F.PolicyLossFunction.apply(x, tok, old, adv, None, (0.2, 0.2), 0.0, -1, reduction), (B, T)),
                   (lambda: F.PreferenceLossFunction.apply(x, tok, ref, 0.1, 0.0, -1, reduction)[0], (B // 2,))):
        dy = torch.linspace(0.5, 2.0, n[0] * (n[1] if len(n) > 1 else 1), device=gpu).view(n) if reduction == "none" else torch.full((), 3.0, device=gpu)
        want = _grads(run, x, dy, torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))[0]
        assert torch.equal(_grads(run, x, dy, HOOKS[hooks]())[0], want)
